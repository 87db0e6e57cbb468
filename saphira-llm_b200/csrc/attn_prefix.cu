// attn_prefix.cu -- decode attention of sequences that share a prefix, over a
// paged cache.

#include "attn_simt.cuh"

namespace sllm {
namespace {

struct PrefixParams {
    const void* q;                  // [n][n_q][n_head][128]
    void* out;
    const void* kp;                 // the layer's slice of page 0
    const void* vp;
    size_t page_stride;
    const int32_t* slots;
    int n, n_q, n_head, n_kv, group, prefix;
    int32_t* status;
};

// the tokens a sequence's slot holds; -1 when the slot or its length is wrong
__device__ __forceinline__ int seq_len(const PagesDev& pg, const PrefixParams& p, int b, int* slot) {
    const int s = p.slots[b];
    *slot = s;
    if (s < 0 || s >= pg.n_slots) return -1;
    const int len = pg.lens[s];
    if (len < 0 || len > pg.cap) return -1;
    if (p.prefix > 0 && len - p.n_q + 1 < p.prefix) return -1;
    return len;
}

template <class T, class O>
__global__ void __launch_bounds__(kSimtThreads)
attn_prefix_simt_kernel(const PagesDev pg, const __grid_constant__ PrefixParams p) {
    extern __shared__ float sm[];
    const int b = blockIdx.x, kvh = blockIdx.y, rows = p.n_q * p.group, r0 = blockIdx.z * kSimtRows;
    int slot;
    const int len = seq_len(pg, p, b, &slot);
    if (len < 0) {
        if (threadIdx.x == 0) raise(p.status, SLLM_CUDA_ERR_ARG);
        return;
    }
    // row r is query token r / group, head kvh * group + r % group
    auto row_off = [&](int r) {
        return (((size_t)b * p.n_q + r / p.group) * p.n_head + kvh * p.group + r % p.group) * kServeDim;
    };
    simt_load_q<T>(sm, [&](int r) {
        return r0 + r < rows ? static_cast<const T*>(p.q) + row_off(r0 + r) : nullptr;
    });
    SimtState st;
    simt_init(st);
    const int ty = threadIdx.x >> 4;
    int lim[4];
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = r0 + 4 * ty + i;
        lim[i] = r < rows ? max(0, len - p.n_q + 1 + r / p.group) : 0;
    }
    const int32_t* row = pg.tables + (size_t)slot * pg.width;
    auto addr = [&](const void* pool, int j) -> const T* {
        if (j >= len) return nullptr;
        int id = row[j / pg.page];
        if (id < 0 || id >= pg.n_pages) {
            raise(p.status, SLLM_CUDA_ERR_ARG);
            return nullptr;
        }
        return static_cast<const T*>(pool) + (size_t)id * p.page_stride + ((size_t)kvh * pg.page + j % pg.page) * kServeDim;
    };
    for (int j0 = 0; j0 < len; j0 += kSimtKeys)
        simt_tile<T>(sm, st, j0, lim, [&](int j) { return addr(p.kp, j); }, [&](int j) { return addr(p.vp, j); });
    #pragma unroll
    for (int i = 0; i < 4; ++i)
        if (r0 + 4 * ty + i < rows) simt_store(st, i, static_cast<O*>(p.out) + row_off(r0 + 4 * ty + i));
}

template <class T, class O>
cudaError_t launch_simt(const PagesDev& pg, const PrefixParams& p, cudaStream_t st) {
    auto* kern = attn_prefix_simt_kernel<T, O>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSimtSmem);
    if (e != cudaSuccess) return e;
    const unsigned z = (unsigned)((p.n_q * p.group + kSimtRows - 1) / kSimtRows);
    return launch(kern, dim3((unsigned)p.n, (unsigned)p.n_kv, z), dim3(kSimtThreads), kSimtSmem, st, false, pg, p);
}

int check_shape(const sllm_cuda_kv_pages* p, int n, int n_q, int n_head, int prefix, const char* who) {
    const int rc = check_pages(p, who);
    if (rc != SLLM_CUDA_OK) return rc;
    if (n < 0 || n > 4096 || n_q < 1 || n_q > 16 || n_head < 1 || n_head > 1024 || n_head % p->n_head_kv != 0 ||
        prefix < 0 || prefix % p->page_size != 0 || prefix / p->page_size > p->table_width)
        return fail(SLLM_CUDA_ERR_ARG, "%s: %d sequences, %d query tokens (1 to 16), %d heads over %d, prefix of %d "
                    "(whole pages of %d)", who, n, n_q, n_head, p->n_head_kv, prefix, p->page_size);
    return SLLM_CUDA_OK;
}

}  // namespace
}  // namespace sllm

using namespace sllm;

extern "C" size_t sllm_cuda_attn_prefix_work_bytes(const sllm_cuda_kv_pages* p, int32_t n, int32_t n_q, int32_t n_head,
                                                   int32_t prefix_len) {
    if (check_shape(p, n, n_q, n_head, prefix_len, "attn_prefix_work_bytes") != SLLM_CUDA_OK) return 0;
    return 16;
}

extern "C" int sllm_cuda_attn_prefix(const sllm_cuda_kv_pages* p, int32_t layer, const void* q, const int32_t* slots,
                                     int32_t n, int32_t n_q, int32_t n_head, int32_t prefix_len, void* out,
                                     int32_t out_type, void* work, size_t work_bytes, int32_t* status,
                                     void* stream) {
    int rc = check_shape(p, n, n_q, n_head, prefix_len, "attn_prefix");
    if (rc != SLLM_CUDA_OK) return rc;
    if (q == nullptr || slots == nullptr || out == nullptr || work == nullptr || layer < 0 || layer >= p->n_layer)
        return fail(SLLM_CUDA_ERR_ARG, "attn_prefix: a NULL array, or layer %d of %d", layer, p->n_layer);
    if ((out_type != SLLM_CUDA_KV_F32 && out_type != SLLM_CUDA_KV_F16) ||
        (p->kv_type == SLLM_CUDA_KV_F32 && out_type == SLLM_CUDA_KV_F16))
        return fail(SLLM_CUDA_ERR_ARG, "attn_prefix: output type %d (f32, or f16 from an f16 cache)", out_type);
    if (!aligned16(q) || !aligned16(out) || !aligned16(work) ||
        work_bytes < sllm_cuda_attn_prefix_work_bytes(p, n, n_q, n_head, prefix_len))
        return fail(SLLM_CUDA_ERR_ARG, "attn_prefix: workspace of %zu bytes (%zu needed), arrays 16-byte aligned",
                    work_bytes, sllm_cuda_attn_prefix_work_bytes(p, n, n_q, n_head, prefix_len));
    const void* ptr[] = {p->k, p->v, p->tables, p->lens, q, slots, out, work, status};
    const char* name[] = {"k", "v", "tables", "lens", "q", "slots", "out", "work", "status"};
    for (int i = 0; i < 9; ++i)
        if (ptr[i] != nullptr && (rc = need_device(ptr[i], "attn_prefix", name[i])) != SLLM_CUDA_OK) return rc;
    if (n == 0) return SLLM_CUDA_OK;
    const size_t layer_elts = (size_t)p->n_head_kv * p->page_size * kServeDim;
    const size_t off = (size_t)layer * layer_elts * kv_elt_bytes(p->kv_type);
    PrefixParams a{};
    a.q = q; a.out = out;
    a.kp = static_cast<const uint8_t*>(p->k) + off;
    a.vp = static_cast<const uint8_t*>(p->v) + off;
    a.page_stride = (size_t)p->n_layer * layer_elts;
    a.slots = slots;
    a.n = n; a.n_q = n_q; a.n_head = n_head; a.n_kv = p->n_head_kv; a.group = n_head / p->n_head_kv;
    a.prefix = prefix_len;
    a.status = status;
    const PagesDev pg = pages_dev(*p);
    const cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = p->kv_type == SLLM_CUDA_KV_F32 ? launch_simt<float, float>(pg, a, st)
                          : out_type == SLLM_CUDA_KV_F32 ? launch_simt<__half, float>(pg, a, st)
                                                         : launch_simt<__half, __half>(pg, a, st);
    CK(e, "attn_prefix launch");
    count_launches(1);
    return SLLM_CUDA_OK;
}
