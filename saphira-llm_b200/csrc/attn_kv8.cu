// attn_kv8.cu -- decode attention over an 8-bit paged cache.

#include "serve.cuh"

namespace sllm {
namespace {

struct Attn8Params {
    const void* q;                  // [n][n_q][n_head][128]
    void* out;
    const int8_t* kp;               // the layer's slice of page 0
    const int8_t* vp;
    const float* ksc;
    const float* vsc;
    size_t page_stride, scale_stride;
    const int32_t* slots;
    int n, n_q, n_head, n_kv, group;
    int32_t* status;
};

// one warp per query row: a lane has four dimensions, one key after the other
template <class Q, class O>
__global__ void __launch_bounds__(256)
attn_kv8_rows_kernel(const __grid_constant__ PagesDev pg, const __grid_constant__ Attn8Params p) {
    const int lane = threadIdx.x & 31;
    const long long x = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (x >= (long long)p.n * p.n_q * p.n_head) return;
    const int h = (int)(x % p.n_head), j = (int)(x / p.n_head % p.n_q), b = (int)(x / p.n_head / p.n_q);
    const int slot = p.slots[b], kvh = h / p.group;
    const int len = slot >= 0 && slot < pg.n_slots ? pg.lens[slot] : -1;
    if (len < 0 || len > pg.cap) {
        if (lane == 0) raise(p.status, SLLM_CUDA_ERR_ARG);
        return;
    }
    const float4 q = ld4(static_cast<const Q*>(p.q) + (size_t)x * kServeDim + 4 * lane);
    const int seen = len - p.n_q + 1 + j;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int t = 0; t < seen; ++t) {
        const int id = pg.tables[(size_t)slot * pg.width + t / pg.page];
        if (id < 0 || id >= pg.n_pages) {
            if (lane == 0) raise(p.status, SLLM_CUDA_ERR_ARG);
            return;
        }
        const int in = t % pg.page;
        const size_t at = (size_t)id * p.page_stride + ((size_t)kvh * pg.page + in) * kServeDim + 4 * lane;
        const size_t sat = (size_t)id * p.scale_stride + (size_t)kvh * (pg.page / kKvBlock) + in / kKvBlock;
        const char4 k = *reinterpret_cast<const char4*>(p.kp + at), v = *reinterpret_cast<const char4*>(p.vp + at);
        float s = q.x * (float)k.x + q.y * (float)k.y + q.z * (float)k.z + q.w * (float)k.w;
        #pragma unroll
        for (int y = 16; y > 0; y >>= 1) s += __shfl_xor_sync(0xffffffffu, s, y);
        s = s * p.ksc[sat] * kServeScale;
        const float m2 = fmaxf(m, s), f = m == -INFINITY ? 0.f : expf(m - m2), e = expf(s - m2), w = e * p.vsc[sat];
        l = l * f + e;
        o.x = o.x * f + w * (float)v.x;
        o.y = o.y * f + w * (float)v.y;
        o.z = o.z * f + w * (float)v.z;
        o.w = o.w * f + w * (float)v.w;
        m = m2;
    }
    const float inv = seen > 0 ? 1.f / l : 0.f;
    st4(static_cast<O*>(p.out) + (size_t)x * kServeDim + 4 * lane, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

int check_shape8(const sllm_cuda_kv_pages* p, int n, int n_q, int n_head, const char* who) {
    const int rc = check_pages(p, who, true);
    if (rc != SLLM_CUDA_OK) return rc;
    if (n < 0 || n > 4096 || n_q < 1 || n_q > 16 || n_head < 1 || n_head > 1024 || n_head % p->n_head_kv != 0)
        return fail(SLLM_CUDA_ERR_ARG, "%s: %d sequences, %d query tokens (1 to 16), %d heads over %d", who, n, n_q, n_head,
                    p->n_head_kv);
    return SLLM_CUDA_OK;
}

size_t work8_bytes(int, int, int) { return 16; }

}  // namespace
}  // namespace sllm

using namespace sllm;

extern "C" size_t sllm_cuda_attn_kv8_work_bytes(const sllm_cuda_kv_pages* p, int32_t n, int32_t n_q, int32_t n_head) {
    if (check_shape8(p, n, n_q, n_head, "attn_kv8_work_bytes") != SLLM_CUDA_OK) return 0;
    return work8_bytes(n, n_q, n_head);
}

extern "C" int sllm_cuda_attn_kv8(const sllm_cuda_kv_pages* p, int32_t layer, const void* q, int32_t q_type,
                                  const int32_t* slots, int32_t n, int32_t n_q, int32_t n_head, void* out,
                                  int32_t out_type, void* work, size_t work_bytes, int32_t* status, void* stream) {
    int rc = check_shape8(p, n, n_q, n_head, "attn_kv8");
    if (rc != SLLM_CUDA_OK) return rc;
    if (q == nullptr || slots == nullptr || out == nullptr || work == nullptr || layer < 0 || layer >= p->n_layer)
        return fail(SLLM_CUDA_ERR_ARG, "attn_kv8: a NULL array, or layer %d of %d", layer, p->n_layer);
    if ((q_type != SLLM_CUDA_KV_F32 && q_type != SLLM_CUDA_KV_F16) ||
        (out_type != SLLM_CUDA_KV_F32 && out_type != SLLM_CUDA_KV_F16) ||
        (q_type == SLLM_CUDA_KV_F32 && out_type == SLLM_CUDA_KV_F16))
        return fail(SLLM_CUDA_ERR_ARG, "attn_kv8: query type %d, output type %d (f32, or f16 from f16)", q_type, out_type);
    const size_t need = work8_bytes(n, n_q, n_head);
    if (!aligned16(q) || !aligned16(out) || !aligned16(work) || work_bytes < need)
        return fail(SLLM_CUDA_ERR_ARG, "attn_kv8: workspace of %zu bytes (%zu needed), arrays 16-byte aligned", work_bytes, need);
    const void* ptr[] = {p->k, p->v, p->tables, p->lens, p->k_scale, p->v_scale, q, slots, out, work, status};
    const char* name[] = {"k", "v", "tables", "lens", "k_scale", "v_scale", "q", "slots", "out", "work", "status"};
    for (int i = 0; i < 11; ++i)
        if (ptr[i] != nullptr && (rc = need_device(ptr[i], "attn_kv8", name[i])) != SLLM_CUDA_OK) return rc;
    if (n == 0) return SLLM_CUDA_OK;
    Attn8Params a{};
    a.q = q; a.out = out;
    const size_t layer_codes = (size_t)p->n_head_kv * kServeDim * p->page_size;
    const size_t layer_scales = (size_t)p->n_head_kv * (p->page_size / kKvBlock);
    a.kp = static_cast<const int8_t*>(p->k) + layer * layer_codes;
    a.vp = static_cast<const int8_t*>(p->v) + layer * layer_codes;
    a.ksc = p->k_scale + layer * layer_scales;
    a.vsc = p->v_scale + layer * layer_scales;
    a.page_stride = p->n_layer * layer_codes;
    a.scale_stride = p->n_layer * layer_scales;
    a.slots = slots;
    a.n = n; a.n_q = n_q; a.n_head = n_head; a.n_kv = p->n_head_kv; a.group = n_head / p->n_head_kv;
    a.status = status;
    const dim3 grid((unsigned)(((long long)n * n_q * n_head + 7) / 8));
    const PagesDev pg = pages_dev(*p);
    const cudaStream_t st = (cudaStream_t)stream;
    CK(q_type == SLLM_CUDA_KV_F32     ? launch(attn_kv8_rows_kernel<float, float>, grid, dim3(256), 0, st, false, pg, a)
       : out_type == SLLM_CUDA_KV_F32 ? launch(attn_kv8_rows_kernel<__half, float>, grid, dim3(256), 0, st, false, pg, a)
                                      : launch(attn_kv8_rows_kernel<__half, __half>, grid, dim3(256), 0, st, false, pg, a),
       "attn_kv8 launch");
    count_launches(1);
    return SLLM_CUDA_OK;
}
