// attn_prompt.cu -- causal attention over packed whole prompts, grouped heads.
//
// Sequence s holds tokens cu[s] .. cu[s + 1] - 1 of the packed arrays; token i
// of a sequence sees its tokens 0 .. i.

#include "attn_simt.cuh"

namespace sllm {
namespace {

struct PromptParams {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    size_t qs, ks, vs, os;          // elements from a token to the next
    const int32_t* cu;
    int n_seq, n_tokens, n_head, group;
};

// the sequence and its tile for linear tile x of tiles of R rows: a warp's
// scan over the lengths. Bounds are clamped to the arrays, so a wrong cu
// stays inside them.
template <int R>
__device__ __forceinline__ bool find_tile(const PromptParams& p, int x, int* start, int* len, int* tile) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += 32) {
        const int s = s0 + lane;
        int a = 0, n = 0;
        if (s < p.n_seq) {
            a = min(max(p.cu[s], 0), p.n_tokens);
            n = min(max(p.cu[s + 1], a), p.n_tokens) - a;
        }
        const int tiles = (n + R - 1) / R;
        int inc = tiles;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, x < before + inc);
        if (hit != 0) {
            const int l = __ffs(hit) - 1;
            *start = __shfl_sync(0xffffffffu, a, l);
            *len = __shfl_sync(0xffffffffu, n, l);
            *tile = x - before - __shfl_sync(0xffffffffu, inc - tiles, l);
            return true;
        }
        before += __shfl_sync(0xffffffffu, inc, 31);
    }
    return false;
}

template <class T, class O>
__global__ void __launch_bounds__(kSimtThreads)
attn_prompt_simt_kernel(const __grid_constant__ PromptParams p) {
    extern __shared__ float sm[];
    int start, len, tile;
    if (!find_tile<kSimtRows>(p, blockIdx.x, &start, &len, &tile)) return;
    const int h = blockIdx.y, kvh = h / p.group, r0 = tile * kSimtRows;
    const T* q = static_cast<const T*>(p.q) + (size_t)h * kServeDim;
    const T* k = static_cast<const T*>(p.k) + (size_t)kvh * kServeDim;
    const T* v = static_cast<const T*>(p.v) + (size_t)kvh * kServeDim;
    simt_load_q<T>(sm, [&](int r) { return r0 + r < len ? q + (size_t)(start + r0 + r) * p.qs : nullptr; });
    SimtState st;
    simt_init(st);
    const int ty = threadIdx.x >> 4;
    int lim[4];
    #pragma unroll
    for (int i = 0; i < 4; ++i) lim[i] = min(r0 + 4 * ty + i + 1, len);
    const int end = min(r0 + kSimtRows, len);
    for (int j0 = 0; j0 < end; j0 += kSimtKeys)
        simt_tile<T>(sm, st, j0, lim,
                     [&](int j) { return j < end ? k + (size_t)(start + j) * p.ks : nullptr; },
                     [&](int j) { return j < end ? v + (size_t)(start + j) * p.vs : nullptr; });
    #pragma unroll
    for (int i = 0; i < 4; ++i)
        if (r0 + 4 * ty + i < len)
            simt_store(st, i, static_cast<O*>(p.out) + (size_t)(start + r0 + 4 * ty + i) * p.os + (size_t)h * kServeDim);
}

template <class T, class O>
cudaError_t launch_simt(const PromptParams& p, cudaStream_t st) {
    auto* kern = attn_prompt_simt_kernel<T, O>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSimtSmem);
    if (e != cudaSuccess) return e;
    // every sequence may end inside a tile
    const long long tiles = (p.n_tokens + kSimtRows - 1) / kSimtRows + (long long)p.n_seq;
    return launch(kern, dim3((unsigned)tiles, (unsigned)p.n_head), dim3(kSimtThreads), kSimtSmem, st, false, p);
}

}  // namespace
}  // namespace sllm

using namespace sllm;

extern "C" int sllm_cuda_attn_prompt(const void* q, size_t q_stride, const void* k, size_t k_stride, const void* v,
                                     size_t v_stride, int32_t type, const int32_t* cu_seqlens, int32_t n_seq,
                                     int32_t n_tokens, int32_t n_head, int32_t n_head_kv, void* out,
                                     size_t out_stride, int32_t out_type, void* stream) {
    if (q == nullptr || k == nullptr || v == nullptr || cu_seqlens == nullptr || out == nullptr)
        return fail(SLLM_CUDA_ERR_ARG, "attn_prompt: a NULL array");
    if ((type != SLLM_CUDA_KV_F32 && type != SLLM_CUDA_KV_F16) ||
        (out_type != SLLM_CUDA_KV_F32 && out_type != SLLM_CUDA_KV_F16) ||
        (type == SLLM_CUDA_KV_F32 && out_type == SLLM_CUDA_KV_F16))
        return fail(SLLM_CUDA_ERR_ARG, "attn_prompt: types %d, %d (f32 to f32, f16 to f16 or f32)", type, out_type);
    if (n_seq < 0 || n_seq > (1 << 20) || n_tokens < 0 || n_tokens > (1 << 24) || n_head < 1 || n_head > 1024 ||
        n_head_kv < 1 || n_head % n_head_kv != 0)
        return fail(SLLM_CUDA_ERR_ARG, "attn_prompt: %d sequences, %d tokens, %d heads over %d", n_seq, n_tokens, n_head,
                    n_head_kv);
    const size_t per = type == SLLM_CUDA_KV_F16 ? 8 : 4, oper = out_type == SLLM_CUDA_KV_F16 ? 8 : 4;
    const size_t qn = (size_t)n_head * kServeDim, kn = (size_t)n_head_kv * kServeDim, most = (size_t)1 << 30;
    if (q_stride < qn || k_stride < kn || v_stride < kn || out_stride < qn || q_stride > most || k_stride > most ||
        v_stride > most || out_stride > most || (q_stride | k_stride | v_stride) % per != 0 || out_stride % oper != 0 ||
        !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
        return fail(SLLM_CUDA_ERR_ARG, "attn_prompt: token strides %zu %zu %zu %zu (at least the heads, rows and arrays "
                    "16-byte aligned)", q_stride, k_stride, v_stride, out_stride);
    const void* ptr[] = {q, k, v, cu_seqlens, out};
    const char* name[] = {"q", "k", "v", "cu_seqlens", "out"};
    for (int i = 0; i < 5; ++i) {
        const int rc = need_device(ptr[i], "attn_prompt", name[i]);
        if (rc != SLLM_CUDA_OK) return rc;
    }
    if (n_seq == 0 || n_tokens == 0) return SLLM_CUDA_OK;
    PromptParams p{};
    p.q = q; p.k = k; p.v = v; p.out = out;
    p.qs = q_stride; p.ks = k_stride; p.vs = v_stride; p.os = out_stride;
    p.cu = cu_seqlens;
    p.n_seq = n_seq; p.n_tokens = n_tokens; p.n_head = n_head; p.group = n_head / n_head_kv;
    const cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = type == SLLM_CUDA_KV_F32 ? launch_simt<float, float>(p, st)
                          : out_type == SLLM_CUDA_KV_F32 ? launch_simt<__half, float>(p, st)
                                                         : launch_simt<__half, __half>(p, st);
    CK(e, "attn_prompt launch");
    count_launches(1);
    return SLLM_CUDA_OK;
}
