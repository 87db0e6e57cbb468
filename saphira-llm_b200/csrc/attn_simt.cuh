// attn_simt.cuh -- one tile of attention in 32-bit arithmetic on the ordinary
// pipes: 16 query rows of one head against 64 keys at a time, with the running
// maximum and sum of a softmax. For so few rows the tensor cores' tiles of 128
// would be all padding.
//
//   s_ij = q_i . k_j / sqrt(128);  m' = max(m, max_j s_ij)
//   p_ij = exp(s_ij - m');  l = l exp(m - m') + sum_j p_ij
//   o_i  = o_i exp(m - m') + sum_j p_ij v_j;  result o_i / l
//
// The caller gives the rows (row_q: a pointer, or NULL for no row), each
// row's number of visible keys, and the keys' addresses. 256 threads: thread
// (ty, tx) holds row ty, keys tx, tx + 16, .. of the scores and dimensions
// 4 tx .. + 3 and 64 + 4 tx .. + 3 of the outputs; both products run two
// multiply-adds at a time (f32x2). f32 keys and values come by asynchronous
// copies, the values under the scores' product. A masked key's value is never
// multiplied: an infinity or NaN there stays out.
//
// Bound: for a few tiles the latency of their loads. The weights lie where the
// keys were, so that two CTAs fit an SM.
#pragma once

#include "serve.cuh"

namespace sllm {

constexpr int kSimtRows = 16, kSimtKeys = 64, kSimtThreads = 256;
constexpr int kSimtDPad = kServeDim + 4;            // q and k rows: eight rows apart in all banks
constexpr int kSimtPPad = kSimtRows + 4;
constexpr int kSimtSmem = 4 * (kSimtRows * kSimtDPad + kSimtKeys * kSimtDPad + kSimtKeys * kServeDim);
static_assert(kSimtKeys * kSimtPPad <= kSimtKeys * kSimtDPad, "the weights fit the keys' place");

// two f32 at a time (sm_100's packed pipe): x += a * b
__device__ __forceinline__ void mad2(float2& x, float a0, float a1, float b0, float b1) {
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\t"
        "mov.b64 b, {%4, %5};\n\t"
        "mov.b64 d, {%0, %1};\n\t"
        "fma.rn.f32x2 d, a, b, d;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "+f"(x.x), "+f"(x.y)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}

struct SimtState {
    float m, l;
    float2 o[4];
};

// a row's 4 elements into shared memory, zeros for a NULL row: f32 by an
// asynchronous copy, f16 through registers
__device__ __forceinline__ void simt_copy(float* dst, const float* src, int c) {
    if (src != nullptr)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst + 4 * c)),
                     "l"(src + 4 * c)
                     : "memory");
    else
        st4(dst + 4 * c, make_float4(0.f, 0.f, 0.f, 0.f));
}
__device__ __forceinline__ void simt_copy(float* dst, const __half* src, int c) {
    st4(dst + 4 * c, src != nullptr ? ld4(src + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f));
}
__device__ __forceinline__ void simt_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void simt_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <class T, class RowQ>
__device__ __forceinline__ void simt_load_q(float* sm, RowQ row_q) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    #pragma unroll
    for (int i = 0; i < kSimtRows / 8; ++i) simt_copy(sm + (warp + 8 * i) * kSimtDPad, row_q(warp + 8 * i), lane);
    simt_commit();
}

__device__ __forceinline__ void simt_init(SimtState& st) {
    st.m = -INFINITY;
    st.l = 0.f;
    #pragma unroll
    for (int d = 0; d < 4; ++d) st.o[d] = make_float2(0.f, 0.f);
}

// keys [j0, j0 + 64): key_k(j) / key_v(j) give a key's address, or NULL past
// the end; lim is the number of keys that row ty sees
template <class T, class KeyK, class KeyV>
__device__ __forceinline__ void simt_tile(float* sm, SimtState& st, int j0, int lim, KeyK key_k, KeyV key_v) {
    float* const qs = sm;
    float* const ks = qs + kSimtRows * kSimtDPad;
    float* const vs = ks + kSimtKeys * kSimtDPad;
    float* const pt = ks;                           // [key][row]
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();                                // the tile before is done with its weights and values
    {
        const T* at[kSimtKeys / 8];
        #pragma unroll
        for (int i = 0; i < kSimtKeys / 8; ++i) at[i] = key_k(j0 + warp + 8 * i);
        #pragma unroll
        for (int i = 0; i < kSimtKeys / 8; ++i) simt_copy(ks + (warp + 8 * i) * kSimtDPad, at[i], lane);
        simt_commit();
        #pragma unroll
        for (int i = 0; i < kSimtKeys / 8; ++i) at[i] = key_v(j0 + warp + 8 * i);
        #pragma unroll
        for (int i = 0; i < kSimtKeys / 8; ++i) simt_copy(vs + (warp + 8 * i) * kServeDim, at[i], lane);
        simt_commit();
    }
    simt_wait<1>();                                 // q and this tile's keys
    __syncthreads();
    float2 acc[4];
    #pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = make_float2(0.f, 0.f);
    #pragma unroll 8
    for (int d = 0; d < kServeDim; d += 4) {
        const float4 q = *reinterpret_cast<const float4*>(qs + ty * kSimtDPad + d);
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4 k = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * kSimtDPad + d);
            mad2(acc[j], q.x, q.y, k.x, k.y);
            mad2(acc[j], q.z, q.w, k.z, k.w);
        }
    }
    float p[4], mx = -INFINITY;
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool seen = j0 + tx + 16 * j < lim;
        p[j] = seen ? __fmul_rn(__fadd_rn(acc[j].x, acc[j].y), kServeScale) : -INFINITY;
        mx = fmaxf(mx, p[j]);
    }
    #pragma unroll
    for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float m = fmaxf(st.m, mx);
    // a row that has seen nothing yet keeps its zeros
    const float f = m == -INFINITY ? 1.f : expf(__fsub_rn(st.m, m));
    float sum = 0.f;
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool seen = j0 + tx + 16 * j < lim;
        p[j] = seen ? expf(__fsub_rn(p[j], m)) : 0.f;
        sum = __fadd_rn(sum, p[j]);
    }
    #pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, o));
    st.l = __fmaf_rn(st.l, f, sum);
    st.m = m;
    #pragma unroll
    for (int d = 0; d < 4; ++d) {
        st.o[d].x = __fmul_rn(st.o[d].x, f);
        st.o[d].y = __fmul_rn(st.o[d].y, f);
    }
    __syncthreads();                                // the keys have been read: the weights take their place
    #pragma unroll
    for (int j = 0; j < 4; ++j) pt[(tx + 16 * j) * kSimtPPad + ty] = p[j];
    simt_wait<0>();
    __syncthreads();
    auto add = [&](auto masked) {
        #pragma unroll 8
        for (int j = 0; j < kSimtKeys; ++j) {
            const float w = pt[j * kSimtPPad + ty];
            const float4 v0 = *reinterpret_cast<const float4*>(vs + j * kServeDim + 4 * tx);
            const float4 v1 = *reinterpret_cast<const float4*>(vs + j * kServeDim + 64 + 4 * tx);
            const float vv[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
            const bool seen = !decltype(masked)::value || j0 + j < lim;
            #pragma unroll
            for (int d = 0; d < 4; ++d) mad2(st.o[d], w, w, seen ? vv[2 * d] : 0.f, seen ? vv[2 * d + 1] : 0.f);
        }
    };
    if (j0 + kSimtKeys <= lim) add(std::false_type{});
    else add(std::true_type{});
}

// out: dimension-contiguous row of 128 values
__device__ __forceinline__ void simt_store(const SimtState& st, float* out) {
    const int tx = threadIdx.x & 15;
    st4(out + 4 * tx, make_float4(st.o[0].x, st.o[0].y, st.o[1].x, st.o[1].y));
    st4(out + 64 + 4 * tx, make_float4(st.o[2].x, st.o[2].y, st.o[3].x, st.o[3].y));
}

}  // namespace sllm
