// attn_simt.cuh -- one tile of attention in 32-bit arithmetic on the ordinary
// pipes: 64 or 16 query rows of one head against 64 keys at a time, with the
// running maximum and sum of a softmax.
//
//   s_ij = q_i . k_j / sqrt(128);  m' = max(m, max_j s_ij)
//   p_ij = exp(s_ij - m');  l = l exp(m - m') + sum_j p_ij
//   o_i  = o_i exp(m - m') + sum_j p_ij v_j;  result o_i / l
//
// The caller gives the rows (row_q: a pointer, or NULL for no row), each
// row's number of visible keys, and the keys' addresses. 256 threads: thread
// (ty, tx) holds rows R ty .. + R - 1 (R = 4 or 1), keys tx, tx + 16, .. of the
// scores and dimensions 4 tx .. + 3 and 64 + 4 tx .. + 3 of the outputs; both
// products run two multiply-adds at a time (f32x2). Keys and values come by
// asynchronous copies, the values under the scores' product. A masked key's
// value is never multiplied: an infinity or NaN there stays out.
//
// Bound: the multiply-add pipe. The weights lie where the keys were, so that
// two CTAs fit an SM and one's loads and softmax run under the other's
// products.
#pragma once

#include "serve.cuh"

namespace sllm {

constexpr int kSimtKeys = 64, kSimtThreads = 256;
constexpr int kSimtDPad = kServeDim + 4;            // q and k rows: eight rows apart in all banks
template <int R> constexpr int kSimtRows = 16 * R;
template <int R> constexpr int kSimtPPad = 16 * R + 4;
template <int R>
constexpr int kSimtSmem = 4 * (kSimtRows<R> * kSimtDPad + kSimtKeys * kSimtDPad + kSimtKeys * kServeDim);
static_assert(kSimtKeys * kSimtPPad<4> <= kSimtKeys * kSimtDPad, "the weights fit the keys' place");

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

template <int R>
struct SimtState {
    float m[R], l[R];
    float2 o[R][4];
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

template <int R, class T, class RowQ>
__device__ __forceinline__ void simt_load_q(float* sm, RowQ row_q) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    #pragma unroll
    for (int i = 0; i < kSimtRows<R> / 8; ++i) {
        const T* q = row_q(warp + 8 * i);
        simt_copy(sm + (warp + 8 * i) * kSimtDPad, q, lane);
    }
    simt_commit();
}

template <int R>
__device__ __forceinline__ void simt_init(SimtState<R>& st) {
    #pragma unroll
    for (int i = 0; i < R; ++i) {
        st.m[i] = -INFINITY;
        st.l[i] = 0.f;
        #pragma unroll
        for (int d = 0; d < 4; ++d) st.o[i][d] = make_float2(0.f, 0.f);
    }
}

// keys [j0, j0 + 64): key_k(j) / key_v(j) give a key's address, or NULL past
// the end; lim[i] is the number of keys that row R ty + i sees
template <int R, class T, class KeyK, class KeyV>
__device__ __forceinline__ void simt_tile(float* sm, SimtState<R>& st, int j0, const int (&lim)[R], KeyK key_k,
                                          KeyV key_v) {
    float* const qs = sm;
    float* const ks = qs + kSimtRows<R> * kSimtDPad;
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
    float2 acc[R][4];
    #pragma unroll
    for (int i = 0; i < R; ++i)
        #pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = make_float2(0.f, 0.f);
    #pragma unroll 4
    for (int d = 0; d < kServeDim; d += 4) {
        float4 q[R], k[4];
        #pragma unroll
        for (int i = 0; i < R; ++i) q[i] = *reinterpret_cast<const float4*>(qs + (R * ty + i) * kSimtDPad + d);
        #pragma unroll
        for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * kSimtDPad + d);
        #pragma unroll
        for (int i = 0; i < R; ++i)
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                mad2(acc[i][j], q[i].x, q[i].y, k[j].x, k[j].y);
                mad2(acc[i][j], q[i].z, q[i].w, k[j].z, k[j].w);
            }
    }
    bool whole = true;
    float p[R][4];
    #pragma unroll
    for (int i = 0; i < R; ++i) {
        float mx = -INFINITY;
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool seen = j0 + tx + 16 * j < lim[i];
            p[i][j] = seen ? __fmul_rn(__fadd_rn(acc[i][j].x, acc[i][j].y), kServeScale) : -INFINITY;
            mx = fmaxf(mx, p[i][j]);
        }
        #pragma unroll
        for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float m = fmaxf(st.m[i], mx);
        // a row that has seen nothing yet keeps its zeros
        const float f = m == -INFINITY ? 1.f : expf(__fsub_rn(st.m[i], m));
        float sum = 0.f;
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool seen = j0 + tx + 16 * j < lim[i];
            p[i][j] = seen ? expf(__fsub_rn(p[i][j], m)) : 0.f;
            sum = __fadd_rn(sum, p[i][j]);
        }
        #pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, o));
        st.l[i] = __fmaf_rn(st.l[i], f, sum);
        st.m[i] = m;
        #pragma unroll
        for (int d = 0; d < 4; ++d) {
            st.o[i][d].x = __fmul_rn(st.o[i][d].x, f);
            st.o[i][d].y = __fmul_rn(st.o[i][d].y, f);
        }
        whole = whole && j0 + kSimtKeys <= lim[i];
    }
    __syncthreads();                                // the keys have been read: the weights take their place
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        float* at = pt + (tx + 16 * j) * kSimtPPad<R> + R * ty;
        if constexpr (R == 4) st4(at, make_float4(p[0][j], p[1][j], p[2][j], p[3][j]));
        else at[0] = p[0][j];
    }
    simt_wait<0>();
    __syncthreads();
    auto add = [&](auto masked) {
        #pragma unroll 4
        for (int j = 0; j < kSimtKeys; ++j) {
            float w[R];
            if constexpr (R == 4) {
                const float4 x = *reinterpret_cast<const float4*>(pt + j * kSimtPPad<R> + R * ty);
                w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
            } else {
                w[0] = pt[j * kSimtPPad<R> + ty];
            }
            const float4 v0 = *reinterpret_cast<const float4*>(vs + j * kServeDim + 4 * tx);
            const float4 v1 = *reinterpret_cast<const float4*>(vs + j * kServeDim + 64 + 4 * tx);
            const float vv[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
            #pragma unroll
            for (int i = 0; i < R; ++i) {
                const bool seen = !decltype(masked)::value || j0 + j < lim[i];
                #pragma unroll
                for (int d = 0; d < 4; ++d)
                    mad2(st.o[i][d], w[i], w[i], seen ? vv[2 * d] : 0.f, seen ? vv[2 * d + 1] : 0.f);
            }
        }
    };
    if (whole) add(std::false_type{});
    else add(std::true_type{});
}

// out: dimension-contiguous row of 128 values, scaled
template <int R, class O>
__device__ __forceinline__ void simt_store(const SimtState<R>& st, int i, float f, O* out) {
    const int tx = threadIdx.x & 15;
    st4(out + 4 * tx, make_float4(__fmul_rn(st.o[i][0].x, f), __fmul_rn(st.o[i][0].y, f), __fmul_rn(st.o[i][1].x, f),
                                  __fmul_rn(st.o[i][1].y, f)));
    st4(out + 64 + 4 * tx, make_float4(__fmul_rn(st.o[i][2].x, f), __fmul_rn(st.o[i][2].y, f),
                                       __fmul_rn(st.o[i][3].x, f), __fmul_rn(st.o[i][3].y, f)));
}

}  // namespace sllm
