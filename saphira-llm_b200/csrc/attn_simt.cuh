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
// (ty, tx) holds rows R ty .. + R - 1 (R = 4 or 1), columns 4 tx .. + 3 of the
// scores and dimensions 4 tx .. + 3 and 64 + 4 tx .. + 3 of the outputs. A masked key's
// value is never multiplied: an infinity or NaN there stays out.
#pragma once

#include "serve.cuh"

namespace sllm {

constexpr int kSimtKeys = 64, kSimtThreads = 256;
constexpr int kSimtPad = kSimtKeys + 4;
template <int R> constexpr int kSimtRows = 16 * R;
template <int R> constexpr int kSimtQPad = 16 * R + 4;
// q and k transposed ([dim][row], so that a thread's four rows are one
// 16-byte read), v as it is, p transposed ([key][row])
template <int R>
constexpr int kSimtSmem = 4 * (kServeDim * kSimtQPad<R> + kServeDim * kSimtPad + kSimtKeys * kServeDim + kSimtKeys * kSimtQPad<R>);
constexpr float kServeScale = 0.08838834764831845f;     // 1 / sqrt(128)

template <int R>
struct SimtState {
    float m[R], l[R], o[R][8];
};

template <int R>
__device__ __forceinline__ void ld_rows(const float* p, float (&v)[R]) {
    if constexpr (R == 4) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
        v[0] = p[0];
    }
}

template <int R, class T, class RowQ>
__device__ __forceinline__ void simt_load_q(float* sm, RowQ row_q) {
    float* qt = sm;
    for (int x = threadIdx.x; x < kSimtRows<R> * 32; x += kSimtThreads) {
        const int r = x % kSimtRows<R>, c = x / kSimtRows<R>;   // neighbouring threads: neighbouring rows
        const T* q = row_q(r);
        const float4 v = q != nullptr ? ld4(q + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
        qt[(4 * c) * kSimtQPad<R> + r] = v.x;
        qt[(4 * c + 1) * kSimtQPad<R> + r] = v.y;
        qt[(4 * c + 2) * kSimtQPad<R> + r] = v.z;
        qt[(4 * c + 3) * kSimtQPad<R> + r] = v.w;
    }
}

template <int R>
__device__ __forceinline__ void simt_init(SimtState<R>& st) {
    #pragma unroll
    for (int i = 0; i < R; ++i) {
        st.m[i] = -INFINITY;
        st.l[i] = 0.f;
        #pragma unroll
        for (int d = 0; d < 8; ++d) st.o[i][d] = 0.f;
    }
}

// keys [j0, j0 + 64): key_k(j) / key_v(j) give a key's address, or NULL past
// the end; lim[i] is the number of keys that row R ty + i sees
template <int R, class T, class KeyK, class KeyV>
__device__ __forceinline__ void simt_tile(float* sm, SimtState<R>& st, int j0, const int (&lim)[R], KeyK key_k,
                                          KeyV key_v) {
    float* const qt = sm;
    float* const kt = qt + kServeDim * kSimtQPad<R>;
    float* const vs = kt + kServeDim * kSimtPad;
    float* const pt = vs + kSimtKeys * kServeDim;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    __syncthreads();                                // the tile before is done with kt, vs and pt
    for (int x = threadIdx.x; x < kSimtKeys * 32; x += kSimtThreads) {
        const int r = x & 63, c = x >> 6;
        const T* k = key_k(j0 + r);
        const float4 v = k != nullptr ? ld4(k + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
        kt[(4 * c) * kSimtPad + r] = v.x;
        kt[(4 * c + 1) * kSimtPad + r] = v.y;
        kt[(4 * c + 2) * kSimtPad + r] = v.z;
        kt[(4 * c + 3) * kSimtPad + r] = v.w;
    }
    for (int x = threadIdx.x; x < kSimtKeys * 32; x += kSimtThreads) {
        const int r = x >> 5, c = x & 31;
        const T* v = key_v(j0 + r);
        st4(vs + r * kServeDim + 4 * c, v != nullptr ? ld4(v + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f));
    }
    __syncthreads();
    float s[R][4] = {};
    #pragma unroll 8
    for (int d = 0; d < kServeDim; ++d) {
        float av[R];
        ld_rows<R>(qt + d * kSimtQPad<R> + R * ty, av);
        const float4 b = *reinterpret_cast<const float4*>(kt + d * kSimtPad + 4 * tx);
        const float bv[4] = {b.x, b.y, b.z, b.w};
        #pragma unroll
        for (int i = 0; i < R; ++i)
            #pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = __fmaf_rn(av[i], bv[j], s[i][j]);
    }
    bool whole = true;
    #pragma unroll
    for (int i = 0; i < R; ++i) {
        float mx = -INFINITY;
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool seen = j0 + 4 * tx + j < lim[i];
            s[i][j] = seen ? __fmul_rn(s[i][j], kServeScale) : -INFINITY;
            mx = fmaxf(mx, s[i][j]);
        }
        #pragma unroll
        for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float m = fmaxf(st.m[i], mx);
        // a row that has seen nothing yet keeps its zeros
        const float f = m == -INFINITY ? 1.f : expf(__fsub_rn(st.m[i], m));
        float sum = 0.f;
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool seen = j0 + 4 * tx + j < lim[i];
            const float p = seen ? expf(__fsub_rn(s[i][j], m)) : 0.f;
            pt[(4 * tx + j) * kSimtQPad<R> + R * ty + i] = p;
            sum = __fadd_rn(sum, p);
        }
        #pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, o));
        st.l[i] = __fmaf_rn(st.l[i], f, sum);
        st.m[i] = m;
        #pragma unroll
        for (int d = 0; d < 8; ++d) st.o[i][d] = __fmul_rn(st.o[i][d], f);
        whole = whole && j0 + kSimtKeys <= lim[i];
    }
    __syncthreads();
    auto add = [&](auto masked) {
        #pragma unroll 4
        for (int j = 0; j < kSimtKeys; ++j) {
            float pv[R];
            ld_rows<R>(pt + j * kSimtQPad<R> + R * ty, pv);
            const float4 v0 = *reinterpret_cast<const float4*>(vs + j * kServeDim + 4 * tx);
            const float4 v1 = *reinterpret_cast<const float4*>(vs + j * kServeDim + 64 + 4 * tx);
            const float vv[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
            #pragma unroll
            for (int i = 0; i < R; ++i) {
                const bool seen = !decltype(masked)::value || j0 + j < lim[i];
                #pragma unroll
                for (int d = 0; d < 8; ++d) st.o[i][d] = __fmaf_rn(pv[i], seen ? vv[d] : 0.f, st.o[i][d]);
            }
        }
    };
    if (whole) add(std::false_type{});
    else add(std::true_type{});
}

// out: dimension-contiguous row of 128 values
template <int R, class O>
__device__ __forceinline__ void simt_store(const SimtState<R>& st, int i, O* out) {
    const int tx = threadIdx.x & 15;
    // a row that saw no key: zeros
    const float inv = st.m[i] == -INFINITY && st.l[i] == 0.f ? 0.f : __fdiv_rn(1.f, st.l[i]);
    st4(out + 4 * tx, make_float4(__fmul_rn(st.o[i][0], inv), __fmul_rn(st.o[i][1], inv), __fmul_rn(st.o[i][2], inv),
                                  __fmul_rn(st.o[i][3], inv)));
    st4(out + 64 + 4 * tx, make_float4(__fmul_rn(st.o[i][4], inv), __fmul_rn(st.o[i][5], inv),
                                       __fmul_rn(st.o[i][6], inv), __fmul_rn(st.o[i][7], inv)));
}

}  // namespace sllm
