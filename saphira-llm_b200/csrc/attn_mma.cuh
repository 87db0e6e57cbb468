// attn_mma.cuh -- what the tensor-core attention kernels share: barriers'
// names, the softmax of one 128-key tile of scores held in tensor memory, and
// the slow path of a tile whose unseen values are no numbers.
#pragma once

#include "serve.cuh"
#include "umma.cuh"

namespace sllm {

constexpr int kAtRows = 128;                    // query rows of a tile: the TMEM lanes
constexpr int kAtKeys = 128;                    // keys of a tile
constexpr int kAtHalf = 128 * 128;              // bytes of 128 rows x 64 f16 in the 128-byte swizzle
constexpr int kAtTile = 2 * kAtHalf;            // ... x 128 f16
// softmax in base 2: exp(s / sqrt(128)) = 2^(s c)
constexpr float kAtScale2 = 0.08838834764831845f * 1.4426950408889634f;
// the running maximum a row's weights stand against may lag behind by this
// many doublings before its sums are rescaled: weights stay below 2^8, far
// from f16's limit, and most tiles need no pass over the outputs
constexpr float kAtLag = 8.0f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// two f32 at a time (sm_100's packed pipe): a * b + c, x += a
__device__ __forceinline__ void fma2v(float& x, float& y, float a0, float a1, float b0, float b1, float c0, float c1) {
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\t"
        "mov.b64 b, {%4, %5};\n\t"
        "mov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "=f"(x), "=f"(y)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void add2(float& x, float& y, float a0, float a1) {
    asm("{\n\t.reg .b64 a, d;\n\t"
        "mov.b64 a, {%2, %3};\n\t"
        "mov.b64 d, {%0, %1};\n\t"
        "add.rn.f32x2 d, d, a;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(a0), "f"(a1));
}

template <int N>
__device__ __forceinline__ void reg_dealloc() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_alloc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// The bounded waits of umma.cuh, in line: a kernel that splits its registers
// between its warps cannot call functions.
__device__ __forceinline__ bool at_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* error) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = gtimer();
    #pragma unroll 1
    while (!mbar_try_wait(bar, parity)) {
        if (*abort_flag) return false;
        if (gtimer() - t0 > kGmWaitNs) {
            *abort_flag = 1;
            atomicExch(error, GM_TIMEOUT);
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ bool at_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* error) {
    return __all_sync(0xffffffffu, at_wait(bar, parity, abort_flag, error));
}
__device__ __forceinline__ void at_drain(uint64_t* bar, uint32_t parity) {
    const uint64_t t0 = gtimer();
    #pragma unroll 1
    while (!mbar_try_wait(bar, parity))
        if (gtimer() - t0 > kGmWaitNs) return;
}

// (the maxima keep a NaN, so that a row which sees one becomes NaN)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float row_max(const float (&s)[128]) {
    float a = max3(s[0], s[1], s[2]), b = max3(s[3], s[4], s[5]), c = max3(s[6], s[7], s[8]), d = s[9];
    #pragma unroll
    for (int i = 10; i < 122; i += 8) {
        a = max3(a, s[i], s[i + 1]);
        b = max3(b, s[i + 2], s[i + 3]);
        c = max3(c, s[i + 4], s[i + 5]);
        d = max3(d, s[i + 6], s[i + 7]);
    }
    a = max3(a, s[122], s[123]);
    b = max3(b, s[124], s[125]);
    c = max3(c, s[126], s[127]);
    return max3(a, b, max3(c, d, d));
}
// a non-finite f16 in two packed ones
__device__ __forceinline__ bool odd_half2(uint32_t u) {
    return (u & 0x7c00u) == 0x7c00u || (u & 0x7c000000u) == 0x7c000000u;
}

// the weights of 64 of a row's scores: two f16 per word, and their sums
// before the rounding. All exponentials go through the special-function pipe:
// moving 1/8, 1/4 or 3/8 of them to a degree-4 polynomial on the multiply-add
// pipe measured slower (one prompt of 16384 tokens, 16 heads: 871 us without,
// 889, 898, 919 us).
__device__ __forceinline__ void half_weights(const float* s, float mc, uint32_t (&u)[32], float (&sum)[4]) {
    #pragma unroll
    for (int i = 0; i < 32; ++i) {
        float x0, x1;
        fma2v(x0, x1, s[2 * i], s[2 * i + 1], kAtScale2, kAtScale2, mc, mc);
        x0 = ex2(x0);
        x1 = ex2(x1);
        if (i & 1) add2(sum[0], sum[1], x0, x1);
        else add2(sum[2], sum[3], x0, x1);
        u[i] = pack_half2(x0, x1);
    }
}
// what the scaled scores are offset by: -m in base 2. A row that has only
// seen -inf has weights 0; one that has seen +inf is no number.
__device__ __forceinline__ float weight_offset(float m) {
    return m == -INFINITY ? 0.f : m == INFINITY ? NAN : -m * kAtScale2;
}

// a row's 128 scores from tensor memory
__device__ __forceinline__ void load_scores(uint32_t s_tmem, float (&s)[128]) {
    #pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint32_t r[32];
        tmem_ld32(s_tmem + 32 * c, r);
        #pragma unroll
        for (int i = 0; i < 32; ++i) s[32 * c + i] = __uint_as_float(r[i]);
    }
    tmem_ld_wait();
}

// the tensor-memory outputs of one row, scaled, to global memory: f16 or f32
__device__ __forceinline__ void store_row(uint32_t o_tmem, float f, bool live, __half* out) {
    #pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint32_t r[32];
        tmem_ld32(o_tmem + 32 * c, r);
        tmem_ld_wait();
        if (live) {
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint4 u;
                uint32_t* w = &u.x;
                #pragma unroll
                for (int e = 0; e < 4; ++e)
                    w[e] = pack_half2(__uint_as_float(r[8 * i + 2 * e]) * f, __uint_as_float(r[8 * i + 2 * e + 1]) * f);
                *reinterpret_cast<uint4*>(out + 32 * c + 8 * i) = u;
            }
        }
    }
}
__device__ __forceinline__ void store_row(uint32_t o_tmem, float f, bool live, float* out) {
    #pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint32_t r[32];
        tmem_ld32(o_tmem + 32 * c, r);
        tmem_ld_wait();
        if (live) {
            #pragma unroll
            for (int i = 0; i < 8; ++i)
                *reinterpret_cast<float4*>(out + 32 * c + 4 * i) =
                    make_float4(__uint_as_float(r[4 * i]) * f, __uint_as_float(r[4 * i + 1]) * f,
                                __uint_as_float(r[4 * i + 2]) * f, __uint_as_float(r[4 * i + 3]) * f);
        }
    }
}

}  // namespace sllm
