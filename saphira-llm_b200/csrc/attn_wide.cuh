// attn_wide.cuh -- attention of 32-bit operands on the tensor cores.
//
// An f32 is the sum of three bf16, 24 bits in all, with f32's range: x = x1 +
// x2 + x3, x1 = x rounded to bf16, x2 = the first eight bits of x - x1, x3 = the
// rest (the differences are exact). A product is the six partial products whose size is
// above 2^-25 of it,
//     x y = x1 y1 + x1 y2 + x2 y1 + x2 y2 + x1 y3 + x3 y1,
// each exact in the tensor core's f32 accumulator: as good as 32-bit
// multiply-adds, at a sixth of the bf16 rate, which is still four times the
// ordinary pipe's.
//
// One CTA: 128 query rows of one head against 64 keys at a time.
//
//   warps 0-3        softmax, one thread per row (warp 0 finds the item first).
//   warps 4-11, 12-19  the operands: the keys' and the values' tiles from
//                    global memory (the next tile waits in registers), split,
//                    into shared memory in the layouts the products want.
//                    Sixteen warps: with eight the splitting took twice the
//                    products' time. At the start all twenty split Q; at the
//                    end these sixteen store the outputs, 32 x 32 each.
//   warp 20, 1 lane  tcgen05.mma: 6 x 8 products of N = 64 for a tile's scores,
//                    6 x 4 of N = 128 for the outputs, with the weights' planes
//                    from tensor memory. The scores of tile j + 1 are made
//                    under the softmax of tile j, which reads its own first.
//
// Q's first plane, which three of the six products take, lies in tensor memory:
// those read 2 KB of shared memory instead of 6 (32 clocks instead of 48), and
// the place it leaves holds a second tile of keys.
//
// Products of different shapes are not ordered among themselves, so none
// touches tensor memory that one of the other shape reads or writes, except
// across a commit: scores 64 columns, Q 64, weights 96, outputs 2 x 128. (One
// product of N = 192 over a key tile's three planes, the softmax adding the
// column groups, would save a quarter of the scores' time, but partial sums of
// three shapes would lean on an order that is not promised.)
//
// Bound by the products and, at half their time each, the softmax and the
// splitting that run beside them: 24 x 32 + 24 x 48 + 24 x 64 = 3456 clocks a
// tile of 4.2 MFLOP, 323 TFLOP/s over 148 SMs at 1.8 GHz. Measured 2.6 us a
// tile (4096 tokens, 20 heads: 372 us, 231 TFLOP/s); with the splitting left out
// 2.4 us, with the products cut to a sixth besides 1.7 us. An item's start and
// end cost about 9 us: 1.2 to find it among several prompts, 2.6 to read and
// split Q and the first tile, 2.6 for the first scores and softmax, 1.6 for the
// last products, 1.4 to store. Four prompts of 320, 1, 777 and 256 tokens: 42.4
// us, the longest row tile's 36 us among them. 32 heads of 8 against a prefix of
// 16384: 59 us.
//
// Registers: 768 threads x 80 at launch; 152 (softmax) + 4 x 72 (operands) + 40
// = 480 = 6 x 80 after the split.
//
// Masks as in attn_mma.cuh: rows behind the keys are stored as zeros, and so is
// a value that is no number, among keys that not every row sees; add_odd brings
// it to the rows that do. A key that a row does see and that is no finite number
// makes that row no number, a value its dimension.
#pragma once

#include <type_traits>

#include "attn_mma.cuh"

namespace sllm {

constexpr int kWdKeys = 64;
constexpr int kWdQPlane = kAtTile;                      // 128 rows x 128 bf16
constexpr int kWdHalf = kWdKeys * 128, kWdPlane = 2 * kWdHalf;      // 64 rows x 64 bf16, x 128
// shared memory: the queries' second and third plane, two tiles of keys, one of values
constexpr int kWdK = 2 * kWdQPlane, kWdV = kWdK + 6 * kWdPlane, kWdEnd = kWdV + 3 * kWdPlane;
constexpr int kWdStage = kWdK + 3 * kWdPlane;           // where the first plane waits for its way into tensor memory
static_assert(kWdQPlane <= 3 * kWdPlane, "in the place of the second tile of keys");
// tensor memory columns behind the scores: the queries' first plane, weights,
// outputs, their total
constexpr int kWdQ1 = 64, kWdP = 128, kWdO = 224, kWdT = 352;
// The tensor core cuts a sum's last bits instead of rounding, always towards
// zero: 1.3e-7 of an output per key tile, 8e-6 after 4000 keys. So the outputs
// of every kWdFold key tiles are summed by themselves, and added to their total
// by ordinary additions (error after 4000 keys 6.6e-7; one tile 3.3e-7 and 3%
// more time, four 1.2e-6; a plain 32-bit computation is 7.9e-7 off).
constexpr int kWdFold = 2;
constexpr int kWdSmem = kWdEnd + 1024;
constexpr int kWdThreads = 32 * 24;

__host__ __device__ constexpr uint32_t umma_idesc_bf16(int M, int N, bool b_mn) {
    return umma_idesc_f16(M, N, b_mn) | (1u << 7) | (1u << 10);
}

__device__ __forceinline__ uint32_t pack_bf2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// two f32 into three words of two bf16 (finite ones; of others only the first
// word means something)
__device__ __forceinline__ uint32_t upper2(float lo, float hi) {
    return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
}
__device__ __forceinline__ float upper(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// (the differences are exact, so a multiply-add by -1 is one)
__device__ __forceinline__ void minus2(float& a, float& b, float x, float y) { fma2v(a, b, x, y, -1.f, -1.f, a, b); }
__device__ __forceinline__ void split2(float a, float b, uint32_t& p1, uint32_t& p2, uint32_t& p3) {
    p1 = pack_bf2(a, b);
    minus2(a, b, __uint_as_float(p1 << 16), __uint_as_float(p1 & 0xffff0000u));
    p2 = upper2(a, b);
    minus2(a, b, upper(a), upper(b));
    p3 = upper2(a, b);
}

// t, or the largest of |x|; NaN when one is
__device__ __forceinline__ float top4(float4 x, float t) {
    return max3(fabsf(x.z), fabsf(x.w), max3(fabsf(x.x), fabsf(x.y), t));
}
// no NaN, no infinity, nothing that bf16 would round to one
__device__ __forceinline__ bool plain(float top) { return !is_odd(top); }

// four elements of a row into its three planes: `at` is the row's 128 bytes of
// the lane's half in the second plane, `first` in the first, r its number in
// the swizzle. What is not plain lies in the first plane alone.
__device__ __forceinline__ void store_planes(uint8_t* at, uint8_t* first, int r, int lane, int plane, float4 x, bool whole) {
    uint32_t a[3], b[3];
    split2(x.x, x.y, a[0], a[1], a[2]);
    split2(x.z, x.w, b[0], b[1], b[2]);
    if (!whole) a[1] = a[2] = b[1] = b[2] = 0u;
    const int in = ((((lane & 15) >> 1) ^ (r & 7)) << 4) + (lane & 1) * 8;
    *reinterpret_cast<uint2*>(first + in) = make_uint2(a[0], b[0]);
    *reinterpret_cast<uint2*>(at + in) = make_uint2(a[1], b[1]);
    *reinterpret_cast<uint2*>(at + in + plane) = make_uint2(a[2], b[2]);
}

// ... of which some are not plain: those lie in the first plane alone, or, where
// they are hidden, nowhere; true: something was hidden
__device__ __forceinline__ bool store_odd(uint8_t* at, uint8_t* first, int r, int lane, int plane, float4 v, bool hidden) {
    const float x[4] = {v.x, v.y, v.z, v.w};
    float y[4];
    #pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = is_odd(x[e]) ? 0.f : x[e];
    store_planes(at, first, r, lane, plane, make_float4(y[0], y[1], y[2], y[3]), true);
    const int in = ((((lane & 15) >> 1) ^ (r & 7)) << 4) + (lane & 1) * 8;
    bool any = false;
    #pragma unroll
    for (int e = 0; e < 4; ++e)
        if (is_odd(x[e])) {
            any = true;
            if (!hidden) *reinterpret_cast<uint16_t*>(first + in + 2 * e) = (uint16_t)pack_bf2(x[e], 0.f);
        }
    return any && hidden;
}

// r[i] without an index into registers
__device__ __forceinline__ float4 pick(const float4 (&r)[8], int i) {
    float4 x = r[0];
    #pragma unroll
    for (int e = 1; e < 8; ++e)
        if (e == i) x = r[e];
    return x;
}

struct WideOut {
    float* base;                    // the first row
    size_t stride;                  // floats from a row to the next
    int n;                          // rows to be written
};

// One warp's 32 rows x 32 columns of outputs, plus their total, times each
// lane's f, to global memory, through the warp's staging: whole lines, four
// rows a store.
__device__ __forceinline__ void store_cols(uint32_t o_tm, uint32_t t_tm, bool total, float f, uint8_t* stage,
                                           const WideOut& to) {
    const int lane = threadIdx.x & 31, sub = lane >> 3;
    #pragma unroll
    for (int c = 0; c < 2; ++c) {
        uint32_t a[16], t[16];
        tmem_ld16(o_tm + 16 * c, a);
        if (total) tmem_ld16(t_tm + 16 * c, t);
        tmem_ld_wait();
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x[4];
            #pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = __uint_as_float(a[4 * i + e]);
                if (total) x[e] = __fadd_rn(x[e], __uint_as_float(t[4 * i + e]));
                x[e] = __fmul_rn(x[e], f);
            }
            *reinterpret_cast<float4*>(stage + lane * kAtStageRow + 64 * c + 16 * i) = make_float4(x[0], x[1], x[2], x[3]);
        }
    }
    __syncwarp();
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float4 u = *reinterpret_cast<const float4*>(stage + (4 * i + sub) * kAtStageRow + 16 * (lane & 7));
        if (4 * i + sub < to.n) st4(to.base + (size_t)(4 * i + sub) * to.stride + 4 * (lane & 7), u);
    }
}

// W: Item; T; find(x, item); keys(item); live(item, row); seen(item, row) (at
// most keys, least for row 0); q_row(item, row); Rows (one warp's keys or values:
// tile(key, n): the next are keys key, key + 8, .. below n; row(i): the i-th of
// them); scale(l) (what the outputs are multiplied by), out(item, row) (where the
// rows from `row` on go), finish(item, row, m, l) (the rest of a row's result),
// value(item, key) (a row of values), check() (one warp of each CTA), wait_limit(),
// gave_up().
template <class W>
__device__ __forceinline__ void attn_wide_core(const W w) {
    using T = typename W::T;
    extern __shared__ __align__(1024) uint8_t sm[];
    struct Shared {
        // q: split; q1: the first plane in tensor memory; k, v: tile split; vf:
        // its products done; s: scores (and the keys' place free; by tile
        // parity, since a wait may come two tiles late); sf: scores read; p:
        // weights; f: the rows' factors; o: all
        uint64_t bar_q, bar_q1, bar_k[2], bar_v, bar_vf, bar_s[2], bar_sf, bar_p, bar_f, bar_o;
        typename W::Item item;
        float f[kAtRows];
        uint32_t tmem;
        int abort_flag, odd, none;
    };
    static_assert(sizeof(Shared) <= kWdSmem - kWdEnd, "the part behind the planes");
    Shared& sh = *reinterpret_cast<Shared*>(sm + kWdEnd);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if ((smem_u32(sm) & 1023u) != 0) {
        if (threadIdx.x == 0) atomicExch(&g_attn_error, 2);
        return;
    }
    if (warp == 0) {                    // (by every warp it took twice as long)
        typename W::Item it;
        const bool found = w.find(blockIdx.x, &it) && !it.last();       // the grid is an upper bound
        if (lane == 0) {
            sh.item = it;
            sh.none = !found;
        }
    }
    if (warp == 23) w.check();
    if (threadIdx.x == 32) {
        mbar_init(&sh.bar_q, 20);
        mbar_init(&sh.bar_q1, 4);
        mbar_init(&sh.bar_k[0], 8);
        mbar_init(&sh.bar_k[1], 8);
        mbar_init(&sh.bar_v, 8);
        mbar_init(&sh.bar_vf, 1);
        mbar_init(&sh.bar_s[0], 1);
        mbar_init(&sh.bar_s[1], 1);
        mbar_init(&sh.bar_sf, 4);
        mbar_init(&sh.bar_p, 4);
        mbar_init(&sh.bar_f, 4);
        mbar_init(&sh.bar_o, 1);
        sh.abort_flag = 0;
        sh.odd = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 20) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    if (sh.none) {
        if (warp == 20)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
        return;
    }
    const typename W::Item it = sh.item;
    volatile int* const ab = &sh.abort_flag;
    const int keys = w.keys(it), n = (keys + kWdKeys - 1) / kWdKeys;

    const int half = lane >> 4;
    auto arrive = [&](uint64_t* bar) {      // what this warp wrote is the products'
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    // a row without anything
    auto store_none = [&](uint8_t* at, uint8_t* first, int r, int plane) {
        const int in = ((((lane & 15) >> 1) ^ (r & 7)) << 4) + (lane & 1) * 8;
        *reinterpret_cast<uint2*>(first + in) = make_uint2(0u, 0u);
        *reinterpret_cast<uint2*>(at + in) = make_uint2(0u, 0u);
        *reinterpret_cast<uint2*>(at + in + plane) = make_uint2(0u, 0u);
    };
    // N rows of Q, all their loads in flight: the softmax warps take the upper
    // half, the operands' warps the lower
    auto split_q = [&](auto count, int from, int step) {
        constexpr int N = decltype(count)::value;
        uint8_t* const at = sm + half * kAtHalf;
        if (w.live(it, from + (N - 1) * step)) {
            float4 x[N];
            #pragma unroll
            for (int i = 0; i < N; ++i) x[i] = ld4(w.q_row(it, from + i * step) + 4 * lane);
            #pragma unroll
            for (int i = 0; i < N; ++i) {
                const int row = from + i * step;
                store_planes(at + row * 128, at + kWdStage + row * 128, row, lane, kWdQPlane, x[i], plain(top4(x[i], 0.f)));
            }
        } else {
            // the rows behind the last are zeros
            #pragma unroll 2
            for (int i = 0; i < N; ++i) {
                const int row = from + i * step;
                if (w.live(it, row)) {
                    const float4 x = ld4(w.q_row(it, row) + 4 * lane);
                    store_planes(at + row * 128, at + kWdStage + row * 128, row, lane, kWdQPlane, x, plain(top4(x, 0.f)));
                } else {
                    store_none(at + row * 128, at + kWdStage + row * 128, row, kWdQPlane);
                }
            }
        }
        arrive(&sh.bar_q);
    };

    if (warp < 4) {
        // ---------------- softmax ----------------
        reg_alloc<152>();
        const int row = threadIdx.x;
        const uint32_t lanes = (uint32_t)(32 * warp) << 16, p_tm = tmem + lanes + kWdP, o_tm = tmem + lanes + kWdO,
                       t_tm = tmem + lanes + kWdT;
        const bool live = w.live(it, row);
        const int seen = w.seen(it, row);
        float m = -INFINITY, l = 0.f;
        split_q(std::integral_constant<int, 16>{}, kAtRows / 2 + 16 * warp, 1);
        // this row's first plane of Q, from the staging place
        bool ok = at_wait_warp(&sh.bar_q, 0, ab, w);
        if (ok) {
            #pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t a[32];
                #pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const uint4 x = *reinterpret_cast<const uint4*>(sm + kWdStage + h * kAtHalf + row * 128 +
                                                                    ((c ^ (row & 7)) << 4));
                    a[4 * c] = x.x;
                    a[4 * c + 1] = x.y;
                    a[4 * c + 2] = x.z;
                    a[4 * c + 3] = x.w;
                }
                tmem_st32(tmem + lanes + kWdQ1 + 32 * h, a);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.bar_q1);
        }
        // this row's outputs go into their total (`total`: there is one), which
        // is then scaled by f
        auto fold = [&](bool total, float f) {
            const bool scale = __any_sync(0xffffffffu, f != 1.f);
            if (!total && !scale) {
                #pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t a[32];
                    tmem_ld32(o_tm + 32 * c, a);
                    tmem_ld_wait();
                    tmem_st32(t_tm + 32 * c, a);
                }
                return;
            }
            #pragma unroll 1
            for (int c = 0; c < 4; ++c) {
                uint32_t a[32], t[32];
                tmem_ld32(o_tm + 32 * c, a);
                if (total) tmem_ld32(t_tm + 32 * c, t);
                tmem_ld_wait();
                if (total) {
                    #pragma unroll
                    for (int e = 0; e < 32; ++e)
                        a[e] = __float_as_uint(__fadd_rn(__uint_as_float(a[e]), __uint_as_float(t[e])));
                }
                if (scale) {
                    #pragma unroll
                    for (int e = 0; e < 32; ++e) a[e] = __float_as_uint(__fmul_rn(__uint_as_float(a[e]), f));
                }
                tmem_st32(t_tm + 32 * c, a);
            }
        };
        auto scale = [&](uint32_t at, float f) {
            #pragma unroll 1
            for (int c = 0; c < 4; ++c) {
                uint32_t a[32];
                tmem_ld32(at + 32 * c, a);
                tmem_ld_wait();
                #pragma unroll
                for (int e = 0; e < 32; ++e) a[e] = __float_as_uint(__fmul_rn(__uint_as_float(a[e]), f));
                tmem_st32(at + 32 * c, a);
            }
        };
        for (int j = 0; j < n && ok; ++j) {
            const uint32_t s_tm = tmem + lanes;
            if (!(ok = at_wait_warp(&sh.bar_s[j & 1], (j >> 1) & 1, ab, w))) break;
            tc_fence_after();
            float s[64];
            {
                uint32_t a[32], b[32];
                tmem_ld32(s_tm, a);
                tmem_ld32(s_tm + 32, b);
                tmem_ld_wait();
                #pragma unroll
                for (int i = 0; i < 32; ++i) {
                    s[i] = __uint_as_float(a[i]);
                    s[32 + i] = __uint_as_float(b[i]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.bar_sf);
            const int lim = seen - j * kWdKeys;
            if (__any_sync(0xffffffffu, lim < kWdKeys)) {
                #pragma unroll
                for (int c = 0; c < 64; ++c) s[c] = c < lim ? s[c] : -INFINITY;
            }
            float mx = max3(s[0], s[1], s[2]);
            #pragma unroll
            for (int c = 3; c < 63; c += 2) mx = max3(mx, s[c], s[c + 1]);
            mx = max3(mx, s[63], s[63]);
            // (a row that is none may hold anything: it never asks for more)
            const bool fine = (mx - m) * kAtScale2 <= kAtLag || mx == -INFINITY || !live;
            const float m1 = fine ? m : max3(m, mx, mx), f = fine ? 1.f : ex2((m - m1) * kAtScale2);
            m = m1;
            l *= f;
            const float mc = weight_offset(m);
            float sum0 = 0.f, sum1 = 0.f;
            uint32_t u[3][32];
            #pragma unroll
            for (int i = 0; i < 32; ++i) {
                float x0, x1;
                fma2v(x0, x1, s[2 * i], s[2 * i + 1], kAtScale2, kAtScale2, mc, mc);
                x0 = ex2(x0);
                x1 = ex2(x1);
                add2(sum0, sum1, x0, x1);
                split2(x0, x1, u[0][i], u[1][i], u[2][i]);
            }
            l += sum0 + sum1;
            // the products before are complete when the values' place is free:
            // then the weights' place is, too, and the outputs may be touched
            if (j > 0) {
                if (!(ok = at_wait_warp(&sh.bar_vf, (j - 1) & 1, ab, w))) break;
                tc_fence_after();
            }
            #pragma unroll
            for (int q = 0; q < 3; ++q) tmem_st32(p_tm + 32 * q, u[q]);
            if (j > 0) {
                if (j % kWdFold == 0) {
                    fold(j > kWdFold, f);
                } else if (__any_sync(0xffffffffu, !fine)) {
                    scale(o_tm, f);
                    if (j > kWdFold) scale(t_tm, f);
                }
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.bar_p);
        }
        sh.f[row] = w.scale(l);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.bar_f);
        if (ok && at_wait_warp(&sh.bar_o, 0, ab, w)) {
            if (live) w.finish(it, row, m, l);
        }
    } else if (warp < 20) {
        // ---------------- operands ----------------
        reg_dealloc<72>();
        const int cw = (warp - 4) & 7, every = w.seen(it, 0);
        const bool is_v = warp >= 12;
        const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
        float4 r[8];                    // this warp's rows cw, cw + 8, .. of a tile
        typename W::Rows rows(w, it, is_v);
        auto load = [&](int j) {
            const int key = j * kWdKeys + cw;
            rows.tile(key, keys);
            if ((j + 1) * kWdKeys <= keys) {
                #pragma unroll
                for (int i = 0; i < 8; ++i) r[i] = ld4(rows.row(i) + 4 * lane);
            } else {
                #pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const T* at = rows.row(i) + 4 * lane;
                    r[i] = key + 8 * i < keys ? ld4(at) : none;
                }
            }
        };
        load(0);
        split_q(std::integral_constant<int, 4>{}, warp - 4, 16);
        #pragma unroll 1
        for (int j = 0; j < n; ++j) {
            // the place is free: values when the products before are done, keys
            // when the scores two tiles before are (the second place: when the
            // queries' first plane has left it)
            if (is_v) {
                if (j > 0 && !at_wait_warp(&sh.bar_vf, (j - 1) & 1, ab, w)) break;
            } else if (j > 0) {
                if (!at_wait_warp(j > 1 ? &sh.bar_s[j & 1] : &sh.bar_q1, j > 1 ? ((j >> 1) - 1) & 1 : 0, ab, w)) break;
            }
            uint8_t* const tile = sm + (is_v ? kWdV : kWdK + (j & 1) * 3 * kWdPlane) + half * kWdHalf;
            float top = 0.f;
            #pragma unroll
            for (int i = 0; i < 8; ++i) top = top4(r[i], top);
            const int rows = keys - j * kWdKeys - cw;           // this warp's are those at 8 i < rows
            const bool ordinary = __all_sync(0xffffffffu, plain(top));
            if (ordinary && rows > 56) {
                #pragma unroll
                for (int i = 0; i < 8; ++i)
                    store_planes(tile + kWdPlane + (cw + 8 * i) * 128, tile + (cw + 8 * i) * 128, cw, lane, kWdPlane, r[i], true);
            } else if (ordinary) {
                #pragma unroll
                for (int i = 0; i < 8; ++i) {
                    uint8_t *const first = tile + (cw + 8 * i) * 128, *const at = first + kWdPlane;
                    if (8 * i < rows) store_planes(at, first, cw, lane, kWdPlane, r[i], true);
                    else store_none(at, first, cw, kWdPlane);
                }
            } else {
                bool odd = false;
                #pragma unroll 1
                for (int i = 0; i < 8; ++i) {
                    uint8_t* const first = tile + (cw + 8 * i) * 128;
                    const bool hidden = is_v && j * kWdKeys + cw + 8 * i >= every;
                    odd = store_odd(first + kWdPlane, first, cw, lane, kWdPlane, pick(r, i), hidden) || odd;
                }
                if (odd) sh.odd = 1;
            }
            arrive(is_v ? &sh.bar_v : &sh.bar_k[j & 1]);
            if (j + 1 < n) load(j + 1);
        }
        // the outputs: sixteen warps, 32 rows x 32 columns each (the query
        // planes' place is free)
        if (at_wait_warp(&sh.bar_f, 0, ab, w) && at_wait_warp(&sh.bar_o, 0, ab, w)) {
            tc_fence_after();
            const int first = 32 * (warp & 3), col = 32 * ((warp - 4) >> 2);
            const uint32_t at = tmem + ((uint32_t)first << 16) + col;
            WideOut to = w.out(it, first);
            to.base += col;
            if (to.n > 0) {
                store_cols(at + kWdO, at + kWdT, n > kWdFold, sh.f[first + lane], sm + (warp - 4) * kAtStage, to);
                if (*(volatile int*)&sh.odd != 0) {
                    const typename W::Item o = sh.item;         // (again, so that it takes no registers till then)
                    add_odd<1>(w.seen(o, 0), w.keys(o), min(32, to.n), [&](int key) { return w.value(o, key) + col + lane; },
                               [&](int r) { return w.seen(o, first + r); },
                               [&](int r) { return to.base + (size_t)r * to.stride + lane; });
                }
            }
        }
    } else {
        reg_dealloc<40>();
        if (warp == 20 && elect_one()) {
            // ---------------- products ----------------
            const uint32_t q0 = umma_desc_lo(smem_u32(sm), 16), k0 = umma_desc_lo(smem_u32(sm + kWdK), 16),
                           v0 = umma_desc_lo(smem_u32(sm + kWdV), kWdHalf);
            // the six pairs of planes, a hex digit each, the small products
            // first; loops, since unrolled their 72 descriptors leave the registers
            constexpr uint32_t kFirst = 0x001102u, kSecond = 0x010120u;
            auto scores = [&](int j) {
                const uint32_t kj = k0 + (j & 1) * (3 * kWdPlane >> 4);
                #pragma unroll 1
                for (int y = 0; y < 6; ++y) {
                    const uint32_t a = kFirst >> (4 * y) & 15u, k = kj + (kSecond >> (4 * y) & 15u) * (kWdPlane >> 4);
                    if (a == 0) {
                        #pragma unroll
                        for (int x = 0; x < 8; ++x)
                            umma_f16_ts(tmem, tmem + kWdQ1 + 8 * x, k + (((x >> 2) * kWdHalf + (x & 3) * 32) >> 4),
                                        umma_idesc_bf16(128, 64, false), x > 0 || y > 0);
                    } else {
                        const uint32_t q = q0 + (a - 1) * (kWdQPlane >> 4);
                        #pragma unroll
                        for (int x = 0; x < 8; ++x)
                            umma_f16_ss(tmem, q + (((x >> 2) * kAtHalf + (x & 3) * 32) >> 4),
                                        k + (((x >> 2) * kWdHalf + (x & 3) * 32) >> 4), umma_idesc_bf16(128, 64, false),
                                        x > 0 || y > 0);
                    }
                }
                umma_commit(&sh.bar_s[j & 1]);
            };
            auto outputs = [&](int j) {
                const uint32_t d = tmem + kWdO;
                #pragma unroll 1
                for (int y = 0; y < 6; ++y) {
                    const uint32_t p = tmem + kWdP + 32 * (kFirst >> (4 * y) & 15u),
                                   v = v0 + (kSecond >> (4 * y) & 15u) * (kWdPlane >> 4);
                    #pragma unroll
                    for (int x = 0; x < 4; ++x)
                        umma_f16_ts(d, p + 8 * x, v + (x * 2048 >> 4), umma_idesc_bf16(128, 128, true),
                                    j % kWdFold != 0 || x > 0 || y > 0);
                }
                umma_commit(&sh.bar_vf);
            };
            bool ok = at_wait_start(&sh.bar_q, 0, ab, w) && at_wait(&sh.bar_q1, 0, ab, w) &&
                      at_wait(&sh.bar_k[0], 0, ab, w);
            if (ok) {
                tc_fence_after();
                scores(0);
            }
            #pragma unroll 1
            for (int j = 0; j < n && ok; ++j) {
                if (j + 1 < n) {
                    if (!(ok = at_wait(&sh.bar_k[(j + 1) & 1], ((j + 1) >> 1) & 1, ab, w) &&
                               at_wait(&sh.bar_sf, j & 1, ab, w)))
                        break;
                    tc_fence_after();
                    scores(j + 1);
                }
                if (!(ok = at_wait(&sh.bar_v, j & 1, ab, w) && at_wait(&sh.bar_p, j & 1, ab, w))) break;
                tc_fence_after();
                outputs(j);
            }
            umma_commit(&sh.bar_o);
            at_drain(&sh.bar_o, 0);
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && sh.abort_flag != 0) w.gave_up();
    if (warp == 20) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace sllm
