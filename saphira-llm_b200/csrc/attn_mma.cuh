// attn_mma.cuh -- what the tensor-core attention kernels share: barriers'
// names, the softmax of one 128-key tile of scores held in tensor memory, and
// the way of values that are no numbers around the products.
#pragma once

#include "serve.cuh"
#include "umma.cuh"

namespace sllm {

constexpr int kAtRows = 128;                    // query rows of a tile: the TMEM lanes
constexpr int kAtKeys = 128;                    // keys of a tile
constexpr int kAtHalf = 128 * 128;              // bytes of 128 rows x 64 f16 in the 128-byte swizzle
constexpr int kAtTile = 2 * kAtHalf;            // ... x 128 f16
constexpr int kAtStages = 4;                    // key and value tiles in flight
constexpr int kAtThreads = 512;
constexpr int kAtStageRow = 128 + 16;           // an output warp's staging: 32 rows of 128 bytes, 16 apart
constexpr int kAtStage = 32 * kAtStageRow;
// two query tiles, the ring, the staging of four warps, barriers and sums
constexpr int kAtSmem = (2 + kAtStages) * kAtTile + 4 * kAtStage + 3 * 1024;
// softmax in base 2: exp(s / sqrt(128)) = 2^(s c)
constexpr float kAtScale2 = 0.08838834764831845f * 1.4426950408889634f;
// the running maximum a row's weights stand against may lag behind by this
// many doublings before its sums are rescaled: most tiles need no pass over
// the outputs
constexpr float kAtLag = 8.0f;
// f16 weights stand against 2^-7 of that maximum: up to 2^15 with the lag,
// within f16's 65504, and a weight keeps its 11 bits down to 2^-21 of the
// largest, some bits down to 2^-31. (Against the maximum itself a weight 2^-26
// of the largest, as many keys beside a sink have it, came out as 0.)
constexpr float kAtShift = 7.0f, kAtBelow = kAtShift / kAtScale2;

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

// why a bounded wait gave up (0: none did), in each file with such a kernel
static __device__ int g_attn_error;

// The bounded waits of umma.cuh, in line: a kernel that splits its registers
// between its warps cannot call functions. Their limit is the launch's: a test
// sets one that runs out. For it to do so, one wait of each item (at_wait_start)
// takes the length of a try's sleep from the launch, too; in all of them that
// cost 2% of many short prompts.
// (`w`: the launch, asked where a wait goes on.)
template <class W>
__device__ __forceinline__ bool at_wait_on(uint64_t* bar, uint32_t parity, volatile int* abort_flag, const W& w, uint32_t nap) {
    const uint64_t t0 = gtimer();
    #pragma unroll 1
    while (!mbar_try_wait_for(bar, parity, nap)) {
        if (*abort_flag) return false;
        if (gtimer() - t0 > w.wait_limit().ns) {
            *abort_flag = 1;
            atomicExch(&g_attn_error, GM_TIMEOUT);
            return false;
        }
    }
    return true;
}
template <class W>
__device__ __forceinline__ bool at_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, const W& w) {
    return mbar_try_wait(bar, parity) || at_wait_on(bar, parity, abort_flag, w, 65536u);
}
template <class W>
__device__ __forceinline__ bool at_wait_start(uint64_t* bar, uint32_t parity, volatile int* abort_flag, const W& w) {
    return at_wait_on(bar, parity, abort_flag, w, w.wait_limit().nap);
}
template <class W>
__device__ __forceinline__ bool at_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag, const W& w) {
    return __all_sync(0xffffffffu, at_wait(bar, parity, abort_flag, w));
}
// ... with something to try meanwhile
template <class W, class F>
__device__ __forceinline__ bool at_wait_while(uint64_t* bar, uint32_t parity, volatile int* abort_flag, const W& w, F f) {
    const uint64_t t0 = gtimer();
    #pragma unroll 1
    while (!mbar_test(bar, parity)) {
        f();
        if (*abort_flag) return false;
        if (gtimer() - t0 > w.wait_limit().ns) {
            *abort_flag = 1;
            atomicExch(&g_attn_error, GM_TIMEOUT);
            return false;
        }
    }
    return true;
}
// what must complete (copies and products in flight), whatever the limit
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
// ... and the two with zeros in such places
__device__ __forceinline__ uint32_t clean_half2(uint32_t u) {
    if ((u & 0x7c00u) == 0x7c00u) u &= 0xffff0000u;
    if ((u & 0x7c000000u) == 0x7c000000u) u &= 0xffffu;
    return u;
}

// What counts as no number: NaN, infinities, and what bf16 would round to one.
__device__ __forceinline__ bool is_odd(float x) { return !(fabsf(x) < 0x1.ffp127f); }

// A value that is no number would reach every row of a tile through its zero
// weights. So the products meet zeros in the places of those that not every row
// sees, and the rows that do see one get it here, when this warp has stored
// them: a weight is positive, so the sum becomes the value itself. Keys `key`
// .. end - 1 (few: those that a causal mask takes from some rows of a tile),
// rows 0 .. rows - 1, E dimensions a lane: v(key), out(row): the lane's first.
template <int E, class V, class S, class O>
__device__ __forceinline__ void add_odd(int key, int end, int rows, V v, S seen, O out) {
    __syncwarp();
    #pragma unroll 1
    for (; key < end; ++key) {
        const auto* const at = v(key);
        float x[E];
        bool any = false;
        #pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = to_f32(at[e]);
            any = any || is_odd(x[e]);
        }
        if (!any) continue;
        #pragma unroll 1
        for (int r = 0; r < rows; ++r) {
            if (seen(r) <= key) continue;
            auto* const to = out(r);
            #pragma unroll
            for (int e = 0; e < E; ++e)
                if (is_odd(x[e])) {
                    const float y = to_f32(to[e]) + (x[e] != x[e] ? x[e] : copysignf(INFINITY, x[e]));
                    from_f32_to(to + e, y);
                }
        }
    }
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

// One warp's 32 rows of outputs, scaled by each lane's f, to global memory:
// 128 bytes of every row at a time through the warp's staging, so that a store
// writes whole lines (row by row, 32 partial sectors a store, a tile of f32
// rows took 2 us). Row r of the warp starts at base + r * stride; the first n
// are to be written.
__device__ __forceinline__ void pack_out(const uint32_t (&r)[32], float f, uint8_t* at, const __half*) {
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint4 u;
        uint32_t* w = &u.x;
        #pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = pack_half2(__uint_as_float(r[8 * i + 2 * e]) * f, __uint_as_float(r[8 * i + 2 * e + 1]) * f);
        *reinterpret_cast<uint4*>(at + 16 * i) = u;
    }
}
__device__ __forceinline__ void pack_out(const uint32_t (&r)[32], float f, uint8_t* at, const float*) {
    #pragma unroll
    for (int i = 0; i < 8; ++i)
        *reinterpret_cast<float4*>(at + 16 * i) =
            make_float4(__uint_as_float(r[4 * i]) * f, __uint_as_float(r[4 * i + 1]) * f,
                        __uint_as_float(r[4 * i + 2]) * f, __uint_as_float(r[4 * i + 3]) * f);
}
template <class O>
__device__ __forceinline__ void store_rows(uint32_t o_tmem, float f, uint8_t* stage, O* base, size_t stride, int n) {
    constexpr int kCols = 128 / (int)sizeof(O);         // of 128 bytes
    const int lane = threadIdx.x & 31, sub = lane >> 3;
    uint8_t* to = reinterpret_cast<uint8_t*>(base + (size_t)sub * stride) + 16 * (lane & 7);
    const size_t four = 4 * stride * sizeof(O);
    uint32_t r[32];
    tmem_ld32(o_tmem, r);
    #pragma unroll 1
    for (int c = 0; c < kServeDim; c += kCols) {
        #pragma unroll
        for (int x = 0; x < kCols; x += 32) {
            tmem_ld_wait();
            pack_out(r, f, stage + lane * kAtStageRow + x * (int)sizeof(O), static_cast<const O*>(nullptr));
            // the next columns come while these leave
            if (c + x + 32 < kServeDim) tmem_ld32(o_tmem + c + x + 32, r);
        }
        __syncwarp();
        #pragma unroll 4
        for (int i = 0; i < 8; ++i) {                   // four rows a store
            const uint4 u = *reinterpret_cast<const uint4*>(stage + (4 * i + sub) * kAtStageRow + 16 * (lane & 7));
            if (4 * i + sub < n) *reinterpret_cast<uint4*>(to + i * four) = u;
        }
        to += 128;
        __syncwarp();
    }
    tmem_ld_wait();
}

// ---------------------------------------------------------------------------
// The core of the f16 kernels. One CTA per SM walks items: up to two tiles of
// 128 query rows that share every key tile. Scores, weights and outputs
// stay in tensor memory (512 columns: S0 S1 O0 O1, 128 each; a tile's f16
// weights overwrite the first 64 columns of its scores).
//
//   warps 0-3, 4-7   softmax of tile 0, 1: one thread per row. S from tensor
//                    memory, mask, weights back. The weights stand against the
//                    running maximum of the tiles before; the tile's own
//                    maximum is found meanwhile and only checked: where it is
//                    more than kAtLag doublings higher (rare after the first
//                    tiles) the warp rescales its rows of O and starts over.
//   warps 8-11       outputs to global memory, under the next item's products.
//   warp 12, 1 lane  tcgen05.mma: S_t = Q_t K^T (both from shared memory) and
//                    O_t += P_t V (P from tensor memory, V MN-major as it
//                    lies), the first 64 keys as soon as their weights are
//                    there. The order P0 V, S0', P1 V, S1' lets one tile's
//                    softmax run under the other tile's products.
//   warp 13          TMA: Q per item, K and V tiles through a ring of four.
//   warp 14          the items, one ahead.
//
// What bounds it: per key tile and row tile 1024 clocks of products, and the
// chain S -> softmax -> P V -> S', whose softmax is 16384 exponentials at 16
// a clock, shared by the two tiles. Measured: one prompt of 16384 tokens, 16
// heads, 845 us (1302 TFLOP/s, 78% of a library GEMM's best); 4096 tokens, 36
// heads, 134 us (1153); 1024 tokens, 64 heads, 30 us (571: an item's start and
// end are 2-3 us, and here most items have four key tiles); 17 tokens 8 us.
// Part of the exponentials as polynomials on the ordinary pipes: slower (889 to
// 919 us against 871 where it was tried).
//
// Masks: a row sees the item's first so many keys, so only an item's last key
// tiles are masked. A value row behind the item's keys is zeroed in shared
// memory before it meets its zero weight. A value among the keys that is no
// number would leak the same way into rows of the tile that do not see it: the
// softmax warps put zeros in the places of such values in the masked tiles, and
// warps 8-11 add them to the rows that see them (add_odd).
//
// `W` says what the items are: a Finder (number(w, r): the number of the CTA's
// r-th item; item(w, x, item): false: there is no item x, but later ones may
// be), tiles(item, t) (0: no such row tile), keys(item),
// seen(item, t, row) (not above keys, and least for row 0), live(item, t, row)
// (a row to be written), a Loader, store(...), odd(...) (add_odd for a warp's
// rows), check() (one idle warp of each CTA), wait_limit() and gave_up() (a wait ran
// out).
//
// Registers: 512 threads x 128 at launch; 2 x 184 (softmax) + 80 (outputs) +
// 64 (the issuing warps) = 512 = 4 x 128 after the split.
// ---------------------------------------------------------------------------
// a fixed share of the item numbers: every other round backwards, so that the
// CTA that got the longest item of one round gets the shortest of the next
__device__ __forceinline__ long long dealt_number(int r) {
    return (long long)r * gridDim.x + ((r & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

static inline int take_attn_error() {
    int v = 0;
    const int zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_attn_error, sizeof v) != cudaSuccess ||
        cudaMemcpyToSymbol(g_attn_error, &zero, sizeof zero) != cudaSuccess)
        return -1;
    return v;
}

template <class W>
__device__ __forceinline__ void attn_core(const W w) {
    using Item = typename W::Item;
    extern __shared__ __align__(1024) uint8_t sm[];
    // [2]: per row tile. q, qf: Q there / free; s: scores there; h, p: the
    // first half of the weights there, all; l: sums there; o: outputs
    // complete; of: outputs read
    struct Shared {
        uint64_t bar_full[kAtStages], bar_free[kAtStages], bar_q[2], bar_qf[2], bar_s[2], bar_h[2], bar_p[2], bar_l[2],
            bar_o[2], bar_of[2], bar_item, bar_itemf, bar_done;
        float sum[2][kAtRows], top[2][kAtRows];
        Item item;
        int odd[2][4];
        uint32_t tmem;
        int abort_flag;
    };
    uint8_t* const stages = sm + (2 + kAtStages) * kAtTile;
    static_assert(sizeof(Shared) <= 3 * 1024, "the part behind the tiles");
    Shared& sh = *reinterpret_cast<Shared*>(stages + 4 * kAtStage);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if ((smem_u32(sm) & 1023u) != 0) {           // the swizzled layouts need it; the compiler was told to
        if (threadIdx.x == 0) atomicExch(&g_attn_error, 2);
        return;
    }
    if (warp == 15) w.check();
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.bar_q[i], 1);
            mbar_init(&sh.bar_qf[i], 1);
            mbar_init(&sh.bar_s[i], 1);
            mbar_init(&sh.bar_h[i], 4);
            mbar_init(&sh.bar_p[i], 4);
            mbar_init(&sh.bar_l[i], 4);
            mbar_init(&sh.bar_o[i], 1);
            mbar_init(&sh.bar_of[i], 4);
        }
        for (int i = 0; i < kAtStages; ++i) {
            mbar_init(&sh.bar_full[i], 1);
            mbar_init(&sh.bar_free[i], 1);
        }
        mbar_init(&sh.bar_item, 1);
        mbar_init(&sh.bar_itemf, 14);           // 8 softmax, 4 output warps, the products and the loads
        mbar_init(&sh.bar_done, 1);
        sh.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    volatile int* const ab = &sh.abort_flag;

    auto next_warp = [&](int i, Item* it) {       // false: no more, or a wait gave up
        if (!at_wait_warp(&sh.bar_item, i & 1, ab, w)) return false;
        *it = sh.item;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.bar_itemf);
        return !it->last();
    };
    auto next_lane = [&](int i, Item* it) {
        if (!at_wait(&sh.bar_item, i & 1, ab, w)) return false;
        *it = sh.item;
        mbar_arrive(&sh.bar_itemf);
        return !it->last();
    };

    if (warp < 8) {
        // ---------------- softmax ----------------
        reg_alloc<184>();
        const int t = warp >> 2, row = 32 * (warp & 3) + lane;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t s_tm = tmem + lanes + 128 * t, o_tm = s_tm + 256;
        int steps = 0, uses = 0, ring = 0;              // score tiles, items with this row tile, ring tiles so far
        bool ok = true;
        Item it;
        for (int i = 0; ok && next_warp(i, &it); ++i) {
            const int n0 = w.tiles(it, 0), n1 = w.tiles(it, 1), n = t == 0 ? n0 : n1;
            const int keys = w.keys(it), seen = w.seen(it, t, row);
            // all rows of this row tile see the keys below `every`
            const int every = n > 0 ? w.seen(it, t, 0) : 0;
            // a warp without rows only keeps the others' pace; a row that is none
            // (what lies in its place may be anything) never asks for a second pass
            const bool live = n > 0 && w.live(it, t, row), idle = !__any_sync(0xffffffffu, live);
            float m = -INFINITY, l = 0.f;
            bool odd = false;
            #pragma unroll 1
            for (int j = 0; j < n; ++j, ++steps) {
                const bool edge = (j + 1) * kAtKeys > every;
                if (edge) {
                    // this row of the masked tile's values: zeros behind the
                    // sequence, and where no number stands inside it
                    const int x = ring + 2 * j + 1, slot = x % kAtStages;
                    if (!(ok = at_wait_warp(&sh.bar_full[slot], (x / kAtStages) & 1, ab, w))) break;
                    uint8_t* v = sm + (2 + slot) * kAtTile + row * 128;
                    const int key = j * kAtKeys + row;
                    if (key >= keys) {
                        #pragma unroll 4
                        for (int c = 0; c < 16; ++c)
                            *reinterpret_cast<uint4*>(v + (c >> 3) * kAtHalf + 16 * (c & 7)) = make_uint4(0, 0, 0, 0);
                    } else if (key >= every) {
                        // (a short loop: its code runs once an item)
                        __half2 top = __half2half2(__ushort_as_half(0));
                        #pragma unroll 4
                        for (int c = 0; c < 16; ++c) {
                            const uint4 u = *reinterpret_cast<const uint4*>(v + (c >> 3) * kAtHalf + 16 * ((c ^ row) & 7));
                            const __half2* x = reinterpret_cast<const __half2*>(&u);
                            top = __hmax2_nan(top, __hmax2_nan(__hmax2_nan(__habs2(x[0]), __habs2(x[1])),
                                                               __hmax2_nan(__habs2(x[2]), __habs2(x[3]))));
                        }
                        if (odd_half2(*reinterpret_cast<const uint32_t*>(&top))) {
                            odd = true;
                            #pragma unroll 1
                            for (int c = 0; c < 16; ++c) {
                                uint4* const at = reinterpret_cast<uint4*>(v + (c >> 3) * kAtHalf + 16 * (c & 7));
                                const uint4 u = *at;
                                *at = make_uint4(clean_half2(u.x), clean_half2(u.y), clean_half2(u.z), clean_half2(u.w));
                            }
                        }
                    }
                    fence_proxy_async_smem();
                }
                if (!(ok = at_wait_warp(&sh.bar_s[t], steps & 1, ab, w))) break;
                tc_fence_after();
                if (idle) {
                    if (lane == 0) {
                        mbar_arrive(&sh.bar_h[t]);
                        mbar_arrive(&sh.bar_p[t]);
                    }
                    continue;
                }
                float s[128];
                load_scores(s_tm, s);
                if (edge) {
                    const int lim = seen - j * kAtKeys;
                    #pragma unroll
                    for (int c = 0; c < 128; ++c) s[c] = c < lim ? s[c] : -INFINITY;
                }
                if (j == 0) m = row_max(s) - kAtBelow;
                float sum[4];
                uint32_t u[32];
                #pragma unroll 1
                for (int pass = 0;; ++pass) {
                    sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
                    half_weights(s, weight_offset(m), u, sum);
                    const float mx = row_max(s);
                    // (false for a NaN)
                    const bool fine = (mx - m) * kAtScale2 <= kAtLag + kAtShift || mx == -INFINITY || !live;
                    if (pass == 1 || __all_sync(0xffffffffu, fine)) break;
                    // (all of O's earlier products are complete: they precede this tile's scores)
                    const float m1 = fine ? m : max3(m, mx - kAtBelow, mx - kAtBelow);
                    const float f = fine ? 1.f : ex2((m - m1) * kAtScale2);
                    m = m1;
                    l *= f;
                    if (j > 0) {
                        #pragma unroll 1
                        for (int c = 0; c < 8; ++c) {
                            uint32_t r[16];
                            tmem_ld16(o_tm + 16 * c, r);
                            tmem_ld_wait();
                            #pragma unroll
                            for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * f);
                            tmem_st16(o_tm + 16 * c, r);
                        }
                    }
                }
                auto arrive = [&](uint64_t* bar) {
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar);
                };
                tmem_st32(s_tm, u);
                arrive(&sh.bar_h[t]);
                half_weights(s + 64, weight_offset(m), u, sum);
                tmem_st32(s_tm + 32, u);
                arrive(&sh.bar_p[t]);
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            }
            if (!ok) break;
            ring += 2 * max(n0, n1);
            if (n == 0) continue;
            // the sums of the item before have been read
            if (uses > 0 && !(ok = at_wait_warp(&sh.bar_of[t], (uses - 1) & 1, ab, w))) break;
            ++uses;
            sh.sum[t][row] = l;
            sh.top[t][row] = m;
            odd = __any_sync(0xffffffffu, odd);
            if (lane == 0) sh.odd[t][warp & 3] = odd ? 1 : 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.bar_l[t]);
        }
    } else if (warp < 12) {
        // ---------------- outputs ----------------
        reg_dealloc<80>();
        const int row = 32 * (warp & 3) + lane;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        int uses[2] = {0, 0};
        bool ok = true;
        Item it;
        for (int i = 0; ok && next_warp(i, &it); ++i) {
            bool odd = false;               // (tile 1 meets the zeros that tile 0's warps have put)
            #pragma unroll 1
            for (int t = 0; t < 2; ++t) {
                if (w.tiles(it, t) == 0) break;
                const int par = uses[t] & 1;
                ++uses[t];
                if (!(ok = at_wait_warp(&sh.bar_l[t], par, ab, w) && at_wait_warp(&sh.bar_o[t], par, ab, w))) break;
                tc_fence_after();
                odd = odd || (sh.odd[t][0] | sh.odd[t][1] | sh.odd[t][2] | sh.odd[t][3]) != 0;
                w.store(it, t, row, tmem + lanes + 256 + 128 * t, sh.top[t][row], sh.sum[t][row],
                        stages + (warp & 3) * kAtStage);
                if (odd) w.odd(it, t, 32 * (warp & 3));
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.bar_of[t]);
            }
        }
    } else {
        reg_dealloc<64>();
        if (warp == 12) {
            if (elect_one()) {
                // ---------------- products ----------------
                constexpr uint32_t idesc_s = umma_idesc_f16(128, 128, false), idesc_o = umma_idesc_f16(128, 128, true);
                const uint32_t tiles = smem_u32(sm + 2 * kAtTile), q0 = umma_desc_lo(smem_u32(sm), 16);
                // the ring's next key and value tiles: slot and parity
                int ks = 0, kp = 0, vs = 1, vp = 0;
                auto step = [](int& slot, int& parity, int by) {
                    slot += by;
                    if (slot >= kAtStages) {
                        slot -= kAtStages;
                        parity ^= 1;
                    }
                };
                auto scores = [&](int t) {                       // S_t = Q_t K^T
                    const uint32_t q = q0 + t * (kAtTile >> 4), k = umma_desc_lo(tiles + ks * kAtTile, 16);
                    #pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const uint32_t off = (x >> 2) * (kAtHalf >> 4) + (x & 3) * 2;
                        umma_f16_ss(tmem + 128 * t, q + off, k + off, idesc_s, x > 0);
                    }
                    umma_commit(&sh.bar_s[t]);
                };
                auto outputs = [&](int t, int half, bool add) {  // O_t (+)= P_t V, 64 keys
                    const uint32_t v = umma_desc_lo(tiles + vs * kAtTile, kAtHalf) + half * (8192 >> 4);
                    #pragma unroll
                    for (int x = 0; x < 4; ++x)
                        umma_f16_ts(tmem + 256 + 128 * t, tmem + 128 * t + 32 * half + 8 * x, v + x * (2048 >> 4),
                                    idesc_o, add || x > 0);
                };
                int steps0 = 0, steps1 = 0, uses0 = 0, uses1 = 0;
                bool ok = true;
                // the next item, and whether its first scores have been issued:
                // that is tried while the last products of this one wait for
                // their weights, so that its softmax starts under them
                Item it, nx;
                bool known = false, ahead = false;
                for (int i = 0; ok; ++i) {
                    if (known) it = nx;
                    else if (!next_lane(i, &it)) break;
                    if (it.last()) break;
                    known = false;
                    const int n0 = w.tiles(it, 0), n1 = w.tiles(it, 1), nt = max(n0, n1);
                    if (!ahead) {
                        ok = at_wait_start(&sh.bar_q[0], uses0 & 1, ab, w) && at_wait(&sh.bar_full[ks], kp, ab, w);
                        if (!ok) break;
                        scores(0);
                        if (n0 == 1) umma_commit(&sh.bar_qf[0]);
                    }
                    ahead = false;
                    if (n1 > 0) {
                        if (!(ok = at_wait(&sh.bar_q[1], uses1 & 1, ab, w))) break;
                        scores(1);
                        if (n1 == 1) umma_commit(&sh.bar_qf[1]);
                    }
                    umma_commit(&sh.bar_free[ks]);
                    step(ks, kp, 2);
                    auto look = [&] {
                        if (!known) {
                            if (!mbar_test(&sh.bar_item, (i + 1) & 1)) return;
                            nx = sh.item;
                            mbar_arrive(&sh.bar_itemf);
                            known = true;
                        }
                        if (ahead || nx.last() || !mbar_test(&sh.bar_q[0], (uses0 + 1) & 1) || !mbar_test(&sh.bar_full[ks], kp))
                            return;
                        scores(0);
                        if (w.tiles(nx, 0) == 1) umma_commit(&sh.bar_qf[0]);
                        ahead = true;
                    };
                    #pragma unroll 1
                    for (int j = 0; j < nt && ok; ++j) {
                        const bool more = j + 1 < nt;
                        ok = at_wait(&sh.bar_full[vs], vp, ab, w) && (!more || at_wait(&sh.bar_full[ks], kp, ab, w));
                        #pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const int n = t == 0 ? n0 : n1, uses = t == 0 ? uses0 : uses1;
                            int& steps = t == 0 ? steps0 : steps1;
                            if (!ok || j >= n) continue;
                            // the item before has left O (of) before the first product overwrites it
                            ok = j > 0 || uses == 0 || at_wait(&sh.bar_of[t], (uses - 1) & 1, ab, w);
                            if (t == 1 && !more) ok = ok && at_wait_while(&sh.bar_h[1], steps & 1, ab, w, look);
                            else ok = ok && at_wait(&sh.bar_h[t], steps & 1, ab, w);
                            if (!ok) continue;
                            tc_fence_after();
                            outputs(t, 0, j > 0);
                            if (!(ok = at_wait(&sh.bar_p[t], steps & 1, ab, w))) continue;
                            tc_fence_after();
                            outputs(t, 1, true);
                            ++steps;
                            if (j + 1 < n) {
                                scores(t);
                                if (j + 2 == n) umma_commit(&sh.bar_qf[t]);
                            } else {
                                umma_commit(&sh.bar_o[t]);
                            }
                        }
                        umma_commit(&sh.bar_free[vs]);
                        step(vs, vp, 2);
                        if (more) {
                            umma_commit(&sh.bar_free[ks]);
                            step(ks, kp, 2);
                        }
                    }
                    ++uses0;
                    uses1 += n1 > 0 ? 1 : 0;
                }
                umma_commit(&sh.bar_done);
                at_drain(&sh.bar_done, 0);
            }
            __syncwarp();
        } else if (warp == 13) {
            // ---------------- loads ----------------
            int x = 0, uses[2] = {0, 0};
            bool ok = true;
            Item it;
            for (int i = 0; ok && next_warp(i, &it); ++i) {
                const int n1 = w.tiles(it, 1), nt = max(w.tiles(it, 0), n1);
                typename W::Loader load;
                load.start(w, it, lane);
                #pragma unroll 1
                for (int j = -1; j < 2 * nt; ++j) {
                    // Q0, K0, Q1, V0, K1, V1, ...
                    const int t = j < 0 ? 0 : 1;
                    if (j < 0 || (j == 1 && n1 > 0)) {
                        if (uses[t] > 0 && !(ok = at_wait_warp(&sh.bar_qf[t], (uses[t] - 1) & 1, ab, w))) break;
                        ++uses[t];
                        load.q(w, it, t, sm + t * kAtTile, &sh.bar_q[t], lane);
                    }
                    if (j < 0) continue;
                    const int s = x % kAtStages, use = x / kAtStages;
                    if (use > 0 && !(ok = at_wait_warp(&sh.bar_free[s], (use - 1) & 1, ab, w))) break;
                    load.kv(w, it, j >> 1, (j & 1) != 0, sm + (size_t)(2 + s) * kAtTile, &sh.bar_full[s], lane);
                    ++x;
                }
            }
            // no copy may be in flight when the CTA ends
            for (int t = 0; t < 2; ++t)
                if (uses[t] > 0) at_drain(&sh.bar_q[t], (uses[t] - 1) & 1);
            for (int y = max(0, x - kAtStages); y < x; ++y) at_drain(&sh.bar_full[y % kAtStages], (y / kAtStages) & 1);
            __syncwarp();
        } else if (warp == 14) {
            // ---------------- items ----------------
            typename W::Finder find;
            find.start(w);
            #pragma unroll 1
            for (int r = 0, i = 0;; ++r) {
                // every warp has taken the item before
                if (i > 0 && !at_wait_warp(&sh.bar_itemf, (i - 1) & 1, ab, w)) break;
                Item it;
                if (!find.item(w, find.number(w, r), &it)) continue;    // no item has this number
                if (lane == 0) {
                    sh.item = it;
                    mbar_arrive(&sh.bar_item);
                }
                if (it.last()) break;
                ++i;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && sh.abort_flag != 0) w.gave_up();
    if (warp == 12) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace sllm
