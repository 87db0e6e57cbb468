// attn_prompt.cu -- causal attention over packed whole prompts, grouped heads.
//
// Sequence s holds tokens cu[s] .. cu[s + 1] - 1 of the packed arrays; token i
// of a sequence sees its tokens 0 .. i.

//
// f16: attn_prompt_mma_kernel, on the tensor cores. f32: the 32-bit kernel
// of attn_simt.cuh.

#include "../../include/sllm_cuda_testing.h"
#include "attn_mma.cuh"
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

// ---------------------------------------------------------------------------
// The f16 kernel. One CTA per SM walks items of 256 query rows of one head:
// two tiles of 128 rows that share every key tile. Scores, weights and outputs
// stay in tensor memory (512 columns: S0 S1 O0 O1, 128 each; a tile's f16
// weights overwrite the first 64 columns of its scores).
//
//   warps 0-3, 4-7   softmax of tile 0, 1: one thread per row. S from tensor
//                    memory, mask, weights back. The weights stand against the
//                    running maximum of the tiles before; the tile's own
//                    maximum is found meanwhile and only checked: where it is
//                    more than kAtLag doublings higher (rare after the first
//                    tiles) the warp rescales its rows of O and starts over.
//   warps 8-11       O / l to global memory, under the next item's products.
//   warp 12, 1 lane  tcgen05.mma: S_t = Q_t K^T (both from shared memory) and
//                    O_t += P_t V (P from tensor memory, V MN-major as it
//                    lies), the first 64 keys as soon as their weights are
//                    there. The order P0 V, S0', P1 V, S1' lets one tile's
//                    softmax run under the other tile's products.
//   warp 13, 1 lane  TMA: Q per item, K and V tiles through a ring of five.
//   warp 14          the items, longest first, two ahead.
//
// What bounds it: per key tile and row tile 1024 clocks of products, and the
// chain S -> softmax -> P V -> S', whose softmax is 16384 exponentials at 16
// a clock, shared by the two tiles.
//
// Causal: only the last key tile of a row tile is masked. A value row past the
// end of the sequence is zeroed in shared memory before it meets its zero
// weight. A value inside the sequence that is no number would leak the same
// way into rows of the tile that do not see it: the softmax warps look for
// such values in that last key tile, and if there are any warps 8-11 recompute
// the tile's rows one by one.
//
// Registers: 512 threads x 128 at launch; 2 x 192 (softmax) + 64 (outputs) +
// 64 (the issuing warps) = 512 = 4 x 128 after the split.
// ---------------------------------------------------------------------------
constexpr int kPmRows = 2 * kAtRows;
constexpr int kPmStages = 5;
constexpr int kPmThreads = 512;
constexpr int kPmSmem = (2 + kPmStages) * kAtTile + 1024;

__device__ int g_prompt_error;      // why a bounded wait gave up (0: none did)

// tile x of the call's tiles of R rows in descending order of their position
// in their sequence (the later, the more keys they see): the longest work
// first. F(t) = tiles at positions >= t; a binary search for the position,
// then the sequence among those that long. One warp.
template <int R>
__device__ __forceinline__ bool find_long_first(const PromptParams& p, int x, int* start, int* len, int* tile) {
    const int lane = threadIdx.x & 31;
    auto seq = [&](int s, int* a) {
        *a = min(max(p.cu[s], 0), p.n_tokens);
        return min(max(p.cu[s + 1], *a), p.n_tokens) - *a;
    };
    auto at_least = [&](int t) {
        int f = 0, a;
        for (int s = lane; s < p.n_seq; s += 32) f += max((seq(s, &a) + R - 1) / R - t, 0);
        return __reduce_add_sync(0xffffffffu, f);
    };
    int lo = 0, hi = (p.n_tokens + R - 1) / R;          // F(lo) > x >= F(hi), if x is a tile at all
    if (at_least(0) <= x) return false;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (at_least(mid) > x) lo = mid;
        else hi = mid;
    }
    int r = x - at_least(lo + 1);                       // the r-th sequence with a tile at lo
    for (int s0 = 0; s0 < p.n_seq; s0 += 32) {
        int a = 0, n = 0;
        if (s0 + lane < p.n_seq) n = seq(s0 + lane, &a);
        const unsigned has = __ballot_sync(0xffffffffu, (n + R - 1) / R > lo);
        const int c = __popc(has);
        if (r < c) {
            const int l = __fns(has, 0, r + 1);
            *start = __shfl_sync(0xffffffffu, a, l);
            *len = __shfl_sync(0xffffffffu, n, l);
            *tile = lo;
            return true;
        }
        r -= c;
    }
    return false;
}

// rows [first, first + 128) of a sequence, one warp per row at a time, in
// 32-bit arithmetic: the way out for values that are no numbers
template <class O>
__device__ __forceinline__ void slow_rows(const PromptParams& p, int h, int start, int len, int first, int warp) {
    const int lane = threadIdx.x & 31, kvh = h / p.group;
    const __half* K = static_cast<const __half*>(p.k) + (size_t)kvh * kServeDim + 4 * lane;
    const __half* V = static_cast<const __half*>(p.v) + (size_t)kvh * kServeDim + 4 * lane;
    for (int r = warp; r < kAtRows; r += 4) {
        const int i = first + r;
        if (i >= len) return;
        const float4 q = ld4(static_cast<const __half*>(p.q) + (size_t)(start + i) * p.qs + (size_t)h * kServeDim + 4 * lane);
        float m = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int j = 0; j <= i; ++j) {
            const float4 k = ld4(K + (size_t)(start + j) * p.ks), v = ld4(V + (size_t)(start + j) * p.vs);
            float s = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, q.w * k.w)));
            #pragma unroll
            for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            s *= kServeScale;
            const float mn = fmaxf(m, s), f = mn == -INFINITY ? 1.f : expf(m - mn), e = expf(s - mn);
            m = mn;
            l = fmaf(l, f, e);
            o.x = fmaf(e, v.x, o.x * f);
            o.y = fmaf(e, v.y, o.y * f);
            o.z = fmaf(e, v.z, o.z * f);
            o.w = fmaf(e, v.w, o.w * f);
        }
        const float inv = 1.f / l;
        st4(static_cast<O*>(p.out) + (size_t)(start + i) * p.os + (size_t)h * kServeDim + 4 * lane,
            make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    }
}

struct PromptItem {
    int start, len, tile, head;         // tile < 0: no more items
};

template <class O>
__global__ void __launch_bounds__(kPmThreads, 1)
attn_prompt_mma_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PromptParams p) {
    extern __shared__ uint8_t pm_raw[];
    // [2]: per row tile. q, qf: Q there / free; s: scores there; h, p: the
    // first half of the weights there, all; l: sums there; o: outputs
    // complete; of: outputs read
    __shared__ uint64_t bar_full[kPmStages], bar_free[kPmStages], bar_q[2], bar_qf[2], bar_s[2], bar_h[2], bar_p[2],
        bar_l[2], bar_o[2], bar_of[2], bar_item[2], bar_itemf[2], bar_done;
    __shared__ float s_sum[2][kAtRows];
    __shared__ PromptItem s_item[2];
    __shared__ int s_odd[2][4];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    uint8_t* const sm = pm_raw + ((1024u - (smem_u32(pm_raw) & 1023u)) & 1023u);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar_q[i], 1);
            mbar_init(&bar_qf[i], 1);
            mbar_init(&bar_s[i], 1);
            mbar_init(&bar_h[i], 4);
            mbar_init(&bar_p[i], 4);
            mbar_init(&bar_l[i], 4);
            mbar_init(&bar_o[i], 1);
            mbar_init(&bar_of[i], 4);
            mbar_init(&bar_item[i], 1);
            mbar_init(&bar_itemf[i], 14);       // 8 softmax, 4 output warps, the MMA's and the loads' lanes
        }
        for (int i = 0; i < kPmStages; ++i) {
            mbar_init(&bar_full[i], 1);
            mbar_init(&bar_free[i], 1);
        }
        mbar_init(&bar_done, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    volatile int* const ab = &abort_flag;
    int* const err = &g_prompt_error;

    // the i-th item, and its key tiles: up to each row tile's diagonal, or the
    // sequence's end (none for a second tile without rows)
    struct Shape {
        int start, len, r0, head, nt0, nt1, nt;
    };
    auto shape = [](const PromptItem& it) {
        Shape s;
        s.start = it.start;
        s.len = it.len;
        s.r0 = it.tile * kPmRows;
        s.head = it.head;
        const int last = (it.len - 1) / kAtKeys;
        s.nt0 = min(2 * it.tile, last) + 1;
        s.nt1 = s.r0 + kAtRows < it.len ? min(2 * it.tile + 1, last) + 1 : 0;
        s.nt = max(s.nt0, s.nt1);
        return s;
    };
    auto next_warp = [&](int i, PromptItem* it) {       // false: no more, or a wait gave up
        if (!at_wait_warp(&bar_item[i & 1], (i >> 1) & 1, ab, err)) return false;
        *it = s_item[i & 1];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_itemf[i & 1]);
        return it->tile >= 0;
    };
    auto next_lane = [&](int i, PromptItem* it) {
        if (!at_wait(&bar_item[i & 1], (i >> 1) & 1, ab, err)) return false;
        *it = s_item[i & 1];
        mbar_arrive(&bar_itemf[i & 1]);
        return it->tile >= 0;
    };

    if (warp < 8) {
        // ---------------- softmax ----------------
        reg_alloc<192>();
        const int t = warp >> 2, row = 32 * (warp & 3) + lane;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t s_tm = tmem + lanes + 128 * t, o_tm = s_tm + 256;
        int steps = 0, uses = 0, ring = 0;              // score tiles, items with this row tile, ring tiles so far
        bool ok = true;
        PromptItem it;
        for (int i = 0; ok && next_warp(i, &it); ++i) {
            const Shape w = shape(it);
            const int n = t == 0 ? w.nt0 : w.nt1;
            const int seen = min(w.r0 + kAtRows * t + row + 1, w.len);
            float m = -INFINITY, l = 0.f;
            bool odd = false;
            #pragma unroll 1
            for (int j = 0; j < n; ++j, ++steps) {
                const bool edge = j == n - 1;
                if (edge) {
                    // this row of the masked tile's values: zeros behind the
                    // sequence; no number inside it
                    const int x = ring + 2 * j + 1, slot = x % kPmStages;
                    if (!(ok = at_wait_warp(&bar_full[slot], (x / kPmStages) & 1, ab, err))) break;
                    uint8_t* v = sm + (2 + slot) * kAtTile + row * 128;
                    const bool inside = j * kAtKeys + row < w.len;
                    #pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        uint4* at = reinterpret_cast<uint4*>(v + (c >> 3) * kAtHalf + 16 * ((c ^ row) & 7));
                        if (inside) {
                            const uint4 u = *at;
                            odd = odd || odd_half2(u.x) || odd_half2(u.y) || odd_half2(u.z) || odd_half2(u.w);
                        } else {
                            *at = make_uint4(0, 0, 0, 0);
                        }
                    }
                    fence_proxy_async_smem();
                }
                if (!(ok = at_wait_warp(&bar_s[t], steps & 1, ab, err))) break;
                tc_fence_after();
                float s[128];
                load_scores(s_tm, s);
                if (edge) {
                    const int lim = seen - j * kAtKeys;
                    #pragma unroll
                    for (int c = 0; c < 128; ++c) s[c] = c < lim ? s[c] : -INFINITY;
                }
                if (j == 0) m = row_max(s);
                float sum[4];
                uint32_t u[32];
                #pragma unroll 1
                for (int pass = 0;; ++pass) {
                    sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
                    half_weights(s, weight_offset(m), u, sum);
                    const float mx = row_max(s);
                    const bool fine = (mx - m) * kAtScale2 <= kAtLag;      // (false for a NaN)
                    if (pass == 1 || __all_sync(0xffffffffu, fine)) break;
                    // (all of O's earlier products are complete: they precede this tile's scores)
                    const float m1 = fine ? m : max3(m, mx, mx);
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
                arrive(&bar_h[t]);
                half_weights(s + 64, weight_offset(m), u, sum);
                tmem_st32(s_tm + 32, u);
                arrive(&bar_p[t]);
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            }
            if (!ok) break;
            ring += 2 * w.nt;
            if (n == 0) continue;
            // the sums of the item before have been read
            if (uses > 0 && !(ok = at_wait_warp(&bar_of[t], (uses - 1) & 1, ab, err))) break;
            ++uses;
            s_sum[t][row] = l;
            odd = __any_sync(0xffffffffu, odd);
            if (lane == 0) s_odd[t][warp & 3] = odd ? 1 : 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_l[t]);
        }
    } else if (warp < 12) {
        // ---------------- outputs ----------------
        reg_dealloc<64>();
        const int row = 32 * (warp & 3) + lane;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        int uses[2] = {0, 0};
        bool ok = true;
        PromptItem it;
        for (int i = 0; ok && next_warp(i, &it); ++i) {
            const Shape w = shape(it);
            #pragma unroll 1
            for (int t = 0; t < 2; ++t) {
                if (t == 1 && w.nt1 == 0) break;
                const int par = uses[t] & 1;
                ++uses[t];
                if (!(ok = at_wait_warp(&bar_l[t], par, ab, err) && at_wait_warp(&bar_o[t], par, ab, err))) break;
                tc_fence_after();
                const int x = w.r0 + kAtRows * t + row;
                if ((s_odd[t][0] | s_odd[t][1] | s_odd[t][2] | s_odd[t][3]) != 0)
                    slow_rows<O>(p, w.head, w.start, w.len, w.r0 + kAtRows * t, warp & 3);
                else
                    store_row(tmem + lanes + 256 + 128 * t, 1.f / s_sum[t][row], x < w.len,
                              static_cast<O*>(p.out) + (size_t)(w.start + x) * p.os + (size_t)w.head * kServeDim);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_of[t]);
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
                    if (slot >= kPmStages) {
                        slot -= kPmStages;
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
                    umma_commit(&bar_s[t]);
                };
                auto outputs = [&](int t, int half, bool add) {  // O_t (+)= P_t V, 64 keys
                    const uint32_t v = umma_desc_lo(tiles + vs * kAtTile, kAtHalf) + half * (8192 >> 4);
                    #pragma unroll
                    for (int x = 0; x < 4; ++x)
                        umma_f16_ts(tmem + 256 + 128 * t, tmem + 128 * t + 32 * half + 8 * x, v + x * (2048 >> 4),
                                    idesc_o, add || x > 0);
                };
                int steps[2] = {0, 0}, uses[2] = {0, 0};
                bool ok = true;
                PromptItem it;
                for (int i = 0; ok && next_lane(i, &it); ++i) {
                    const Shape w = shape(it);
                    ok = at_wait(&bar_q[0], uses[0] & 1, ab, err) && at_wait(&bar_full[ks], kp, ab, err);
                    if (!ok) break;
                    scores(0);
                    if (w.nt0 == 1) umma_commit(&bar_qf[0]);
                    if (w.nt1 > 0) {
                        if (!(ok = at_wait(&bar_q[1], uses[1] & 1, ab, err))) break;
                        scores(1);
                        if (w.nt1 == 1) umma_commit(&bar_qf[1]);
                    }
                    umma_commit(&bar_free[ks]);
                    step(ks, kp, 2);
                    #pragma unroll 1
                    for (int j = 0; j < w.nt && ok; ++j) {
                        const bool more = j + 1 < w.nt;
                        ok = at_wait(&bar_full[vs], vp, ab, err) && (!more || at_wait(&bar_full[ks], kp, ab, err));
                        #pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const int n = t == 0 ? w.nt0 : w.nt1;
                            if (!ok || j >= n) continue;
                            // the item before has left O (of) before the first product overwrites it
                            ok = (j > 0 || uses[t] == 0 || at_wait(&bar_of[t], (uses[t] - 1) & 1, ab, err)) &&
                                 at_wait(&bar_h[t], steps[t] & 1, ab, err);
                            if (!ok) continue;
                            tc_fence_after();
                            outputs(t, 0, j > 0);
                            if (!(ok = at_wait(&bar_p[t], steps[t] & 1, ab, err))) continue;
                            tc_fence_after();
                            outputs(t, 1, true);
                            ++steps[t];
                            if (j + 1 < n) {
                                scores(t);
                                if (j + 2 == n) umma_commit(&bar_qf[t]);
                            } else {
                                umma_commit(&bar_o[t]);
                            }
                        }
                        umma_commit(&bar_free[vs]);
                        step(vs, vp, 2);
                        if (more) {
                            umma_commit(&bar_free[ks]);
                            step(ks, kp, 2);
                        }
                    }
                    ++uses[0];
                    uses[1] += w.nt1 > 0 ? 1 : 0;
                }
                umma_commit(&bar_done);
                at_drain(&bar_done, 0);
            }
            __syncwarp();
        } else if (warp == 13) {
            if (elect_one()) {
                // ---------------- loads ----------------
                int x = 0, uses[2] = {0, 0};
                bool ok = true;
                auto load = [&](uint8_t* dst, const CUtensorMap* tm, int head, int token, uint64_t* bar) {
                    mbar_expect_tx(bar, kAtTile);
                    tma_load_3d(dst, tm, 0, head, token, bar);
                    tma_load_3d(dst + kAtHalf, tm, 64, head, token, bar);
                };
                PromptItem it;
                for (int i = 0; ok && next_lane(i, &it); ++i) {
                    const Shape w = shape(it);
                    const int kvh = w.head / p.group;
                    #pragma unroll 1
                    for (int j = -1; j < 2 * w.nt; ++j) {
                        // Q0, K0, Q1, V0, K1, V1, ...
                        const int t = j < 0 ? 0 : 1;
                        if (j < 0 || (j == 1 && w.nt1 > 0)) {
                            if (uses[t] > 0 && !(ok = at_wait(&bar_qf[t], (uses[t] - 1) & 1, ab, err))) break;
                            ++uses[t];
                            load(sm + t * kAtTile, &tm_q, w.head, w.start + w.r0 + kAtRows * t, &bar_q[t]);
                        }
                        if (j < 0) continue;
                        const int s = x % kPmStages, use = x / kPmStages;
                        if (use > 0 && !(ok = at_wait(&bar_free[s], (use - 1) & 1, ab, err))) break;
                        load(sm + (size_t)(2 + s) * kAtTile, (j & 1) == 0 ? &tm_k : &tm_v, kvh,
                             w.start + (j >> 1) * kAtKeys, &bar_full[s]);
                        ++x;
                    }
                }
                // no copy may be in flight when the CTA ends
                for (int t = 0; t < 2; ++t)
                    if (uses[t] > 0) at_drain(&bar_q[t], (uses[t] - 1) & 1);
                for (int y = max(0, x - kPmStages); y < x; ++y) at_drain(&bar_full[y % kPmStages], (y / kPmStages) & 1);
            }
            __syncwarp();
        } else if (warp == 14) {
            // ---------------- items ----------------
            #pragma unroll 1
            for (int i = 0;; ++i) {
                // every other round backwards: the CTA that got the longest
                // item of one round gets the shortest of the next
                const int x = i * (int)gridDim.x + ((i & 1) ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
                PromptItem it{0, 0, -1, x % p.n_head};
                if (!find_long_first<kPmRows>(p, x / p.n_head, &it.start, &it.len, &it.tile)) it.tile = -1;
                if (i >= 2 && !at_wait_warp(&bar_itemf[i & 1], ((i >> 1) - 1) & 1, ab, err)) break;
                if (lane == 0) {
                    s_item[i & 1] = it;
                    mbar_arrive(&bar_item[i & 1]);
                }
                if (it.tile < 0) break;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// [tokens][heads][128] f16 as (64 dims of a half, head, token) boxes of
// 128 tokens of one head
bool encode_heads(CUtensorMap* tm, const void* base, int heads, int tokens, size_t stride) {
    PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
    if (enc == nullptr) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)kServeDim, (cuuint64_t)heads, (cuuint64_t)tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)kServeDim * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, 1, kAtRows};
    const cuuint32_t estr[3] = {1, 1, 1};
    return enc(tm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class O>
cudaError_t launch_mma(const PromptParams& p, cudaStream_t st) {
    CUtensorMap tq, tk, tv;
    const int n_kv = p.n_head / p.group;
    if (!encode_heads(&tq, p.q, p.n_head, p.n_tokens, p.qs) || !encode_heads(&tk, p.k, n_kv, p.n_tokens, p.ks) ||
        !encode_heads(&tv, p.v, n_kv, p.n_tokens, p.vs))
        return cudaErrorInvalidValue;
    auto* kern = attn_prompt_mma_kernel<O>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kPmSmem);
    if (e != cudaSuccess) return e;
    int dev = 0;
    if ((e = cudaGetDevice(&dev)) != cudaSuccess) return e;
    // at most this many items: every sequence may end inside one
    const long long items = (p.n_tokens / kPmRows + (long long)p.n_seq) * p.n_head;
    const int grid = (int)(items < num_sms_of(dev) ? items : num_sms_of(dev));
    return launch(kern, dim3((unsigned)grid), dim3(kPmThreads), kPmSmem, st, false, tq, tk, tv, p);
}

}  // namespace
}  // namespace sllm

using namespace sllm;

extern "C" int sllm_cuda_test_attn_error(void) {
    int v = 0;
    if (cudaDeviceSynchronize() != cudaSuccess ||
        cudaMemcpyFromSymbol(&v, g_prompt_error, sizeof v) != cudaSuccess)
        return -1;
    const int zero = 0;
    cudaMemcpyToSymbol(g_prompt_error, &zero, sizeof zero);
    return v;
}

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
                          : out_type == SLLM_CUDA_KV_F32 ? launch_mma<float>(p, st)
                                                         : launch_mma<__half>(p, st);
    CK(e, "attn_prompt launch");
    count_launches(1);
    return SLLM_CUDA_OK;
}
