// attn_kv8_wide.cuh -- decode attention over the 8-bit cache for 17 rows and more
// (query tokens times heads of the group) of f16 queries: blocks of 32 rows on
// tcgen05.
//
// Feeding mma.sync, every 16 rows unpack the codes again and every 16 keys end in
// 64 multiply-adds that scale their outputs. Here a tile of 128 keys is unpacked
// once, into f16 tiles in shared memory, and the scales go into the exponents:
//     S^T [128 keys][32 rows] = C Q^T                 (codes: 128 lanes of tensor memory)
//     w = 2^(s log2 e / sqrt 128 * scale_k + log2 scale_v - ref)
//     O^T [128 dimensions][32 rows] += C'^T W         (W: f16, in shared memory)
//     l += 2^(s log2 e / sqrt 128 * scale_k - ref)
// so w stands for a key's weight times its value scale, against a reference per row
// that is no lower than the row's largest such product over 2^8 (as in the form of
// 16 rows, products keep 11 bits down to 2^-21 of the largest). The sums have exponents
// of their own: w / scale_v would be lost where scales are 2^110 apart. A block of
// scale_v 0 has zeros for values, whatever its codes, and in the exponents the lowest
// scale there is, 2^-100, so that it moves no reference that matters. A sum's terms are
// up to 2^115 then: sums are held 2^8 lower, so that 2^21 keys of no value fit. (The
// other end: of keys whose scales are 2^104 and more, those count that are above 2^-21
// of the largest. Subnormal terms as well, by exp2f, cost 5%.)
//
// Two CTAs a SM. Warps 0-3 and 4-7 (a key a lane, 16 of the rows each group):
// exponentials. 8-11 (32 keys each): codes to f16, K's into tensor memory, V's into
// shared memory, K a tile ahead of V. 12: the products. 13: which tile comes next, its
// scales, and its codes into a ring of 16 KB a half tile.
//
// Bound: neither memory nor the tensor cores but the chains between the roles, two
// of them a SM, with half of the issue slots taken (32 sequences of up to 4096 keys,
// four tokens of 64/8 heads, 139 MB: 60 us, 22 at the memory's rate). Tried, same
// case: one CTA a SM with 18 warps and tiles double buffered 77 us; two with the
// codes loaded into registers, a block ahead, 68 us (49 without the loads: their
// latency was the bound, hence the ring); outputs read after the next tile's
// weights 66 us for 62; row maxima by shuffles instead of redux 84 for 72; queries
// loaded before a pair's first tile instead of under it 63; K's codes left 1152 too
// large, and the exponentials correcting it, 67; sums as w / scale_v while scales are
// within 2^50, or exponents prepared while the scores are made, 61 to 63.
#pragma once

#include "attn_kv8.cuh"

namespace sllm {

constexpr int kW8Rows = 32;                         // rows of a block
constexpr int kW8Mine = kW8Rows / 2;                // of a group of softmax warps
constexpr int kW8Soft = 8, kW8Load = 4;             // warps of exponentials, of codes
constexpr int kW8Products = kW8Soft + kW8Load, kW8Plan = kW8Products + 1;       // single warps
constexpr int kW8Threads = 32 * (kW8Plan + 1), kW8Ctas = 2;                     // CTAs a SM
constexpr int kW8Half = kE8Keys * 128;              // 64 of the dimensions of a tile, f16
constexpr int kW8Extra = 2;                         // what a pair's start and end cost, in tiles (with 1 or 3: 72 and 70 us for 68)
constexpr float kW8Zero = -100.f;                   // log2 of a scale of 0
constexpr float kW8Sum = 8.f, kW8SumDown = 0x1p-8f; // what sums are held lower by, in powers of two
constexpr int kW8Plans = 8;                         // tiles planned ahead, some of them in use
constexpr int kW8Ring = 3;                          // K or V of a tile each
constexpr uint32_t kW8Cols = 256, kW8O = 2 * kW8Rows, kW8K = 128;       // tensor memory: two S tiles, the outputs, two K tiles

struct Plan8 {
    Meta meta;
    __align__(8) float ks[kE8Blocks], vs[kE8Blocks];             // of each block of 16 keys; without one 0 and 1
};

struct __align__(1024) SharedW8 {
    uint8_t raw[kW8Ring][kE8Tile];                  // [key][128], 128-byte swizzle
    uint8_t v[2 * kW8Half];                         // [half of the dimensions][key][64] f16, likewise
    uint8_t p[kE8Keys * 128];                       // [key][32 rows of an even tile, of an odd one], likewise
    uint8_t q[2 * kW8Rows * 128];                   // [half][row][64], likewise
    Plan8 plan[kW8Plans];
    float ref[kW8Soft][kW8Mine], alpha[kW8Soft][kW8Mine];       // each warp has its own copy
    int lim[kW8Soft][kW8Mine];
    float most[kW8Soft][kW8Mine], sum[kW8Soft][kW8Mine];
    uint64_t raw_full[kW8Ring], raw_free[kW8Ring], k_full[2], v_full, v_free, s_full[2], s_free[2], p_full[2], p_free[2], o_free, done;
    uint64_t plan_full[kW8Plans], plan_free[kW8Plans];
    RunStart run;
    uint32_t tmem;
    int abort;
};
static_assert(kW8Ctas * (sizeof(SharedW8) + 1024) <= 228 * 1024, "shared memory");

// whether any of a group's 128 threads says so; all of them come here
__device__ __forceinline__ bool soft_any(int group, bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.or.pred q, %2, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)x), "r"(1 + group)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ void soft_sync(int group) { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); }

__device__ __forceinline__ float warp_top(float x) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}

// 16 bytes of f16 at chunk c of row r of a swizzled tile
__device__ __forceinline__ uint8_t* swizzled(uint8_t* tile, int r, int c) { return tile + r * 128 + ((c ^ (r & 7)) << 4); }

// 16 codes as f16
__device__ __forceinline__ void codes16(const uint4& c, uint32_t* f) {
    const uint32_t w[4] = {c.x ^ 0x80808080u, c.y ^ 0x80808080u, c.z ^ 0x80808080u, c.w ^ 0x80808080u};
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = two_codes(w[i], false);
        f[2 * i + 1] = two_codes(w[i], true);
    }
}

template <class O>
__global__ void __launch_bounds__(kW8Threads, kW8Ctas)
attn_kv8_wide_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ PagesDev pg, const __grid_constant__ Attn8Params p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    SharedW8& sh = *reinterpret_cast<SharedW8*>(smem_raw);
    pdl_trigger();
    const int t = threadIdx.x, lane = t & 31, warp = __shfl_sync(0xffffffffu, t >> 5, 0);
    volatile int* const ab = &sh.abort;
    if ((smem_u32(smem_raw) & 1023u) != 0) {        // (the swizzle counts from a 1024-byte boundary)
        if (t == 0) {
            raise(p.status, SLLM_CUDA_ERR_DEVICE);
            if ((int)blockIdx.x < p.n_notes) p.notes[blockIdx.x] = make_int4(-1, 0, 0, 0);
        }
        return;
    }
    if (t == 0) {
        for (int i = 0; i < kW8Ring; ++i) {
            mbar_init(&sh.raw_full[i], 1);
            mbar_init(&sh.raw_free[i], kW8Load);
        }
        mbar_init(&sh.v_full, kW8Load);
        mbar_init(&sh.v_free, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.k_full[i], kW8Load);
            mbar_init(&sh.p_full[i], kW8Soft);
            mbar_init(&sh.s_free[i], kW8Soft);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_free[i], 1);
        }
        for (int i = 0; i < kW8Plans; ++i) {
            mbar_init(&sh.plan_full[i], 33);        // a warp's scales, and the rest
            mbar_init(&sh.plan_free[i], kW8Soft + kW8Load);
        }
        mbar_init(&sh.o_free, kW8Soft);
        mbar_init(&sh.done, 1);
        sh.abort = 0;
        sh.run.at.tiles = 0;
        fence_proxy_async_smem();
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    Walk8<kW8Extra> walk(pg, p);
    if (!walk.find<kW8Threads>(sh.run)) return;
    if (warp == kW8Products) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(kW8Cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;                  // S at columns 0 and 32
    const Waits w{p};
    bool ok = true;

    if (warp < kW8Soft) {
        // ---- exponentials: lane's key of the tile, the group's 16 rows
        constexpr int R = kW8Mine;
        const int group = warp >> 2, first_row = R * group, key = 32 * (warp & 3) + lane, g0 = 4 * group;
        const uint32_t tm = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + first_row;
        float* const ref = sh.ref[warp];
        float l[R];
        size_t out_at = 0;                          // of row `lane`
        constexpr float LIFT = e8_lift(1);
        for (uint32_t n = 0;; ++n) {
            const int b = n & 1;
            const uint32_t par = n >> 1 & 1;
            ok = (n == 0 ? __all_sync(0xffffffffu, at_wait_start(&sh.s_full[b], 0, ab, w)) : at_wait_warp(&sh.s_full[b], par, ab, w)) && ok;
            ok = at_wait_warp(&sh.plan_full[n % kW8Plans], n / kW8Plans & 1, ab, w) && ok;         // (it is; for its scales)
            const Meta mt = sh.plan[n % kW8Plans].meta;
            const bool stop = !ok || (mt.flags & E8_END) != 0;
            tc_fence_after();
            float z[R], top = -INFINITY;
            auto scores = [&] {
                uint32_t s[R];
                tmem_ld16(tm + kW8Rows * b, s);
                tmem_ld_wait();
                #pragma unroll
                for (int i = 0; i < R; ++i) z[i] = u2f(s[i]);
            };
            const int row0 = mt.row_block * kW8Rows + first_row, j = mt.key0 + key;
            if (mt.flags & E8_FIRST) {
                if (lane < R) {
                    const int row = row0 + lane;
                    ref[lane] = kE8None;
                    sh.lim[warp][lane] = mt.len - p.n_q + 1 + (row < p.rows ? p.token(row) : p.n_q - 1);
                    out_at = p.row_at(mt.b, mt.head, row < p.rows ? row : 0);
                }
                #pragma unroll
                for (int i = 0; i < R; ++i) l[i] = 0.f;
                __syncwarp();
            }
            const float ks = sh.plan[n % kW8Plans].ks[key / kKvBlock], vs = sh.plan[n % kW8Plans].vs[key / kKvBlock];
            const float base = ks * kE8Log2, lsv = vs != 0.f ? __log2f(vs) : kW8Zero;
            const bool masked = mt.key0 + kE8Keys > mt.len - p.n_q + 1;
            // exponents of two against the references
            auto exponents = [&] {
                scores();
                #pragma unroll
                for (int i = 0; i < R; i += 4) {
                    const float4 r = *reinterpret_cast<const float4*>(ref + i);
                    z[i] = __fmaf_rn(z[i], base, __fsub_ru(lsv + LIFT, r.x));
                    z[i + 1] = __fmaf_rn(z[i + 1], base, __fsub_ru(lsv + LIFT, r.y));
                    z[i + 2] = __fmaf_rn(z[i + 2], base, __fsub_ru(lsv + LIFT, r.z));
                    z[i + 3] = __fmaf_rn(z[i + 3], base, __fsub_ru(lsv + LIFT, r.w));
                }
                if (masked) {
                    #pragma unroll
                    for (int i = 0; i < R; ++i)
                        if (j >= sh.lim[warp][i]) z[i] = -INFINITY;
                }
            };
            exponents();
            #pragma unroll
            for (int i = 0; i < R; ++i) top = fmaxf(top, z[i]);
            if (soft_any(group, top > kE8Most || stop)) {
                // (the group's warps leave together: they meet at barriers without a limit)
                if (soft_any(group, stop)) break;
                // the references move to the rows' maxima, and what stands against the
                // old ones with them
                scores();
                float mine = kE8None;               // row `lane`
                #pragma unroll
                for (int i = 0; i < R; ++i) {
                    const float m = warp_top(!masked || j < sh.lim[warp][i] ? __fmaf_rd(z[i], base, lsv) : kE8None);
                    if (lane == i) mine = m;
                }
                if (lane < R) sh.most[warp][lane] = mine;
                soft_sync(group);
                if (lane < R) {
                    const float was = ref[lane];
                    const float now = fmaxf(fmaxf(was, fmaxf(sh.most[g0][lane], sh.most[g0 + 1][lane])),
                                            fmaxf(sh.most[g0 + 2][lane], sh.most[g0 + 3][lane]));
                    ref[lane] = now;
                    sh.alpha[warp][lane] = ex2(was - now);
                }
                __syncwarp();
                const float* const alpha = sh.alpha[warp];
                if (!(mt.flags & E8_FIRST)) {
                    ok = at_wait_warp(&sh.p_free[b ^ 1], (n - 1) >> 1 & 1, ab, w) && ok;
                    tc_fence_after();
                    if (ok) {
                        uint32_t o[R];
                        tmem_ld16(tm + kW8O, o);
                        tmem_ld_wait();
                        #pragma unroll
                        for (int i = 0; i < R; ++i) o[i] = f2u(u2f(o[i]) * alpha[i]);
                        tmem_st16(tm + kW8O, o);
                        tmem_st_wait();
                    }
                }
                #pragma unroll
                for (int i = 0; i < R; ++i) l[i] *= alpha[i];
                exponents();
                #pragma unroll
                for (int i = 0; i < R; ++i) z[i] = ended(z[i]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh.s_free[b]);
                mbar_arrive(&sh.plan_free[n % kW8Plans]);
            }
            const float lsum = lsv + kW8Sum;
            #pragma unroll
            for (int i = 0; i < R; ++i) {
                l[i] += ex2(z[i] - lsum);
                z[i] = ex2(z[i]);
            }
            if (n >= 2) ok = at_wait_warp(&sh.p_free[b], par ^ 1, ab, w) && ok;
            if (ok) {
                #pragma unroll
                for (int c = 0; c < R / 8; ++c)
                    *reinterpret_cast<uint4*>(swizzled(sh.p, key, 4 * b + 2 * group + c)) =
                        make_uint4(pack2(z[8 * c], z[8 * c + 1]), pack2(z[8 * c + 2], z[8 * c + 3]), pack2(z[8 * c + 4], z[8 * c + 5]),
                                   pack2(z[8 * c + 6], z[8 * c + 7]));
            }
            fence_proxy_async_smem();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.p_full[b]);
            if (!(mt.flags & E8_LAST)) continue;
            // ---- the outputs: lane's dimension, the group's rows
            ok = at_wait_warp(&sh.p_free[b], par, ab, w) && ok;
            tc_fence_after();
            uint32_t o[R];
            tmem_ld16(tm + kW8O, o);
            // the rows' sums over the warp's keys: half of the values with each shuffle,
            // lanes i and i + 16 end with row i's
            #pragma unroll
            for (int i = 0; i < R; ++i) l[i] += __shfl_xor_sync(0xffffffffu, l[i], R);
            #pragma unroll
            for (int h = R / 2; h > 0; h >>= 1) {
                const bool up = (lane & h) != 0;
                #pragma unroll
                for (int i = 0; i < h; ++i) {
                    const float give = up ? l[i] : l[i + h], keep = up ? l[i + h] : l[i];
                    l[i] = keep + __shfl_xor_sync(0xffffffffu, give, h);
                }
            }
            if (lane < R) sh.sum[warp][lane] = l[0];
            tmem_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.o_free);
            soft_sync(group);
            const int rl = lane & (R - 1);
            const float sum = (sh.sum[g0][rl] + sh.sum[g0 + 1][rl]) + (sh.sum[g0 + 2][rl] + sh.sum[g0 + 3][rl]);
            const int part = mt.flags & E8_PART0 ? 2 * (int)blockIdx.x : mt.flags & E8_PART1 ? 2 * (int)blockIdx.x + 1 : -1;
            const int live = min(p.rows - row0, R);
            if (!ok) continue;
            if (part >= 0) {
                const size_t at = (size_t)part * kW8Rows + first_row;
                float* const to = p.part_o + at * kServeDim + key;
                if ((warp & 3) == 0 && lane < live) p.part_ml[at + lane] = make_float2(ref[lane], sum);
                #pragma unroll
                for (int i = 0; i < R; ++i)
                    if (i < live) to[i * kServeDim] = u2f(o[i]) * kW8SumDown;
            } else {
                const float inv = sum == 0.f ? 0.f : __fdiv_rn(kW8SumDown, sum);   // (0: the row has seen nothing)
                #pragma unroll
                for (int i = 0; i < R; ++i) {
                    const size_t at = __shfl_sync(0xffffffffu, (unsigned long long)out_at, i);
                    const float f = __shfl_sync(0xffffffffu, inv, i);
                    if (i < live) from_f32_to(static_cast<O*>(p.out) + at + key, u2f(o[i]) * f);
                }
            }
        }
    } else if (warp < kW8Products) {
        // ---- codes: this warp's 32 keys of each tile: K of tile 0, of 1, V of 0, K of 2, V of 1, ...
        const int cw = warp - kW8Soft, key = 32 * cw + lane;
        const uint32_t tm = tmem + ((uint32_t)(32 * cw) << 16) + kW8K;
        uint32_t unit = 0;                          // of the ring
        auto arrived = [&] { return at_wait_warp(&sh.raw_full[unit % kW8Ring], unit / kW8Ring & 1, ab, w); };
        auto consumed = [&] {
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.raw_free[unit % kW8Ring]);
            ++unit;
        };
        // K of tile n (its plan is there)
        auto put_k = [&](uint32_t n) {
            const Meta mt = sh.plan[n % kW8Plans].meta;
            const int b = n & 1;
            if (!(mt.flags & E8_END)) {
                // (the scores of two tiles before are there: its keys have been read)
                if (n >= 2 && !at_wait_warp(&sh.s_full[b], ((n >> 1) - 1) & 1, ab, w)) return false;
                if (mt.flags & E8_FIRST) {          // the pair's queries; those before have been read
                    if (n >= 1 && !at_wait_warp(&sh.s_full[b ^ 1], (n - 1) >> 1 & 1, ab, w)) return false;
                    const int r0 = mt.row_block * kW8Rows;
                    #pragma unroll
                    for (int i = 0; i < kW8Rows * 16 / (32 * kW8Load); ++i) {
                        const int y = (i * kW8Load + cw) * 32 + lane, r = y >> 4, c = y & 15;
                        const bool there = r0 + r < p.rows;         // (else zeros)
                        const __half* const from = static_cast<const __half*>(p.q) + p.row_at(mt.b, mt.head, there ? r0 + r : r0) + 8 * c;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                         smem_u32(swizzled(sh.q + (c >> 3) * kW8Rows * 128, r, c & 7))),
                                     "l"(from), "r"(there ? 16 : 0)
                                     : "memory");
                    }
                }
                if (!arrived()) return false;
                uint8_t* const raw = sh.raw[unit % kW8Ring];
                tc_fence_after();
                #pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint4 c[4];
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) c[i] = *reinterpret_cast<const uint4*>(swizzled(raw, key, 4 * h + i));
                    uint32_t f[32];
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) codes16(c[i], f + 8 * i);
                    tmem_st32(tm + 64 * b + 32 * h, f);
                }
                consumed();
                if (mt.flags & E8_FIRST) {
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    fence_proxy_async_smem();
                }
                tmem_st_wait();
                tc_fence_before();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.k_full[b]);
            return true;
        };
        auto planned = [&](uint32_t n) { return at_wait_warp(&sh.plan_full[n % kW8Plans], n / kW8Plans & 1, ab, w); };
        // lane's piece of a row: of rows r and r ^ 5, so that eight lanes load and store
        // eight different 16 bytes of the swizzle
        const int vrow = 32 * cw + ((lane >> 3) ^ (lane & 4 ? 5 : 0)), piece = lane & 3;
        ok = planned(0) && put_k(0);
        bool end = ok && (sh.plan[0].meta.flags & E8_END) != 0;
        for (uint32_t n = 0; ok && !end; ++n) {
            ok = planned(n + 1) && put_k(n + 1) && (n == 0 || at_wait_warp(&sh.v_free, (n - 1) & 1, ab, w)) && arrived();
            if (!ok) break;
            end = (sh.plan[(n + 1) % kW8Plans].meta.flags & E8_END) != 0;
            uint8_t* const raw = sh.raw[unit % kW8Ring];
            const float2 sv = *reinterpret_cast<const float2*>(sh.plan[n % kW8Plans].vs + 2 * cw);
            #pragma unroll
            for (int g = 0; g < 2; ++g) {           // a block of 16 keys
                uint4 c[4];
                #pragma unroll
                for (int i = 0; i < 4; ++i)
                    c[i] = *reinterpret_cast<const uint4*>(swizzled(raw, vrow + 16 * g + 8 * (i >> 1), 4 * (i & 1) + piece));
                // (a scale of 0 is zeros, whatever the codes are)
                if ((g == 0 ? sv.x : sv.y) == 0.f) c[0] = c[1] = c[2] = c[3] = make_uint4(0, 0, 0, 0);
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t f[8];
                    codes16(c[i], f);
                    #pragma unroll
                    for (int j = 0; j < 2; ++j)
                        *reinterpret_cast<uint4*>(swizzled(sh.v + (i & 1) * kW8Half, vrow + 16 * g + 8 * (i >> 1), 2 * piece + j)) =
                            make_uint4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
                }
            }
            consumed();
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh.v_full);
                mbar_arrive(&sh.plan_free[n % kW8Plans]);
            }
        }
    } else if (warp == kW8Plan) {
        // ---- plans and loads
        // lane i: the page of the tile's i-th load
        auto ids = [&](const Place& x) {
            const int at = x.tile * kE8Keys + (lane << p.page_log2);
            int id = 0;
            if (lane < (kE8Keys >> p.page_log2) && at < x.len) {
                id = pg.tables[(size_t)x.slot * pg.width + (at >> p.page_log2)];
                if (id < 0 || id >= pg.n_pages) {
                    raise(p.status, SLLM_CUDA_ERR_ARG);
                    id = 0;
                }
            }
            return id;
        };
        uint32_t unit = 0;                          // of the ring
        auto load = [&](const CUtensorMap* tm, int loads, int head, int id) {
            const int slot = unit % kW8Ring;
            if (unit >= kW8Ring && !at_wait_warp(&sh.raw_free[slot], (unit / kW8Ring - 1) & 1, ab, w)) return false;
            if (lane == 0) mbar_expect_tx(&sh.raw_full[slot], (uint32_t)(loads << p.page_log2) * kServeDim);
            __syncwarp();
            if (lane < loads) tma_load_4d(sh.raw[slot] + (lane * kServeDim << p.page_log2), tm, 0, 0, head, id, &sh.raw_full[slot]);
            ++unit;
            return true;
        };
        // each lane's arrival when its scales are there, and one for what the lanes have written
        auto plan_ready = [&](int slot) {
            cp_async_arrive(&sh.plan_full[slot]);
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.plan_full[slot]);
        };
        bool more = walk.start(sh.run);
        int id = more ? ids(walk.cur) : 0;
        int first = 1, started = more && walk.cur.tile == 0;    // of the segment: its first tile here; whether the pair starts here
        int v_id = 0, v_head = 0, v_loads = 0;      // of the tile before: its V is to be loaded
        int4 note = make_int4(-1, 0, 0, 0);
        uint32_t n = 0;
        while (more) {
            const Place cur = walk.cur;
            const bool ends = cur.tile + 1 == cur.tiles;
            more = walk.advance();
            const int nid = more ? ids(walk.cur) : 0;
            const int slot = n % kW8Plans;
            if (n >= kW8Plans && !(ok = at_wait_warp(&sh.plan_free[slot], (n / kW8Plans - 1) & 1, ab, w))) break;
            const bool last = ends || !more;
            const int key0 = cur.tile * kE8Keys, keys = min(kE8Keys, cur.len - key0);
            const int loads = (keys + (1 << p.page_log2) - 1) >> p.page_log2;
            const int blk = lane & (kE8Blocks - 1), from = __shfl_sync(0xffffffffu, id, (blk * kKvBlock) >> p.page_log2);
            if (lane < 2 * kE8Blocks) {
                float* const to = lane < kE8Blocks ? sh.plan[slot].ks + blk : sh.plan[slot].vs + blk;
                if (blk * kKvBlock < keys)
                    cp_async4(to, (lane < kE8Blocks ? p.ksc : p.vsc) + (size_t)from * p.scale_stride + cur.head * (pg.page / kKvBlock) +
                                      ((key0 + blk * kKvBlock) & (pg.page - 1)) / kKvBlock);
                else
                    *to = lane < kE8Blocks ? 0.f : 1.f;
            }
            if (lane == 0) {
                const int flags = (first ? E8_FIRST : 0) | (last ? E8_LAST : 0) |
                                  (!last || (ends && started) ? 0 : started ? E8_PART1 : E8_PART0);
                sh.plan[slot].meta = Meta{cur.b, cur.head, cur.row_block, cur.len, key0, flags};
            }
            plan_ready(slot);
            if (!(ok = load(&tm_k, loads, cur.head, id) && (n == 0 || load(&tm_v, v_loads, v_head, v_id)))) break;
            v_id = id;
            v_head = cur.head;
            v_loads = loads;
            if (last && started) {
                const int4 x = walk.note(cur);
                if (!ends) note = x;
                if (p.by_pair && lane == 0) p.notes[cur.b * walk.pairs + cur.pair] = x;
            }
            first = last;
            started = last ? 1 : started;
            id = nid;
            ++n;
        }
        if (ok && n > 0) ok = load(&tm_v, v_loads, v_head, v_id);
        if (ok && n >= kW8Plans) ok = at_wait_warp(&sh.plan_free[n % kW8Plans], (n / kW8Plans - 1) & 1, ab, w);
        if (ok) {
            if (lane == 0) sh.plan[n % kW8Plans].meta = Meta{0, 0, 0, 0, 0, E8_END};
            plan_ready(n % kW8Plans);
        }
        if (lane == 0 && !p.by_pair) p.notes[blockIdx.x] = note;
        // copies in flight end before the CTA does, also where the others gave up
        for (uint32_t i = unit > kW8Ring ? unit - kW8Ring : 0; i < unit; ++i) at_drain(&sh.raw_full[i % kW8Ring], (i / kW8Ring) & 1);
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (elect_one()) {
        // ---- products
        constexpr uint32_t A_MN = 1u << 15;         // the first operand's rows are contiguous
        constexpr uint32_t idesc_s = umma_idesc_f16(128, kW8Rows, false), idesc_o = umma_idesc_f16(128, kW8Rows, true) | A_MN;
        uint32_t seg = 0;
        int before = 0;                             // the tile before: its flags
        for (uint32_t n = 0;; ++n) {
            const int b = n & 1;
            const uint32_t par = n >> 1 & 1;
            if (!(ok = at_wait(&sh.k_full[b], par, ab, w))) break;
            const int flags = sh.plan[n % kW8Plans].meta.flags;
            if (n >= 2 && !(ok = at_wait(&sh.s_free[b], par ^ 1, ab, w))) break;
            if (flags & E8_END) mbar_arrive(&sh.s_full[b]);
            else {
                tc_fence_after();
                const uint32_t q = umma_desc_lo(smem_u32(sh.q), 16);
                #pragma unroll
                for (int x = 0; x < 8; ++x)
                    umma_f16_ts(tmem + kW8Rows * b, tmem + kW8K + 64 * b + 8 * x, q + (x >> 2) * (kW8Rows * 128 >> 4) + (x & 3) * 2,
                                idesc_s, x > 0);
                umma_commit(&sh.s_full[b]);
            }
            if (n >= 1) {                           // the tile before: its outputs
                if (before & E8_FIRST) {
                    if (seg > 0 && !(ok = at_wait(&sh.o_free, (seg - 1) & 1, ab, w))) break;
                    ++seg;
                }
                if (!(ok = at_wait(&sh.v_full, (n - 1) & 1, ab, w) && at_wait(&sh.p_full[b ^ 1], (n - 1) >> 1 & 1, ab, w))) break;
                tc_fence_after();
                const uint32_t v = umma_desc_lo(smem_u32(sh.v), kW8Half), pp = umma_desc_lo(smem_u32(sh.p) + 64 * (b ^ 1), kW8Half);
                #pragma unroll
                for (int x = 0; x < 8; ++x)
                    umma_f16_ss(tmem + kW8O, v + x * (2048 >> 4), pp + x * (2048 >> 4), idesc_o, x > 0 || !(before & E8_FIRST));
                umma_commit(&sh.p_free[b ^ 1]);
                umma_commit(&sh.v_free);
            }
            if (flags & E8_END) break;
            before = flags;
        }
        umma_commit(&sh.done);
        at_drain(&sh.done, 0);
    }
    __syncwarp();
    if (!ok && lane == 0) raise(p.status, SLLM_CUDA_ERR_TIMEOUT);
    tc_fence_before();
    __syncthreads();
    if (t == 0 && sh.abort != 0) raise(p.status, SLLM_CUDA_ERR_TIMEOUT);
    if (warp == kW8Products) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kW8Cols) : "memory");
    }
}

}  // namespace sllm
