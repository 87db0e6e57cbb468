// attn_kv8.cuh -- shared by the two forms of decode attention over an 8-bit cache
// (attn_kv8.cu, attn_kv8_wide.cuh): the parameters, how the work is cut, and
// codes as f16.
#pragma once

#include "attn_mma.cuh"
#include "serve.cuh"

namespace sllm {

constexpr int kE8Keys = 128;                        // keys of a tile
constexpr int kE8Blocks = kE8Keys / kKvBlock;
constexpr int kE8Tile = kE8Keys * kServeDim;        // bytes of one of K or V
// Weights stand against 2^-lift of a reference and are 2^15 at most. Pairs of f16: the
// reference is the running maximum, or a little below. One f16: the maximum when it
// last grew by more than 2^8, so that the outputs are seldom rescaled; weights keep 11
// bits down to 2^-21 of the largest. That adds a tenth to the error of f16 outputs
// (2.1e-4 of their own rounding, 2.3e-4; the wide form, which rounds weight times value
// scale, 2.5e-4); pairs double the products: 64 sequences of up to 8192 keys, 64/8
// heads, 129 us with f32 queries, 97 with f16. A row that has seen nothing has the
// reference kE8None.
// An exponent is one multiply-add of the exact product against the rounded reference.
// References are rounded down and what is taken off up, so that a row's largest key
// never vanishes; where a score is so far from zero (2^23) that the rounding shows,
// exponents end at kE8Top.
constexpr float kE8None = -3.402823466e38f;
constexpr float kE8Most = 15.f, kE8Top = 15.9f;     // of exponents: the reference moves above the one; f16 holds the other
constexpr float kE8Grow = 8.f;
__host__ __device__ constexpr float e8_lift(int planes) { return planes == 1 ? 15.f - kE8Grow : 15.f; }
__host__ __device__ constexpr float e8_down(int planes) { return planes == 1 ? 0x1p-7f : 0x1p-15f; }         // 2^-lift
__device__ __forceinline__ float ended(float z) { return z > kE8Top ? kE8Top : z; }      // (NaN stays)
constexpr float kE8Log2 = kServeScale * 1.4426950408889634f;

struct Attn8Params {
    const void* q;                  // [n][n_q][n_head][128]
    void* out;
    const int8_t* kp;               // the layer's slice of page 0
    const int8_t* vp;
    const float* ksc;
    const float* vsc;
    size_t page_codes, scale_stride;                // codes, scales from a page to the next
    const int32_t* slots;
    int n, n_q, n_head, n_kv, group, rows;          // rows: n_q * group
    int rg, row_blocks, block_rows;                 // row groups of a CTA; row blocks of a pair, and rows of one
    int q_bufs;                     // buffers of a row block's queries
    int page_log2;                  // rows of a page, and of a load
    WaitLimit wait;
    int32_t* status;
    float* part_o;                  // [2 * CTAs][block_rows][128]
    float2* part_ml;                // [2 * CTAs][block_rows]
    // notes for the join: sequence (-1: nothing to join), pair, first and last CTA. Of each
    // pair where there are no more pairs than CTAs (by_pair), else of the pair that starts
    // in a CTA's run and ends in another's
    int4* notes;
    int by_pair, n_notes, ctas;
    uint32_t over_group;            // ceil(2^32 / group), 0 for 1: exact below 2^22 (rows are under 2^14, groups up to 2^10)

    __device__ __forceinline__ int token(int row) const { return over_group == 0 ? row : (int)__umulhi((uint32_t)row, over_group); }
    // row `row` of a sequence's kv head, in q and out
    __device__ __forceinline__ size_t row_at(int b, int head, int row) const {
        const int j = token(row);
        return (((size_t)b * n_q + j) * n_head + (size_t)head * group + (row - j * group)) * kServeDim;
    }
};

struct Meta {                       // of a tile in a stage
    int b, head, row_block, len, key0, flags;
};
enum { E8_FIRST = 1, E8_LAST = 2, E8_PART0 = 4, E8_PART1 = 8, E8_END = 16 };

// The loading warp's place in its run, tile by tile; pair: head * row blocks + row
// block of a sequence
struct Place {
    int b, slot, len, tiles, pair, head, row_block, tile;
    unsigned long long unit;        // its number among all
};

struct RunStart {                   // what finding a run leaves in shared memory
    unsigned long long scan[16];
    unsigned long long rest;
    Place at;
};

struct Waits {                      // for the bounded waits
    const Attn8Params& p;
    __device__ __forceinline__ WaitLimit wait_limit() const { return p.wait; }
};

__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// two codes, of bytes 0 and 1 or 2 and 3 of u (with 128 added to each), as f16:
// 0x6400 + byte is 1024 + byte. (K's codes left 1152 too large, with 1152 times the
// row's sum taken off its scores, were half an instruction a code less, but the f32
// sums then cancelled numbers far larger than a score: scores off by 1e-3 for
// queries of mean 10.)
__device__ __forceinline__ uint32_t two_codes(uint32_t u, bool upper) {
    const uint32_t x = __byte_perm(u, 0x64646464u, upper ? 0x4342 : 0x4140);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t pack2(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

// the tiles of a sequence (one at least: without keys it has zeros to write); 0
// where its slot or length is wrong
__device__ __forceinline__ int seq_tiles(const PagesDev& pg, const Attn8Params& p, int b, int* slot, int* len) {
    const int s = p.slots[b];
    *slot = s;
    *len = 0;
    if (s < 0 || s >= pg.n_slots) return 0;
    const int n = pg.lens[s];
    if (n < 0 || n > pg.cap) return 0;
    *len = n;
    return max(1, (n + kE8Keys - 1) / kE8Keys);
}

// A CTA's run of tiles. All tiles of all pairs are numbered in order, a pair with one
// number more than it has tiles, at its end: what its start and end cost.
template <int EXTRA>
struct Walk8 {
    const PagesDev& pg;
    const Attn8Params& p;
    const int pairs;                // of a sequence
    unsigned long long all, G, u0, u1;              // numbers; runs; this run's numbers
    Place cur;

    __device__ __forceinline__ Walk8(const PagesDev& pages, const Attn8Params& params)
        : pg(pages), p(params), pairs(params.n_kv * params.row_blocks) {}

    // by a prefix sum over the sequences, each of the CTA's THREADS threads some of
    // them; false: there is no run for this CTA. (sh.at.tiles is 0 before.)
    template <int THREADS>
    __device__ __forceinline__ bool find(RunStart& sh) {
        static_assert(THREADS <= 32 * 16, "a sum of each warp");
        const int t = threadIdx.x, lane = t & 31, warp = t >> 5, per = (p.n + THREADS - 1) / THREADS;
        const int b0 = min(t * per, p.n), b1 = min(b0 + per, p.n);
        unsigned long long mine = 0;
        for (int b = b0; b < b1; ++b) {
            int slot, len;
            const int tiles = seq_tiles(pg, p, b, &slot, &len);
            if (tiles == 0 && blockIdx.x == 0) {
                raise(p.status, SLLM_CUDA_ERR_ARG);
                if (p.by_pair)
                    for (int i = 0; i < pairs; ++i) p.notes[b * pairs + i] = make_int4(-1, 0, 0, 0);
            }
            if (tiles > 0) mine += (unsigned long long)(tiles + EXTRA) * pairs;
        }
        unsigned long long upto = mine;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        if (lane == 31) sh.scan[warp] = upto;
        __syncthreads();
        all = 0;
        #pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) upto += sh.scan[w];
            all += sh.scan[w];
        }
        G = gridDim.x < all ? gridDim.x : all;
        const unsigned long long c = blockIdx.x;
        if (c >= G) {
            if (t == 0 && !p.by_pair) p.notes[c] = make_int4(-1, 0, 0, 0);
            return false;
        }
        u0 = c * all / G;
        u1 = (c + 1) * all / G;
        if (u0 >= upto - mine && u0 < upto) {
            unsigned long long rest = u0 - (upto - mine);
            for (int b = b0; b < b1; ++b) {
                Place x;
                x.tiles = seq_tiles(pg, p, b, &x.slot, &x.len);
                const unsigned long long units = x.tiles > 0 ? (unsigned long long)(x.tiles + EXTRA) * pairs : 0;
                if (rest < units) {
                    x.b = b;
                    sh.at = x;
                    sh.rest = rest;
                    break;
                }
                rest -= units;
            }
        }
        __syncthreads();
        return true;
    }

    __device__ __forceinline__ bool next_pair() {
        cur.tile = 0;
        if (++cur.row_block == p.row_blocks) {
            cur.row_block = 0;
            ++cur.head;
        }
        if (++cur.pair < pairs) return true;
        cur.pair = cur.head = 0;
        int b = cur.b + 1;
        for (cur.tiles = 0; b < p.n && cur.tiles == 0; ++b) {       // the next sequence that has tiles
            cur.b = b;
            cur.tiles = seq_tiles(pg, p, b, &cur.slot, &cur.len);
        }
        return cur.tiles > 0;
    }

    // cur: the run's first tile; false: it has none. (Lengths that somebody writes to
    // meanwhile end a run early, inside the arrays.)
    __device__ __forceinline__ bool start(const RunStart& sh) {
        cur = sh.at;
        if (cur.tiles <= 0) return false;
        cur.pair = (int)(sh.rest / (cur.tiles + EXTRA));
        cur.tile = (int)(sh.rest % (cur.tiles + EXTRA));
        cur.head = cur.pair / p.row_blocks;
        cur.row_block = cur.pair % p.row_blocks;
        cur.unit = u0;
        if (cur.tile < cur.tiles) return true;
        cur.unit += cur.tiles + EXTRA - cur.tile;
        return cur.unit < u1 && next_pair();
    }
    __device__ __forceinline__ bool advance() {
        const bool ends = cur.tile + 1 == cur.tiles;
        const unsigned long long to = cur.unit + (ends ? 1 + EXTRA : 1);
        if (to >= u1) return false;
        cur.unit = to;
        if (ends) return next_pair();
        ++cur.tile;
        return true;
    }
    // for the join, from the last tile here of a pair that starts here: other runs
    // go on with it up to its last tile's
    __device__ __forceinline__ int4 note(const Place& x) const {
        const unsigned long long end = x.unit + (unsigned long long)(x.tiles - x.tile);
        return make_int4(x.tile + 1 == x.tiles ? -1 : x.b, x.pair, (int)blockIdx.x, (int)min((end * G - 1) / all, G - 1));
    }
};

}  // namespace sllm
