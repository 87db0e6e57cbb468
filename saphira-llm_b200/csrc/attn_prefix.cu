// attn_prefix.cu -- decode attention of sequences that share a prefix, over a
// paged cache.
//
// The rows of a kv head are all (sequence, query token, query head of the
// group). Against the prefix they are one matrix, so each of its keys is read
// once and multiplied with all of them; against a sequence's own tokens only
// that sequence's rows are. Both kinds of work are split along the keys into
// items of about one size; an item leaves, for each of its rows, the softmax's
// maximum m and sum l over its keys and the unscaled output, and a second
// launch (overlapped by programmatic dependent launch) joins a row's parts:
//     M = max m_i,  out = sum_i e^(m_i - M) o_i / sum_i e^(m_i - M) l_i.
//
// f16: the tensor-core core of attn_mma.cuh. f32, and groups of more than 128
// heads: that of attn_wide.cuh, one item per CTA.
//
// Bound: HBM (the keys and values once) for few rows; the products for many
// (n * n_q * group rows share each key: above about 250 of them); under about
// 8000 keys the two launches and the chain of dependent reads in them, 12 us.
// Measured, f16: 16 sequences of up to 300 tokens behind 4096, 20 heads of 5,
// 19 us; 64 of up to 1000 behind 32768, four query tokens each, 64 heads of 8,
// 288 us (969 TFLOP/s). f32: two of 64 behind 256, 20 heads of 5, 13.4 us; four
// behind 16384, 32 heads of 8, 59 us.
// The cut is made on the host, from sizes alone: made on the device, from the
// lengths, it put two dependent reads before the first item (27.6 us against
// 18.0 us for the 16 sequences).

#include <algorithm>

#include "attn_mma.cuh"
#include "attn_wide.cuh"

namespace sllm {
namespace {

// how the work is cut
struct Plan {
    int key_tile;                   // keys of a tile
    int rt, per;                    // rows of a row tile, row tiles of an item
    int ptiles, sp;                 // key tiles of the prefix, and its splits
    int ct, cm;                     // key tiles of a chunk of a sequence's own keys; chunks at most
    int ri_all, ri_seq;             // row items of all sequences, of one
    int* next;                      // the next item's number, or NULL: numbers are dealt
};

struct PrefixParams {
    const void* q;                  // [n][n_q][n_head][128]
    void* out;
    const void* kp;                 // the layer's slice of page 0
    const void* vp;
    size_t page_stride;             // elements
    const int32_t* slots;
    int n, n_q, n_head, n_kv, group, prefix;
    WaitLimit wait;
    int32_t* status;
    float* part_o;                  // [n_kv][rows][sp + cm][128]
    float2* part_ml;                // [n_kv][rows][sp + cm]
    Plan plan;
};

// the tokens a sequence's slot holds; -1 when the slot or its length is wrong
__device__ __forceinline__ int seq_len(const PagesDev& pg, const PrefixParams& p, int b, int* slot) {
    const int s = p.slots[b];
    *slot = s;
    if (s < 0 || s >= pg.n_slots) return -1;
    const int len = pg.lens[s];
    if (len < 0 || len > pg.cap) return -1;
    if (p.prefix > 0 && len - p.n_q + 1 < p.prefix) return -1;
    return len;
}

__device__ __forceinline__ int own_tiles(const PrefixParams& p, int len) {
    return (max(0, len - p.prefix) + p.plan.key_tile - 1) / p.plan.key_tile;
}

__device__ __forceinline__ int own_chunks(const PrefixParams& p, int tiles) {
    return min(p.plan.cm, (tiles + p.plan.ct - 1) / p.plan.ct);
}

// Keys a .. a + keys - 1 of `slot` for rows row0 .. of kv head kvh (at most
// row_end); row r (token r / group) sees lim0 + r / group - tok0 of them.
struct PrefixItem {
    int slot, kvh, row0, row_end, a, keys, lim0, tok0, part;    // part < 0: no more items
    __device__ bool last() const { return part < 0; }
};

// item x: the prefix's splits first, then the sequences' own chunks; false
// where a sequence has fewer chunks than its share of numbers
__device__ __forceinline__ bool find_item(const PagesDev& pg, const PrefixParams& p, long long x, PrefixItem* it) {
    const Plan& pl = p.plan;
    const long long pre = (long long)p.n_kv * pl.ri_all * pl.sp;
    if (x < pre) {
        const int ri = (int)(x % pl.ri_all), u = (int)(x / pl.ri_all);
        it->kvh = u % p.n_kv;
        const int s = u / p.n_kv;
        const int t0 = (int)((long long)s * pl.ptiles / pl.sp), t1 = (int)((long long)(s + 1) * pl.ptiles / pl.sp);
        it->slot = p.slots[0];
        it->row0 = ri * pl.per * pl.rt;
        it->row_end = p.n * p.n_q * p.group;
        it->a = t0 * pl.key_tile;
        it->keys = min(t1 * pl.key_tile, p.prefix) - it->a;
        it->lim0 = it->keys;
        it->tok0 = 0;
        it->part = s;
        return true;
    }
    x -= pre;
    if (x >= (long long)p.n * pl.cm * p.n_kv * pl.ri_seq) {
        it->part = -1;
        return true;
    }
    const int ri = (int)(x % pl.ri_seq);
    x /= pl.ri_seq;
    it->kvh = (int)(x % p.n_kv);
    x /= p.n_kv;
    const int b = (int)(x % p.n), c = (int)(x / p.n);
    int slot;
    const int len = seq_len(pg, p, b, &slot), tiles = own_tiles(p, len), chunks = own_chunks(p, tiles);
    if (c >= chunks) return false;
    const int t0 = (int)((long long)c * tiles / chunks), t1 = (int)((long long)(c + 1) * tiles / chunks);
    it->slot = slot;
    it->row0 = (b * p.n_q) * p.group + ri * pl.per * pl.rt;
    it->row_end = (b + 1) * p.n_q * p.group;
    it->a = p.prefix + t0 * pl.key_tile;
    it->keys = min(p.prefix + t1 * pl.key_tile, len) - it->a;
    it->tok0 = b * p.n_q;
    it->lim0 = len - p.n_q + 1 - it->a;
    it->part = pl.sp + c;
    return true;
}

__device__ __forceinline__ int row_seen(const PrefixParams& p, const PrefixItem& it, int r) {
    return min(max(it.lim0 + r / p.group - it.tok0, 0), it.keys);
}

// a row of q or out: token r / group, head kvh * group + r % group
__device__ __forceinline__ size_t row_off(const PrefixParams& p, int kvh, int r) {
    return ((size_t)(r / p.group) * p.n_head + kvh * p.group + r % p.group) * kServeDim;
}

__device__ __forceinline__ size_t part_at(const PrefixParams& p, const PrefixItem& it, int r) {
    return ((size_t)it.kvh * p.n * p.n_q * p.group + r) * (p.plan.sp + p.plan.cm) + it.part;
}

// the page that holds key j of a slot; a wrong one is reported and replaced
__device__ __forceinline__ int page_of(const PagesDev& pg, const PrefixParams& p, int slot, int index) {
    int id = -1;
    if (slot >= 0 && slot < pg.n_slots && index < pg.width) id = pg.tables[(size_t)slot * pg.width + index];
    if (id < 0 || id >= pg.n_pages) {
        raise(p.status, SLLM_CUDA_ERR_ARG);
        id = 0;
    }
    return id;
}

// one warp's rows of the row tile at r0, from tensor memory, as parts
__device__ __forceinline__ void store_parts(const PrefixParams& p, const PrefixItem& it, int r0, int row, uint32_t o_tm,
                                            float m, float l, uint8_t* stage) {
    const int lane = row & 31, r = r0 + row - lane;         // the warp's first row
    const int n = min(p.plan.rt - (row - lane), it.row_end - r);
    if (n <= 0) return;                                     // a warp without rows
    const int parts = p.plan.sp + p.plan.cm;
    const size_t at = part_at(p, it, r);
    if (lane < n) p.part_ml[at + (size_t)lane * parts] = make_float2(m * kServeScale, l);
    store_rows(o_tm, 1.f, stage, p.part_o + at * kServeDim, (size_t)parts * kServeDim, n);
}

// value row `key` of an item
template <class T>
__device__ __forceinline__ const T* value_row(const PagesDev& pg, const PrefixParams& p, const PrefixItem& it, int key) {
    const int id = page_of(pg, p, it.slot, (it.a + key) / pg.page);
    return static_cast<const T*>(p.vp) + (size_t)id * p.page_stride +
           ((size_t)it.kvh * pg.page + (it.a + key) % pg.page) * kServeDim;
}

// ---------------------------------------------------------------------------
// f16 on the tensor cores
// ---------------------------------------------------------------------------
struct PrefixWork {
    using Item = PrefixItem;
    const PagesDev& pg;
    const PrefixParams& p;
    const CUtensorMap &tm_q, &tm_k, &tm_v;

    struct Finder {
        __device__ __forceinline__ void start(const PrefixWork&) {}
        __device__ __forceinline__ long long number(const PrefixWork& w, int r) {
            if (w.p.plan.next == nullptr) return dealt_number(r);
            int x = 0;
            if ((threadIdx.x & 31) == 0) x = atomicAdd(w.p.plan.next, 1);
            return __shfl_sync(0xffffffffu, x, 0);
        }
        __device__ __forceinline__ bool item(const PrefixWork& w, long long x, Item* it) {
            return find_item(w.pg, w.p, x, it);
        }
    };
    __device__ __forceinline__ WaitLimit wait_limit() const { return p.wait; }
    __device__ __forceinline__ void check() const {}
    __device__ __forceinline__ void gave_up() const { raise(p.status, SLLM_CUDA_ERR_TIMEOUT); }
    __device__ __forceinline__ int tiles(const Item& it, int t) const {
        return it.row0 + t * p.plan.rt < it.row_end ? (it.keys + kAtKeys - 1) / kAtKeys : 0;
    }
    __device__ __forceinline__ int keys(const Item& it) const { return it.keys; }
    __device__ __forceinline__ int seen(const Item& it, int t, int row) const {
        return live(it, t, row) ? row_seen(p, it, it.row0 + t * p.plan.rt + row) : it.keys;
    }
    __device__ __forceinline__ bool live(const Item& it, int t, int row) const {
        return row < p.plan.rt && it.row0 + t * p.plan.rt + row < it.row_end;
    }
    // One lane per page of a tile; the ids of 32 pages at a time, the next 32
    // on their way.
    struct Loader {
        int cur, nxt, base;
        __device__ __forceinline__ int ids(const PrefixWork& w, const Item& it, int at, int lane) {
            const int pages = (it.keys + w.pg.page - 1) / w.pg.page;
            return at + lane < pages ? page_of(w.pg, w.p, it.slot, it.a / w.pg.page + at + lane) : 0;
        }
        __device__ __forceinline__ void start(const PrefixWork& w, const Item& it, int lane) {
            base = 0;
            cur = ids(w, it, 0, lane);
            nxt = ids(w, it, 32, lane);
        }
        __device__ __forceinline__ void q(const PrefixWork& w, const Item& it, int t, uint8_t* dst, uint64_t* bar, int lane) {
            if (lane == 0) {
                const int token = it.row0 / w.p.group + t * (w.p.plan.rt / w.p.group);
                mbar_expect_tx(bar, (uint32_t)w.p.plan.rt * 256u);
                tma_load_4d(dst, &w.tm_q, 0, 0, it.kvh, token, bar);
                tma_load_4d(dst + kAtHalf, &w.tm_q, 64, 0, it.kvh, token, bar);
            }
        }
        __device__ __forceinline__ void kv(const PrefixWork& w, const Item& it, int j, bool v, uint8_t* dst, uint64_t* bar,
                                           int lane) {
            const int per = kAtKeys / w.pg.page, first = j * per;
            if (first >= base + 32) {
                base += 32;
                cur = nxt;
                nxt = ids(w, it, base + 32, lane);
            }
            const int n = min(per, (it.keys - j * kAtKeys + w.pg.page - 1) / w.pg.page);
            const int id = __shfl_sync(0xffffffffu, cur, (first - base + lane) & 31);
            if (lane == 0) mbar_expect_tx(bar, (uint32_t)(n * w.pg.page) * 256u);
            __syncwarp();
            if (lane < n) {
                const CUtensorMap* tm = v ? &w.tm_v : &w.tm_k;
                uint8_t* at = dst + lane * w.pg.page * 128;
                tma_load_4d(at, tm, 0, 0, it.kvh, id, bar);
                tma_load_4d(at + kAtHalf, tm, 64, 0, it.kvh, id, bar);
            }
            __syncwarp();
        }
    };
    __device__ __forceinline__ void store(const Item& it, int t, int row, uint32_t o_tm, float m, float l,
                                          uint8_t* stage) const {
        store_parts(p, it, it.row0 + t * p.plan.rt, row, o_tm, m, l, stage);
    }
    __device__ __forceinline__ void odd(const Item& it, int t, int row) const {
        const int lane4 = 4 * (threadIdx.x & 31), r0 = it.row0 + t * p.plan.rt + row;
        add_odd<4>(row_seen(p, it, it.row0), it.keys, min(min(32, p.plan.rt - row), it.row_end - r0),
                   [&](int key) { return value_row<__half>(pg, p, it, key) + lane4; },
                   [&](int r) { return row_seen(p, it, r0 + r); },
                   [&](int r) { return p.part_o + part_at(p, it, r0 + r) * kServeDim + lane4; });
    }
};

__global__ void __launch_bounds__(kAtThreads, 1)
attn_prefix_mma_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PagesDev pg,
                       const __grid_constant__ PrefixParams p) {
    pdl_trigger();
    attn_core(PrefixWork{pg, p, tm_q, tm_k, tm_v});
}

// ---------------------------------------------------------------------------
// 32-bit on the tensor cores: one item of up to 128 rows per CTA. Groups of
// more than 128 f16 heads come here too.
// ---------------------------------------------------------------------------
template <class KV>
struct PrefixWide {
    using T = KV;
    using Item = PrefixItem;
    const PagesDev& pg;
    const PrefixParams& p;

    __device__ __forceinline__ WaitLimit wait_limit() const { return p.wait; }
    __device__ __forceinline__ void check() const {}
    __device__ __forceinline__ void gave_up() const { raise(p.status, SLLM_CUDA_ERR_TIMEOUT); }
    __device__ __forceinline__ bool find(long long x, Item* it) const { return find_item(pg, p, x, it); }
    __device__ __forceinline__ int keys(const Item& it) const { return it.keys; }
    __device__ __forceinline__ bool live(const Item& it, int row) const { return it.row0 + row < it.row_end; }
    __device__ __forceinline__ int seen(const Item& it, int row) const {
        return live(it, row) ? row_seen(p, it, it.row0 + row) : it.keys;
    }
    __device__ __forceinline__ const T* q_row(const Item& it, int row) const {
        return static_cast<const T*>(p.q) + row_off(p, it.kvh, it.row0 + row);
    }
    struct Rows {                   // lane i looks up row i's page
        const PagesDev& pg;
        const PrefixParams& p;
        const T* pool;
        int slot, a, shift, lane;
        size_t mine;
        __device__ __forceinline__ Rows(const PrefixWide& w, const Item& it, bool is_v) : pg(w.pg), p(w.p) {
            pool = static_cast<const T*>(is_v ? p.vp : p.kp) + (size_t)it.kvh * pg.page * kServeDim;
            slot = it.slot;
            a = it.a;
            shift = __ffs(pg.page) - 1;
            lane = threadIdx.x & 31;
            mine = 0;
        }
        __device__ __forceinline__ void tile(int key, int n) {
            const int k = key + 8 * lane;
            if (lane < 8 && k < n)
                mine = (size_t)page_of(pg, p, slot, (a + k) >> shift) * p.page_stride +
                       (size_t)(((a + k) & (pg.page - 1)) * kServeDim);
            __syncwarp();
        }
        __device__ __forceinline__ const T* row(int i) const {
            return pool + __shfl_sync(0xffffffffu, (unsigned long long)mine, i);
        }
    };
    __device__ __forceinline__ float scale(float) const { return 1.f; }
    __device__ __forceinline__ WideOut out(const Item& it, int row) const {
        const int parts = p.plan.sp + p.plan.cm;
        return WideOut{p.part_o + part_at(p, it, it.row0 + row) * kServeDim, (size_t)parts * kServeDim,
                       it.row_end - (it.row0 + row)};
    }
    __device__ __forceinline__ void finish(const Item& it, int row, float m, float l) const {
        p.part_ml[part_at(p, it, it.row0 + row)] = make_float2(m * kServeScale, l);
    }
    __device__ __forceinline__ const T* value(const Item& it, int key) const { return value_row<T>(pg, p, it, key); }
};

template <class KV>
__global__ void __launch_bounds__(kWdThreads, 1)
attn_prefix_wide_kernel(const __grid_constant__ PagesDev pg, const __grid_constant__ PrefixParams p) {
    pdl_trigger();
    attn_wide_core(PrefixWide<KV>{pg, p});
}

// ---------------------------------------------------------------------------
// the join: one warp per row, a lane four dimensions
// ---------------------------------------------------------------------------
template <class O>
__global__ void __launch_bounds__(256)
attn_prefix_join_kernel(const __grid_constant__ PagesDev pg, const __grid_constant__ PrefixParams p) {
    const int lane = threadIdx.x & 31;
    const long long x = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int rows = p.n * p.n_q * p.group;
    if (x >= (long long)rows * p.n_kv) {
        pdl_wait();                 // (this grid must not end before the parts' does)
        return;
    }
    const int kvh = (int)(x / rows), r = (int)(x % rows), b = r / (p.n_q * p.group);
    int slot;
    const int len = seq_len(pg, p, b, &slot);
    if (len < 0) {
        pdl_wait();
        if (lane == 0) raise(p.status, SLLM_CUDA_ERR_ARG);
        return;
    }
    const int parts = p.plan.sp + own_chunks(p, own_tiles(p, len));
    pdl_wait();
    const size_t at = (size_t)x * (p.plan.sp + p.plan.cm);
    const float2* ml = p.part_ml + at;
    const float* po = p.part_o + at * kServeDim + 4 * lane;
    float M = -INFINITY;
    for (int i = lane; i < parts; i += 32) M = fmaxf(M, ml[i].x);
    M = warp_max(M);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < parts; i0 += 32) {
        float f = 0.f, part_l = 0.f;
        if (i0 + lane < parts) {
            const float2 v = ml[i0 + lane];
            f = v.x == -INFINITY ? 0.f : expf(v.x - M);     // a part whose rows saw nothing adds nothing
            part_l = v.x == -INFINITY ? 0.f : f * v.y;
        }
        #pragma unroll
        for (int y = 16; y > 0; y >>= 1) part_l += __shfl_xor_sync(0xffffffffu, part_l, y);
        l += part_l;
        // eight parts' outputs in flight; past the last, its own again with weight 0
        const int n = min(32, parts - i0);
        for (int i = 0; i < n; i += 8) {
            float4 v[8];
            #pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = __ldcg(reinterpret_cast<const float4*>(po + (size_t)(i0 + min(i + e, n - 1)) * kServeDim));
            #pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float g = __shfl_sync(0xffffffffu, f, (i + e) & 31);
                if (i + e < n) {        // (a part too small to count still brings its infinities)
                    o.x = fmaf(g, v[e].x, o.x);
                    o.y = fmaf(g, v[e].y, o.y);
                    o.z = fmaf(g, v[e].z, o.z);
                    o.w = fmaf(g, v[e].w, o.w);
                }
            }
        }
    }
    const float inv = M == -INFINITY && l == 0.f ? 0.f : __fdiv_rn(1.f, l);
    st4(static_cast<O*>(p.out) + row_off(p, kvh, r) + 4 * lane, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Rows: whole tokens per row tile where TMA gathers them. Splits of the prefix:
// with an item of its own keys for each sequence besides, all of it in one
// round of the SMs where that makes splits of at most twelve key tiles, or of
// at most eight where the sequences' items alone are more than a round. Longer:
// the number, of those that make up to 32 tiles a split, that ends first on
// the SMs when a split costs three tiles' time for its start and its parts
// (all SMs write their parts at about one time, 128 KB each).
// One round or that number, f16, 32 heads of 8: 4 sequences, prefix 4096 (three
// tiles a split) 16.7 and 21.6 us, 16384 (nine) 26.2 and 33.2 us, 20480 (twelve)
// 30.5 and 38.8 us; 32 sequences (256 items of their own), prefix 4096 (four)
// 26.7 and 28.8 us, 12288 (eleven) 42.2 and 36.9 us.
// No more splits than eight rounds of the SMs take (f32, with half the rows an
// item: sixteen), if a split has at most 32 tiles then: that bounds the
// workspace (work_parts). Shapes that would take more otherwise (one in 30 of
// those drawn at random), f16, 8 query tokens, with the limit and without: 107
// sequences, prefix 47872, 32 heads of 8 (12 and 13 splits) 645 and 653 us; 203,
// 19328 (5 and 7) 519 and 543 us; 59, 35072, 64 heads of 8 (9 and 11) 517 and 508 us.
// A sequence's own keys: chunks of as many tiles, at least two; no more than
// two items per SM over all sequences, and no more than 64 chunks.
int most_rounds(int per) { return per == 2 ? 8 : 16; }
Plan make_plan(const sllm_cuda_kv_pages& p, int n, int n_q, int n_head, int prefix, int sms) {
    const int group = n_head / p.n_head_kv, rows = n * n_q * group;
    const bool mma = p.kv_type == SLLM_CUDA_KV_F16 && group <= kAtRows;
    Plan pl{};
    pl.key_tile = mma ? kAtKeys : kWdKeys;
    pl.rt = mma ? kAtRows / group * group : kAtRows;
    pl.per = mma ? 2 : 1;
    auto items = [&](int r) { return (r + pl.rt * pl.per - 1) / (pl.rt * pl.per); };
    pl.ri_all = items(rows);
    pl.ri_seq = items(n_q * group);
    pl.ptiles = (prefix + pl.key_tile - 1) / pl.key_tile;
    const long long base = (long long)p.n_head_kv * pl.ri_all, own = (long long)n * p.n_head_kv * pl.ri_seq;
    const long long room = sms - own > sms / 2 ? sms - own : sms / 2;
    const long long one = (base * pl.ptiles + room - 1) / room;        // tiles a split in one round
    if (one <= (own <= sms ? 12 : 8)) {
        pl.ct = one < 1 ? 1 : (int)one;
        pl.sp = (pl.ptiles + pl.ct - 1) / pl.ct;
    } else {
        long long best = 0;
        const int least = (pl.ptiles + 31) / 32;
        const long long most = std::max<long long>((long long)most_rounds(pl.per) * sms / base, least);
        for (int s = least; s <= pl.ptiles && s <= most && (s <= 32 || pl.sp == 0); ++s) {
            const long long tiles = (pl.ptiles + s - 1) / s, cost = ((base * s + sms - 1) / sms) * (tiles + 3);
            if (pl.sp == 0 || cost < best) {
                best = cost;
                pl.sp = s;
                pl.ct = (int)tiles;
            }
        }
    }
    if (pl.ct < 2) pl.ct = 2;
    const long long cm = own > 0 ? (2LL * sms + own - 1) / own : 1;
    pl.cm = (int)(cm < 1 ? 1 : cm > 64 ? 64 : cm);
    return pl;
}

size_t part_count(const Plan& pl, int n, int n_q, int n_head) {
    return (size_t)n * n_q * n_head * (pl.sp + pl.cm);
}

// part_count of this call and of every one with no more sequences, query tokens
// and prefix, by a form that rises with each (the splits themselves do not: a
// second tile in a split halves their number). R rows, `item` of a kv head in an
// item at most. Splits of the prefix: its tiles at most; in one round of the SMs
// room / base and one more, so R + sms * item; else as many as tiles of 32, or
// most_rounds' worth. Chunks: 64, or 2 sms / own and one more.
size_t work_parts(const Plan& pl, int n, int n_q, int n_head, int group, int sms) {
    const size_t R = (size_t)n * n_q * n_head, item = (size_t)pl.rt * pl.per;
    const size_t rows = std::min(item, (size_t)n * n_q * group), own = std::min(item, (size_t)n_q * group);
    const size_t splits = std::min(R * pl.ptiles, std::max({R * ((pl.ptiles + 31) / 32), R + sms * rows, most_rounds(pl.per) * sms * rows}));
    return splits + std::min(64 * R, R + 2 * sms * own);
}

size_t part_bytes(size_t parts) { return parts * (kServeDim * sizeof(float) + sizeof(float2)) + 16; }

bool encode_q(CUtensorMap* tm, const void* base, int tokens, int n_kv, int group) {
    PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
    if (enc == nullptr) return false;
    const cuuint64_t row = kServeDim * 2;
    const cuuint64_t dims[4] = {(cuuint64_t)kServeDim, (cuuint64_t)group, (cuuint64_t)n_kv, (cuuint64_t)tokens};
    const cuuint64_t strides[3] = {row, row * group, row * group * n_kv};
    const cuuint32_t box[4] = {64, (cuuint32_t)group, 1, (cuuint32_t)(kAtRows / group)};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    return enc(tm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// one layer of a pool: a page's rows of one kv head per box
bool encode_pool(CUtensorMap* tm, const void* base, const sllm_cuda_kv_pages& p) {
    PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
    if (enc == nullptr) return false;
    const cuuint64_t row = kServeDim * 2, head = row * p.page_size, page = head * p.n_head_kv * p.n_layer;
    const cuuint64_t dims[4] = {(cuuint64_t)kServeDim, (cuuint64_t)p.page_size, (cuuint64_t)p.n_head_kv,
                                (cuuint64_t)p.n_pages};
    const cuuint64_t strides[3] = {row, head, page};
    const cuuint32_t box[4] = {64, (cuuint32_t)p.page_size, 1, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    return enc(tm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

long long item_numbers(const PrefixParams& p) {
    return (long long)p.n_kv * p.plan.ri_all * p.plan.sp + (long long)p.n * p.plan.cm * p.n_kv * p.plan.ri_seq;
}

cudaError_t launch_mma(const sllm_cuda_kv_pages& pages, const PagesDev& pg, const PrefixParams& p, int sms, cudaStream_t st) {
    CUtensorMap tq, tk, tv;
    if (!encode_q(&tq, p.q, p.n * p.n_q, p.n_kv, p.group) || !encode_pool(&tk, p.kp, pages) ||
        !encode_pool(&tv, p.vp, pages))
        return cudaErrorInvalidValue;
    const cudaError_t e = allow_smem<attn_prefix_mma_kernel>(kAtSmem);
    if (e != cudaSuccess) return e;
    const long long items = item_numbers(p);
    if (p.plan.next != nullptr) {
        const cudaError_t z = cudaMemsetAsync(p.plan.next, 0, sizeof(int), st);
        if (z != cudaSuccess) return z;
    }
    return launch(attn_prefix_mma_kernel, dim3((unsigned)(items < sms ? items : sms)), dim3(kAtThreads), kAtSmem, st, false,
                  tq, tk, tv, pg, p);
}

template <class T>
cudaError_t launch_32(const PagesDev& pg, const PrefixParams& p, cudaStream_t st) {
    const cudaError_t e = allow_smem<attn_prefix_wide_kernel<T>>(kWdSmem);
    return e != cudaSuccess ? e
                            : launch(attn_prefix_wide_kernel<T>, dim3((unsigned)item_numbers(p)), dim3(kWdThreads), kWdSmem,
                                     st, false, pg, p);
}

int check_shape(const sllm_cuda_kv_pages* p, int n, int n_q, int n_head, int prefix, const char* who) {
    const int rc = check_pages(p, who, false);
    if (rc != SLLM_CUDA_OK) return rc;
    if (n < 0 || n > 4096 || n_q < 1 || n_q > 16 || n_head < 1 || n_head > 1024 || n_head % p->n_head_kv != 0 ||
        prefix < 0 || prefix % p->page_size != 0 || prefix / p->page_size > p->table_width)
        return fail(SLLM_CUDA_ERR_ARG, "%s: %d sequences, %d query tokens (1 to 16), %d heads over %d, prefix of %d "
                    "(whole pages of %d)", who, n, n_q, n_head, p->n_head_kv, prefix, p->page_size);
    return SLLM_CUDA_OK;
}

}  // namespace
}  // namespace sllm

using namespace sllm;

int sllm::take_prefix_error() { return take_attn_error(); }

extern "C" size_t sllm_cuda_attn_prefix_work_bytes(const sllm_cuda_kv_pages* p, int32_t n, int32_t n_q, int32_t n_head,
                                                   int32_t prefix_len) {
    if (check_shape(p, n, n_q, n_head, prefix_len, "attn_prefix_work_bytes") != SLLM_CUDA_OK) return 0;
    const int sms = current_sms();
    return part_bytes(work_parts(make_plan(*p, n, n_q, n_head, prefix_len, sms), n, n_q, n_head, n_head / p->n_head_kv, sms));
}

extern "C" int sllm_cuda_attn_prefix(const sllm_cuda_kv_pages* p, int32_t layer, const void* q, const int32_t* slots,
                                     int32_t n, int32_t n_q, int32_t n_head, int32_t prefix_len, void* out,
                                     int32_t out_type, void* work, size_t work_bytes, int32_t* status,
                                     void* stream) {
    int rc = check_shape(p, n, n_q, n_head, prefix_len, "attn_prefix");
    if (rc != SLLM_CUDA_OK) return rc;
    if (q == nullptr || slots == nullptr || out == nullptr || work == nullptr || layer < 0 || layer >= p->n_layer)
        return fail(SLLM_CUDA_ERR_ARG, "attn_prefix: a NULL array, or layer %d of %d", layer, p->n_layer);
    if ((out_type != SLLM_CUDA_KV_F32 && out_type != SLLM_CUDA_KV_F16) ||
        (p->kv_type == SLLM_CUDA_KV_F32 && out_type == SLLM_CUDA_KV_F16))
        return fail(SLLM_CUDA_ERR_ARG, "attn_prefix: output type %d (f32, or f16 from an f16 cache)", out_type);
    const int sms = current_sms();
    const Plan plan = make_plan(*p, n, n_q, n_head, prefix_len, sms);
    const size_t parts = part_count(plan, n, n_q, n_head);
    if (!aligned16(q) || !aligned16(out) || !aligned16(work) || work_bytes < part_bytes(parts))
        return fail(SLLM_CUDA_ERR_ARG, "attn_prefix: workspace of %zu bytes (%zu needed), arrays 16-byte aligned",
                    work_bytes, part_bytes(parts));
    const void* ptr[] = {p->k, p->v, p->tables, p->lens, q, slots, out, work, status};
    const char* name[] = {"k", "v", "tables", "lens", "q", "slots", "out", "work", "status"};
    for (int i = 0; i < 9; ++i)
        if (ptr[i] != nullptr && (rc = need_device(ptr[i], "attn_prefix", name[i])) != SLLM_CUDA_OK) return rc;
    if (n == 0) return SLLM_CUDA_OK;
    const size_t layer_elts = (size_t)p->n_head_kv * p->page_size * kServeDim;
    const size_t off = (size_t)layer * layer_elts * kv_elt_bytes(p->kv_type);
    PrefixParams a{};
    a.q = q; a.out = out;
    a.kp = static_cast<const uint8_t*>(p->k) + off;
    a.vp = static_cast<const uint8_t*>(p->v) + off;
    a.page_stride = (size_t)p->n_layer * layer_elts;
    a.slots = slots;
    a.n = n; a.n_q = n_q; a.n_head = n_head; a.n_kv = p->n_head_kv; a.group = n_head / p->n_head_kv;
    a.prefix = prefix_len;
    a.status = status;
    a.wait = attn_wait_limit();
    a.plan = plan;
    a.part_o = static_cast<float*>(work);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + parts * kServeDim);
    // many items per SM: each CTA takes the next one when it is free, for one
    // more launch, to clear the counter; few: they are dealt. Taken and dealt,
    // f16, 32 heads of 8, own lengths of 1 to 4096 at random: 16 sequences (256
    // items) 62 and 57 us, 64 (512) 149 and 156 us, 192 (1536) 336 and 375 us;
    // lengths up to 1024, so that the items are short: 192 behind a prefix of
    // 2048 149 and 130 us. (The lengths are the device's, so the rule is on the
    // number alone.)
    if (item_numbers(a) > 3LL * sms)
        a.plan.next = reinterpret_cast<int*>(a.part_ml + parts);
    if (item_numbers(a) > 0x3fffffffLL) return fail(SLLM_CUDA_ERR_TOO_LARGE, "attn_prefix: %d sequences", n);
    const PagesDev pg = pages_dev(*p);
    const cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = p->kv_type == SLLM_CUDA_KV_F32 ? launch_32<float>(pg, a, st)
                          : a.group > kAtRows            ? launch_32<__half>(pg, a, st)
                                                         : launch_mma(*p, pg, a, sms, st);
    CK(e, "attn_prefix launch");
    const dim3 grid((unsigned)(((long long)n * n_q * n_head + 7) / 8));
    CK(out_type == SLLM_CUDA_KV_F32 ? launch(attn_prefix_join_kernel<float>, grid, dim3(256), 0, st, true, pg, a)
                                    : launch(attn_prefix_join_kernel<__half>, grid, dim3(256), 0, st, true, pg, a),
       "attn_prefix join");
    count_launches(2);
    return SLLM_CUDA_OK;
}
