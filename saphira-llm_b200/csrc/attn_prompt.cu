// attn_prompt.cu -- causal attention over packed whole prompts, grouped heads.
//
// Sequence s holds tokens cu[s] .. cu[s + 1] - 1 of the packed arrays; token i
// of a sequence sees its tokens 0 .. i.
//
// f16: attn_prompt_mma_kernel over attn_mma.cuh, one CTA per SM that walks items
// dealt longest first. f32: attn_prompt_wide_kernel over attn_wide.cuh, one CTA
// per item, the longest launched first where sequences are few. What bounds the two stands there.
// Measured: prompts of 8192, 1, 300, 1021, 0, 2048, 513 and 64 tokens together,
// 64 heads of 8, f16: 0.95 to 1.03 ms (1250 to 1158 TFLOP/s); of 320, 1, 777 and
// 256, 20 heads of 5, f32: 42.4 us.

#include "attn_mma.cuh"
#include "attn_wide.cuh"

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
    WaitLimit wait;
    int32_t* status;
};

// Offsets that descend or leave the arrays are reported; one warp of each CTA, a
// share each.
__device__ __forceinline__ void check_offsets(const PromptParams& p) {
    if (p.status == nullptr) return;
    bool bad = false;
    for (long long s = 32LL * blockIdx.x + (threadIdx.x & 31); s <= p.n_seq; s += 32LL * gridDim.x) {
        const int at = p.cu[s];
        bad = bad || at < 0 || at > p.n_tokens || (s < p.n_seq && p.cu[s + 1] < at);
    }
    if (bad) raise(p.status, SLLM_CUDA_ERR_ARG);
}

// sequence s; its bounds are clamped to the arrays, so a wrong cu stays inside
__device__ __forceinline__ int seq_len(const PromptParams& p, int s, int* start) {
    *start = min(max(p.cu[s], 0), p.n_tokens);
    return min(max(p.cu[s + 1], *start), p.n_tokens) - *start;
}

// the place of the n-th bit (from 0) that is set, by a whole warp; it is there
__device__ __forceinline__ int nth_bit(unsigned bits, int n) {
    const unsigned lane = threadIdx.x & 31, below = bits & ((1u << lane) - 1u);
    return __ffs(__ballot_sync(0xffffffffu, (bits >> lane & 1u) != 0 && __popc(below) == n)) - 1;
}

// The call's tiles of R rows in descending order of their position in their
// sequence (the later, the more keys they see): the longest work first. One
// warp; what it asks for only ever rises, so all of a CTA's searches together
// walk the sequences once per position. (With a search from the start for each
// item 256 prompts of 100 to 200 tokens, 20 heads, took 270 us instead of 198,
// 2048 of 32 to 64 tokens 6.0 ms instead of 1.05.) Positions that the same
// sequences reach are passed over after one walk: 65535 prompts of 8 tokens and
// one of 131072 take 6.6 ms; with a walk for each of its tiles, behind which the
// other warps wait, 256 ms.
template <int R>
struct LongFirst {
    int pos;                        // the position
    int before;                     // tiles at later positions, and at this one in sequences below s0
    int s0;
    int at, below;                  // `before` at this walk's start; the most tiles of sequences that end before pos (by lanes)
    int2 cur, nxt;                  // the offsets of sequences s0 .. s0 + 31, and of the 32 that are looked at after them
    __device__ __forceinline__ int2 offsets(const PromptParams& p, int s) const {
        s = min(s + (int)(threadIdx.x & 31), p.n_seq - 1);
        return make_int2(p.cu[s], p.cu[s + 1]);
    }
    __device__ __forceinline__ int after(const PromptParams& p, int s) const { return s + 32 < p.n_seq ? s + 32 : 0; }
    __device__ __forceinline__ void start(const PromptParams& p) {
        int most = 0, a;
        before = s0 = pos = at = below = 0;
        if (p.n_seq == 1) return;
        for (int s = threadIdx.x & 31; s < p.n_seq; s += 32) most = max(most, (seq_len(p, s, &a) + R - 1) / R);
        pos = __reduce_max_sync(0xffffffffu, most) - 1;
        cur = offsets(p, 0);
        nxt = offsets(p, after(p, 0));
    }
    // tile x; false: there is none, nor any after it
    __device__ __forceinline__ bool find(const PromptParams& p, int x, int* start, int* len, int* tile) {
        const int lane = threadIdx.x & 31;
        if (p.n_seq == 1) {
            *len = seq_len(p, 0, start);
            *tile = (*len + R - 1) / R - 1 - x;
            return *tile >= 0;
        }
        if (x >= p.n_tokens / R + p.n_seq) return false;        // ascending offsets have no more
        while (pos >= 0) {
            const int a = min(max(cur.x, 0), p.n_tokens);
            const int n = s0 + lane < p.n_seq ? min(max(cur.y, a), p.n_tokens) - a : 0, tiles = (n + R - 1) / R;
            const unsigned has = __ballot_sync(0xffffffffu, tiles > pos);
            const int c = __popc(has), r = x - before;
            if (r < c) {
                const int l = nth_bit(has, r);
                *start = __shfl_sync(0xffffffffu, a, l);
                *len = __shfl_sync(0xffffffffu, n, l);
                *tile = pos;
                return true;
            }
            before += c;
            if (tiles <= pos) below = max(below, tiles);
            s0 = after(p, s0);
            cur = nxt;
            if (p.n_seq > 32) nxt = offsets(p, after(p, s0));
            if (s0 != 0) continue;
            // (never 0, unless somebody writes the offsets meanwhile; the search ends all the same)
            const int each = max(before - at, 1), same = pos - __reduce_max_sync(0xffffffffu, below);
            const int skip = min(same, (x - before) / each);
            pos -= skip + 1;
            before += skip * each;
            at = before;
            below = 0;
        }
        return false;
    }
};

// ... for a single search among up to 32 sequences: F(t) = tiles at positions
// >= t; a binary search for the position, then the sequence
template <int R>
__device__ __forceinline__ bool find_long_first(const PromptParams& p, int x, int* start, int* len, int* tile) {
    const int lane = threadIdx.x & 31;
    int a = 0, n = 0;
    if (lane < p.n_seq) n = seq_len(p, lane, &a);
    const int tiles = (n + R - 1) / R;
    if (__reduce_add_sync(0xffffffffu, tiles) <= x) return false;
    int lo = 0, hi = __reduce_max_sync(0xffffffffu, tiles), f_hi = 0;      // F(lo) > x >= F(hi) = f_hi
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2, f = __reduce_add_sync(0xffffffffu, max(tiles - mid, 0));
        if (f > x) {
            lo = mid;
        } else {
            hi = mid;
            f_hi = f;
        }
    }
    const int l = nth_bit(__ballot_sync(0xffffffffu, tiles > lo), x - f_hi);
    *start = __shfl_sync(0xffffffffu, a, l);
    *len = __shfl_sync(0xffffffffu, n, l);
    *tile = lo;
    return true;
}

// Tile x of R rows in the order of the sequences: sequence s has the numbers
// from cu[s] / R + s on, of which the last may be nobody's (false). One warp,
// 32 sequences a probe: for a single search among many.
template <int R>
__device__ __forceinline__ bool find_in_order(const PromptParams& p, int x, int* start, int* len, int* tile) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = p.n_seq, first = 0;
    for (int step = hi; step > 1;) {
        step = (hi - lo + 31) / 32;
        const int s = lo + lane * step;
        first = s < hi ? min(max(p.cu[s], 0), p.n_tokens) / R + s : 0x7fffffff;
        const unsigned at = __ballot_sync(0xffffffffu, first <= x);
        if ((at & 1u) == 0) return false;
        lo += (31 - __clz(at)) * step;
        hi = min(hi, lo + step);
    }
    *len = seq_len(p, lo, start);
    *tile = x - (*start / R + lo);
    return *tile >= 0 && *tile < (*len + R - 1) / R;
}

// ---------------------------------------------------------------------------
// The f16 kernel: attn_mma.cuh's core over items of 256 query rows of one
// head, from the start of the sequence to the diagonal.
// ---------------------------------------------------------------------------
constexpr int kPmRows = 2 * kAtRows;

template <class O>
struct PromptWork {
    struct Item {
        int start, len, tile, head;             // tile < 0: no more items
        __device__ bool last() const { return tile < 0; }
    };
    const PromptParams& p;
    const CUtensorMap &tm_q, &tm_k, &tm_v;

    struct Finder {
        LongFirst<kPmRows> order;
        __device__ __forceinline__ void start(const PromptWork& w) { order.start(w.p); }
        __device__ __forceinline__ long long number(const PromptWork&, int r) { return dealt_number(r); }
        __device__ __forceinline__ bool item(const PromptWork& w, long long x, Item* it) {
            *it = Item{0, 0, -1, (int)(x % w.p.n_head)};
            if (!order.find(w.p, (int)(x / w.p.n_head), &it->start, &it->len, &it->tile)) it->tile = -1;
            return true;
        }
    };
    __device__ __forceinline__ WaitLimit wait_limit() const { return p.wait; }
    __device__ __forceinline__ void check() const { check_offsets(p); }
    __device__ __forceinline__ void gave_up() const { raise(p.status, SLLM_CUDA_ERR_TIMEOUT); }
    // key tiles of row tile t: up to its diagonal, or the sequence's end
    __device__ __forceinline__ int tiles(const Item& it, int t) const {
        if (it.tile * kPmRows + kAtRows * t >= it.len) return 0;
        return min(2 * it.tile + t, (it.len - 1) / kAtKeys) + 1;
    }
    __device__ __forceinline__ int keys(const Item& it) const { return it.len; }
    __device__ __forceinline__ int seen(const Item& it, int t, int row) const {
        return min(it.tile * kPmRows + kAtRows * t + row + 1, it.len);
    }
    __device__ __forceinline__ bool live(const Item& it, int t, int row) const {
        return it.tile * kPmRows + kAtRows * t + row < it.len;
    }
    struct Loader {
        __device__ __forceinline__ void start(const PromptWork&, const Item&, int) {}
        __device__ __forceinline__ void q(const PromptWork& w, const Item& it, int t, uint8_t* dst, uint64_t* bar, int lane) {
            load(&w.tm_q, it.head, it.start + it.tile * kPmRows + kAtRows * t, dst, bar, lane);
        }
        __device__ __forceinline__ void kv(const PromptWork& w, const Item& it, int j, bool v, uint8_t* dst, uint64_t* bar,
                                           int lane) {
            load(v ? &w.tm_v : &w.tm_k, it.head / w.p.group, it.start + j * kAtKeys, dst, bar, lane);
        }
        __device__ __forceinline__ void load(const CUtensorMap* tm, int head, int token, uint8_t* dst, uint64_t* bar,
                                             int lane) {
            if (lane == 0) {
                mbar_expect_tx(bar, kAtTile);
                tma_load_3d(dst, tm, 0, head, token, bar);
                tma_load_3d(dst + kAtHalf, tm, 64, head, token, bar);
            }
        }
    };
    __device__ __forceinline__ void store(const Item& it, int t, int row, uint32_t o_tm, float, float l, uint8_t* stage) const {
        const int x0 = it.tile * kPmRows + kAtRows * t + (row & ~31);       // the warp's first row
        store_rows(o_tm, 1.f / l, stage, static_cast<O*>(p.out) + (size_t)(it.start + x0) * p.os + (size_t)it.head * kServeDim,
                   p.os, it.len - x0);
    }
    __device__ __forceinline__ void odd(const Item& it, int t, int row) const {
        const int lane = threadIdx.x & 31, x0 = it.tile * kPmRows + kAtRows * t + row;
        const __half* const v = static_cast<const __half*>(p.v) + (size_t)it.start * p.vs +
                                (size_t)(it.head / p.group) * kServeDim + 4 * lane;
        O* const out = static_cast<O*>(p.out) + (size_t)(it.start + x0) * p.os + (size_t)it.head * kServeDim + 4 * lane;
        add_odd<4>(seen(it, 0, 0), min(x0 + 32, it.len), min(32, it.len - x0),
                   [&](int key) { return v + (size_t)key * p.vs; }, [&](int r) { return x0 + r + 1; },
                   [&](int r) { return out + (size_t)r * p.os; });
    }
};

template <class O>
__global__ void __launch_bounds__(kAtThreads, 1)
attn_prompt_mma_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PromptParams p) {
    attn_core(PromptWork<O>{p, tm_q, tm_k, tm_v});
}

// ---------------------------------------------------------------------------
// The f32 kernel: attn_wide.cuh's core, 128 query rows a CTA.
// ---------------------------------------------------------------------------
struct PromptWide {
    using T = float;
    struct Item {
        int start, len, tile, head;
        __device__ bool last() const { return tile < 0; }
    };
    const PromptParams& p;

    __device__ __forceinline__ WaitLimit wait_limit() const { return p.wait; }
    __device__ __forceinline__ void check() const { check_offsets(p); }
    __device__ __forceinline__ void gave_up() const { raise(p.status, SLLM_CUDA_ERR_TIMEOUT); }
    // longest first; of more than 32 sequences in their order, which takes no
    // walk over all of them and leaves each SM many items to even out (2048
    // prompts of 32 to 64 tokens, 20 heads: 4.9 ms longest first, 2.9 ms in order;
    // 256 of 100 to 200: 940 us and 843 us)
    __device__ __forceinline__ bool find(long long x, Item* it) const {
        const int t = (int)(x / p.n_head);
        it->head = (int)(x % p.n_head);
        return p.n_seq > 32 ? find_in_order<kAtRows>(p, t, &it->start, &it->len, &it->tile)
                            : find_long_first<kAtRows>(p, t, &it->start, &it->len, &it->tile);
    }
    __device__ __forceinline__ int keys(const Item& it) const { return min((it.tile + 1) * kAtRows, it.len); }
    __device__ __forceinline__ int seen(const Item& it, int row) const { return min(it.tile * kAtRows + row + 1, it.len); }
    __device__ __forceinline__ bool live(const Item& it, int row) const { return it.tile * kAtRows + row < it.len; }
    __device__ __forceinline__ const float* q_row(const Item& it, int row) const {
        return static_cast<const float*>(p.q) + (size_t)(it.start + it.tile * kAtRows + row) * p.qs +
               (size_t)it.head * kServeDim;
    }
    struct Rows {
        const float* base;
        size_t stride;
        __device__ __forceinline__ Rows(const PromptWide& w, const Item& it, bool is_v) {
            stride = is_v ? w.p.vs : w.p.ks;
            base = static_cast<const float*>(is_v ? w.p.v : w.p.k) + (size_t)it.start * stride +
                   (size_t)(it.head / w.p.group) * kServeDim;
            at = base;
        }
        const float* at;
        __device__ __forceinline__ void tile(int key, int) { at = base + (size_t)key * stride; }
        __device__ __forceinline__ const float* row(int i) const { return at + (size_t)(8 * i) * stride; }
    };
    __device__ __forceinline__ float scale(float l) const { return 1.f / l; }
    __device__ __forceinline__ WideOut out(const Item& it, int row) const {
        const int x0 = it.tile * kAtRows + row;
        return WideOut{static_cast<float*>(p.out) + (size_t)(it.start + x0) * p.os + (size_t)it.head * kServeDim, p.os,
                       it.len - x0};
    }
    __device__ __forceinline__ void finish(const Item&, int, float, float) const {}
    // value row `key`
    __device__ __forceinline__ const float* value(const Item& it, int key) const {
        return static_cast<const float*>(p.v) + (size_t)(it.start + key) * p.vs + (size_t)(it.head / p.group) * kServeDim;
    }
};

__global__ void __launch_bounds__(kWdThreads, 1) attn_prompt_wide_kernel(const __grid_constant__ PromptParams p) {
    attn_wide_core(PromptWide{p});
}

cudaError_t launch_wide(const PromptParams& p, cudaStream_t st) {
    const cudaError_t e = allow_smem<attn_prompt_wide_kernel>(kWdSmem);
    if (e != cudaSuccess) return e;
    // every sequence may end inside a tile
    const long long tiles = p.n_tokens / kAtRows + (long long)p.n_seq;
    return launch(attn_prompt_wide_kernel, dim3((unsigned)(tiles * p.n_head)), dim3(kWdThreads), kWdSmem, st, false, p);
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
    const cudaError_t e = allow_smem<attn_prompt_mma_kernel<O>>(kAtSmem);
    if (e != cudaSuccess) return e;
    // at most this many items: every sequence may end inside one
    const long long items = (p.n_tokens / kPmRows + (long long)p.n_seq) * p.n_head;
    const int sms = current_sms();
    return launch(attn_prompt_mma_kernel<O>, dim3((unsigned)(items < sms ? items : sms)), dim3(kAtThreads), kAtSmem, st,
                  false, tq, tk, tv, p);
}

}  // namespace
}  // namespace sllm

using namespace sllm;

int sllm::take_prompt_error() { return take_attn_error(); }

extern "C" int sllm_cuda_attn_prompt(const void* q, size_t q_stride, const void* k, size_t k_stride, const void* v,
                                     size_t v_stride, int32_t type, const int32_t* cu_seqlens, int32_t n_seq,
                                     int32_t n_tokens, int32_t n_head, int32_t n_head_kv, void* out,
                                     size_t out_stride, int32_t out_type, void* stream) {
    return sllm_cuda_attn_prompt_checked(q, q_stride, k, k_stride, v, v_stride, type, cu_seqlens, n_seq, n_tokens, n_head,
                                         n_head_kv, out, out_stride, out_type, nullptr, stream);
}

extern "C" int sllm_cuda_attn_prompt_checked(const void* q, size_t q_stride, const void* k, size_t k_stride, const void* v,
                                             size_t v_stride, int32_t type, const int32_t* cu_seqlens, int32_t n_seq,
                                             int32_t n_tokens, int32_t n_head, int32_t n_head_kv, void* out,
                                             size_t out_stride, int32_t out_type, int32_t* status, void* stream) {
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
    const void* ptr[] = {q, k, v, cu_seqlens, out, status};
    const char* name[] = {"q", "k", "v", "cu_seqlens", "out", "status"};
    for (int i = 0; i < 6; ++i) {
        if (ptr[i] == nullptr) continue;
        const int rc = need_device(ptr[i], "attn_prompt", name[i]);
        if (rc != SLLM_CUDA_OK) return rc;
    }
    if (n_seq == 0 || n_tokens == 0) return SLLM_CUDA_OK;
    PromptParams p{};
    p.q = q; p.k = k; p.v = v; p.out = out;
    p.qs = q_stride; p.ks = k_stride; p.vs = v_stride; p.os = out_stride;
    p.cu = cu_seqlens;
    p.wait = attn_wait_limit();
    p.status = status;
    p.n_seq = n_seq; p.n_tokens = n_tokens; p.n_head = n_head; p.group = n_head / n_head_kv;
    const cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = type == SLLM_CUDA_KV_F32 ? launch_wide(p, st)
                          : out_type == SLLM_CUDA_KV_F32 ? launch_mma<float>(p, st)
                                                         : launch_mma<__half>(p, st);
    CK(e, "attn_prompt launch");
    count_launches(1);
    return SLLM_CUDA_OK;
}
