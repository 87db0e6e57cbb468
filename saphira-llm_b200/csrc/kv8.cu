// kv8.cu -- the 8-bit paged cache: the quantising store of new tokens, and
// reading them back.
//
// A block is 16 tokens of one head: 2048 codes c in [-127, 127] and one scale
// s; a value is c * s. With m the largest |value| stored in the block,
//     s = max(m / 127, 2^-100)   (0 while m = 0),    c = rint(x * (1 / s)).
// A token that needs a larger scale s' has the block's earlier codes follow:
// c' = rint(c * (s * (1 / s'))). Simulated on normal values stored one at a
// time that happens 2.4 times a block and leaves 1.04% rms error, against 0.77%
// of a block stored at once; a margin on the scale (1/16 to 1) gained 3% at
// best and cost 2 to 60% on values with heavier tails, so there is none.

#include "serve.cuh"

namespace sllm {
namespace {

constexpr int kK8Warps = 8;
constexpr int kK8Entries = 16;      // list entries of a CTA
constexpr float kK8Least = 0x1p-100f;

struct Append8Params {
    const int32_t* slot;
    const int32_t* pos;
    const float* q;
    const float* k;
    const float* v;
    size_t qs, ks, vs;              // floats from a token to the next
    const float* cs;
    const float* sn;
    void* qo;
    void* ko;
    void* vo;
    int8_t* kp;                     // the layer's slice of page 0
    int8_t* vp;
    float* ksc;                     // its scales
    float* vsc;
    size_t page_stride, scale_stride;       // codes, scales from a page to the next
    int n_tokens, n_head, n_kv, n_ctx;
    int kv_ctas, kv_rows;           // CTAs of k and v (those of q behind them), and the heads of k and v that one has
    int32_t* status;
};

struct RotPair {                    // elements 4l .. 4l + 3 of a row, and 64 + 4l ..
    float4 lo, hi;
};

__device__ __forceinline__ void rotate(RotPair& r, float4 c, float4 s) {
    const float4 x = r.lo, y = r.hi;
    r.lo.x = __fsub_rn(__fmul_rn(x.x, c.x), __fmul_rn(y.x, s.x));
    r.lo.y = __fsub_rn(__fmul_rn(x.y, c.y), __fmul_rn(y.y, s.y));
    r.lo.z = __fsub_rn(__fmul_rn(x.z, c.z), __fmul_rn(y.z, s.z));
    r.lo.w = __fsub_rn(__fmul_rn(x.w, c.w), __fmul_rn(y.w, s.w));
    r.hi.x = __fadd_rn(__fmul_rn(x.x, s.x), __fmul_rn(y.x, c.x));
    r.hi.y = __fadd_rn(__fmul_rn(x.y, s.y), __fmul_rn(y.y, c.y));
    r.hi.z = __fadd_rn(__fmul_rn(x.z, s.z), __fmul_rn(y.z, c.z));
    r.hi.w = __fadd_rn(__fmul_rn(x.w, s.w), __fmul_rn(y.w, c.w));
}

// the largest finite magnitude so far; odd: something was no finite number
__device__ __forceinline__ float most4(float m, float4 v, bool* odd) {
    const float a[4] = {fabsf(v.x), fabsf(v.y), fabsf(v.z), fabsf(v.w)};
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool fine = a[i] < INFINITY;
        *odd = *odd || !fine;
        m = fmaxf(m, fine ? a[i] : 0.f);
    }
    return m;
}

__device__ __forceinline__ int code_of(float x, float inv) {
    if (!(inv > 0.f) || x != x) return 0;                   // a block of zeros; no number
    return __float2int_rn(fminf(fmaxf(__fmul_rn(x, inv), -127.f), 127.f));
}

__device__ __forceinline__ uint32_t codes4(float4 v, float inv) {
    uint32_t u = 0;
    const float x[4] = {v.x, v.y, v.z, v.w};
    #pragma unroll
    for (int i = 0; i < 4; ++i) u |= (uint32_t)(code_of(x[i], inv) & 255) << (8 * i);
    return u;
}

// four codes again at another scale, f = old scale / new scale <= 1
__device__ __forceinline__ uint32_t recode4(uint32_t u, float f) {
    uint32_t r = 0;
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float c = (float)(int)(int8_t)(u >> (8 * i));
        r |= (uint32_t)(__float2int_rn(__fmul_rn(c, f)) & 255) << (8 * i);
    }
    return r;
}

// the page of a token, -1 where slot, position or page is wrong
__device__ __forceinline__ int page_at(const PagesDev& p, int slot, int pos) {
    if (slot < 0 || slot >= p.n_slots || pos < 0 || pos >= p.cap || pos >= p.lens[slot]) return -1;
    const int id = p.tables[(size_t)slot * p.width + pos / p.page];
    return id >= 0 && id < p.n_pages ? id : -1;
}

// ---------------------------------------------------------------------------
// append. Of the list's tokens those of one block are a run; a warp takes one
// run of one head of k or of v, all of its (up to 16) tokens in registers: lane
// l of a half-warp holds elements 4l .. and 64 + 4l .. of a token, the
// rotation's pairs. A CTA has 16 entries of the list and some heads, and its eight
// warps share the runs times heads: one or two runs in a prompt, 16 in a
// decode step. With one head a CTA a step of few tokens has one such pair a warp;
// with eight a long prompt has (one head a CTA left six warps of eight idle: 67 us
// for 4099 tokens of 8 heads). The pages are looked up once for all pairs, a lane
// per entry, behind the first pair's loads. The q rows are rotated by CTAs of
// their own, eight rows a warp.
// Bound: HBM for a prompt (4099 tokens of 64/8 heads, f16 outputs, 270 MB: 48 us, 5.6
// TB/s), else the chain of page id, values, old scale and codes, stores (16 tokens of
// 20/5 heads: 7 us).
// ---------------------------------------------------------------------------
struct Run {
    RotPair r[8];

    __device__ __forceinline__ void load(const Append8Params& a, int e0, int count, int h, bool is_v) {
        const int lane = threadIdx.x & 31, half = lane >> 4, l4 = 4 * (lane & 15);
        const float* const x = (is_v ? a.v : a.k) + h * kServeDim + l4;
        const size_t xs = is_v ? a.vs : a.ks;
        #pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int t = 2 * i + half;
            if (t < count) {
                const float* row = x + (size_t)(e0 + t) * xs;
                r[i].lo = __ldcs(reinterpret_cast<const float4*>(row));
                r[i].hi = __ldcs(reinterpret_cast<const float4*>(row + 64));
            }
        }
    }
};

// tokens e0 .. e0 + count - 1 into page `id`, their first position pos0
template <class O>
__device__ __forceinline__ void append_run(const PagesDev& p, const Append8Params& a, Run& run, int e0, int count, int id, int pos0,
                                           int h, bool is_v) {
    RotPair (&r)[8] = run.r;
    const int lane = threadIdx.x & 31, half = lane >> 4, l4 = 4 * (lane & 15);
    const int block = pos0 % p.page / kKvBlock, row0 = pos0 % kKvBlock;
    float* const sc = (is_v ? a.vsc : a.ksc) + (size_t)id * a.scale_stride + (size_t)h * (p.page / kKvBlock) + block;
    int8_t* const codes = (is_v ? a.vp : a.kp) + (size_t)id * a.page_stride + ((size_t)h * p.page + block * kKvBlock) * kServeDim;
    float old = row0 > 0 ? *sc : 0.f;
    if (!(old > 0.f && old < INFINITY)) old = 0.f;
    float m = 0.f;
    bool odd = false;
    O* const out = static_cast<O*>(is_v ? a.vo : a.ko);
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int t = 2 * i + half;
        if (t < count) {
            if (!is_v) {
                const int pos = a.pos[e0 + t];
                rotate(r[i], ld4(a.cs + (size_t)pos * 64 + l4), ld4(a.sn + (size_t)pos * 64 + l4));
            }
            m = most4(most4(m, r[i].lo, &odd), r[i].hi, &odd);
            if (out != nullptr) {
                O* o = out + ((size_t)(e0 + t) * a.n_kv + h) * kServeDim + l4;
                st4(o, r[i].lo);
                st4(o + 64, r[i].hi);
            }
        }
    }
    m = warp_max(m);
    if (__any_sync(0xffffffffu, odd) && lane == 0) raise(a.status, SLLM_CUDA_ERR_ARG);
    const bool grows = m > __fmul_rn(old, 127.f);
    const float s = grows ? fmaxf(__fdiv_rn(m, 127.f), kK8Least) : old;
    const float inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
    if (grows && row0 > 0) {
        const float f = __fmul_rn(old, inv);
        uint4* const c16 = reinterpret_cast<uint4*>(codes);
        for (int i = lane; i < row0 * (kServeDim / 16); i += 32) {
            uint4 u = c16[i];
            u.x = recode4(u.x, f);
            u.y = recode4(u.y, f);
            u.z = recode4(u.z, f);
            u.w = recode4(u.w, f);
            c16[i] = u;
        }
    }
    if (lane == 0) *sc = s;
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int t = 2 * i + half;
        if (t < count) {
            int8_t* const c = codes + (size_t)(a.pos[e0 + t] % kKvBlock) * kServeDim + l4;
            *reinterpret_cast<uint32_t*>(c) = codes4(r[i].lo, inv);
            *reinterpret_cast<uint32_t*>(c + 64) = codes4(r[i].hi, inv);
        }
    }
}

template <class O>
__global__ void __launch_bounds__(32 * kK8Warps)
kv8_append_kernel(const __grid_constant__ PagesDev p, const __grid_constant__ Append8Params a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if ((int)blockIdx.x < a.kv_ctas) {
        const int groups = (2 * a.n_kv + a.kv_rows - 1) / a.kv_rows;
        const int row0 = (int)blockIdx.x % groups * a.kv_rows, e0 = (int)blockIdx.x / groups * kK8Entries;
        const int heads = min(a.kv_rows, 2 * a.n_kv - row0);
        // lane l looks at entry e0 + l: a run starts at one of the first 16 and
        // ends among all 32
        const int e = e0 + lane;
        const bool in = e < a.n_tokens;
        const int slot = in ? a.slot[e] : -1, pos = in ? a.pos[e] : 0;
        int before = __shfl_up_sync(0xffffffffu, slot, 1), bpos = __shfl_up_sync(0xffffffffu, pos, 1);
        if (lane == 0) {
            before = e0 > 0 ? a.slot[e0 - 1] : -1;
            bpos = e0 > 0 ? a.pos[e0 - 1] : 0;
        }
        const bool same = slot >= 0 && slot == before && (pos >> 4) == (bpos >> 4);
        const unsigned starts = __ballot_sync(0xffffffffu, in && slot >= 0 && !same && lane < kK8Entries);
        const unsigned goes_on = __ballot_sync(0xffffffffu, same && pos > bpos), again = __ballot_sync(0xffffffffu, same);
        const int pairs = __popc(starts) * heads;
        // pair w of this CTA: run w / heads, head w % heads
        auto run_of = [&](int w, int* l, int* count) {
            *l = (int)__fns(starts, 0, w / heads + 1);
            const unsigned rest = goes_on >> 1 >> *l;           // bit i: entry l + 1 + i follows its predecessor
            *count = __ffs(~rest);                              // (at most 16: positions ascend in a block)
        };
        if (warp >= pairs) return;
        int l, count;
        run_of(warp, &l, &count);
        Run run;
        run.load(a, e0 + l, count, (row0 + warp % heads) % a.n_kv, row0 + warp % heads >= a.n_kv);
        // Each entry's page, -1: none, or a shared one, which is never written (its other
        // owners would change). Tokens behind the slot's end or the angles' are left out.
        const bool fine = slot >= 0 && slot < p.n_slots && pos >= 0 && pos < a.n_ctx && pos < p.cap && pos < p.lens[slot];
        int id = fine ? p.tables[(size_t)slot * p.width + pos / p.page] : -1;
        if (id < 0 || id >= p.n_pages || p.refs[id] != 1) id = -1;
        const unsigned good = __ballot_sync(0xffffffffu, fine && id >= 0);
        for (int w = warp; w < pairs; w += kK8Warps) {
            if (w != warp) run_of(w, &l, &count);
            const int row = row0 + w % heads;
            const unsigned mine = (count < 32 ? (1u << count) - 1u : 0xffffffffu) << l;
            // those that count end where the positions pass a limit; what comes after
            // its place in the list is wrong, too
            const int live = __popc(good & mine);
            const bool wrong = live < count || (l + count < 32 && (again >> (l + count) & 1) != 0);
            if (wrong && lane == 0) raise(a.status, SLLM_CUDA_ERR_ARG);
            const int page = __shfl_sync(0xffffffffu, id, l), p0 = __shfl_sync(0xffffffffu, pos, l);
            if (live == 0) continue;
            const bool is_v = row >= a.n_kv;
            if (w != warp) run.load(a, e0 + l, live, row - (is_v ? a.n_kv : 0), is_v);
            append_run<O>(p, a, run, e0 + l, live, page, p0, row - (is_v ? a.n_kv : 0), is_v);
        }
        return;
    }
    // q: eight rows of one token a warp, two at a time
    const int units = (a.n_head + 7) / 8;
    const long long u = (long long)(blockIdx.x - a.kv_ctas) * kK8Warps + warp;
    const int tok = (int)(u / units);
    if (tok >= a.n_tokens) return;
    const int r0 = (int)(u - (long long)tok * units) * 8 + (lane >> 4), l4 = 4 * (lane & 15);
    const int slot = a.slot[tok], pos = a.pos[tok];
    RotPair r[4];
    #pragma unroll
    for (int i = 0; i < 4; ++i)
        if (r0 + 2 * i < a.n_head) {
            const float* x = a.q + tok * a.qs + (size_t)(r0 + 2 * i) * kServeDim + l4;
            r[i].lo = __ldcs(reinterpret_cast<const float4*>(x));
            r[i].hi = __ldcs(reinterpret_cast<const float4*>(x + 64));
        }
    if (slot < 0) return;
    const int id = pos < a.n_ctx ? page_at(p, slot, pos) : -1;
    if (id < 0 || p.refs[id] != 1) {
        if (lane == 0) raise(a.status, SLLM_CUDA_ERR_ARG);
        return;
    }
    const float4 c = ld4(a.cs + (size_t)pos * 64 + l4), s = ld4(a.sn + (size_t)pos * 64 + l4);
    #pragma unroll
    for (int i = 0; i < 4; ++i)
        if (r0 + 2 * i < a.n_head) {
            rotate(r[i], c, s);
            O* o = static_cast<O*>(a.qo) + ((size_t)tok * a.n_head + r0 + 2 * i) * kServeDim + l4;
            st4(o, r[i].lo);
            st4(o + 64, r[i].hi);
        }
}

// ---------------------------------------------------------------------------
// read. A warp takes one head of k or of v of up to 32 tokens of the list; the
// tokens' pages are looked up first, a lane each. A lane's values leave in 16
// bytes, so 16 lanes share an f16 row and 32 an f32 one; eight such loads are in
// flight.
// Bound: the writes, two to four bytes for each one read (32768 tokens of 8 heads
// to f16, 201 MB: 37 us, where filling the outputs alone takes 35), else the chain
// of page id, scale and codes, stores (4 us).
// ---------------------------------------------------------------------------
struct Read8Params {
    const int32_t* slot;
    const int32_t* pos;
    const int8_t* kp;
    const int8_t* vp;
    const float* ksc;
    const float* vsc;
    size_t page_stride, scale_stride;
    void* ko;
    void* vo;
    int n_tokens, n_kv;
    int per, first, rows;           // tokens of a warp; the first row (k heads, then v heads) and their number
    int32_t* status;
};

__device__ __forceinline__ float value_of(uint32_t u, int i, float s) {
    return __fmul_rn((float)(int)(int8_t)(u >> (8 * i)), s);
}

template <class O>
__global__ void __launch_bounds__(32 * kK8Warps)
kv8_read_kernel(const __grid_constant__ PagesDev p, const __grid_constant__ Read8Params a) {
    constexpr int PER = 16 / (int)sizeof(O), ROWS = PER / 4, FLY = 8;  // elements of a lane; tokens at once; loads in flight
    const int lane = threadIdx.x & 31;
    const long long u = (long long)blockIdx.x * kK8Warps + (threadIdx.x >> 5);
    const long long c = u / a.rows;
    const int row = a.first + (int)(u - c * a.rows), h = row < a.n_kv ? row : row - a.n_kv;
    if (c * a.per >= a.n_tokens) return;
    const int e0 = (int)c * a.per, n = min(a.per, a.n_tokens - e0);
    // this lane's token: where its row of head 0 and the scale of that are, -1: nowhere
    int id = -1, in = 0;
    bool wrong = false;
    if (lane < n) {
        const int slot = a.slot[e0 + lane], pos = a.pos[e0 + lane];
        if (slot >= 0) {
            id = page_at(p, slot, pos);
            wrong = id < 0;
            in = pos & (p.page - 1);
        }
    }
    if (__any_sync(0xffffffffu, wrong) && lane == 0) raise(a.status, SLLM_CUDA_ERR_ARG);
    const bool is_v = row >= a.n_kv;
    const int sub = lane / (32 / ROWS), col = lane % (32 / ROWS) * PER;
    const int8_t* const codes = (is_v ? a.vp : a.kp) + (size_t)h * p.page * kServeDim + col;
    const float* const scales = (is_v ? a.vsc : a.ksc) + (size_t)h * (p.page / kKvBlock);
    O* const out = static_cast<O*>(is_v ? a.vo : a.ko) + ((size_t)e0 * a.n_kv + h) * kServeDim + col;
    for (int i0 = 0; i0 < n; i0 += ROWS * FLY) {
        uint2 x[FLY];
        float s[FLY];
        bool live[FLY];
        #pragma unroll
        for (int i = 0; i < FLY; ++i) {
            const int t = i0 + i * ROWS + sub;
            const int page = __shfl_sync(0xffffffffu, id, t & 31), at = __shfl_sync(0xffffffffu, in, t & 31);
            live[i] = t < n && page >= 0;
            if (live[i]) {
                const int8_t* from = codes + (size_t)page * a.page_stride + at * kServeDim;
                if (PER == 8) x[i] = __ldg(reinterpret_cast<const uint2*>(from));
                else x[i].x = __ldg(reinterpret_cast<const uint32_t*>(from));
                s[i] = __ldg(scales + (size_t)page * a.scale_stride + at / kKvBlock);
            }
        }
        #pragma unroll
        for (int i = 0; i < FLY; ++i) {
            if (!live[i]) continue;
            O* const to = out + (size_t)(i0 + i * ROWS + sub) * a.n_kv * kServeDim;
            if constexpr (PER == 8) {
                __half2 y[4];
                #pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w = e < 2 ? x[i].x : x[i].y;
                    y[e] = __floats2half2_rn(value_of(w, 2 * (e & 1), s[i]), value_of(w, 2 * (e & 1) + 1, s[i]));
                }
                __stcs(reinterpret_cast<uint4*>(to), *reinterpret_cast<const uint4*>(y));
            } else {
                __stcs(reinterpret_cast<float4*>(to), make_float4(value_of(x[i].x, 0, s[i]), value_of(x[i].x, 1, s[i]),
                                                                  value_of(x[i].x, 2, s[i]), value_of(x[i].x, 3, s[i])));
            }
        }
    }
}

}  // namespace
}  // namespace sllm

using namespace sllm;

extern "C" int sllm_cuda_kv8_append(const sllm_cuda_kv_pages* p, int32_t layer, int32_t n_tokens, const int32_t* slot,
                                    const int32_t* pos, int32_t n_head, const float* q, size_t q_stride,
                                    const float* k, size_t k_stride, const float* v, size_t v_stride,
                                    const float* rope_cos, const float* rope_sin, int32_t n_ctx, void* q_out,
                                    void* k_out, void* v_out, int32_t out_type, int32_t* status, void* stream) {
    int rc = check_pages(p, "kv8_append", true);
    if (rc != SLLM_CUDA_OK) return rc;
    if (slot == nullptr || pos == nullptr || k == nullptr || v == nullptr || rope_cos == nullptr ||
        rope_sin == nullptr || (q == nullptr) != (q_out == nullptr))
        return fail(SLLM_CUDA_ERR_ARG, "kv8_append: a NULL array (q and q_out go together)");
    const size_t kvn = (size_t)p->n_head_kv * kServeDim, qn = (size_t)(n_head > 0 ? n_head : 0) * kServeDim;
    if (layer < 0 || layer >= p->n_layer || n_tokens < 0 || n_tokens > (1 << 24) || n_ctx < 1 ||
        (q != nullptr && (n_head < 1 || n_head > 1024 || n_head % p->n_head_kv != 0 || q_stride < qn)) ||
        k_stride < kvn || v_stride < kvn || q_stride > (1u << 30) || k_stride > (1u << 30) || v_stride > (1u << 30) ||
        (out_type != SLLM_CUDA_KV_F32 && out_type != SLLM_CUDA_KV_F16))
        return fail(SLLM_CUDA_ERR_ARG, "kv8_append: layer %d, %d tokens, %d heads, strides %zu %zu %zu, outputs of type %d",
                    layer, n_tokens, n_head, q_stride, k_stride, v_stride, out_type);
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(q_out) || !aligned16(k_out) || !aligned16(v_out) ||
        !aligned16(rope_cos) || !aligned16(rope_sin) || (q_stride | k_stride | v_stride) % 4 != 0)
        return fail(SLLM_CUDA_ERR_ARG, "kv8_append: arrays must be 16-byte aligned, strides a multiple of 4 floats");
    const void* ptr[] = {p->k, p->v, p->refs, p->tables, p->lens, p->k_scale, p->v_scale, slot, pos, q, k, v, rope_cos,
                         rope_sin, q_out, k_out, v_out, status};
    const char* name[] = {"k", "v", "refs", "tables", "lens", "k_scale", "v_scale", "slot", "pos", "q", "k", "v",
                          "rope_cos", "rope_sin", "q_out", "k_out", "v_out", "status"};
    for (int i = 0; i < 18; ++i)
        if (ptr[i] != nullptr && (rc = need_device(ptr[i], "kv8_append", name[i])) != SLLM_CUDA_OK) return rc;
    if (n_tokens == 0) return SLLM_CUDA_OK;
    Append8Params a{};
    a.slot = slot; a.pos = pos;
    a.q = q; a.k = k; a.v = v;
    a.qs = q_stride; a.ks = k_stride; a.vs = v_stride;
    a.cs = rope_cos; a.sn = rope_sin;
    a.qo = q_out; a.ko = k_out; a.vo = v_out;
    const size_t layer_codes = kvn * p->page_size, layer_scales = (size_t)p->n_head_kv * (p->page_size / kKvBlock);
    a.kp = static_cast<int8_t*>(p->k) + layer * layer_codes;
    a.vp = static_cast<int8_t*>(p->v) + layer * layer_codes;
    a.ksc = p->k_scale + layer * layer_scales;
    a.vsc = p->v_scale + layer * layer_scales;
    a.page_stride = p->n_layer * layer_codes;
    a.scale_stride = p->n_layer * layer_scales;
    a.n_tokens = n_tokens; a.n_head = n_head; a.n_kv = p->n_head_kv; a.n_ctx = n_ctx;
    a.status = status;
    // one head of k or v a CTA while that makes no more than four CTAs an SM, else eight
    const long long chunks = (n_tokens + kK8Entries - 1) / kK8Entries;
    a.kv_rows = chunks * 2 * p->n_head_kv <= 4LL * current_sms() ? 1 : 8;
    const long long kv = chunks * ((2 * p->n_head_kv + a.kv_rows - 1) / a.kv_rows);
    const long long units = q != nullptr ? (long long)n_tokens * ((n_head + 7) / 8) : 0;
    const long long ctas = kv + (units + kK8Warps - 1) / kK8Warps;
    if (ctas > 0x7fffffffLL) return fail(SLLM_CUDA_ERR_TOO_LARGE, "kv8_append: %d tokens", n_tokens);
    a.kv_ctas = (int)kv;
    if (out_type == SLLM_CUDA_KV_F16)
        kv8_append_kernel<__half><<<(unsigned)ctas, 32 * kK8Warps, 0, (cudaStream_t)stream>>>(pages_dev(*p), a);
    else
        kv8_append_kernel<float><<<(unsigned)ctas, 32 * kK8Warps, 0, (cudaStream_t)stream>>>(pages_dev(*p), a);
    CK(cudaGetLastError(), "kv8_append launch");
    count_launches(1);
    return SLLM_CUDA_OK;
}

extern "C" int sllm_cuda_kv8_read(const sllm_cuda_kv_pages* p, int32_t layer, int32_t n_tokens, const int32_t* slot,
                                  const int32_t* pos, void* k_out, void* v_out, int32_t out_type, int32_t* status,
                                  void* stream) {
    int rc = check_pages(p, "kv8_read", true);
    if (rc != SLLM_CUDA_OK) return rc;
    if (slot == nullptr || pos == nullptr) return fail(SLLM_CUDA_ERR_ARG, "kv8_read: a NULL list");
    if (layer < 0 || layer >= p->n_layer || n_tokens < 0 || n_tokens > (1 << 24) ||
        (out_type != SLLM_CUDA_KV_F32 && out_type != SLLM_CUDA_KV_F16) || !aligned16(k_out) || !aligned16(v_out))
        return fail(SLLM_CUDA_ERR_ARG, "kv8_read: layer %d, %d tokens, outputs of type %d (16-byte aligned)", layer, n_tokens,
                    out_type);
    const void* ptr[] = {p->k, p->v, p->tables, p->lens, p->k_scale, p->v_scale, slot, pos, k_out, v_out, status};
    const char* name[] = {"k", "v", "tables", "lens", "k_scale", "v_scale", "slot", "pos", "k_out", "v_out", "status"};
    for (int i = 0; i < 11; ++i)
        if (ptr[i] != nullptr && (rc = need_device(ptr[i], "kv8_read", name[i])) != SLLM_CUDA_OK) return rc;
    if (n_tokens == 0 || (k_out == nullptr && v_out == nullptr)) return SLLM_CUDA_OK;
    Read8Params a{};
    a.slot = slot; a.pos = pos;
    const size_t layer_codes = (size_t)p->n_head_kv * kServeDim * p->page_size;
    const size_t layer_scales = (size_t)p->n_head_kv * (p->page_size / kKvBlock);
    a.kp = static_cast<const int8_t*>(p->k) + layer * layer_codes;
    a.vp = static_cast<const int8_t*>(p->v) + layer * layer_codes;
    a.ksc = p->k_scale + layer * layer_scales;
    a.vsc = p->v_scale + layer * layer_scales;
    a.page_stride = p->n_layer * layer_codes;
    a.scale_stride = p->n_layer * layer_scales;
    a.ko = k_out; a.vo = v_out;
    a.n_tokens = n_tokens; a.n_kv = p->n_head_kv;
    a.status = status;
    a.first = k_out != nullptr ? 0 : p->n_head_kv;
    a.rows = ((k_out != nullptr) + (v_out != nullptr)) * p->n_head_kv;
    // 32 tokens a warp where that still makes 16 warps an SM, else eight
    a.per = (long long)n_tokens * a.rows / 32 >= 16LL * current_sms() ? 32 : 8;
    const long long units = ((long long)n_tokens + a.per - 1) / a.per * a.rows;
    const long long ctas = (units + kK8Warps - 1) / kK8Warps;
    if (ctas > 0x7fffffffLL) return fail(SLLM_CUDA_ERR_TOO_LARGE, "kv8_read: %d tokens", n_tokens);
    if (out_type == SLLM_CUDA_KV_F16)
        kv8_read_kernel<__half><<<(unsigned)ctas, 32 * kK8Warps, 0, (cudaStream_t)stream>>>(pages_dev(*p), a);
    else
        kv8_read_kernel<float><<<(unsigned)ctas, 32 * kK8Warps, 0, (cudaStream_t)stream>>>(pages_dev(*p), a);
    CK(cudaGetLastError(), "kv8_read launch");
    count_launches(1);
    return SLLM_CUDA_OK;
}
