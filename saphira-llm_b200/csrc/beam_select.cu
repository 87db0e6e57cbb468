// beam_select.cu -- one step of beam search: the `beams` best continuations
// among beams * n_vocab candidates
//     score[b] + logits[b][x] - lse[b],    lse[b] = ln sum_y exp(logits[b][y]).
//
// The values are compared in 64 bits. Within a beam the order is that of the
// logits, so each beam needs its own best `beams` logits only, and its lse.
//
// One cluster of CTAs per request; each CTA has a share of the vocabulary of
// all beams, 8192 words of one beam at a time, 16 in the registers of a thread.
// One pass gives the sum of exponentials (against the running maximum; terms
// in 32 bits, sums of four of them in 64) and the few words that can be among
// the best: those not below the least of `beams` or more disjoint parts' maxima,
// about three per part for random logits. A list that overflows all the same
// (many equal logits) is made again word by word. The first CTA of the cluster
// gets the lists through distributed shared memory and merges them.
//
// Bound: HBM, the logits once; for one request the chain load, maximum, list,
// merge.

#include <cooperative_groups.h>

#include "serve.cuh"

namespace cg = cooperative_groups;

namespace sllm {
namespace {

constexpr int kBmThreads = 512;
constexpr int kBmWarps = kBmThreads / 32;
constexpr int kBmPer = 16;                          // words of a thread
constexpr int kBmPiece = kBmThreads * kBmPer;
constexpr int kBmMost = 16;                         // beams
constexpr int kBmList = 256;                        // words kept of a beam by a CTA
constexpr int kBmNone = 0x7fffffff;

struct BeamParams {
    const float* logits;
    size_t stride;                  // floats from a row to the next
    const float* score;
    const int32_t* done;
    const int32_t* slots;
    int n, beams, V, eos, per;      // per: words of a CTA
    float* score_out;
    int32_t* parent;
    int32_t* token;
    int32_t* done_out;
    int32_t* src;
    int32_t* status;
};

struct Word {
    float v;
    int x;
};

struct BeamShared {
    float wmax[2][kBmWarps];
    double part[kBmMost][kBmWarps];                 // a warp's sum of exponentials, against top[b]
    float top[kBmMost];                             // the largest logit of this CTA's share
    int count[kBmMost];
    int odd;
    Word list[kBmMost][kBmList];
    Word best[16][kBmMost][kBmMost];                // [CTA][beam][rank], of the cluster's first CTA
    double sum[16][kBmMost];
    float tops[16][kBmMost];
    Word merged[kBmMost][kBmMost];
    double lse[kBmMost];
};

__device__ __forceinline__ bool before(float av, int ax, float bv, int bx) { return av > bv || (av == bv && ax < bx); }

// 16 words of a thread: by fours where rows are 16-byte aligned, one by one
// where not; a share of under 2048 words dealt out among the warps, so that each
// has some (parts without words give no bound)
enum { BM_VEC = 0, BM_WORDS = 1, BM_DEALT = 2 };
constexpr int kBmDealt = 4 * kBmThreads;
template <int MODE>
__device__ __forceinline__ int word_at(int e, int t) {
    if (MODE == BM_VEC) return 4 * (t + kBmThreads * (e >> 2)) + (e & 3);
    if (MODE == BM_WORDS) return t + kBmThreads * e;
    return (t >> 5) + kBmWarps * (t & 31) + kBmThreads * e;
}

template <int MODE>
__device__ __forceinline__ void load_piece(const float* row, int lo, int hi, float (&x)[kBmPer]) {
    constexpr bool VEC = MODE == BM_VEC;
    const int t = threadIdx.x;
    #pragma unroll
    for (int e = 0; e < kBmPer; e += VEC ? 4 : 1) {
        const int i = lo + word_at<MODE>(e, t);
        if (VEC && i + 4 <= hi) {
            const float4 v = __ldcs(reinterpret_cast<const float4*>(row + i));
            x[e] = v.x;
            x[e + (VEC ? 1 : 0)] = v.y;
            x[e + (VEC ? 2 : 0)] = v.z;
            x[e + (VEC ? 3 : 0)] = v.w;
        } else {
            #pragma unroll
            for (int j = 0; j < (VEC ? 4 : 1); ++j) x[e + j] = i + j < hi ? __ldg(row + i + j) : -INFINITY;
        }
    }
}

// the best of a row's words that come after (pv, px), over the CTA; for lists
// that overflowed
__device__ Word next_word(const float* row, int lo, int hi, float pv, int px, Word* scratch) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    Word w{-INFINITY, kBmNone};
    for (int i = lo + t; i < hi; i += kBmThreads) {
        float v = row[i];
        if (!(v < INFINITY)) v = -INFINITY;
        if (v > -INFINITY && before(pv, px, v, i) && before(v, i, w.v, w.x)) w = Word{v, i};
    }
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, w.v, o);
        const int x = __shfl_xor_sync(0xffffffffu, w.x, o);
        if (before(v, x, w.v, w.x)) w = Word{v, x};
    }
    if (lane == 0) scratch[warp] = w;
    __syncthreads();
    w = scratch[0];
    for (int i = 1; i < kBmWarps; ++i)
        if (before(scratch[i].v, scratch[i].x, w.v, w.x)) w = scratch[i];
    __syncthreads();
    return w;
}

template <int MODE>
__global__ void __launch_bounds__(kBmThreads, 2)
beam_select_kernel(const __grid_constant__ BeamParams a) {
    extern __shared__ __align__(16) uint8_t smem[];
    BeamShared& sh = *reinterpret_cast<BeamShared*>(smem);
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int req = blockIdx.x / C, t = threadIdx.x, lane = t & 31, warp = t >> 5, B = a.beams;
    const int lo = (int)min((long long)rank * a.per, (long long)a.V), hi = min(a.V, lo + a.per);
    const float* const rows = a.logits + (size_t)req * B * a.stride;
    if (t < kBmMost) {
        sh.count[t] = 0;
        sh.top[t] = -INFINITY;
    }
    if (t == 0) sh.odd = 0;
    // beams that have words to offer: not done, of a score above -inf
    unsigned live = 0;
    bool odd = false;
    for (int b = 0; b < B; ++b) {
        const float s = a.score[(size_t)req * B + b];
        odd = odd || !(s < INFINITY);
        if (s > -INFINITY && s < INFINITY && (a.done == nullptr || a.done[(size_t)req * B + b] == 0)) live |= 1u << b;
    }
    // parts of 32 to 512 threads whose maxima bound the beams-th best
    const int span = B <= 4 ? 128 : B <= 8 ? 64 : 32;
    float x[kBmPer], next[kBmPer];
    int b = live != 0 ? __ffs(live) - 1 : B, at = lo, buf = 0;
    if (b < B && lo < hi) load_piece<MODE>(rows + (size_t)b * a.stride, lo, hi, x);
    float top = -INFINITY, floor = -INFINITY;       // of the beam so far: its largest; what `beams` of its words reach
    double sum = 0.0;
    __syncthreads();
    while (b < B && lo < hi) {
        int nb = b, nat = at + kBmPiece;
        if (nat >= hi) {
            const unsigned rest = live >> b >> 1;
            nb = rest != 0 ? b + __ffs(rest) : B;
            nat = lo;
        }
        if (nb < B) load_piece<MODE>(rows + (size_t)nb * a.stride, nat, hi, next);
        float m = -INFINITY;
        #pragma unroll
        for (int e = 0; e < kBmPer; ++e) {
            const bool fine = x[e] < INFINITY;      // NaN and +inf count as -inf
            odd = odd || !fine;
            x[e] = fine ? x[e] : -INFINITY;
            m = fmaxf(m, x[e]);
        }
        const float mine = m;
        m = warp_max(m);
        if (lane == 0) sh.wmax[buf][warp] = m;
        __syncthreads();
        // parts of span threads: span / 32 warps each
        float w = sh.wmax[buf][lane & (kBmWarps - 1)];
        for (int o = 1; o < span / 32; o <<= 1) w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, o));
        float least = w, most = w;
        #pragma unroll
        for (int o = 1; o < kBmWarps; o <<= 1) {
            least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        floor = fmaxf(floor, least);
        if (mine >= floor && mine > -INFINITY) {
            #pragma unroll
            for (int e = 0; e < kBmPer; ++e)
                if (x[e] >= floor && x[e] > -INFINITY) {
                    const int i = atomicAdd(&sh.count[b], 1);
                    if (i < kBmList) sh.list[b][i] = Word{x[e], at + word_at<MODE>(e, t)};
                }
        }
        if (most > top) {
            sum = top > -INFINITY ? sum * exp((double)top - (double)most) : 0.0;
            top = most;
        }
        if (top > -INFINITY) {
            #pragma unroll
            for (int e = 0; e < kBmPer; e += 4)
                sum += (double)((expf(x[e] - top) + expf(x[e + 1] - top)) + (expf(x[e + 2] - top) + expf(x[e + 3] - top)));
        }
        if (nb != b) {
            const double all = warp_sum_d(sum);
            if (lane == 0) sh.part[b][warp] = all;
            if (t == 0) sh.top[b] = top;
            sum = 0.0;
            top = floor = -INFINITY;
        }
        buf ^= 1;
        b = nb;
        at = nat;
        #pragma unroll
        for (int e = 0; e < kBmPer; ++e) x[e] = next[e];
    }
    if (odd) sh.odd = 1;
    __syncthreads();
    if (t == 0 && sh.odd != 0) raise(a.status, SLLM_CUDA_ERR_ARG);
    // this CTA's best words of each beam, in order, into the first CTA's memory
    BeamShared& sh0 = *cl.map_shared_rank(&sh, 0);
    cl.sync();                      // (the first CTA runs)
    for (int r = warp; r < B; r += kBmWarps) {
        const int c = sh.count[r];
        if (lane == 0) {
            double s = 0.0;
            if (sh.top[r] > -INFINITY)
                for (int i = 0; i < kBmWarps; ++i) s += sh.part[r][i];
            sh0.sum[rank][r] = s;
            sh0.tops[rank][r] = sh.top[r];
        }
        if (c > kBmList) continue;
        for (int i = lane; i < c || i < B; i += 32) {
            if (i >= c) {
                sh0.best[rank][r][i] = Word{-INFINITY, kBmNone};
                continue;
            }
            const Word w = sh.list[r][i];
            int place = 0;
            for (int j = 0; j < c; ++j) {
                const Word o = sh.list[r][j];
                place += before(o.v, o.x, w.v, w.x) ? 1 : 0;
            }
            if (place < B) sh0.best[rank][r][place] = w;
        }
    }
    __syncthreads();
    for (int r = 0; r < B; ++r) {
        if (sh.count[r] <= kBmList) continue;       // the same for every thread
        float pv = INFINITY;
        int px = -1;
        for (int i = 0; i < B; ++i) {
            const Word w = next_word(rows + (size_t)r * a.stride, lo, hi, pv, px, sh.list[r]);
            if (t == 0) sh0.best[rank][r][i] = w;
            pv = w.v;
            px = w.x;
        }
    }
    cl.sync();
    if (rank != 0) return;
    // merge: a warp per beam, a lane per CTA's list
    for (int r = warp; r < B; r += kBmWarps) {
        if ((live >> r & 1) == 0) continue;
        int head = 0;
        for (int i = 0; i < B; ++i) {
            Word w{-INFINITY, kBmNone};
            if (lane < C && head < B) w = sh.best[lane][r][head];
            Word m = w;
            #pragma unroll
            for (int o = 8; o > 0; o >>= 1) {
                const float v = __shfl_xor_sync(0xffffffffu, m.v, o);
                const int y = __shfl_xor_sync(0xffffffffu, m.x, o);
                if (before(v, y, m.v, m.x)) m = Word{v, y};
            }
            if (w.x == m.x && w.x != kBmNone) ++head;
            if (lane == 0) sh.merged[r][i] = m;
        }
        float top_r = lane < C ? sh.tops[lane][r] : -INFINITY;
        const float all = warp_max(top_r);
        double s = lane < C && top_r > -INFINITY ? sh.sum[lane][r] * exp((double)top_r - (double)all) : 0.0;
        s = warp_sum_d(s);
        if (lane == 0) sh.lse[r] = (double)all + log(s);
    }
    __syncthreads();
    if (warp != 0) return;
    // the best of the beams' heads, `beams` times: a lane per beam
    const bool mine = lane < B;
    const float score = mine ? a.score[(size_t)req * B + lane] : -INFINITY;
    const bool is_done = mine && a.done != nullptr && a.done[(size_t)req * B + lane] != 0;
    const bool offers = (live >> (lane & 31) & 1) != 0 && mine;
    const bool one = is_done && score > -INFINITY && score < INFINITY;
    int head = 0, px = -1, pb = -1;
    double pv = 0.0;
    int got = 0;
    auto value = [&](int i) -> double {             // of this lane's i-th candidate
        if (one) return i == 0 ? (double)score : -INFINITY;
        if (!offers || i >= B || sh.merged[lane][i].x == kBmNone) return -INFINITY;
        return (double)score + ((double)sh.merged[lane][i].v - sh.lse[lane]);
    };
    for (int i = 0; i < B; ++i) {
        const double v = value(head);
        double m = v;
        int who = lane;
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double ov = __shfl_xor_sync(0xffffffffu, m, o);
            const int ow = __shfl_xor_sync(0xffffffffu, who, o);
            if (ov > m || (ov == m && ow < who)) {
                m = ov;
                who = ow;
            }
        }
        if (!(m > -INFINITY)) break;
        int word = 0;
        if (lane == who) {
            word = one ? a.eos : sh.merged[lane][head].x;
            ++head;
        }
        word = __shfl_sync(0xffffffffu, word, who);
        if (lane == i) {
            pv = m;
            pb = who;
            px = word;
        }
        got = i + 1;
    }
    // too few of weight: the first candidates of value -inf
    if (got < B) {
        int cb = 0, cx = 0;
        for (int i = got; i < B; ++i) {
            for (;;) {
                const bool d = a.done != nullptr && a.done[(size_t)req * B + cb] != 0;
                if (d && cx <= a.eos) cx = a.eos;
                else if (d) cx = a.V;
                if (cx >= a.V) {
                    ++cb;
                    cx = 0;
                    continue;
                }
                const bool taken = __any_sync(0xffffffffu, lane < i && pb == cb && px == cx);
                if (!taken) break;
                ++cx;
            }
            if (lane == i) {
                pv = -INFINITY;
                pb = cb;
                px = cx;
            }
            ++cx;
        }
    }
    if (mine) {
        const size_t o = (size_t)req * B + lane;
        a.score_out[o] = (float)pv;
        a.parent[o] = pb;
        a.token[o] = px;
        if (a.done_out != nullptr)
            a.done_out[o] = (a.done != nullptr && a.done[(size_t)req * B + pb] != 0) || px == a.eos ? 1 : 0;
        if (a.src != nullptr) a.src[o] = a.slots[(size_t)req * B + pb];
    }
}

int beam_cluster(int n, int beams, int n_vocab, int sms) {
    int C = 1;
    while (C < 16 && (long long)n * C * 2 <= 4LL * sms && n_vocab / C > kBmPiece) C *= 2;
    return C;
}

}  // namespace
}  // namespace sllm

using namespace sllm;

extern "C" int sllm_cuda_beam_select(const float* logits, size_t row_stride, const float* score, const int32_t* done,
                                     const int32_t* slots, int32_t n, int32_t beams, int32_t n_vocab, int32_t eos,
                                     float* score_out, int32_t* parent, int32_t* token, int32_t* done_out, int32_t* src,
                                     int32_t* status, void* stream) {
    if (logits == nullptr || score == nullptr || score_out == nullptr || parent == nullptr || token == nullptr ||
        (slots == nullptr) != (src == nullptr))
        return fail(SLLM_CUDA_ERR_ARG, "beam_select: a NULL array (slots and src go together)");
    if (n < 0 || n > 65536 || beams < 1 || beams > kBmMost || n_vocab < 1 || n_vocab > (1 << 20) ||
        row_stride < (size_t)n_vocab || row_stride > (1u << 30))
        return fail(SLLM_CUDA_ERR_ARG, "beam_select: %d requests of %d beams (1 to %d), %d words, rows %zu apart", n, beams,
                    kBmMost, n_vocab, row_stride);
    if (eos >= n_vocab || (eos < 0 && (done != nullptr || done_out != nullptr)))
        return fail(SLLM_CUDA_ERR_ARG, "beam_select: eos %d of %d words (none: no done, no done_out)", eos, n_vocab);
    const void* ptr[] = {logits, score, done, slots, score_out, parent, token, done_out, src, status};
    const char* name[] = {"logits", "score", "done", "slots", "score_out", "parent", "token", "done_out", "src", "status"};
    for (int i = 0; i < 10; ++i) {
        if (ptr[i] == nullptr) continue;
        const int rc = need_device(ptr[i], "beam_select", name[i]);
        if (rc != SLLM_CUDA_OK) return rc;
    }
    if (n == 0) return SLLM_CUDA_OK;
    BeamParams a{};
    a.logits = logits; a.stride = row_stride;
    a.score = score; a.done = done; a.slots = slots;
    a.n = n; a.beams = beams; a.V = n_vocab; a.eos = eos < 0 ? -1 : eos;
    a.score_out = score_out; a.parent = parent; a.token = token; a.done_out = done_out; a.src = src;
    a.status = status;
    const int C = beam_cluster(n, beams, n_vocab, current_sms());
    a.per = ((n_vocab + C - 1) / C + 3) / 4 * 4;
    const int mode = a.per < kBmDealt ? BM_DEALT : row_stride % 4 == 0 && aligned16(logits) ? BM_VEC : BM_WORDS;
    constexpr int kBytes = (int)sizeof(BeamShared);
    const cudaError_t e[6] = {allow_smem<beam_select_kernel<BM_VEC>>(kBytes), allow_smem<beam_select_kernel<BM_WORDS>>(kBytes),
                              allow_smem<beam_select_kernel<BM_DEALT>>(kBytes), allow_cluster<beam_select_kernel<BM_VEC>>(),
                              allow_cluster<beam_select_kernel<BM_WORDS>>(), allow_cluster<beam_select_kernel<BM_DEALT>>()};
    for (int i = 0; i < 6; ++i) CK(e[i], "beam_select attributes");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(n * C));
    cfg.blockDim = dim3(kBmThreads);
    cfg.dynamicSmemBytes = kBytes;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = C;
    at.val.clusterDim.y = 1;
    at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    CK(mode == BM_VEC     ? cudaLaunchKernelEx(&cfg, beam_select_kernel<BM_VEC>, a)
       : mode == BM_WORDS ? cudaLaunchKernelEx(&cfg, beam_select_kernel<BM_WORDS>, a)
                          : cudaLaunchKernelEx(&cfg, beam_select_kernel<BM_DEALT>, a),
       "beam_select launch");
    count_launches(1);
    return SLLM_CUDA_OK;
}
