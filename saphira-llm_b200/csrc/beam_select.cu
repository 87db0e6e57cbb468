// beam_select.cu -- one step of beam search: the `beams` best continuations
// among beams * n_vocab candidates
//     score[b] + logits[b][x] - lse[b],    lse[b] = ln sum_y exp(logits[b][y]).
//
// The values are compared in 64 bits. Within a beam the order is that of the
// logits, so each beam needs its own best `beams` logits only, and its lse.
//
// One cluster of CTAs per request; each CTA has a share of the vocabulary of
// all beams, a piece of 8192 words of one beam at a time, 16 in the registers of
// a thread, the pieces behind it on their way into shared memory (a thread
// copies and reads its own words, so that needs no barrier, and 4-byte copies
// where rows are not aligned). One pass gives the sum of exponentials (against
// the warp's running maximum; terms in 32 bits, sums of more than 16 in 64) and
// the few words that can be among the best: those not below the least of
// `beams` or more disjoint parts' maxima, about three per part for random
// logits. A list that overflows all the same (many equal logits) is made again
// word by word. The first CTA of the cluster gets the lists through distributed
// shared memory and merges them.
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
constexpr int kBmRing = 2;                          // pieces in shared memory or on their way

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

// A word of a beam as one integer: its logit's order, then the words before it first.
// 0 is none.
using Word = unsigned long long;
__device__ __forceinline__ uint32_t key_of(float v) {       // (+0 and -0 are equal)
    const uint32_t u = __float_as_uint(v + 0.f);
    return (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) != 0 ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ Word word_of(float v, int x) { return (Word)key_of(v) << 32 | (0xffffffffu - (uint32_t)x); }
__device__ __forceinline__ int index_of(Word w) { return (int)(0xffffffffu - (uint32_t)w); }

struct BeamShared {
    uint32_t wmax[2][kBmWarps];                     // keys of the warps' largest logits of the beam so far
    double part[kBmMost][kBmWarps];                 // a warp's sum of e^(x - ref)
    float ref[kBmMost][kBmWarps];                   // and that ref, whole; -inf: no words
    uint32_t floor[kBmMost];                        // key: at least `beams` words reach it
    int count[kBmMost];
    int odd;
    float score[kBmMost];
    int done[kBmMost], slots[kBmMost];
    double sum[16][kBmMost];                        // [CTA][beam], of the cluster's first CTA, as are `best` and what follows
    float refs[16][kBmMost];
    Word merged[kBmMost][kBmMost];
    double value[kBmMost * kBmMost];
    double powers[96];                              // of kPowers

    __device__ __forceinline__ double down_by(float d) const { return d < 96.f ? powers[(int)d] : 0.0; }
    int pick[kBmMost];                              // the chosen: beam * beams + rank
    Word list[kBmMost][kBmList];
    union {
        float4 ring[kBmRing][kBmPiece / 4];
        Word best[16][kBmMost][kBmMost];            // [CTA][beam][rank]
    };
};

// e^-i: references are whole, so sums against two of them differ by such a factor
struct Powers {
    double v[96];
    constexpr Powers() : v() {
        v[0] = 1.0;
        for (int i = 1; i < 96; ++i) v[i] = v[i - 1] * 0.36787944117144232160;
    }
};
__device__ const Powers kPowers;

// the sum of e^(x - ref) over a thread's words
__device__ __forceinline__ float sum_exp(const float (&x)[kBmPer], float ref) {
    float e[kBmPer];
    #pragma unroll
    for (int i = 0; i < kBmPer; ++i)
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e[i]) : "f"((x[i] - ref) * 1.4426950408889634f));
    #pragma unroll
    for (int n = kBmPer / 2; n > 0; n >>= 1)
        #pragma unroll
        for (int i = 0; i < n; ++i) e[i] += e[i + n];
    return e[0];
}

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

// a thread's words of the piece at `lo`, on their way into its places of a ring entry
template <int MODE>
__device__ __forceinline__ void fetch_piece(const float* row, int lo, int hi, float4* to) {
    const int t = threadIdx.x;
    #pragma unroll
    for (int e = 0; e < kBmPer; e += MODE == BM_VEC ? 4 : 1) {
        const int i = lo + word_at<MODE>(e, t);
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to + (e / 4) * kBmThreads + t) + 4 * (e & 3);
        if (MODE == BM_VEC && i + 4 <= hi)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(row + i) : "memory");
        else
            #pragma unroll
            for (int j = 0; j < (MODE == BM_VEC ? 4 : 1); ++j)
                if (i + j < hi) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 4 * j), "l"(row + i + j) : "memory");
    }
}
__device__ __forceinline__ void fetch_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int MODE>
__device__ __forceinline__ void take_piece(const float4* from, int lo, int hi, float (&x)[kBmPer]) {
    const int t = threadIdx.x;
    #pragma unroll
    for (int e = 0; e < kBmPer; e += 4) {
        const float4 v = from[(e / 4) * kBmThreads + t];
        x[e] = v.x;
        x[e + 1] = v.y;
        x[e + 2] = v.z;
        x[e + 3] = v.w;
    }
    if (lo + kBmPiece > hi) {
        #pragma unroll
        for (int e = 0; e < kBmPer; ++e)
            if (lo + word_at<MODE>(e, t) >= hi) x[e] = -INFINITY;
    }
}

// the best of a row's words behind `last`, over the CTA; for lists that overflowed
__device__ Word next_word(const float* row, int lo, int hi, Word last, Word* scratch) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    Word w = 0;
    for (int i = lo + t; i < hi; i += kBmThreads) {
        const float v = row[i];
        if (!(v < INFINITY && v > -INFINITY)) continue;
        const Word x = word_of(v, i);
        if (x < last && x > w) w = x;
    }
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) w = max(w, __shfl_xor_sync(0xffffffffu, w, o));
    if (lane == 0) scratch[warp] = w;
    __syncthreads();
    for (int i = 0; i < kBmWarps; ++i) w = max(w, scratch[i]);
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
    if (t < kBmMost) sh.count[t] = 0;
    if (t >= kBmThreads - 96) sh.powers[t - (kBmThreads - 96)] = kPowers.v[t - (kBmThreads - 96)];
    if (t < kBmMost * kBmWarps) sh.ref[t / kBmWarps][t % kBmWarps] = -INFINITY;
    if (t == 0) sh.odd = 0;
    // beams that have words to offer: not done, of a score above -inf
    float my_score = 0.f;
    int my_done = 0, my_slot = 0;
    if (lane < B) {
        my_score = a.score[(size_t)req * B + lane];
        if (a.done != nullptr) my_done = a.done[(size_t)req * B + lane];
        if (warp == 0 && a.slots != nullptr) my_slot = a.slots[(size_t)req * B + lane];
    }
    const unsigned live = __ballot_sync(0xffffffffu, lane < B && my_done == 0 && my_score > -INFINITY && my_score < INFINITY);
    bool odd = lane < B && !(my_score < INFINITY);
    if (warp == 0 && lane < B) {
        sh.score[lane] = my_score;
        sh.done[lane] = my_done;
        sh.slots[lane] = my_slot;
    }
    // parts of 1 to 4 warps whose maxima bound the beams-th best
    const int parts = B <= 4 ? 4 : B <= 8 ? 8 : 16, span = kBmWarps / parts;
    // the pieces of this CTA in order: beam by beam
    struct Piece {
        int b, at;
    };
    auto after = [&](Piece p) {
        p.at += kBmPiece;
        if (p.at >= hi) {
            const unsigned rest = live >> p.b >> 1;
            p.b = rest != 0 ? p.b + __ffs(rest) : B;
            p.at = lo;
        }
        return p;
    };
    float x[kBmPer];
    Piece cur{live != 0 && lo < hi ? __ffs(live) - 1 : B, lo}, ahead = cur;
    int buf = 0, entry = 0, fill = 0;
    #pragma unroll
    for (int i = 0; i < kBmRing - 1; ++i) {
        if (ahead.b < B) {
            fetch_piece<MODE>(rows + (size_t)ahead.b * a.stride, ahead.at, hi, sh.ring[fill]);
            ahead = after(ahead);
        }
        fetch_end();
        fill = i + 1;
    }
    // of the beam so far: this warp's reference, its sum, its largest logit
    float ref = -INFINITY;
    double sum = 0.0;
    uint32_t run = 0;
    __syncthreads();
    while (cur.b < B) {
        const int b = cur.b, at = cur.at;
        fetch_wait<kBmRing - 2>();
        const float4* const here = sh.ring[entry];
        take_piece<MODE>(here, at, hi, x);
        // (this thread's places of the entry that it read last are free)
        if (ahead.b < B) {
            fetch_piece<MODE>(rows + (size_t)ahead.b * a.stride, ahead.at, hi, sh.ring[fill]);
            ahead = after(ahead);
        }
        fetch_end();
        entry = entry + 1 == kBmRing ? 0 : entry + 1;
        fill = fill + 1 == kBmRing ? 0 : fill + 1;
        cur = after(cur);
        float mine = x[0];
        #pragma unroll
        for (int e = 1; e < kBmPer; ++e) mine = fmaxf(mine, x[e]);
        if (!(mine < INFINITY)) {                   // +inf counts as -inf, as a NaN does
            odd = true;
            mine = -INFINITY;
            #pragma unroll
            for (int e = 0; e < kBmPer; ++e) {
                x[e] = x[e] < INFINITY ? x[e] : -INFINITY;
                mine = fmaxf(mine, x[e]);
            }
        }
        run = max(run, __reduce_max_sync(0xffffffffu, key_of(mine)));
        if (lane == 0) sh.wmax[buf][warp] = run;
        // this warp's exponentials, while the maxima of the others come in
        const float want = ceilf(logit_of(run));
        if (want > ref) {
            sum = ref > -INFINITY ? sum * sh.down_by(want - ref) : 0.0;
            ref = want;
        }
        if (ref > -INFINITY) {
            float e = sum_exp(x, ref);
            if (e != e) {                           // a NaN among them
                odd = true;
                #pragma unroll
                for (int i = 0; i < kBmPer; ++i) x[i] = x[i] == x[i] ? x[i] : -INFINITY;
                e = sum_exp(x, ref);
            }
            sum += (double)e;
        } else {                                    // only -inf so far, and perhaps NaN
            #pragma unroll
            for (int i = 0; i < kBmPer; ++i) odd = odd || x[i] != x[i];
        }
        __syncthreads();
        // the least of the parts' maxima is reached by as many words as there are parts
        uint32_t least = 0xffffffffu;
        if (lane < parts) {
            least = sh.wmax[buf][lane * span];
            if (span > 1) least = max(least, sh.wmax[buf][lane * span + 1]);
            if (span > 2) least = max(least, max(sh.wmax[buf][lane * span + 2], sh.wmax[buf][lane * span + 3]));
        }
        least = __reduce_min_sync(0xffffffffu, least);
        const float floor = logit_of(least);
        if (mine >= floor && mine > -INFINITY) {
            unsigned hits = 0;
            #pragma unroll
            for (int e = 0; e < kBmPer; ++e) hits |= x[e] >= floor && x[e] > -INFINITY ? 1u << e : 0u;
            int i = atomicAdd(&sh.count[b], __popc(hits));
            // (few as a rule, and still where they were read from)
            for (; hits != 0 && i < kBmList; hits &= hits - 1, ++i) {
                const int e = __ffs(hits) - 1;
                const float v = reinterpret_cast<const float*>(&here[(e >> 2) * kBmThreads + t])[e & 3];
                sh.list[b][i] = word_of(v, at + word_at<MODE>(e, t));
            }
        }
        if (cur.b != b) {
            const double all = warp_sum_d(sum);
            if (lane == 0) {
                sh.part[b][warp] = all;
                sh.ref[b][warp] = ref;
                if (warp == 0) sh.floor[b] = least;
            }
            sum = 0.0;
            ref = -INFINITY;
            run = 0;
        }
        buf ^= 1;
    }
    fetch_wait<0>();
    if (odd) sh.odd = 1;
    __syncthreads();
    if (t == 0 && sh.odd != 0) raise(a.status, SLLM_CUDA_ERR_ARG);
    // this CTA's best words of each beam, in order, into the first CTA's memory
    BeamShared& sh0 = *cl.map_shared_rank(&sh, 0);
    cl.sync();                      // the first CTA no longer needs its ring
    for (int r = warp; r < B; r += kBmWarps) {
        int c = sh.count[r];
        const float mine = lane < kBmWarps ? sh.ref[r][lane] : -INFINITY, all = warp_max(mine);
        const double s = warp_sum_d(mine > -INFINITY ? sh.part[r][lane] * sh.down_by(all - mine) : 0.0);
        if (lane == 0) {
            sh0.sum[rank][r] = s;
            sh0.refs[rank][r] = all;
        }
        if (c > kBmList) continue;
        // those that the last floor leaves, then each one's place
        Word* const list = sh.list[r];
        const Word least = (Word)sh.floor[r] << 32;
        int kept = 0;
        for (int i0 = 0; i0 < c; i0 += 32) {
            const Word w = i0 + lane < c ? list[i0 + lane] : 0;
            const unsigned m = __ballot_sync(0xffffffffu, w > least && w != 0);
            __syncwarp();
            if (w > least && w != 0) list[kept + __popc(m & ((1u << lane) - 1u))] = w;
            kept += __popc(m);
            __syncwarp();
        }
        c = kept;
        for (int i = lane; i < c || i < B; i += 32) {
            if (i >= c) {
                sh0.best[rank][r][i] = 0;
                continue;
            }
            const Word w = list[i];
            int place = 0;
            #pragma unroll 4
            for (int j = 0; j < c; ++j) place += list[j] > w ? 1 : 0;
            if (place < B) sh0.best[rank][r][place] = w;
        }
    }
    __syncthreads();
    for (int r = 0; r < B; ++r) {
        if (sh.count[r] <= kBmList) continue;       // the same for every thread
        Word last = ~0ull;
        for (int i = 0; i < B; ++i) {
            last = next_word(rows + (size_t)r * a.stride, lo, hi, last, sh.list[r]);
            if (t == 0) sh0.best[rank][r][i] = last;
        }
    }
    cl.sync();
    if (rank != 0) return;
    // merge: a warp per beam, a lane per CTA's list; then the candidates' values
    for (int r = warp; r < B; r += kBmWarps) {
        const bool on = (live >> r & 1) != 0;
        const float mine = on && lane < C ? sh.refs[lane][r] : -INFINITY, all = warp_max(mine);
        const double s = warp_sum_d(mine > -INFINITY ? sh.sum[lane][r] * sh.down_by(all - mine) : 0.0);
        const double lse = (double)all + log(s);
        int head = 0;
        Word w = on && lane < C ? sh.best[lane][r][0] : 0;
        for (int i = 0; i < B; ++i) {
            // of equal logits the first CTA's: its words come first
            const uint32_t key = (uint32_t)(w >> 32), top = __reduce_max_sync(0xffffffffu, key);
            const int who = __ffs(__ballot_sync(0xffffffffu, key == top)) - 1;
            if (lane == who) {
                sh.merged[r][i] = w;
                ++head;
                w = w != 0 && head < B ? sh.best[lane][r][head] : 0;
            }
        }
        __syncwarp();
        if (lane < B) {
            double v = -INFINITY;
            const Word m = sh.merged[r][lane];
            if (m != 0) v = (double)sh.score[r] + ((double)logit_of((uint32_t)(m >> 32)) - lse);
            if (!on && lane == 0 && sh.done[r] != 0 && sh.score[r] < INFINITY) v = (double)sh.score[r];
            sh.value[r * B + lane] = v;
        }
    }
    if (t < B) sh.pick[t] = -1;
    __syncthreads();
    // Each candidate's place among them: its beam's order is its rank's, so equal ones
    // go by number. 2^share threads count for one.
    const int all = B * B;
    int share = 0;
    while (share < 5 && all << (share + 1) <= kBmThreads) ++share;
    const int sub = 1 << share;
    if (t >> share < all) {
        const int i = t >> share;
        const double v = sh.value[i];
        int place = 0;
        for (int j = t & (sub - 1); j < all; j += sub) {
            const double o = sh.value[j];
            place += o > v || (o == v && j < i) ? 1 : 0;
        }
        const int in = all * sub - 32 * warp;       // of this warp's threads
        const unsigned m = in >= 32 ? 0xffffffffu : (1u << in) - 1u;
        for (int o = 1; o < sub; o <<= 1) place += __shfl_xor_sync(m, place, o);
        if ((t & (sub - 1)) == 0 && place < B && v > -INFINITY) sh.pick[place] = i;
    }
    __syncthreads();
    if (warp != 0) return;
    const bool mine = lane < B;
    const int won = mine ? sh.pick[lane] : -1;
    const int got = __popc(__ballot_sync(0xffffffffu, won >= 0));
    double pv = -INFINITY;
    int pb = -1, px = -1;
    if (won >= 0) {
        pb = won / B;
        pv = sh.value[won];
        px = sh.done[pb] != 0 ? a.eos : index_of(sh.merged[pb][won % B]);
    }
    // too few of weight: the first candidates of value -inf
    if (got < B) {
        int cb = 0, cx = 0;
        for (int i = got; i < B; ++i) {
            for (;;) {
                const bool d = sh.done[cb] != 0;
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
            a.done_out[o] = sh.done[pb] != 0 || px == a.eos ? 1 : 0;
        if (a.src != nullptr) a.src[o] = sh.slots[pb];
    }
}

// The CTAs of a request: what ends first when a piece takes 0.6 us, the rest of a
// CTA 6 us, and two CTAs are on an SM at a time.
int beam_cluster(int n, int beams, int n_vocab, int sms) {
    int best = 1;
    double least = 0.0;
    for (int C = 1; C <= 16; C *= 2) {
        const int per = (n_vocab + C - 1) / C, pieces = (per + kBmPiece - 1) / kBmPiece;
        const double cost = (double)(((long long)n * C + 2 * sms - 1) / (2 * sms)) * (0.6 * pieces * beams + 6.0);
        if (C == 1 || cost < least) {
            least = cost;
            best = C;
        }
    }
    return best;
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
