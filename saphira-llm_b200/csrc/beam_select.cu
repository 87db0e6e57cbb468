// beam_select.cu -- one step of beam search: the `beams` best continuations
// among beams * n_vocab candidates
//     score[b] + logits[b][x] - lse[b],    lse[b] = ln sum_y exp(logits[b][y]).
//
// The values are compared in 64 bits. Within a beam the order is that of the
// logits, so each beam needs its own best `beams` logits only, and its lse.
//
// One cluster of CTAs per request; each CTA has a share of the vocabulary of
// all beams and streams it once, a piece of 4096 words of one beam at a time, 16
// in the registers of a thread, the pieces behind it on their way into shared
// memory. A thread copies and reads its own words (4-byte copies where rows are
// not aligned), and keeps of a beam its largest logit and its sum of
// exponentials (terms and sums of 16 in 32 bits, else 64, against its own running
// maximum, rounded up to a power of two, or as it is where it is far from zero), so
// the stream has no barrier in it. What follows is short: of a beam's 256
// largest-of-a-thread the `beams`-th best is a bound that at least as many words
// reach; the few threads that reach it have their words read again (from L2), those
// words are put in order, and the first CTA of the cluster gets the lists through
// distributed shared memory and merges them. A list that overflows (many equal logits)
// is made word by word instead. Keeping lists while streaming, against bounds that the
// warps exchanged at a barrier per piece, took more clocks than the exponentials: 51 us
// for 32 requests of 8 beams.
//
// Bound: for many requests the exponentials and the loads together (32 of 8 beams,
// 128256 words, 118 to 131 MB: 37 us, 3.5 TB/s, a third of the exponential pipe and 45%
// of the issue slots), then the second look; for one request the chain load, bound,
// second look, merge (4 beams 13 us, 2 MB).

#include <cooperative_groups.h>

#include "serve.cuh"

namespace cg = cooperative_groups;

namespace sllm {
namespace {

constexpr int kBmThreads = 256;
constexpr int kBmWarps = kBmThreads / 32;
constexpr int kBmPer = 16;                          // words of a thread
constexpr int kBmPiece = kBmThreads * kBmPer;
constexpr int kBmMost = 16;                         // beams
constexpr int kBmList = 64;                         // words kept of a beam by a CTA

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

struct __align__(16) BeamShared {                 // behind it: most and list of each beam, then the ring
    double part[kBmMost][kBmWarps];                 // a warp's sum of e^(x - ref)
    float ref[kBmMost][kBmWarps];                   // and that ref, whole; -inf: no words
    int count[kBmMost];                             // words in the list
    float score[kBmMost];
    int done[kBmMost], slots[kBmMost];
    double sum[16][kBmMost];                        // [CTA][beam], of the cluster's first CTA, as are `best` and what follows
    float refs[16][kBmMost];
    Word merged[kBmMost][kBmMost];
    double value[kBmMost * kBmMost];
    int pick[kBmMost];                              // the chosen: beam * beams + rank
};
struct __align__(16) BeamRow {
    Word list[kBmList];
    uint32_t most[kBmThreads];      // keys of the threads' largest logits; later the pieces to look at again
    uint32_t next[kBmThreads];      // the piece that has it, and 16 bits of the largest key of the others
};
// [CTA][beam][rank], where the first CTA's ring was
using BeamBest = Word[kBmMost][kBmMost];

// Sums are of 2^(x log2 e - ref) with a whole ref, so those against two references
// differ by a power of two. log2 e is an f32, off by kBmLog2eOff of itself: what that
// makes of the largest logit is put right at the end. A largest logit beyond kBmFar is
// its own reference, m, and sums are of e^(x - m): of x log2 e a rounded reference
// would be off by more than an exponent holds. Such a reference is kept as 2 m,
// beyond all near ones, so that the order is that of the logits. Logits beyond 2^100
// count as that.
constexpr float kBmLog2e = 1.44269502162933349609375f, kBmFar = 0x1p24f, kBmHuge = 0x1p100f;
constexpr double kBmLog2eOff = 1.44269502162933349609375 / 1.4426950408889634074 - 1.0;
__device__ __forceinline__ float held(float x) { return fminf(fmaxf(x, -kBmHuge), kBmHuge); }
__device__ __forceinline__ double limited(uint32_t key) { return (double)held(logit_of(key)); }
__device__ __forceinline__ bool is_far(float ref) { return fabsf(ref) > 1.5f * kBmFar; }        // (a near one is below 1.4427 kBmFar)
__device__ __forceinline__ float ref_of(float most) {
    return fabsf(most) <= kBmFar ? ceilf(most * kBmLog2e) : 2.f * held(most);
}
// what sums against ref count in those against top >= ref
__device__ __forceinline__ double down_to(float top, float ref) {
    const float d = top - ref;
    if (is_far(top)) return (double)exp2f(-0.5f * d * kBmLog2e);
    return d < 1000.f ? __hiloint2double((1023 - (int)d) << 20, 0) : 0.0;
}

// x += a, y += b in one instruction
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
    asm("{\n\t.reg .b64 d, a;\n\t"
        "mov.b64 d, {%0, %1};\n\tmov.b64 a, {%2, %3};\n\t"
        "add.rn.f32x2 d, d, a;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(a), "f"(b));
}

// the sum of 2^((x - from) log2 e - ref) over a thread's words, two at a time
template <bool FROM>
__device__ __forceinline__ float sum_exp(const float (&x)[kBmPer], float from, float ref) {
    float e[kBmPer];
    #pragma unroll
    for (int i = 0; i < kBmPer; ++i) e[i] = x[i];
    #pragma unroll
    for (int i = 0; i < kBmPer; i += 2) {
        if (FROM) add2(e[i], e[i + 1], -from, -from);
        asm("{\n\t.reg .b64 x, l, r;\n\t"
            "mov.b64 x, {%0, %1};\n\tmov.b64 l, {%2, %2};\n\tmov.b64 r, {%3, %3};\n\t"
            "fma.rn.f32x2 x, x, l, r;\n\t"
            "mov.b64 {%0, %1}, x;\n\t}"
            : "+f"(e[i]), "+f"(e[i + 1])
            : "f"(kBmLog2e), "f"(-ref));
        asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e[i]));
        asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e[i + 1]));
    }
    #pragma unroll
    for (int n = kBmPer / 2; n > 1; n >>= 1)
        #pragma unroll
        for (int i = 0; i < n; i += 2) add2(e[i], e[i + 1], e[i + n], e[i + n + 1]);
    return e[0] + e[1];
}

// the largest of a thread's words, NaN if there is one
__device__ __forceinline__ float max_of(const float (&x)[kBmPer]) {
    float m = x[0];
    #pragma unroll
    for (int i = 1; i + 1 < kBmPer; i += 2) asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(x[i]), "f"(x[i + 1]));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(x[kBmPer - 1]));
    return m;
}

// 16 words of a thread: by fours where rows are 16-byte aligned, else one by one
template <bool VEC>
__device__ __forceinline__ int word_at(int e, int t) {
    return VEC ? 4 * (t + kBmThreads * (e >> 2)) + (e & 3) : t + kBmThreads * e;
}

// a thread's words of the piece at `lo`, on their way into its places of a ring entry
template <bool VEC>
__device__ __forceinline__ void fetch_piece(const float* row, int lo, int hi, float4* to) {
    const int t = threadIdx.x;
    #pragma unroll
    for (int e = 0; e < kBmPer; e += VEC ? 4 : 1) {
        const int i = lo + word_at<VEC>(e, t);
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to + (e / 4) * kBmThreads + t) + 4 * (e & 3);
        if (VEC && i + 4 <= hi)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(row + i) : "memory");
        else
            #pragma unroll
            for (int j = 0; j < (VEC ? 4 : 1); ++j)
                if (i + j < hi) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 4 * j), "l"(row + i + j) : "memory");
    }
}
__device__ __forceinline__ void fetch_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <bool VEC>
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
            if (lo + word_at<VEC>(e, t) >= hi) x[e] = -INFINITY;
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

// the words of one beam that are among this CTA's best: a warp
template <bool VEC>
__device__ __forceinline__ int collect(const float* row, int lo, int hi, BeamRow& sr, int B) {
    constexpr uint32_t NONE = 0x007fffffu;          // the key of -inf
    const int lane = threadIdx.x & 31;
    uint32_t k[kBmWarps], left[kBmWarps];
    #pragma unroll
    for (int i = 0; i < kBmWarps; ++i) left[i] = k[i] = sr.most[32 * i + lane];
    static_assert(kBmWarps == 8, "a sorting network of eight");
    constexpr int NET[19][2] = {{0, 1}, {2, 3}, {4, 5}, {6, 7}, {0, 2}, {1, 3}, {4, 6}, {5, 7}, {1, 2}, {5, 6},
                                {0, 4}, {1, 5}, {2, 6}, {3, 7}, {2, 4}, {3, 5}, {1, 2}, {3, 4}, {5, 6}};
    #pragma unroll
    for (int i = 0; i < 19; ++i) {
        const uint32_t x = left[NET[i][0]], y = left[NET[i][1]];
        left[NET[i][0]] = max(x, y);
        left[NET[i][1]] = min(x, y);
    }
    // the B-th largest; any number where there are not so many
    uint32_t floor = 0;
    for (int i = 0; i < B; ++i) {
        const uint32_t top = __reduce_max_sync(0xffffffffu, left[0]);
        floor = max(top, NONE + 1);
        if (top <= NONE) break;
        const bool mine = lane == __ffs(__ballot_sync(0xffffffffu, left[0] == top)) - 1;
        #pragma unroll
        for (int j = 0; j < kBmWarps; ++j) left[j] = mine ? (j + 1 < kBmWarps ? left[j + 1] : 0u) : left[j];
    }
    // the pieces that may hold words as large: of each thread that reaches it the one
    // with its largest, all where another may reach it, too
    const int pieces = (hi - lo + kBmPiece - 1) / kBmPiece;
    int tasks = 0;
    __syncwarp();                                   // (all keys are in registers)
    #pragma unroll
    for (int i = 0; i < kBmWarps; ++i) {
        const bool in = k[i] >= floor;
        const unsigned m = __ballot_sync(0xffffffffu, in);
        if (m == 0) continue;
        const uint32_t nx = sr.next[32 * i + lane], who = (uint32_t)(32 * i + lane) << 16;
        const bool many = in && (nx >> 16) >= (floor >> 16);
        const int n = !in ? 0 : many ? pieces : 1;
        int before = __popc(m & ((1u << lane) - 1u)), total = __popc(m);
        if (__any_sync(0xffffffffu, many)) {
            int upto = n;
            #pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            before = upto - n;
            total = __shfl_sync(0xffffffffu, upto, 31);
        }
        if (tasks + total > kBmThreads) return kBmList + 1;              // many equal ones
        for (int j = 0; j < n; ++j) sr.most[tasks + before + j] = who | (many ? (uint32_t)j : nx & 0xffffu);
        tasks += total;
    }
    __syncwarp();
    // their words again, four to a lane
    const float bound = logit_of(floor);
    const int all = tasks * (kBmPer / 4);
    int count = 0;
    auto place = [&](int i, int* x) {               // the first of lane's four words of batch i, or none
        const bool in = i + lane < all;
        const uint32_t task = in ? sr.most[(i + lane) / (kBmPer / 4)] : 0;
        *x = lo + (int)(task & 0xffffu) * kBmPiece + word_at<VEC>(lane % (kBmPer / 4) * 4, (int)(task >> 16));
        return in;
    };
    auto load = [&](int x, bool in) {
        float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        constexpr int STEP = VEC ? 1 : kBmThreads;
        if (VEC && in && x + 4 <= hi) return __ldg(reinterpret_cast<const float4*>(row + x));
        if (in && x < hi) v.x = __ldg(row + x);
        if (in && x + STEP < hi) v.y = __ldg(row + x + STEP);
        if (in && x + 2 * STEP < hi) v.z = __ldg(row + x + 2 * STEP);
        if (in && x + 3 * STEP < hi) v.w = __ldg(row + x + 3 * STEP);
        return v;
    };
    int x, nx = 0;
    bool in = place(0, &x);
    float4 v = load(x, in), nv = v;
    #pragma unroll 1
    for (int i = 0; i < all; i += 32) {
        if (i + 32 < all) {
            in = place(i + 32, &nx);
            nv = load(nx, in);
        }
        #pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float f = e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w;
            const bool hit = f >= bound && f < INFINITY;
            const unsigned m = __ballot_sync(0xffffffffu, hit);
            const int to = count + __popc(m & ((1u << lane) - 1u));
            if (hit && to < kBmList) sr.list[to] = word_of(f, x + e * (VEC ? 1 : kBmThreads));
            count += __popc(m);
        }
        x = nx;
        v = nv;
    }
    __syncwarp();
    return count;
}

// RING: pieces in shared memory or on their way
template <bool VEC, int RING>
__global__ void __launch_bounds__(kBmThreads, 3)
beam_select_kernel(const __grid_constant__ BeamParams a) {
    extern __shared__ __align__(16) uint8_t smem[];
    BeamShared& sh = *reinterpret_cast<BeamShared*>(smem);
    BeamRow* const by_row = reinterpret_cast<BeamRow*>(smem + sizeof(BeamShared));
    const int B = a.beams;
    float4 (*const ring)[kBmPiece / 4] = reinterpret_cast<float4 (*)[kBmPiece / 4]>(by_row + B);
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int req = blockIdx.x / C, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int lo = (int)min((long long)rank * a.per, (long long)a.V), hi = min(a.V, lo + a.per);
    const float* const rows = a.logits + (size_t)req * B * a.stride;
    // beams that have words to offer: not done, of a score above -inf
    float my_score = 0.f;
    int my_done = 0, my_slot = 0;
    if (lane < B) {
        my_score = a.score[(size_t)req * B + lane];
        if (a.done != nullptr) my_done = a.done[(size_t)req * B + lane];
        if (warp == 0 && a.slots != nullptr) my_slot = a.slots[(size_t)req * B + lane];
    }
    // (a warp's own column: the stream has no barrier)
    if (lane < kBmMost) sh.ref[lane][warp] = -INFINITY;
    __syncwarp();
    const unsigned live = __ballot_sync(0xffffffffu, lane < B && my_done == 0 && my_score > -INFINITY && my_score < INFINITY);
    bool odd = lane < B && !(my_score < INFINITY);
    if (warp == 0 && lane < B) {
        sh.score[lane] = my_score;
        sh.done[lane] = my_done;
        sh.slots[lane] = my_slot;
    }
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
    Piece cur{live != 0 && lo < hi ? __ffs(live) - 1 : B, lo}, ahead = cur;
    int entry = 0, fill = 0;
    #pragma unroll
    for (int i = 0; i < RING - 1; ++i) {
        if (ahead.b < B) {
            fetch_piece<VEC>(rows + (size_t)ahead.b * a.stride, ahead.at, hi, ring[fill]);
            ahead = after(ahead);
        }
        fetch_end();
        fill = i + 1;
    }
    // of the beam so far: the reference, this thread's largest logit, the piece that
    // has it, the largest of the other pieces
    float ref = -INFINITY, most = -INFINITY, other = -INFINITY;
    int piece = 0, at_piece = 0;
    double sum = 0.0;
    while (cur.b < B) {
        const int b = cur.b;
        float x[kBmPer];
        fetch_wait<RING - 2>();
        take_piece<VEC>(ring[entry], cur.at, hi, x);
        // (this thread's places of the entry that it read last are free)
        if (ahead.b < B) {
            fetch_piece<VEC>(rows + (size_t)ahead.b * a.stride, ahead.at, hi, ring[fill]);
            ahead = after(ahead);
        }
        fetch_end();
        entry = entry + 1 == RING ? 0 : entry + 1;
        fill = fill + 1 == RING ? 0 : fill + 1;
        cur = after(cur);
        float mine = max_of(x);
        if (!(mine < INFINITY)) {                   // +inf and NaN count as -inf
            odd = true;
            #pragma unroll
            for (int e = 0; e < kBmPer; ++e) x[e] = x[e] < INFINITY ? x[e] : -INFINITY;
            mine = max_of(x);
        }
        other = fmaxf(other, fminf(most, mine));
        if (mine > most) {
            most = mine;
            at_piece = piece;
        }
        ++piece;
        if (most > -INFINITY) {
            const float want = ref_of(most);
            if (want > ref) {
                sum = ref > -INFINITY ? sum * down_to(want, ref) : 0.0;
                ref = want;
            }
        }
        // (a thread without words yet: its terms are 0 against any reference; together, as
        // far words among near ones would else take both ways)
        const bool far = is_far(ref) && ref > -INFINITY;
        if (!__any_sync(0xffffffffu, far)) {
            sum += (double)sum_exp<false>(x, 0.f, ref > -INFINITY ? ref : 0.f);
        } else {
            const float from = far ? 0.5f * ref : 0.f;
            if (fabsf(from) == kBmHuge) {
                #pragma unroll
                for (int e = 0; e < kBmPer; ++e) x[e] = x[e] > -INFINITY ? held(x[e]) : x[e];
            }
            sum += (double)sum_exp<true>(x, from, far || !(ref > -INFINITY) ? 0.f : ref);
        }
        if (cur.b != b) {
            by_row[b].most[t] = key_of(most);
            by_row[b].next[t] = (key_of(other) & 0xffff0000u) | (uint32_t)at_piece;
            const float top = logit_of(__reduce_max_sync(0xffffffffu, key_of(ref)));
            const double all = warp_sum_d(ref > -INFINITY ? sum * down_to(top, ref) : 0.0);
            if (lane == 0) {
                sh.part[b][warp] = all;
                sh.ref[b][warp] = top;
            }
            sum = 0.0;
            ref = most = other = -INFINITY;
            piece = at_piece = 0;
        }
    }
    fetch_wait<0>();
    if (__any_sync(0xffffffffu, odd) && lane == 0) raise(a.status, SLLM_CUDA_ERR_ARG);
    cl.sync();                      // the first CTA no longer needs its ring (and this CTA's shared memory is written)
    // this CTA's best words of each beam, in order, into the first CTA's memory
    BeamShared& sh0 = *cl.map_shared_rank(&sh, 0);
    BeamBest* const best = reinterpret_cast<BeamBest*>(ring);
    BeamBest& best0 = *cl.map_shared_rank(best + rank, 0);
    for (int r = warp; r < B; r += kBmWarps) {
        const bool on = (live >> r & 1) != 0 && lo < hi;
        const int c = on ? collect<VEC>(rows + (size_t)r * a.stride, lo, hi, by_row[r], B) : 0;
        const float mine = lane < kBmWarps ? sh.ref[r][lane] : -INFINITY, all = warp_max(mine);
        const double s = warp_sum_d(mine > -INFINITY ? sh.part[r][lane] * down_to(all, mine) : 0.0);
        if (lane == 0) {
            sh.count[r] = c;
            sh0.sum[rank][r] = s;
            sh0.refs[rank][r] = all;
        }
        if (c > kBmList) continue;
        const Word* const list = by_row[r].list;
        for (int i = lane; i < c || i < B; i += 32) {
            if (i >= c) {
                best0[r][i] = 0;
                continue;
            }
            const Word w = list[i];
            int place = 0;
            #pragma unroll 4
            for (int j = 0; j < c; ++j) place += list[j] > w ? 1 : 0;
            if (place < B) best0[r][place] = w;
        }
    }
    __syncthreads();
    for (int r = 0; r < B; ++r) {
        if (sh.count[r] <= kBmList) continue;       // the same for every thread
        Word last = ~0ull;
        for (int i = 0; i < B; ++i) {
            last = next_word(rows + (size_t)r * a.stride, lo, hi, last, by_row[r].list);
            if (t == 0) best0[r][i] = last;
        }
    }
    cl.sync();
    if (rank != 0) return;
    // merge: a warp per beam, a lane per CTA's list; then the candidates' values
    for (int r = warp; r < B; r += kBmWarps) {
        const bool on = (live >> r & 1) != 0;
        const float mine = on && lane < C ? sh.refs[lane][r] : -INFINITY, all = warp_max(mine);
        const double s = warp_sum_d(mine > -INFINITY ? sh.sum[lane][r] * down_to(all, mine) : 0.0);
        int head = 0;
        Word w = on && lane < C ? best[lane][r][0] : 0;
        for (int i = 0; i < B; ++i) {
            // of equal logits the first CTA's: its words come first
            const uint32_t key = (uint32_t)(w >> 32), top = __reduce_max_sync(0xffffffffu, key);
            const int who = __ffs(__ballot_sync(0xffffffffu, key == top)) - 1;
            if (lane == who) {
                sh.merged[r][i] = w;
                ++head;
                w = w != 0 && head < B ? best[lane][r][head] : 0;
            }
        }
        __syncwarp();
        const double top = limited((uint32_t)(sh.merged[r][0] >> 32));
        // (of far logits both are counted from the largest: lse would round its logarithm away)
        const double from = is_far(all) ? top : 0.0;
        const double lse = is_far(all) ? log(s) : ((double)all + log2(s)) * 0.69314718055994530942 - top * kBmLog2eOff;
        if (lane < B) {
            double v = -INFINITY;
            const Word m = sh.merged[r][lane];
            if (m != 0) v = (double)sh.score[r] + (limited((uint32_t)(m >> 32)) - from - lse);
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

// The CTAs of a request: what ends first when a piece takes 0.25 us, the rest of a
// CTA 6 us, and three CTAs are on an SM at a time; of clusters of 16, which find room
// in few places, two (24 requests of 8 beams, 128256 words: 46 us in clusters of 16, 37
// in clusters of 8; 16 requests of 4 beams 19.0, 21.2). Other sizes than powers of two
// were no better for any of fifteen shapes by more than 3%.
int beam_cluster(int n, int beams, int n_vocab, int sms) {
    int best = 1;
    double least = 0.0;
    for (int C = 1; C <= 16; C *= 2) {
        const int per = (n_vocab + C - 1) / C, pieces = (per + kBmPiece - 1) / kBmPiece;
        const int room = (C == 16 ? 2 : 3) * sms;
        const double cost = (double)(((long long)n * C + room - 1) / room) * (0.25 * pieces * beams + 6.0);
        if (C == 1 || cost < least) {
            least = cost;
            best = C;
        }
    }
    return best;
}

template <bool VEC, int RING>
cudaError_t launch_ring(const BeamParams& a, int C, cudaStream_t st) {
    constexpr int kRing = RING * kBmPiece * (int)sizeof(float), kMost = (int)sizeof(BeamShared) + kBmMost * (int)sizeof(BeamRow) + kRing;
    static_assert(kRing >= (int)(16 * sizeof(BeamBest)) && kBmPiece * 256 >= 1 << 20 && sizeof(BeamShared) % 16 == 0 && sizeof(BeamRow) % 16 == 0, "");
    const cudaError_t e1 = allow_smem<beam_select_kernel<VEC, RING>>(kMost), e2 = allow_cluster<beam_select_kernel<VEC, RING>>();
    if (e1 != cudaSuccess || e2 != cudaSuccess) return e1 != cudaSuccess ? e1 : e2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a.n * C));
    cfg.blockDim = dim3(kBmThreads);
    cfg.dynamicSmemBytes = sizeof(BeamShared) + a.beams * sizeof(BeamRow) + kRing;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = C;
    at.val.clusterDim.y = 1;
    at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, beam_select_kernel<VEC, RING>, a);
}
// where each CTA has an SM of its own (and clusters find room), more of its pieces are on their way
template <bool VEC>
cudaError_t launch_beam(const BeamParams& a, int C, int sms, cudaStream_t st) {
    return 2LL * a.n * C <= sms ? launch_ring<VEC, 8>(a, C, st) : launch_ring<VEC, 3>(a, C, st);
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
    const int sms = current_sms(), C = beam_cluster(n, beams, n_vocab, sms);
    a.per = ((n_vocab + C - 1) / C + 3) / 4 * 4;
    const bool vec = row_stride % 4 == 0 && aligned16(logits);
    const cudaStream_t st = (cudaStream_t)stream;
    CK(vec ? launch_beam<true>(a, C, sms, st) : launch_beam<false>(a, C, sms, st), "beam_select launch");
    count_launches(1);
    return SLLM_CUDA_OK;
}
