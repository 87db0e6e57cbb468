// spec_verify.cu -- drafted tokens against the target's probabilities.
//
// For each sequence: token t of the draft is accepted while
// u_t * q_t(x_t) < p_t(x_t); at the first refusal r the next token is drawn
// from max(p_r - q_r, 0), after the last accepted one from p, by inversion:
// the first index whose running sum exceeds u * total. The sums are held in
// 64 bits, so the order in which threads add them moves a border by about
// 1e-16 of the total: the same token comes out of any order, except for a u
// that lies that close to a border.
//
// One cluster of CTAs per sequence, each warp a contiguous run of the
// vocabulary. One pass over the two rows gives each warp its sum; the cluster
// exchanges its CTAs' sums through distributed shared memory, and the CTA whose
// run holds the draw walks that run again.
// What is rare costs another pass: a residual without mass (p stands in), and
// infinities, which count as nothing.
//
// Bound: for one sequence the chain of dependent reads: lengths and tokens,
// their probabilities, the rows, the run again (measured 9.5 us); for many the
// loads of a row's pass, four of each row in flight a warp, summed before the next
// (64 of 128256 words: 17.3 us, 3.8 TB/s, 10.2 us for the two rows that each needs
// at the memory's rate; 256: 57.5 us, 4.6 TB/s, 41 us).

#include <cooperative_groups.h>

#include "serve.cuh"

namespace cg = cooperative_groups;

namespace sllm {
namespace {

constexpr int kSvThreads = 256;
constexpr int kSvWarps = kSvThreads / 32;
constexpr int kSvMaxDraft = 64;

struct VerifyParams {
    const float* p;                 // [n][k + 1][V]
    const float* q;                 // [n][k][V] or NULL: the draft was certain of its tokens
    const int32_t* draft;           // [n][k]
    const int32_t* n_draft;         // [n] or NULL: k for all
    const float* u_accept;          // [n][k]
    const float* u_draw;            // [n]
    int32_t* tokens;                // [n][k + 1]
    int32_t* count;                 // [n]
    int k, V, vec;                  // vec: rows are 16-byte aligned
    int32_t* status;
};

// what an entry counts for: nothing when negative, NaN or infinite
__device__ __forceinline__ float prob(float x) { return x > 0.0f && x < INFINITY ? x : 0.0f; }

template <bool VEC>
__device__ __forceinline__ float4 row4(const float* row, int i, int hi) {
    if (row == nullptr || i >= hi) return make_float4(0.f, 0.f, 0.f, 0.f);
    if (VEC && i + 4 <= hi) return __ldg(reinterpret_cast<const float4*>(row + i));
    float4 r;
    r.x = __ldg(row + i);
    r.y = i + 1 < hi ? __ldg(row + i + 1) : 0.f;
    r.z = i + 2 < hi ? __ldg(row + i + 2) : 0.f;
    r.w = i + 3 < hi ? __ldg(row + i + 3) : 0.f;
    return r;
}

// the distribution that is drawn from
struct Draw {
    const float* p;
    const float* q;                 // NULL: nothing is subtracted
    int skip;                       // an index without mass (the refused token of a certain draft), or -1
};

__device__ __forceinline__ double mass_at(const Draw& d, float p, float q, int i) {
    if (i == d.skip) return 0.0;
    const float a = prob(p), b = prob(q);
    return a > b ? (double)a - (double)b : 0.0;
}

// the sum over [lo, hi) by one warp. Quick: negatives and NaN count as
// nothing; an infinity comes out as a sum that is not finite, or in *odd.
template <bool VEC, bool QUICK>
__device__ __forceinline__ double run_sum(const Draw& d, int lo, int hi, bool* odd) {
    const int lane = threadIdx.x & 31;
    double s0 = 0.0, s1 = 0.0;
    float top = 0.f;
    for (int i0 = lo; i0 < hi; i0 += 512) {
        float4 pv[4], qv[4];
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = i0 + 128 * j + 4 * lane;
            pv[j] = row4<VEC>(d.p, i, hi);
            qv[j] = row4<VEC>(d.q, i, hi);
        }
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = i0 + 128 * j + 4 * lane;
            const float pe[4] = {pv[j].x, pv[j].y, pv[j].z, pv[j].w};
            const float qe[4] = {qv[j].x, qv[j].y, qv[j].z, qv[j].w};
            #pragma unroll
            for (int e = 0; e < 4; ++e) {
                double m;
                if (QUICK) {
                    const float a = i + e == d.skip ? 0.f : fmaxf(pe[e], 0.f);
                    const float b = fmaxf(qe[e], 0.f);
                    top = fmaxf(top, b);
                    m = (double)a - (double)fminf(a, b);        // exact where a <= b: 0
                } else {
                    m = mass_at(d, pe[e], qe[e], i + e);
                }
                if (e & 1) s1 += m;
                else s0 += m;
            }
        }
    }
    if (QUICK) *odd = __any_sync(0xffffffffu, top == INFINITY);
    return warp_sum_d(s0 + s1);
}

// the last index with mass below hi, by one warp; -1 when there is none
template <bool VEC>
__device__ __noinline__ int last_mass(const Draw& d, int hi) {
    const int lane = threadIdx.x & 31;
    for (int i0 = (hi - 1) & ~31; i0 >= 0; i0 -= 32) {
        const int i = i0 + lane;
        const bool has = i < hi && mass_at(d, d.p[i], d.q != nullptr ? d.q[i] : 0.f, i) > 0.0;
        const unsigned any = __ballot_sync(0xffffffffu, has);
        if (any != 0) return i0 + 31 - __clz(any);
    }
    return -1;
}

// the first index of [lo, hi) with mass whose running sum, from `before`,
// exceeds target, by one warp; -1 when the sums' rounding leaves none
template <bool VEC>
__device__ __forceinline__ int find_in_run(const Draw& d, int lo, int hi, double before, double target) {
    const int lane = threadIdx.x & 31;
    const int per = ((hi - lo + 31) / 32 + 3) & ~3, a = min(lo + lane * per, hi), z = min(a + per, hi);
    double own = 0.0;
    #pragma unroll 4
    for (int i = a; i < z; i += 4) {
        const float4 pv = row4<VEC>(d.p, i, z), qv = row4<VEC>(d.q, i, z);
        own += (mass_at(d, pv.x, qv.x, i) + mass_at(d, pv.y, qv.y, i + 1)) +
               (mass_at(d, pv.z, qv.z, i + 2) + mass_at(d, pv.w, qv.w, i + 3));
    }
    double x = own;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    // lanes from the first that may hold it: a border that rounding moved
    // across a lane's end is found by the next one
    const unsigned may = __ballot_sync(0xffffffffu, own > 0.0 && before + x > target);
    if (may == 0) return -1;
    const int l = __ffs(may) - 1;
    int found = -1;
    if (lane == l) {
        double run = before + (x - own);
        int last = -1;
        #pragma unroll 2
        for (int i = a; i < z && found < 0; i += 4) {
            const float4 pv = row4<VEC>(d.p, i, z), qv = row4<VEC>(d.q, i, z);
            const float pe[4] = {pv.x, pv.y, pv.z, pv.w}, qe[4] = {qv.x, qv.y, qv.z, qv.w};
            #pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double m = mass_at(d, pe[e], qe[e], i + e);
                run += m;
                if (found < 0 && m > 0.0) {         // an entry without mass is never drawn
                    last = i + e;
                    if (run > target) found = i + e;
                }
            }
        }
        if (found < 0) found = last;
    }
    return __shfl_sync(0xffffffffu, found, l);
}

template <bool VEC>
__global__ void __launch_bounds__(kSvThreads, 4)
spec_verify_kernel(const __grid_constant__ VerifyParams a) {
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int b = blockIdx.x / C, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    __shared__ double s_sum[kSvWarps], cta_sum;
    __shared__ int first_refusal, s_odd, cta_odd;
    const int V = a.V, k = a.k;
    const int nd_raw = a.n_draft != nullptr ? a.n_draft[b] : k;
    const int nd = min(max(nd_raw, 0), k);
    if (t == 0) {
        first_refusal = nd;
        if (rank == 0 && nd != nd_raw) raise(a.status, SLLM_CUDA_ERR_ARG);
    }
    __syncthreads();
    const float* P = a.p + (size_t)b * (k + 1) * V;
    const float* Q = a.q != nullptr ? a.q + (size_t)b * k * V : nullptr;
    if (t < nd) {
        const int x = a.draft[(size_t)b * k + t];
        bool ok = false;
        if (x >= 0 && x < V) {
            const double px = (double)prob(P[(size_t)t * V + x]);
            const double qx = Q != nullptr ? (double)prob(Q[(size_t)t * V + x]) : 1.0;
            ok = (double)a.u_accept[(size_t)b * k + t] * qx < px;     // exact in 64 bits
        } else if (rank == 0) {
            raise(a.status, SLLM_CUDA_ERR_ARG);                       // no such token: refused
        }
        if (!ok) atomicMin(&first_refusal, t);
    }
    __syncthreads();
    const int r = first_refusal;
    Draw d{P + (size_t)r * V, nullptr, -1};
    bool residual = r < nd;
    if (residual) {
        if (Q != nullptr) d.q = Q + (size_t)r * V;
        else d.skip = a.draft[(size_t)b * k + r];
    }
    // this warp's run: a multiple of 128 indices, so that a step of the warp
    // reads 512 contiguous bytes
    const int per = ((V + C * kSvWarps - 1) / (C * kSvWarps) + 127) / 128 * 128;
    const int lo = (int)min((long long)(rank * kSvWarps + warp) * per, (long long)V), hi = min(V, lo + min(per, V - lo));
    double total, before = 0.0, target;
    int owner;
    for (bool quick = true;;) {
        bool odd = false;
        const double sum = quick ? run_sum<VEC, true>(d, lo, hi, &odd) : run_sum<VEC, false>(d, lo, hi, &odd);
        if (t == 0) s_odd = 0;
        __syncthreads();
        if (lane == 0) {
            s_sum[warp] = sum;
            if (odd) s_odd = 1;
        }
        __syncthreads();
        if (t == 0) {
            double x = 0.0;
            for (int w = 0; w < kSvWarps; ++w) x += s_sum[w];
            cta_sum = x;
            cta_odd = s_odd;
        }
        cl.sync();
        // every warp adds the CTAs' sums in the same way, a lane per CTA, and
        // finds the one that holds the draw
        const double part = lane < C ? *cl.map_shared_rank(&cta_sum, lane) : 0.0;
        const bool odds = __any_sync(0xffffffffu, lane < C && *cl.map_shared_rank(&cta_odd, lane) != 0);
        double upto = part;
        #pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        total = __shfl_sync(0xffffffffu, upto, C - 1);
        target = fmax((double)a.u_draw[b], 0.0) * total;
        const unsigned hit = __ballot_sync(0xffffffffu, part > 0.0 && upto > target);
        owner = __ffs(hit) - 1;
        before = __shfl_sync(0xffffffffu, upto - part, max(owner, 0));
        cl.sync();                  // remote reads done: the sums may be replaced, a CTA may leave
        if (quick && (odds || !(total < INFINITY))) {
            quick = false;          // the infinities have to be told apart
        } else if (residual && total <= 0.0) {
            residual = false;       // p lies below q everywhere: p itself
            d.q = nullptr;
            d.skip = -1;
        } else {
            break;
        }
    }
    int32_t* const out = a.tokens + (size_t)b * (k + 1);
    // the accepted tokens, and -1 behind the drawn one
    if (rank == 0) {
        if (t <= k && t != r) out[t] = t < r ? a.draft[(size_t)b * k + t] : -1;
        if (t == 0) {
            a.count[b] = r + 1;
            if (total <= 0.0) out[r] = -1;          // no mass at all: no token
        }
    }
    if (total <= 0.0 || (owner >= 0 ? owner != rank : rank != 0)) return;
    // the run that holds it, then which eighth of that run (a warp each, from
    // L2), then the index. Where the rounding of the sums leaves no such run,
    // eighth or index: the last index with mass before the border
    auto pick = [&](const double* sums) {
        int at = -1;
        for (int w = 0; w < kSvWarps && at < 0; ++w) {
            if (sums[w] > 0.0 && before + sums[w] > target) at = w;
            else before += sums[w];
        }
        return at;
    };
    int limit = V, found = -1, leader = 0;
    if (owner >= 0) {
        limit = (int)min((long long)V, (long long)(rank + 1) * kSvWarps * per);
        const int mine = pick(s_sum);
        if (mine >= 0) {
            const int first = (rank * kSvWarps + mine) * per, end = min(V, first + per);
            const int piece = ((end - first + kSvWarps - 1) / kSvWarps + 127) / 128 * 128;
            const int a0 = min(first + warp * piece, end), a1 = min(a0 + piece, end);
            const double sum = run_sum<VEC, false>(d, a0, a1, nullptr);
            __shared__ double s_piece[kSvWarps];
            if (lane == 0) s_piece[warp] = sum;
            __syncthreads();
            const int eighth = pick(s_piece);
            limit = end;
            if (eighth >= 0) {
                leader = eighth;
                limit = min(first + (eighth + 1) * piece, end);
                if (warp == leader) found = find_in_run<VEC>(d, a0, a1, before, target);
            }
        }
    }
    if (warp != leader) return;
    if (found < 0) found = last_mass<VEC>(d, limit);
    if (lane == 0) out[r] = found;
}

// The CTAs of a sequence. Twice as many halve the time of a row's pass, which
// is about 0.35 us per 1000 words of a CTA, and cost what the launch of more
// clusters costs: nothing up to two CTAs per SM, about 2 us up to four, 8 us up
// to eight; clusters of 16 as much as four times their CTAs. Measured, clusters
// of 1, 2, 4, 8, 16, us:
//      1 sequence  of   4096 words   7.7   7.3   7.5   7.3   7.8
//      1              128256        50.2  28.1  15.6  11.4   8.9
//     64               32000        16.7  11.6  10.0  10.8  22.6
//     64              128256        60.6  31.6  20.6  17.2  27.9
//    256                4096         8.7  10.1  17.1  27.1  66.1
//    256              128256        82.7  61.8  60.3  60.9  96.0
int cluster_size(int n, int n_vocab, int sms) {
    int C = 1;
    while (C < 16) {
        const long long ctas = 2LL * C * n * (C == 8 ? 4 : 1);
        const int worth = ctas <= 2LL * sms ? 6144 : ctas <= 4LL * sms ? 12288 : 40960;     // words of a CTA
        if (ctas > 8LL * sms || n_vocab / C < worth) break;
        C *= 2;
    }
    return C;
}

}  // namespace
}  // namespace sllm

using namespace sllm;

extern "C" int sllm_cuda_spec_verify(const float* p, const float* q, const int32_t* draft, const int32_t* n_draft,
                                     const float* u_accept, const float* u_draw, int32_t n, int32_t k,
                                     int32_t n_vocab, int32_t* tokens, int32_t* count, int32_t* status,
                                     void* stream) {
    if (p == nullptr || draft == nullptr || u_accept == nullptr || u_draw == nullptr || tokens == nullptr ||
        count == nullptr)
        return fail(SLLM_CUDA_ERR_ARG, "spec_verify: a NULL array");
    if (n < 0 || n > 65536 || k < 1 || k > kSvMaxDraft || n_vocab < 1 || n_vocab > (1 << 24))
        return fail(SLLM_CUDA_ERR_ARG, "spec_verify: %d sequences, %d drafted tokens (1 to %d), %d words", n, k,
                    kSvMaxDraft, n_vocab);
    const void* ptr[] = {p, q, draft, n_draft, u_accept, u_draw, tokens, count, status};
    const char* name[] = {"p", "q", "draft", "n_draft", "u_accept", "u_draw", "tokens", "count", "status"};
    for (int i = 0; i < 9; ++i) {
        if (ptr[i] == nullptr) continue;
        const int rc = need_device(ptr[i], "spec_verify", name[i]);
        if (rc != SLLM_CUDA_OK) return rc;
    }
    if (n == 0) return SLLM_CUDA_OK;
    VerifyParams a{};
    a.p = p; a.q = q; a.draft = draft; a.n_draft = n_draft;
    a.u_accept = u_accept; a.u_draw = u_draw;
    a.tokens = tokens; a.count = count;
    a.k = k; a.V = n_vocab;
    a.vec = n_vocab % 4 == 0 && aligned16(p) && (q == nullptr || aligned16(q));
    a.status = status;
    const int C = cluster_size(n, n_vocab, current_sms());
    if (C == 16) {
        const cudaError_t e1 = allow_cluster<spec_verify_kernel<true>>(), e2 = allow_cluster<spec_verify_kernel<false>>();
        CK(e1 != cudaSuccess ? e1 : e2, "spec_verify clusters");
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(n * C));
    cfg.blockDim = dim3(kSvThreads);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = C;
    at.val.clusterDim.y = 1;
    at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    CK(a.vec ? cudaLaunchKernelEx(&cfg, spec_verify_kernel<true>, a) : cudaLaunchKernelEx(&cfg, spec_verify_kernel<false>, a),
       "spec_verify launch");
    count_launches(1);
    return SLLM_CUDA_OK;
}
