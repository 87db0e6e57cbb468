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
// vocabulary: one pass over the two rows gives each warp its sums of p and
// of max(p - q, 0) (the second may have no mass, then p stands in), the
// cluster exchanges its CTAs' sums through distributed shared memory, and the
// one warp whose run holds the draw walks it again (from L2). Bound by HBM
// for many sequences and by this chain of dependent steps for one.

#include <cooperative_groups.h>

#include "serve.cuh"

namespace cg = cooperative_groups;

namespace sllm {
namespace {

constexpr int kSvThreads = 512;
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
__device__ __forceinline__ double mass(double x) { return x > 0.0 && x < INFINITY ? x : 0.0; }

__device__ __forceinline__ float prob(float x) { return x > 0.0f && x < INFINITY ? x : 0.0f; }

struct Pair2 {
    double res, all;
};

template <bool VEC>
__device__ __forceinline__ float4 row4(const float* row, int i, int hi) {
    if (row == nullptr) return make_float4(0.f, 0.f, 0.f, 0.f);
    if (VEC && i + 4 <= hi) return __ldg(reinterpret_cast<const float4*>(row + i));
    float4 r;
    r.x = i < hi ? __ldg(row + i) : 0.f;
    r.y = i + 1 < hi ? __ldg(row + i + 1) : 0.f;
    r.z = i + 2 < hi ? __ldg(row + i + 2) : 0.f;
    r.w = i + 3 < hi ? __ldg(row + i + 3) : 0.f;
    return r;
}

// the mass of index i: p alone, p - q, or p without the refused token
__device__ __forceinline__ double mass_at(float p, float q, int i, int refused, bool point, bool residual) {
    const double a = (double)prob(p);
    if (!residual || refused < 0) return a;
    if (point) return i == refused ? 0.0 : a;
    return mass(a - (double)prob(q));
}

template <bool VEC>
__global__ void __launch_bounds__(kSvThreads)
spec_verify_kernel(const __grid_constant__ VerifyParams a) {
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int b = blockIdx.x / C, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    __shared__ double s_res[kSvWarps], s_all[kSvWarps], cta_res, cta_all;
    __shared__ int first_refusal, s_last_res[kSvWarps], s_last_all[kSvWarps], cta_last_res, cta_last_all;
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
    for (int i = t; i < nd; i += kSvThreads) {
        const int x = a.draft[(size_t)b * k + i];
        bool ok = false;
        if (x >= 0 && x < V) {
            const double px = (double)prob(P[(size_t)i * V + x]);
            const double qx = Q != nullptr ? (double)prob(Q[(size_t)i * V + x]) : 1.0;
            ok = (double)a.u_accept[(size_t)b * k + i] * qx < px;     // exact in 64 bits
        } else if (rank == 0) {
            raise(a.status, SLLM_CUDA_ERR_ARG);                       // no such token: refused
        }
        if (!ok) atomicMin(&first_refusal, i);
    }
    __syncthreads();
    const int r = first_refusal;
    // the refused token (V: one that is no token), -1 when none was refused
    int refused = -1;
    if (r < nd) {
        const int x = a.draft[(size_t)b * k + r];
        refused = x >= 0 && x < V ? x : V;
    }
    const bool point = Q == nullptr;
    const float* prow = P + (size_t)r * V;
    const float* qrow = refused >= 0 && !point ? Q + (size_t)r * V : nullptr;

    // this warp's run: a multiple of 128 indices, so that a step of the warp
    // reads 512 contiguous bytes
    const int runs = C * kSvWarps;
    const int per = ((V + runs - 1) / runs + 127) / 128 * 128;
    const long long lo_l = (long long)(rank * kSvWarps + warp) * per;
    const int lo = (int)(lo_l < V ? lo_l : V), hi = min((long long)V, lo_l + per) > lo ? (int)min((long long)V, lo_l + per) : lo;
    Pair2 sum{0.0, 0.0};
    int last_res = -1, last_all = -1;
    for (int i0 = lo; i0 < hi; i0 += 512) {
        float4 pv[4], qv[4];
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = i0 + 128 * j + 4 * lane;
            pv[j] = row4<VEC>(i < hi ? prow : nullptr, i, hi);
            qv[j] = row4<VEC>(i < hi ? qrow : nullptr, i, hi);
        }
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = i0 + 128 * j + 4 * lane;
            const float pe[4] = {pv[j].x, pv[j].y, pv[j].z, pv[j].w};
            const float qe[4] = {qv[j].x, qv[j].y, qv[j].z, qv[j].w};
            #pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double all = (double)prob(pe[e]);
                const double res = mass_at(pe[e], qe[e], i + e, refused, point, true);
                sum.all += all;
                sum.res += res;
                if (all > 0.0) last_all = i + e;
                if (res > 0.0) last_res = i + e;
            }
        }
    }
    sum.res = warp_sum_d(sum.res);
    sum.all = warp_sum_d(sum.all);
    last_res = __reduce_max_sync(0xffffffffu, last_res);
    last_all = __reduce_max_sync(0xffffffffu, last_all);
    if (lane == 0) {
        s_res[warp] = sum.res;
        s_all[warp] = sum.all;
        s_last_res[warp] = last_res;
        s_last_all[warp] = last_all;
    }
    __syncthreads();
    if (t == 0) {
        double x = 0.0, y = 0.0;
        int lr = -1, la = -1;
        for (int w = 0; w < kSvWarps; ++w) {
            x += s_res[w];
            y += s_all[w];
            lr = max(lr, s_last_res[w]);
            la = max(la, s_last_all[w]);
        }
        cta_res = x;
        cta_all = y;
        cta_last_res = lr;
        cta_last_all = la;
    }
    cl.sync();
    // every CTA adds the CTAs' sums in the same order, and finds the one that
    // holds the draw
    double total_res = 0.0, total_all = 0.0;
    int end_res = -1, end_all = -1;
    for (int c = 0; c < C; ++c) {
        total_res += *cl.map_shared_rank(&cta_res, c);
        total_all += *cl.map_shared_rank(&cta_all, c);
        end_res = max(end_res, *cl.map_shared_rank(&cta_last_res, c));
        end_all = max(end_all, *cl.map_shared_rank(&cta_last_all, c));
    }
    const bool residual = refused >= 0 && total_res > 0.0;
    const double total = residual ? total_res : total_all;
    const int end = residual ? end_res : end_all;      // the last index with mass
    const double target = fmax((double)a.u_draw[b], 0.0) * total;
    double before = 0.0;
    int owner = -1;
    for (int c = 0; c < C; ++c) {
        const double m = *cl.map_shared_rank(residual ? &cta_res : &cta_all, c);
        if (owner < 0 && before + m > target) owner = c;
        if (owner < 0) before += m;
    }
    cl.sync();                                          // remote reads done
    // the accepted tokens, and -1 behind the drawn one
    if (rank == 0)
        for (int i = t; i <= k; i += kSvThreads)
            if (i != r) a.tokens[(size_t)b * (k + 1) + i] = i < r ? a.draft[(size_t)b * k + i] : -1;
    if (rank == 0 && t == 0) {
        a.count[b] = r + 1;
        // no mass at all: no token; no index past the draw: the last with mass
        if (total <= 0.0 || owner < 0) a.tokens[(size_t)b * (k + 1) + r] = total <= 0.0 ? -1 : end;
    }
    if (total <= 0.0 || owner != rank) return;
    // the warp of this CTA, then the index; a border that moved by the
    // rounding of the partial sums falls to the last index with mass before it
    int mine = -1;
    for (int w = 0; w < kSvWarps; ++w) {
        const double m = residual ? s_res[w] : s_all[w];
        if (mine < 0 && before + m > target) mine = w;
        if (mine < 0) before += m;
    }
    if (mine < 0) {
        if (t == 0) a.tokens[(size_t)b * (k + 1) + r] = residual ? cta_last_res : cta_last_all;
        return;
    }
    if (warp != mine) return;
    int found = -1;
    for (int i0 = lo; i0 < hi && found < 0; i0 += 128) {
        const int i = i0 + 4 * lane;
        const float4 pv = row4<VEC>(i < hi ? prow : nullptr, i, hi), qv = row4<VEC>(i < hi ? qrow : nullptr, i, hi);
        const float pe[4] = {pv.x, pv.y, pv.z, pv.w}, qe[4] = {qv.x, qv.y, qv.z, qv.w};
        double m[4], x = 0.0;
        #pragma unroll
        for (int e = 0; e < 4; ++e) {
            m[e] = mass_at(pe[e], qe[e], i + e, refused, point, residual);
            x += m[e];
        }
        const double own = x;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        // an entry without mass is never drawn, whatever the sums' rounding
        double run = before + (x - own);
        int hit = -1;
        #pragma unroll
        for (int e = 0; e < 4; ++e) {
            run += m[e];
            if (hit < 0 && m[e] > 0.0 && run > target) hit = e;
        }
        const unsigned any = __ballot_sync(0xffffffffu, hit >= 0);
        if (any != 0) found = __shfl_sync(0xffffffffu, i + hit, __ffs(any) - 1);
        before += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0)
        a.tokens[(size_t)b * (k + 1) + r] = found >= 0 ? found : residual ? s_last_res[warp] : s_last_all[warp];
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
    // few sequences: eight CTAs each, so that the rows are read by many SMs;
    // a small vocabulary needs no cluster
    const int C = n_vocab <= 4096 ? 1 : 8;
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
