// attn_kv8.cu -- decode attention over an 8-bit paged cache.
//
// For a sequence and kv head the rows are its query tokens times the heads of
// the group. A block of 16 keys k_j = s c_j (codes c, scale s) gives
//     scores  S^T = s C Q^T,    outputs  O^T += s' C'^T P^T,
// both as m16n8k16 products with the codes as the first operand (keys, or
// dimensions, down the 16 rows, eight query rows across): codes are exact in
// f16, so a scale only multiplies the f32 sums. With few rows that is no more
// work than eight rows' worth; tcgen05 would want 128 codes down its rows, in
// shared memory as f16, where here they go from the 8-bit tile straight into
// the operand registers (one byte permutation and one subtraction for two).
// The order of the dimensions in a sum, and of the keys, is free: a thread of the
// quad takes 32 dimensions in a row of K, 16 in a row of V^T, and so loads 16
// bytes at a time, without conflicts in the 128-byte swizzle.
//
// f32 queries and weights are pairs of f16, x = hi + 2^-11 lo, with a power of
// two per query row; two products then, 22 bits.
//
// Much work of 17 rows and more of f16 queries goes to attn_kv8_wide.cuh.
//
// The work is cut by the device: the tiles of 128 keys of all (sequence, kv
// head) pairs, in order, are dealt to the CTAs in equal runs. A pair inside one
// run is written at once; of a pair that runs share each leaves its part
// (maximum, sum, outputs), at most two a CTA, and a second launch joins them.
// So the split follows the lengths, whatever they are, and the workspace does not
// depend on them.
//
// Bound: HBM for long contexts (f16, 64/8 heads: one sequence of 131072 keys, 269 MB
// of codes and scales, 54 us; 64 of up to 8192, 539 MB, 97 us, 5.6 TB/s), with the
// issue slots half taken (53%). For little work the chain is the bound: lengths, page
// ids, tile, products, the parts and their join (one sequence of 320 keys 11 us, 2 of
// them the join). Tiles of 128 keys in two stages leave room for three CTAs a SM with
// up to eight rows, each with a warp that loads.

#include <type_traits>

#include "attn_kv8.cuh"
#include "attn_kv8_wide.cuh"

namespace sllm {
namespace {

constexpr int kE8Warps = 4;                         // that multiply; one more loads
constexpr int kE8Threads = 32 * (kE8Warps + 1);
__host__ __device__ constexpr int e8_ctas(int nt) { return nt == 1 ? 3 : 2; }      // per SM

struct __align__(1024) Stage8 {
    uint8_t k[kE8Tile], v[kE8Tile];
};
constexpr int kE8Stages = 2;

struct __align__(1024) Shared8 {    // and the queries' buffers behind it
    Stage8 stage[kE8Stages];
    float sc[kE8Stages][2 * kE8Blocks];             // of K's blocks, of V's
    Meta meta[kE8Stages];
    uint64_t full[kE8Stages], empty[kE8Stages];
    uint64_t q_free[2], done, merged;
    RunStart run;
    int abort;
    float2 ml[kE8Warps][16];
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ... from zero
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

__device__ __forceinline__ uint4 lds16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }

// What a warp holds of its NT tiles of eight rows. Lane 4 g + t: of Q, row g's
// dimensions 32 t ..; of the outputs, rows 2 t and 2 t + 1, dimensions 16 g ..
// (o[tile][j] = dimensions 16 g + 2 j of both rows, then 16 g + 2 j + 1).
template <int P, int NT>
struct Rows8 {
    uint32_t q[P][NT][16];
    float o[NT][8][4], m[NT][2], l[NT][2];
    float mul[NT][2];               // the row's power of two (one f16: 1)
    int lim[NT][2];

    __device__ __forceinline__ void clear() {
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            #pragma unroll
            for (int j = 0; j < 8; ++j)
                #pragma unroll
                for (int c = 0; c < 4; ++c) o[n][j][c] = 0.f;
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                m[n][c] = kE8None;
                l[n][c] = 0.f;
                mul[n][c] = 1.f;
            }
        }
    }

    // query rows r0 .. of the row block that starts at row `first`, from its buffer
    template <class Q>
    __device__ __forceinline__ void load(const Attn8Params& p, const uint8_t* buf, int r0, int first, int len) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            const Q* x = reinterpret_cast<const Q*>(buf) + (r0 + 8 * n + g) * kServeDim + 32 * t;
            if constexpr (P == 1) {
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint4 u = *(reinterpret_cast<const uint4*>(x) + i);
                    q[0][n][4 * i] = u.x;
                    q[0][n][4 * i + 1] = u.y;
                    q[0][n][4 * i + 2] = u.z;
                    q[0][n][4 * i + 3] = u.w;
                }
            } else {
                float4 f[8];
                float most = 0.f;
                #pragma unroll
                for (int i = 0; i < 8; ++i) {
                    f[i] = *(reinterpret_cast<const float4*>(x) + i);
                    most = fmaxf(most, fmaxf(fmaxf(fabsf(f[i].x), fabsf(f[i].y)), fmaxf(fabsf(f[i].z), fabsf(f[i].w))));
                }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                // the row's power of two: its largest value becomes 1 to 2
                int e = (int)(f2u(most) >> 23) - 127;
                e = most > 0.f && most < INFINITY ? min(max(e, -100), 100) : 0;
                const float down = u2f((uint32_t)(127 - e) << 23), up = u2f((uint32_t)(127 + e) << 23);
                #pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float y[4] = {f[i].x * down, f[i].y * down, f[i].z * down, f[i].w * down};
                    #pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t hi = pack2(y[2 * c], y[2 * c + 1]);
                        const float2 z = unpack2(hi);
                        q[0][n][2 * i + c] = hi;
                        q[P - 1][n][2 * i + c] = pack2((y[2 * c] - z.x) * 2048.f, (y[2 * c + 1] - z.y) * 2048.f);
                    }
                }
                #pragma unroll
                for (int c = 0; c < 2; ++c) mul[n][c] = __shfl_sync(0xffffffffu, up, 8 * t + 4 * c);
            }
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int row = first + r0 + 8 * n + 2 * t + c;
                lim[n][c] = len - p.n_q + 1 + (row < p.rows ? p.token(row) : p.n_q - 1);
            }
        }
    }

    // Two blocks of 16 keys, the first keys of each number j0 and j0 + dj; the second
    // counts for nothing where its scales are 0 and its keys are masked.
    __device__ __forceinline__ void blocks(const uint8_t* kt, const uint8_t* vt, int apart, const float (&ks)[2],
                                           const float (&vs)[2], bool masked, int j0, int dj) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        float s[2][P][NT][4];
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
            #pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint8_t* at = kt + k * apart + g * 128 + (((2 * t + i) ^ g) << 4);
                const uint4 ua = lds16(at), ub = lds16(at + 1024);
                const uint32_t wa[4] = {ua.x, ua.y, ua.z, ua.w}, wb[4] = {ub.x, ub.y, ub.z, ub.w};
                #pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t xa = wa[w] ^ 0x80808080u, xb = wb[w] ^ 0x80808080u;
                    const uint32_t a[4] = {two_codes(xa, false), two_codes(xb, false), two_codes(xa, true), two_codes(xb, true)};
                    #pragma unroll
                    for (int n = 0; n < NT; ++n)
                        #pragma unroll
                        for (int x = 0; x < P; ++x) {
                            if (i == 0 && w == 0) mma_f16_zero(s[k][x][n], a, q[x][n][0], q[x][n][1]);
                            else mma_f16(s[k][x][n], a, q[x][n][8 * i + 2 * w], q[x][n][8 * i + 2 * w + 1]);
                        }
                }
            }
        }
        // Exponents against the rows' references, no shuffles: one that is too large is
        // seen by its own lane, and then only the row's maximum is looked for. (With it
        // each time, a tile of eight rows took 65 instructions more for the 32 keys.)
        const float base[2] = {ks[0] * kE8Log2, ks[1] * kE8Log2};
        constexpr float LIFT = e8_lift(P), MOST = P == 1 ? kE8Most : kE8Most + 0.5f;     // (rounding alone moves no reference)
        float z[NT][2][4], top = -INFINITY;
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float ref[2] = {__fsub_ru(LIFT, m[n][0]), __fsub_ru(LIFT, m[n][1])};
            #pragma unroll
            for (int k = 0; k < 2; ++k)
                #pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if constexpr (P == 2) s[k][0][n][c] = __fmaf_rn(s[k][P - 1][n][c], 0x1p-11f, s[k][0][n][c]);
                    z[n][k][c] = __fmaf_rn(s[k][0][n][c], P == 1 ? base[k] : base[k] * mul[n][c & 1], ref[c & 1]);
                }
            if (masked) {
                #pragma unroll
                for (int k = 0; k < 2; ++k)
                    #pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (j0 + k * dj + g + 8 * (c >> 1) >= lim[n][c & 1]) z[n][k][c] = -INFINITY;
            }
            #pragma unroll
            for (int k = 0; k < 2; ++k) top = fmaxf(fmaxf(fmaxf(top, z[n][k][0]), fmaxf(z[n][k][1], z[n][k][2])), z[n][k][3]);
        }
        if (__any_sync(0xffffffffu, top > MOST)) {
            #pragma unroll
            for (int n = 0; n < NT; ++n) {
                float alpha[2];
                #pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float now = kE8None;
                    #pragma unroll
                    for (int k = 0; k < 2; ++k)
                        #pragma unroll
                        for (int i = c; i < 4; i += 2)
                            if (z[n][k][i] > -INFINITY) now = fmaxf(now, __fmul_rd(s[k][0][n][i], P == 1 ? base[k] : base[k] * mul[n][c]));
                    #pragma unroll
                    for (int y = 4; y < 32; y <<= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, y));
                    now = fmaxf(m[n][c], now);
                    alpha[c] = ex2(m[n][c] - now);
                    m[n][c] = now;
                    l[n][c] *= alpha[c];
                    #pragma unroll
                    for (int k = 0; k < 2; ++k)
                        #pragma unroll
                        for (int i = c; i < 4; i += 2)
                            if (z[n][k][i] != -INFINITY)
                                z[n][k][i] = ended(__fmaf_rn(s[k][0][n][i], P == 1 ? base[k] : base[k] * mul[n][c], __fsub_ru(LIFT, now)));
                }
                #pragma unroll
                for (int j = 0; j < 8; ++j)
                    #pragma unroll
                    for (int c = 0; c < 4; ++c) o[n][j][c] *= alpha[c & 1];
            }
        }
        uint32_t pb[2][P][NT][2];
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            #pragma unroll
            for (int k = 0; k < 2; ++k) {
                #pragma unroll
                for (int c = 0; c < 4; ++c) z[n][k][c] = ex2(z[n][k][c]);
                #pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t hi = pack2(z[n][k][2 * c], z[n][k][2 * c + 1]);
                    pb[k][0][n][c] = transpose8(hi);
                    if constexpr (P == 2) {
                        const float2 y = unpack2(hi);
                        pb[k][P - 1][n][c] = transpose8(pack2((z[n][k][2 * c] - y.x) * 2048.f, (z[n][k][2 * c + 1] - y.y) * 2048.f));
                    }
                }
            }
            #pragma unroll
            for (int c = 0; c < 2; ++c) l[n][c] += (z[n][0][c] + z[n][0][c + 2]) + (z[n][1][c] + z[n][1][c + 2]);
        }
        #pragma unroll
        for (int k = 0; k < 2; ++k) {
            uint32_t wv[4][4];
            #pragma unroll
            for (int i = 0; i < 4; ++i) {           // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
                const int r = 2 * t + (i & 1);
                const uint4 u = lds16(vt + k * apart + (r + 8 * (i >> 1)) * 128 + ((g ^ r) << 4));
                wv[i][0] = u.x ^ 0x80808080u;
                wv[i][1] = u.y ^ 0x80808080u;
                wv[i][2] = u.z ^ 0x80808080u;
                wv[i][3] = u.w ^ 0x80808080u;
            }
            #pragma unroll
            for (int w = 0; w < 4; ++w) {
                #pragma unroll
                for (int hi = 0; hi < 2; ++hi) {
                    const uint32_t x = __byte_perm(wv[0][w], wv[1][w], hi ? 0x7362 : 0x5140);
                    const uint32_t z = __byte_perm(wv[2][w], wv[3][w], hi ? 0x7362 : 0x5140);
                    const uint32_t a[4] = {two_codes(x, false), two_codes(x, true), two_codes(z, false), two_codes(z, true)};
                    const int j = 2 * w + hi;
                    #pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float d[P][4];
                        #pragma unroll
                        for (int e = 0; e < P; ++e) mma_f16_zero(d[e], a, pb[k][e][n][0], pb[k][e][n][1]);
                        #pragma unroll
                        for (int c = 0; c < 4; ++c)
                            o[n][j][c] = __fmaf_rn(P == 1 ? d[0][c] : __fmaf_rn(d[P - 1][c], 0x1p-11f, d[0][c]), vs[k], o[n][j][c]);
                    }
                }
            }
        }
    }

    // the sums of a row's keys, over the lanes that share it
    __device__ __forceinline__ void total() {
        #pragma unroll
        for (int n = 0; n < NT; ++n)
            #pragma unroll
            for (int c = 0; c < 2; ++c)
                #pragma unroll
                for (int z = 4; z < 32; z <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], z);
    }

    // This warp's outputs [row][128] into `to`, its maxima and sums into `ml`. The 16-byte
    // columns of row r are permuted by (r / 2) % 4: no two of the lanes that store
    // at once meet in a bank.
    __device__ __forceinline__ void give(float4* to, float2* ml) const {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        #pragma unroll
        for (int n = 0; n < NT; ++n)
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int r = 8 * n + 2 * t + c;
                #pragma unroll
                for (int j = 0; j < 4; ++j)
                    to[r * 32 + ((4 * g + j) ^ t)] =
                        make_float4(o[n][2 * j][c], o[n][2 * j][c + 2], o[n][2 * j + 1][c], o[n][2 * j + 1][c + 2]);
                if (g == 0) ml[r] = make_float2(m[n][c], l[n][c] * e8_down(P));
            }
    }
};

// The rows of a row group from its key groups' warps (`from`: the first warp's, `step`
// float4 from one key group to the next), a share of the rows each: results, or
// the part `part` (>= 0). Lane i weighs row i of the share; then row by row.
template <class O, int NT, int KG>
__device__ __forceinline__ void finish(const Attn8Params& p, const Meta& mt, const float4* from, int step, const float2 (*ml)[16],
                                       int ml_step, int kg, int r0, int part) {
    constexpr int SHARE = 8 * NT / KG;
    const int lane = threadIdx.x & 31, r = kg * SHARE + (lane < SHARE ? lane : 0), row = mt.row_block * p.block_rows + r0 + r;
    float w[KG], M = kE8None, l = 0.f;
    float2 x[KG];
    #pragma unroll
    for (int k = 0; k < KG; ++k) {
        x[k] = ml[k * ml_step][r];
        M = fmaxf(M, x[k].x);
    }
    #pragma unroll
    for (int k = 0; k < KG; ++k) {
        w[k] = ex2(x[k].x - M);
        l = __fmaf_rn(w[k], x[k].y, l);
    }
    const int live = min(max(p.rows - (mt.row_block * p.block_rows + r0 + kg * SHARE), 0), SHARE);
    size_t at;                                      // of this lane's row, in floats of a part or elements of the output
    if (part >= 0) {
        at = ((size_t)part * p.block_rows + r0 + r) * kServeDim;
        if (lane < live) p.part_ml[(size_t)part * p.block_rows + r0 + r] = make_float2(M, l);
    } else {
        const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);     // (0: the row has seen nothing)
        #pragma unroll
        for (int k = 0; k < KG; ++k) w[k] *= inv;
        at = p.row_at(mt.b, mt.head, row);
    }
    #pragma unroll
    for (int i = 0; i < SHARE; ++i) {
        const int ri = kg * SHARE + i;
        const size_t to = __shfl_sync(0xffffffffu, (unsigned long long)at, i) + 4 * lane;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        #pragma unroll
        for (int k = 0; k < KG; ++k) {
            const float4 v = from[(size_t)k * step + ri * 32 + (lane ^ ((ri >> 1) & 3))];
            const float f = __shfl_sync(0xffffffffu, w[k], i);
            o.x = __fmaf_rn(f, v.x, o.x);
            o.y = __fmaf_rn(f, v.y, o.y);
            o.z = __fmaf_rn(f, v.z, o.z);
            o.w = __fmaf_rn(f, v.w, o.w);
        }
        if (i >= live) continue;
        if (part >= 0) st4(p.part_o + to, o);
        else st4(static_cast<O*>(p.out) + to, o);
    }
}

template <class Q, class O, int NT>
__global__ void __launch_bounds__(kE8Threads, e8_ctas(NT))
attn_kv8_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                const __grid_constant__ PagesDev pg, const __grid_constant__ Attn8Params p) {
    constexpr int P = std::is_same<Q, float>::value ? 2 : 1, STAGES = kE8Stages;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Shared8& sh = *reinterpret_cast<Shared8*>(smem_raw);
    uint8_t* const q_buf = smem_raw + sizeof(Shared8);
    const int q_bytes = p.block_rows * kServeDim * (int)sizeof(Q);
    pdl_trigger();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    volatile int* const ab = &sh.abort;
    if ((smem_u32(smem_raw) & 1023u) != 0) {        // (the swizzle counts from a 1024-byte boundary)
        if (t == 0) {
            raise(p.status, SLLM_CUDA_ERR_DEVICE);
            if ((int)blockIdx.x < p.n_notes) p.notes[blockIdx.x] = make_int4(-1, 0, 0, 0);
        }
        return;
    }
    if (t == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&sh.full[i], 1 + 32);
            mbar_init(&sh.empty[i], kE8Warps);
        }
        mbar_init(&sh.q_free[0], kE8Warps);
        mbar_init(&sh.q_free[1], kE8Warps);
        mbar_init(&sh.done, kE8Warps);
        mbar_init(&sh.merged, kE8Warps);
        sh.abort = 0;
        sh.run.at.tiles = 0;
        fence_proxy_async_smem();
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (t == 32 * kE8Warps) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_k)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_v)) : "memory");
    }
    Walk8<1> walk(pg, p);
    if (!walk.find<kE8Threads>(sh.run)) return;

    const Waits w{p};
    bool ok = true;
    if (warp == kE8Warps) {
        // ---- loads
        // lane i: the page of the tile's i-th load
        auto ids = [&](const Place& x) {
            const int key = x.tile * kE8Keys + (lane << p.page_log2);
            int id = 0;
            if (lane < (kE8Keys >> p.page_log2) && key < x.len) {
                id = pg.tables[(size_t)x.slot * pg.width + (key >> p.page_log2)];
                if (id < 0 || id >= pg.n_pages) {
                    raise(p.status, SLLM_CUDA_ERR_ARG);
                    id = 0;
                }
            }
            return id;
        };
        bool more = walk.start(sh.run);
        int id = more ? ids(walk.cur) : 0;
        int first = 1, started = more && walk.cur.tile == 0;    // of the segment: its first tile here; whether the pair starts here
        int4 note = make_int4(-1, 0, 0, 0);
        uint32_t n = 0, seg = 0;
        while (more) {
            const Place cur = walk.cur;
            const bool ends = cur.tile + 1 == cur.tiles;
            more = walk.advance();
            const int nid = more ? ids(walk.cur) : 0;
            const int slot = n % STAGES;
            if (n >= STAGES && !(ok = at_wait_warp(&sh.empty[slot], (n / STAGES - 1) & 1, ab, w))) break;
            const int qb = seg % p.q_bufs;
            if (first && seg >= p.q_bufs && !(ok = at_wait_warp(&sh.q_free[qb], (seg / p.q_bufs - 1) & 1, ab, w))) break;
            const bool last = ends || !more;
            const int key0 = cur.tile * kE8Keys, keys = min(kE8Keys, cur.len - key0);
            const int loads = (keys + (1 << p.page_log2) - 1) >> p.page_log2;
            if (lane == 0) {
                const int flags = (first ? E8_FIRST : 0) | (last ? E8_LAST : 0) |
                                  (!last || (ends && started) ? 0 : started ? E8_PART1 : E8_PART0);
                sh.meta[slot] = Meta{cur.b, cur.head, cur.row_block, cur.len, key0, flags};
                mbar_expect_tx(&sh.full[slot], (uint32_t)(loads << p.page_log2) * 2 * kServeDim);
            }
            __syncwarp();
            if (lane < loads) {
                const int at = lane * kServeDim << p.page_log2;
                tma_load_4d(sh.stage[slot].k + at, &tm_k, 0, 0, cur.head, id, &sh.full[slot]);
                tma_load_4d(sh.stage[slot].v + at, &tm_v, 0, 0, cur.head, id, &sh.full[slot]);
            }
            const int blk = lane & (kE8Blocks - 1), from = __shfl_sync(0xffffffffu, id, (blk * kKvBlock) >> p.page_log2);
            if (lane < 2 * kE8Blocks) {
                if (blk * kKvBlock < keys)
                    cp_async4(&sh.sc[slot][lane], (lane < kE8Blocks ? p.ksc : p.vsc) + (size_t)from * p.scale_stride +
                                                      cur.head * (pg.page / kKvBlock) +
                                                      ((key0 + blk * kKvBlock) & (pg.page - 1)) / kKvBlock);
            }
            if (first) {                            // the pair's queries come with its first tile
                const int r0 = cur.row_block * p.block_rows, rows = min(p.block_rows, p.rows - r0);
                constexpr int PER = kServeDim * (int)sizeof(Q) / 16;
                for (int i = lane; i < rows * PER; i += 32) {
                    cp_async16(q_buf + qb * q_bytes + i * 16,
                               static_cast<const Q*>(p.q) + p.row_at(cur.b, cur.head, r0 + i / PER) + i % PER * (16 / (int)sizeof(Q)));
                }
                ++seg;
            }
            cp_async_arrive(&sh.full[slot]);
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
        if (ok) {
            const int slot = n % STAGES;
            ok = n < STAGES || at_wait_warp(&sh.empty[slot], (n / STAGES - 1) & 1, ab, w);
            if (ok) {
                if (lane == 0) {
                    sh.meta[slot] = Meta{0, 0, 0, 0, 0, E8_END};
                    mbar_arrive(&sh.full[slot]);
                }
                mbar_arrive(&sh.full[slot]);
                ++n;
            }
        }
        if (lane == 0 && !p.by_pair) p.notes[blockIdx.x] = note;
        // copies in flight end before the CTA does, also where the others gave up
        for (uint32_t i = n > STAGES ? n - STAGES : 0; i < n; ++i) at_drain(&sh.full[i % STAGES], (i / STAGES) & 1);
    } else {
        // ---- products. A warp has its share of the blocks of a tile (key group
        // kg) for its share of the rows (row group)
        const int RG = p.rg, KG = kE8Warps / RG, rgrp = warp % RG, kg = warp / RG;
        Rows8<P, NT> rows;
        rows.clear();
        uint32_t seg = 0;
        for (uint32_t n = 0;; ++n) {
            const int slot = n % STAGES;
            ok = n == 0 ? __all_sync(0xffffffffu, at_wait_start(&sh.full[slot], 0, ab, w))
                        : at_wait_warp(&sh.full[slot], (n / STAGES) & 1, ab, w);
            if (!ok) break;
            const Meta mt = sh.meta[slot];
            if (mt.flags & E8_END) break;
            if (mt.flags & E8_FIRST) {
                const int qb = seg % p.q_bufs;
                rows.clear();
                rows.template load<Q>(p, q_buf + qb * q_bytes, rgrp * 8 * NT, mt.row_block * p.block_rows, mt.len);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.q_free[qb]);
            }
            const int keys = min(kE8Keys, mt.len - mt.key0);
            const bool masked = mt.key0 + kE8Keys > mt.len - p.n_q + 1;
            const float* const sc = sh.sc[slot];
            // blocks kg and kg + KG, and so on: a short tile's are shared out, too
            #pragma unroll 1
            for (int blk = kg; blk * kKvBlock < keys; blk += 2 * KG) {
                const bool two = (blk + KG) * kKvBlock < keys;
                const float ks[2] = {sc[blk], two ? sc[blk + KG] : 0.f};
                // (without the weights' lift: outputs overflow no sooner than the values do)
                const float vs[2] = {sc[kE8Blocks + blk] * e8_down(P), two ? sc[kE8Blocks + blk + KG] * e8_down(P) : 0.f};
                rows.blocks(sh.stage[slot].k + blk * kKvBlock * kServeDim, sh.stage[slot].v + blk * kKvBlock * kServeDim,
                            KG * kKvBlock * kServeDim, ks, vs, masked, mt.key0 + blk * kKvBlock, KG * kKvBlock);
            }
            __syncwarp();
            if (!(mt.flags & E8_LAST)) {
                if (lane == 0) mbar_arrive(&sh.empty[slot]);
                continue;
            }
            // the key groups' parts into one, through the tile that nobody needs any more
            const uint32_t par = seg & 1;
            ++seg;
            if (lane == 0) mbar_arrive(&sh.done);
            rows.total();
            if (!(ok = at_wait_warp(&sh.done, par, ab, w))) break;
            float4* const area = reinterpret_cast<float4*>(sh.stage[slot].k);
            rows.give(area + warp * (8 * NT * 32), sh.ml[warp]);
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.merged);
            if (!(ok = at_wait_warp(&sh.merged, par, ab, w))) break;
            const int part = mt.flags & E8_PART0 ? 2 * (int)blockIdx.x : mt.flags & E8_PART1 ? 2 * (int)blockIdx.x + 1 : -1;
            const float4* const from = area + rgrp * (8 * NT * 32);
            const int step = RG * 8 * NT * 32, r0 = rgrp * 8 * NT;
            if (NT == 1 || KG == 4) finish<O, NT, 4>(p, mt, from, step, sh.ml + rgrp, RG, kg, r0, part);
            else if (KG == 2) finish<O, NT, NT == 1 ? 4 : 2>(p, mt, from, step, sh.ml + rgrp, RG, kg, r0, part);
            else finish<O, NT, NT == 1 ? 4 : 1>(p, mt, from, step, sh.ml + rgrp, RG, kg, r0, part);
            fence_proxy_async_smem();               // before the next tile is copied over it
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.empty[slot]);
        }
    }
    if (!ok && lane == 0) raise(p.status, SLLM_CUDA_ERR_TIMEOUT);
}

// ---------------------------------------------------------------------------
// the join of pairs that several runs share: a row per warp, or per several
// where rows are few. Bound: its launch and one round of loads, eight parts in
// flight a warp; launched early, it adds 2 us to a short call, 4 us to one of 32 rows.
// ---------------------------------------------------------------------------
constexpr int kJoinWarps = 8;
template <class O>
__global__ void __launch_bounds__(32 * kJoinWarps)
attn_kv8_join_kernel(const __grid_constant__ Attn8Params p, int per_row) {
    __shared__ float4 so[kJoinWarps][32];
    __shared__ float2 sm[kJoinWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = warp % per_row, in = blockIdx.y * (kJoinWarps / per_row) + warp / per_row;
    pdl_wait();
    const int4 note = p.notes[blockIdx.x];
    const int c = note.z;
    // (a run that gave up leaves notes unwritten: what stood there stays inside the arrays)
    if (note.x < 0 || note.x >= p.n || note.y < 0 || note.y >= p.n_kv * p.row_blocks || c < 0 || note.w < c || note.w >= p.ctas) return;
    const int h = note.y / p.row_blocks, r = note.y % p.row_blocks * p.block_rows + in;
    const bool live = in < p.block_rows && r < p.rows;
    // parts: the second of the first CTA's, then the first of the following CTAs'
    const int parts = note.w - c + 1;
    auto at = [&](int i) { return (size_t)(i == 0 ? 2 * c + 1 : 2 * (c + i)) * p.block_rows + in; };
    float M = kE8None, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) {
        for (int i0 = sub; i0 < parts; i0 += 8 * per_row) {
            float4 v[8];
            float2 ml[8];
            #pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = i0 + e * per_row;
                ml[e] = make_float2(kE8None, 0.f);
                if (i < parts) {
                    ml[e] = __ldcg(p.part_ml + at(i));
                    v[e] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at(i) * kServeDim) + lane);
                }
            }
            float now = M;
            #pragma unroll
            for (int e = 0; e < 8; ++e) now = fmaxf(now, ml[e].x);
            const float f0 = ex2(M - now);
            M = now;
            l *= f0;
            o.x *= f0; o.y *= f0; o.z *= f0; o.w *= f0;
            #pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (i0 + e * per_row >= parts) continue;
                const float f = ex2(ml[e].x - M);
                l = __fmaf_rn(f, ml[e].y, l);
                o.x = __fmaf_rn(f, v[e].x, o.x);
                o.y = __fmaf_rn(f, v[e].y, o.y);
                o.z = __fmaf_rn(f, v[e].z, o.z);
                o.w = __fmaf_rn(f, v[e].w, o.w);
            }
        }
    }
    if (per_row > 1) {
        so[warp][lane] = o;
        if (lane == 0) sm[warp] = make_float2(M, l);
        __syncthreads();
        if (sub != 0) return;
        for (int i = 1; i < per_row; ++i) {
            const float2 b = sm[warp + i];
            const float4 v = so[warp + i][lane];
            const float now = fmaxf(M, b.x), f0 = ex2(M - now), f1 = ex2(b.x - now);
            M = now;
            l = __fmaf_rn(l, f0, b.y * f1);
            o.x = __fmaf_rn(o.x, f0, v.x * f1);
            o.y = __fmaf_rn(o.y, f0, v.y * f1);
            o.z = __fmaf_rn(o.z, f0, v.z * f1);
            o.w = __fmaf_rn(o.w, f0, v.w * f1);
        }
    }
    if (!live) return;
    const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
    st4(static_cast<O*>(p.out) + p.row_at(note.x, h, r) + 4 * lane, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Rows of a CTA: 8 NT a warp, and row groups so that the four warps share them
// and the keys; beyond 64 rows a pair is read once for every 64.
struct Cut8 {
    bool wide;
    int nt, rg, block_rows, row_blocks, ctas;
};
// `keys`: the most that there may be, of all pairs. The wide form's longer chain
// from a CTA's first load to its last result costs 4 us, and its tiles take four
// fifths of the time. Both measured, in us, f16 (wide, this file's): 10 sequences of
// 1000 keys at most, 4 tokens of 64/8 heads (80 thousand keys at most) 22.4, 18.5; 20 of
// 2000 (320) 32.9, 32.8; 64 of 1000 (512) 47.7, 47.3; 30 of 4000, 5 tokens of 20/5 heads
// (600) 40.6, 43.1; one of 60000 (480) 48.3, 56.2; 8 of 8000, 8 tokens (1024) 61.3,
// 71.9; 32 of 8192 (2097) 93, 112. The host knows the tables' width, not the lengths:
// in tables with room for much, short sequences take the wide form too, 4 tokens of
// 64/8 heads: 64 of 200 keys 30.8, 28.7; 16 of 500 22.6, 19.3.
constexpr long long kE8WideKeys = 3000;             // a SM
Cut8 cut8(int rows, bool f16, int sms, long long keys) {
    Cut8 x;
    x.wide = f16 && rows > 16;
    if (x.wide) {
        x.nt = x.rg = 0;
        x.block_rows = kW8Rows;
        x.row_blocks = (rows + kW8Rows - 1) / kW8Rows;
        x.wide = keys * x.row_blocks >= kE8WideKeys * sms;
    }
    if (x.wide) {
        x.ctas = sms * kW8Ctas;
        return x;
    }
    x.nt = rows <= 8 ? 1 : 2;
    x.rg = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    x.block_rows = 8 * x.nt * x.rg;
    x.row_blocks = (rows + x.block_rows - 1) / x.block_rows;
    x.ctas = sms * e8_ctas(x.nt);
    return x;
}

// (f32 rises with the rows: 8 * 3, 16 * 2, 32 * 2, 64 * 2 a SM, and the wide form needs 32 * 2)
size_t work8_bytes(const Cut8& x) {
    return (size_t)x.ctas * (2 * x.block_rows * (kServeDim * sizeof(float) + sizeof(float2)) + sizeof(int4));
}

// two buffers of queries up to 32 rows, one of 64: 16 KB of f16, 32 KB of f32
constexpr int kE8QBytes = 64 * kServeDim * 2;

// one layer of a pool: a page's rows of one kv head per box
bool encode_codes(CUtensorMap* tm, const void* base, const sllm_cuda_kv_pages& p) {
    PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
    if (enc == nullptr) return false;
    const cuuint64_t row = kServeDim, head = row * p.page_size, page = head * p.n_head_kv * p.n_layer;
    const cuuint64_t dims[4] = {(cuuint64_t)kServeDim, (cuuint64_t)p.page_size, (cuuint64_t)p.n_head_kv, (cuuint64_t)p.n_pages};
    const cuuint64_t strides[3] = {row, head, page};
    const cuuint32_t box[4] = {(cuuint32_t)kServeDim, (cuuint32_t)p.page_size, 1, 1}, estr[4] = {1, 1, 1, 1};
    return enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class Q, class O, int NT>
cudaError_t launch8(const CUtensorMap& tk, const CUtensorMap& tv, const PagesDev& pg, const Attn8Params& a, int ctas,
                    cudaStream_t st) {
    constexpr int kMost = (int)sizeof(Shared8) + kE8QBytes * (int)sizeof(Q) / 2;
    const cudaError_t e = allow_smem<attn_kv8_kernel<Q, O, NT>>(kMost);
    const int bytes = (int)sizeof(Shared8) + a.q_bufs * a.block_rows * kServeDim * (int)sizeof(Q);
    return e != cudaSuccess ? e : launch(attn_kv8_kernel<Q, O, NT>, dim3(ctas), dim3(kE8Threads), bytes, st, false, tk, tv, pg, a);
}

template <class O>
cudaError_t launch_wide8(const CUtensorMap& tk, const CUtensorMap& tv, const PagesDev& pg, const Attn8Params& a, int ctas, cudaStream_t st) {
    constexpr int kBytes = (int)sizeof(SharedW8);
    const cudaError_t e = allow_smem<attn_kv8_wide_kernel<O>>(kBytes);
    return e != cudaSuccess ? e : launch(attn_kv8_wide_kernel<O>, dim3(ctas), dim3(kW8Threads), kBytes, st, false, tk, tv, pg, a);
}

int check_shape8(const sllm_cuda_kv_pages* p, int n, int n_q, int n_head, const char* who) {
    const int rc = check_pages(p, who, true);
    if (rc != SLLM_CUDA_OK) return rc;
    if (n < 0 || n > 4096 || n_q < 1 || n_q > 16 || n_head < 1 || n_head > 1024 || n_head % p->n_head_kv != 0)
        return fail(SLLM_CUDA_ERR_ARG, "%s: %d sequences, %d query tokens (1 to 16), %d heads over %d", who, n, n_q, n_head,
                    p->n_head_kv);
    return SLLM_CUDA_OK;
}

}  // namespace
}  // namespace sllm

using namespace sllm;

int sllm::take_kv8_error() { return take_attn_error(); }

extern "C" size_t sllm_cuda_attn_kv8_work_bytes(const sllm_cuda_kv_pages* p, int32_t n, int32_t n_q, int32_t n_head) {
    if (check_shape8(p, n, n_q, n_head, "attn_kv8_work_bytes") != SLLM_CUDA_OK) return 0;
    return work8_bytes(cut8(n_q * (n_head / p->n_head_kv), false, current_sms(), 0));
}

extern "C" int sllm_cuda_attn_kv8(const sllm_cuda_kv_pages* p, int32_t layer, const void* q, int32_t q_type,
                                  const int32_t* slots, int32_t n, int32_t n_q, int32_t n_head, void* out,
                                  int32_t out_type, void* work, size_t work_bytes, int32_t* status, void* stream) {
    int rc = check_shape8(p, n, n_q, n_head, "attn_kv8");
    if (rc != SLLM_CUDA_OK) return rc;
    if (q == nullptr || slots == nullptr || out == nullptr || work == nullptr || layer < 0 || layer >= p->n_layer)
        return fail(SLLM_CUDA_ERR_ARG, "attn_kv8: a NULL array, or layer %d of %d", layer, p->n_layer);
    if ((q_type != SLLM_CUDA_KV_F32 && q_type != SLLM_CUDA_KV_F16) ||
        (out_type != SLLM_CUDA_KV_F32 && out_type != SLLM_CUDA_KV_F16) ||
        (q_type == SLLM_CUDA_KV_F32 && out_type == SLLM_CUDA_KV_F16))
        return fail(SLLM_CUDA_ERR_ARG, "attn_kv8: query type %d, output type %d (f32, or f16 from f16)", q_type, out_type);
    const int sms = current_sms(), rows = n_q * (n_head / p->n_head_kv);
    const Cut8 cut = cut8(rows, q_type == SLLM_CUDA_KV_F16, sms, (long long)n * p->n_head_kv * p->table_width * p->page_size);
    const size_t need = work8_bytes(cut8(rows, false, sms, 0));
    if (!aligned16(q) || !aligned16(out) || !aligned16(work) || work_bytes < need)
        return fail(SLLM_CUDA_ERR_ARG, "attn_kv8: workspace of %zu bytes (%zu needed), arrays 16-byte aligned", work_bytes, need);
    const void* ptr[] = {p->k, p->v, p->tables, p->lens, p->k_scale, p->v_scale, q, slots, out, work, status};
    const char* name[] = {"k", "v", "tables", "lens", "k_scale", "v_scale", "q", "slots", "out", "work", "status"};
    for (int i = 0; i < 11; ++i)
        if (ptr[i] != nullptr && (rc = need_device(ptr[i], "attn_kv8", name[i])) != SLLM_CUDA_OK) return rc;
    if (n == 0) return SLLM_CUDA_OK;
    Attn8Params a{};
    a.q = q; a.out = out;
    const size_t layer_codes = (size_t)p->n_head_kv * kServeDim * p->page_size;
    const size_t layer_scales = (size_t)p->n_head_kv * (p->page_size / kKvBlock);
    a.kp = static_cast<const int8_t*>(p->k) + layer * layer_codes;
    a.vp = static_cast<const int8_t*>(p->v) + layer * layer_codes;
    a.page_codes = p->n_layer * layer_codes;
    a.ksc = p->k_scale + layer * layer_scales;
    a.vsc = p->v_scale + layer * layer_scales;
    a.scale_stride = p->n_layer * layer_scales;
    a.slots = slots;
    a.n = n; a.n_q = n_q; a.n_head = n_head; a.n_kv = p->n_head_kv; a.group = n_head / p->n_head_kv;
    a.rows = n_q * a.group;
    a.over_group = a.group == 1 ? 0 : (uint32_t)(((1ull << 32) + a.group - 1) / a.group);
    a.q_bufs = cut.block_rows <= 32 ? 2 : 1;
    a.ctas = cut.ctas;
    a.rg = cut.rg; a.row_blocks = cut.row_blocks; a.block_rows = cut.block_rows;
    while ((1 << a.page_log2) < p->page_size) ++a.page_log2;
    a.wait = attn_wait_limit();
    a.status = status;
    a.part_o = static_cast<float*>(work);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)2 * cut.ctas * cut.block_rows * kServeDim);
    a.notes = reinterpret_cast<int4*>(a.part_ml + (size_t)2 * cut.ctas * cut.block_rows);
    const long long pairs = (long long)n * p->n_head_kv * cut.row_blocks;
    a.by_pair = pairs <= cut.ctas;
    a.n_notes = a.by_pair ? (int)pairs : cut.ctas;
    const PagesDev pg = pages_dev(*p);
    const cudaStream_t st = (cudaStream_t)stream;
    const bool f32 = q_type == SLLM_CUDA_KV_F32, out32 = out_type == SLLM_CUDA_KV_F32;
    cudaError_t e;
    CUtensorMap tk, tv;
    if (!encode_codes(&tk, a.kp, *p) || !encode_codes(&tv, a.vp, *p))
        return fail(SLLM_CUDA_ERR_DEVICE, "attn_kv8: a tensor map could not be made");
    if (cut.wide)
        e = out32 ? launch_wide8<float>(tk, tv, pg, a, cut.ctas, st) : launch_wide8<__half>(tk, tv, pg, a, cut.ctas, st);
    else if (cut.nt == 1)
        e = f32     ? launch8<float, float, 1>(tk, tv, pg, a, cut.ctas, st)
            : out32 ? launch8<__half, float, 1>(tk, tv, pg, a, cut.ctas, st)
                    : launch8<__half, __half, 1>(tk, tv, pg, a, cut.ctas, st);
    else
        e = f32     ? launch8<float, float, 2>(tk, tv, pg, a, cut.ctas, st)
            : out32 ? launch8<__half, float, 2>(tk, tv, pg, a, cut.ctas, st)
                    : launch8<__half, __half, 2>(tk, tv, pg, a, cut.ctas, st);
    CK(e, "attn_kv8 launch");
    // few pairs have many parts each: warps share a row's
    const int share = cut.ctas / a.n_notes, per_row = !a.by_pair ? 1 : share >= 16 ? 8 : share >= 8 ? 4 : share >= 4 ? 2 : 1;
    const dim3 grid(a.n_notes, (cut.block_rows * per_row + kJoinWarps - 1) / kJoinWarps);
    CK(out32 ? launch(attn_kv8_join_kernel<float>, grid, dim3(32 * kJoinWarps), 0, st, true, a, per_row)
             : launch(attn_kv8_join_kernel<__half>, grid, dim3(32 * kJoinWarps), 0, st, true, a, per_row),
       "attn_kv8 join");
    count_launches(2);
    return SLLM_CUDA_OK;
}
