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
// The work is cut by the device: the tiles of 128 keys of all (sequence, kv
// head) pairs, in order, are dealt to the CTAs in equal runs. A pair inside one
// run is written at once; of a pair that runs share each leaves its part
// (maximum, sum, outputs), at most two a CTA, and a second launch joins them.
// So the split follows the lengths, whatever they are, and the workspace does not
// depend on them.

#include <type_traits>

#include "attn_mma.cuh"
#include "serve.cuh"

namespace sllm {
namespace {

constexpr int kE8Warps = 4;                         // that multiply; one more loads
constexpr int kE8Threads = 32 * (kE8Warps + 1);
constexpr int kE8Keys = 128;                        // keys of a tile
constexpr int kE8Blocks = kE8Keys / kKvBlock;
constexpr int kE8Tile = kE8Keys * kServeDim;        // bytes of one of K or V
constexpr float kE8Lift = 15.f;                     // weights are up to 2^15: f16 keeps 11 bits of them down to 2^-29 of the largest
constexpr float kE8Log2 = kServeScale * 1.4426950408889634f;

__host__ __device__ constexpr int e8_stages(int) { return 2; }
__host__ __device__ constexpr int e8_ctas(int nt) { return nt == 1 ? 3 : 2; }      // per SM

struct Attn8Params {
    const void* q;                  // [n][n_q][n_head][128]
    void* out;
    const float* ksc;               // the layer's slice of page 0
    const float* vsc;
    size_t scale_stride;
    const int32_t* slots;
    int n, n_q, n_head, n_kv, group, rows;          // rows: n_q * group
    int rg, row_blocks, block_rows;                 // row groups of a CTA; row blocks of a pair, and rows of one
    int page_log2;                  // rows of a page, and of a load
    WaitLimit wait;
    int32_t* status;
    float* part_o;                  // [2 * CTAs][block_rows][128]
    float2* part_ml;                // [2 * CTAs][block_rows]
    int4* shared;                   // [CTAs]: the pair that starts in this CTA's run and ends in another's
};

struct Meta {                       // of a tile in a stage
    int b, head, row_block, len, key0, flags;
};
enum { E8_FIRST = 1, E8_LAST = 2, E8_PART0 = 4, E8_PART1 = 8, E8_END = 16 };

template <int NT>
struct __align__(1024) Shared8 {
    uint8_t k[e8_stages(NT)][kE8Tile];
    uint8_t v[e8_stages(NT)][kE8Tile];
    float4 merge[2][NT * 9][32];                    // outputs, maximum and sum of a warp, a lane apart
    float sc[e8_stages(NT)][2 * kE8Blocks];         // of K's blocks, of V's
    Meta meta[e8_stages(NT)];
    uint64_t full[e8_stages(NT)], empty[e8_stages(NT)], merged[2], taken[2], passed;
    unsigned long long scan[kE8Threads / 32];
    unsigned long long start_rest;
    int start_b;
    int abort;
};

struct Waits {                      // for the bounded waits
    const Attn8Params& p;
    __device__ __forceinline__ WaitLimit wait_limit() const { return p.wait; }
};

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ... from zero
__device__ __forceinline__ void mma_f16_new(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// two codes, of bytes 0 and 1 or 2 and 3 of u (with 128 added to each), as f16:
// 0x6400 + byte is 1024 + byte
__device__ __forceinline__ uint32_t two_codes(uint32_t u, bool upper) {
    const uint32_t x = __byte_perm(u, 0x64646464u, upper ? 0x4342 : 0x4140);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));     // 1152
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t pack2(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

__device__ __forceinline__ uint4 lds16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }

// What a warp holds of its NT tiles of eight rows. Lane 4 g + t: of Q, row g's
// dimensions 32 t ..; of the outputs, rows 2 t and 2 t + 1, dimensions 16 g ..
// (o[tile][j] = dimensions 16 g + 2 j of both rows, then 16 g + 2 j + 1).
template <int P, int NT>
struct Rows8 {
    uint32_t q[P][NT][16];
    float o[NT][8][4], m[NT][2], l[NT][2], mul[NT][2];
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
                m[n][c] = -INFINITY;
                l[n][c] = 0.f;
                mul[n][c] = 1.f;
            }
        }
    }

    // query rows r0 .. of sequence b and kv head h
    template <class Q>
    __device__ __forceinline__ void load(const Attn8Params& p, int b, int h, int r0, int len) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = r0 + 8 * n + g;
            const bool in = r < p.rows;
            const Q* x = static_cast<const Q*>(p.q) +
                         (((size_t)b * p.n_q + (in ? r / p.group : 0)) * p.n_head + (size_t)h * p.group + (in ? r % p.group : 0)) * kServeDim + 32 * t;
            if constexpr (P == 1) {
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint4 u = in ? __ldg(reinterpret_cast<const uint4*>(x) + i) : make_uint4(0, 0, 0, 0);
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
                    f[i] = in ? __ldg(reinterpret_cast<const float4*>(x) + i) : make_float4(0.f, 0.f, 0.f, 0.f);
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
                const int row = r0 + 8 * n + 2 * t + c;
                lim[n][c] = len - p.n_q + 1 + (row < p.rows ? row / p.group : p.n_q - 1);
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
                            if (i == 0 && w == 0) mma_f16_new(s[k][x][n], a, q[x][n][0], q[x][n][1]);
                            else mma_f16(s[k][x][n], a, q[x][n][8 * i + 2 * w], q[x][n][8 * i + 2 * w + 1]);
                        }
                }
            }
        }
        const float base[2] = {ks[0] * kE8Log2, ks[1] * kE8Log2};
        uint32_t pb[2][P][NT][2];
        bool moved = false;
        float alpha[NT][2];
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            float y[2][4];
            #pragma unroll
            for (int k = 0; k < 2; ++k)
                #pragma unroll
                for (int c = 0; c < 4; ++c)
                    y[k][c] = P == 1 ? s[k][0][n][c] * base[k]
                                     : __fmaf_rn(s[k][P - 1][n][c], 0x1p-11f, s[k][0][n][c]) * (base[k] * mul[n][c & 1]);
            if (masked) {
                #pragma unroll
                for (int k = 0; k < 2; ++k)
                    #pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (j0 + k * dj + g + 8 * (c >> 1) >= lim[n][c & 1]) y[k][c] = -INFINITY;
            }
            float ref[2];
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                float now = fmaxf(fmaxf(y[0][c], y[0][c + 2]), fmaxf(y[1][c], y[1][c + 2]));
                #pragma unroll
                for (int z = 4; z < 32; z <<= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, z));
                now = fmaxf(m[n][c], now);
                ref[c] = (now == -INFINITY ? 0.f : now) - kE8Lift;
                alpha[n][c] = ex2(m[n][c] - kE8Lift - ref[c]);
                moved = moved || now != m[n][c];
                m[n][c] = now;
            }
            #pragma unroll
            for (int k = 0; k < 2; ++k) {
                #pragma unroll
                for (int c = 0; c < 4; ++c) y[k][c] = ex2(y[k][c] - ref[c & 1]);
                #pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t hi = pack2(y[k][2 * c], y[k][2 * c + 1]);
                    pb[k][0][n][c] = transpose8(hi);
                    if constexpr (P == 2) {
                        const float2 z = unpack2(hi);
                        pb[k][P - 1][n][c] = transpose8(pack2((y[k][2 * c] - z.x) * 2048.f, (y[k][2 * c + 1] - z.y) * 2048.f));
                    }
                }
            }
            #pragma unroll
            for (int c = 0; c < 2; ++c)
                l[n][c] = __fmaf_rn(l[n][c], alpha[n][c], (y[0][c] + y[0][c + 2]) + (y[1][c] + y[1][c + 2]));
        }
        if (__any_sync(0xffffffffu, moved)) {
            #pragma unroll
            for (int n = 0; n < NT; ++n)
                #pragma unroll
                for (int j = 0; j < 8; ++j)
                    #pragma unroll
                    for (int c = 0; c < 4; ++c) o[n][j][c] *= alpha[n][c & 1];
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
                    const uint32_t y = __byte_perm(wv[2][w], wv[3][w], hi ? 0x7362 : 0x5140);
                    const uint32_t a[4] = {two_codes(x, false), two_codes(x, true), two_codes(y, false), two_codes(y, true)};
                    const int j = 2 * w + hi;
                    #pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float d[P][4];
                        #pragma unroll
                        for (int z = 0; z < P; ++z) mma_f16_new(d[z], a, pb[k][z][n][0], pb[k][z][n][1]);
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

    __device__ __forceinline__ void give(float4 (*to)[32]) const {
        const int lane = threadIdx.x & 31;
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            #pragma unroll
            for (int j = 0; j < 8; ++j) to[n * 9 + j][lane] = make_float4(o[n][j][0], o[n][j][1], o[n][j][2], o[n][j][3]);
            to[n * 9 + 8][lane] = make_float4(m[n][0], m[n][1], l[n][0], l[n][1]);
        }
    }
    __device__ __forceinline__ void take(const float4 (*from)[32]) {
        const int lane = threadIdx.x & 31;
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float4 ml = from[n * 9 + 8][lane];
            const float om[2] = {ml.x, ml.y}, ol[2] = {ml.z, ml.w};
            float fa[2], fb[2];
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float now = fmaxf(m[n][c], om[c]), ref = now == -INFINITY ? 0.f : now;
                fa[c] = ex2(m[n][c] - ref);
                fb[c] = ex2(om[c] - ref);
                m[n][c] = now;
                l[n][c] = __fmaf_rn(l[n][c], fa[c], ol[c] * fb[c]);
            }
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float4 v = from[n * 9 + j][lane];
                o[n][j][0] = __fmaf_rn(o[n][j][0], fa[0], v.x * fb[0]);
                o[n][j][1] = __fmaf_rn(o[n][j][1], fa[1], v.y * fb[1]);
                o[n][j][2] = __fmaf_rn(o[n][j][2], fa[0], v.z * fb[0]);
                o[n][j][3] = __fmaf_rn(o[n][j][3], fa[1], v.w * fb[1]);
            }
        }
    }

    // rows r0 .. of the pair as results, or as the part `part` (>= 0)
    template <class O>
    __device__ __forceinline__ void store(const Attn8Params& p, int b, int h, int row_block, int r0, int part) const {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        #pragma unroll
        for (int n = 0; n < NT; ++n)
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int in = r0 + 8 * n + 2 * t + c, r = row_block * p.block_rows + in;
                if (r >= p.rows) continue;
                if (part >= 0) {
                    const size_t at = (size_t)part * p.block_rows + in;
                    float4* to = reinterpret_cast<float4*>(p.part_o + at * kServeDim + 16 * g);
                    #pragma unroll
                    for (int j = 0; j < 8; j += 2)
                        to[j / 2] = make_float4(o[n][j][c], o[n][j][c + 2], o[n][j + 1][c], o[n][j + 1][c + 2]);
                    if (g == 0) p.part_ml[at] = make_float2(m[n][c], l[n][c]);
                    continue;
                }
                const float inv = m[n][c] == -INFINITY && l[n][c] == 0.f ? 0.f : __fdiv_rn(1.f, l[n][c]);
                O* to = static_cast<O*>(p.out) +
                        (((size_t)b * p.n_q + r / p.group) * p.n_head + (size_t)h * p.group + r % p.group) * kServeDim + 16 * g;
                #pragma unroll
                for (int j = 0; j < 8; j += 2)
                    st4(to + 2 * j, make_float4(o[n][j][c] * inv, o[n][j][c + 2] * inv, o[n][j + 1][c] * inv, o[n][j + 1][c + 2] * inv));
            }
    }
};

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

__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// The loading warp's place: unit by unit through its run.
struct Place {
    int b, slot, len, tiles, pair, head, row_block, tile;    // pair: head * row blocks + row block
};

template <class Q, class O, int NT>
__global__ void __launch_bounds__(kE8Threads, e8_ctas(NT))
attn_kv8_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                const __grid_constant__ PagesDev pg, const __grid_constant__ Attn8Params p) {
    constexpr int P = std::is_same<Q, float>::value ? 2 : 1, STAGES = e8_stages(NT);
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Shared8<NT>& sh = *reinterpret_cast<Shared8<NT>*>(smem_raw);
    pdl_trigger();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    volatile int* const ab = &sh.abort;
    if ((smem_u32(smem_raw) & 1023u) != 0) {        // (the swizzle counts from a 1024-byte boundary)
        if (t == 0) {
            raise(p.status, SLLM_CUDA_ERR_DEVICE);
            p.shared[blockIdx.x] = make_int4(-1, 0, 0, 0);
        }
        return;
    }
    if (t == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&sh.full[i], 1 + 2 * kE8Blocks);
            mbar_init(&sh.empty[i], kE8Warps);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.merged[i], 1);
            mbar_init(&sh.taken[i], 1);
        }
        mbar_init(&sh.passed, 1);
        sh.abort = 0;
        sh.start_b = p.n;
        sh.start_rest = 0;
        fence_proxy_async_smem();
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // this CTA's run of units: a prefix sum over the sequences, each thread some of them
    const int pairs = p.n_kv * p.row_blocks, per = (p.n + kE8Threads - 1) / kE8Threads;
    const int b0 = min(t * per, p.n), b1 = min(b0 + per, p.n);
    unsigned long long mine = 0;
    for (int b = b0; b < b1; ++b) {
        int slot, len;
        const int tiles = seq_tiles(pg, p, b, &slot, &len);
        if (tiles == 0 && blockIdx.x == 0) raise(p.status, SLLM_CUDA_ERR_ARG);
        mine += (unsigned long long)tiles * pairs;
    }
    unsigned long long upto = mine;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    if (lane == 31) sh.scan[warp] = upto;
    __syncthreads();
    unsigned long long all = 0;
    #pragma unroll
    for (int w = 0; w < kE8Threads / 32; ++w) {
        if (w < warp) upto += sh.scan[w];
        all += sh.scan[w];
    }
    const unsigned long long G = gridDim.x < all ? gridDim.x : all;     // runs
    const unsigned long long c = blockIdx.x;
    if (c >= G) {
        if (t == 0) p.shared[c] = make_int4(-1, 0, 0, 0);
        return;
    }
    const unsigned long long u0 = c * all / G, u1 = (c + 1) * all / G;
    if (u0 >= upto - mine && u0 < upto) {
        unsigned long long rest = u0 - (upto - mine);
        for (int b = b0; b < b1; ++b) {
            int slot, len;
            const unsigned long long units = (unsigned long long)seq_tiles(pg, p, b, &slot, &len) * pairs;
            if (rest < units) {
                sh.start_b = b;
                sh.start_rest = rest;
                break;
            }
            rest -= units;
        }
    }
    __syncthreads();

    const Waits w{p};
    bool ok = true;
    if (warp == kE8Warps) {
        // ---- loads
        auto enter = [&](Place& x, int b) {         // the next sequence that has tiles; false: none
            for (x.tiles = 0; b < p.n && x.tiles == 0; ++b) {
                x.b = b;
                x.tiles = seq_tiles(pg, p, b, &x.slot, &x.len);
            }
            return x.tiles > 0;
        };
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
        Place cur;
        unsigned long long left = u1 - u0;
        // (lengths that somebody writes to meanwhile end the run early, inside the arrays)
        cur.pair = cur.tile = cur.head = cur.row_block = 0;
        if (!enter(cur, sh.start_b) || sh.start_rest >= (unsigned long long)cur.tiles * pairs) {
            left = 0;
        } else {
            cur.pair = (int)(sh.start_rest / cur.tiles);
            cur.tile = (int)(sh.start_rest % cur.tiles);
            cur.head = cur.pair / p.row_blocks;
            cur.row_block = cur.pair % p.row_blocks;
        }
        int id = left > 0 ? ids(cur) : 0;
        int first = 1, started = cur.tile == 0;     // of the segment: its first tile here; whether the pair starts here
        int4 note = make_int4(-1, 0, 0, 0);
        uint32_t n = 0;
        for (; left > 0 && ok; --left, ++n) {
            Place nxt = cur;
            int nid = 0;
            if (left > 1) {
                if (++nxt.tile == nxt.tiles) {
                    nxt.tile = 0;
                    if (++nxt.row_block == p.row_blocks) {
                        nxt.row_block = 0;
                        ++nxt.head;
                    }
                    if (++nxt.pair == pairs) {
                        nxt.pair = nxt.head = 0;
                        if (!enter(nxt, cur.b + 1)) left = 1;
                    }
                }
                if (left > 1) nid = ids(nxt);
            }
            const int slot = n % STAGES;
            if (n >= STAGES && !(ok = at_wait_warp(&sh.empty[slot], (n / STAGES - 1) & 1, ab, w))) break;
            const bool ends = cur.tile + 1 == cur.tiles, last = ends || left == 1;
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
                tma_load_4d(sh.k[slot] + at, &tm_k, 0, 0, cur.head, id, &sh.full[slot]);
                tma_load_4d(sh.v[slot] + at, &tm_v, 0, 0, cur.head, id, &sh.full[slot]);
            }
            const int blk = lane & (kE8Blocks - 1), from = __shfl_sync(0xffffffffu, id, (blk * kKvBlock) >> p.page_log2);
            if (lane < 2 * kE8Blocks) {
                if (blk * kKvBlock < keys)
                    cp_async4(&sh.sc[slot][lane], (lane < kE8Blocks ? p.ksc : p.vsc) + (size_t)from * p.scale_stride +
                                                      cur.head * (pg.page / kKvBlock) +
                                                      ((key0 + blk * kKvBlock) & (pg.page - 1)) / kKvBlock);
                cp_async_arrive(&sh.full[slot]);
            }
            if (last && !ends && started) {         // other runs go on with this pair
                const unsigned long long end = u1 + (unsigned long long)(cur.tiles - cur.tile - 1);
                note = make_int4(cur.b, cur.head, (int)min((end * G - 1) / all, G - 1), cur.row_block);
            }
            first = last;
            started = last ? 1 : started;
            cur = nxt;
            id = nid;
        }
        if (ok) {
            const int slot = n % STAGES;
            ok = n < STAGES || at_wait_warp(&sh.empty[slot], (n / STAGES - 1) & 1, ab, w);
            if (ok) {
                if (lane == 0) {
                    sh.meta[slot] = Meta{0, 0, 0, 0, 0, E8_END};
                    mbar_arrive(&sh.full[slot]);
                }
                if (lane < 2 * kE8Blocks) mbar_arrive(&sh.full[slot]);
                ++n;
            }
        }
        if (lane == 0) p.shared[c] = note;
        // copies in flight end before the CTA does, also where the others gave up
        for (uint32_t i = n > STAGES ? n - STAGES : 0; i < n; ++i) at_drain(&sh.full[i % STAGES], (i / STAGES) & 1);
    } else {
        // ---- products. A warp has its share of the blocks of a tile (key group
        // kg) for its share of the rows (row group)
        const int RG = p.rg, KG = kE8Warps / RG, rgrp = warp % RG, kg = warp / RG, half = KG / 2;
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
                rows.clear();
                rows.template load<Q>(p, mt.b, mt.head, mt.row_block * p.block_rows + rgrp * 8 * NT, mt.len);
            }
            const int keys = min(kE8Keys, mt.len - mt.key0);
            const bool masked = mt.key0 + kE8Keys > mt.len - p.n_q + 1;
            const float* const sc = sh.sc[slot];
            // blocks kg and kg + KG, and so on: a short tile's are shared out, too
            #pragma unroll 1
            for (int blk = kg; blk * kKvBlock < keys; blk += 2 * KG) {
                const bool two = (blk + KG) * kKvBlock < keys;
                const float ks[2] = {sc[blk], two ? sc[blk + KG] : 0.f};
                const float vs[2] = {sc[kE8Blocks + blk], two ? sc[kE8Blocks + blk + KG] : 0.f};
                rows.blocks(sh.k[slot] + blk * kKvBlock * kServeDim, sh.v[slot] + blk * kKvBlock * kServeDim,
                            KG * kKvBlock * kServeDim, ks, vs, masked, mt.key0 + blk * kKvBlock, KG * kKvBlock);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.empty[slot]);
            if (!(mt.flags & E8_LAST)) continue;
            rows.total();
            const uint32_t par = seg & 1;
            ++seg;
            // the key groups' parts into one: the upper half gives, the lower takes
            if (KG > 1) {
                const int at = (kg >= half ? kg - half : kg) * RG + rgrp;
                if (kg >= half) {
                    if (seg > 1 && !(ok = at_wait_warp(&sh.taken[at], par ^ 1, ab, w))) break;
                    rows.give(sh.merge[at]);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.merged[at]);
                    continue;
                }
                if (!(ok = at_wait_warp(&sh.merged[at], par, ab, w))) break;
                rows.take(sh.merge[at]);
                __syncwarp();
                if (KG == 4 && kg == 1) {           // (its place is free again when warp 0 has read it)
                    rows.give(sh.merge[1]);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.passed);
                    continue;
                }
                if (lane == 0) mbar_arrive(&sh.taken[at]);
                if (KG == 4) {
                    if (!(ok = at_wait_warp(&sh.passed, par, ab, w))) break;
                    rows.take(sh.merge[1]);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.taken[1]);
                }
            }
            const int part = mt.flags & E8_PART0 ? 2 * (int)c : mt.flags & E8_PART1 ? 2 * (int)c + 1 : -1;
            rows.template store<O>(p, mt.b, mt.head, mt.row_block, rgrp * 8 * NT, part);
        }
    }
    if (!ok && lane == 0) raise(p.status, SLLM_CUDA_ERR_TIMEOUT);
}

// ---------------------------------------------------------------------------
// the join of pairs that several runs share: a row per warp, or per several
// where rows are few
// ---------------------------------------------------------------------------
constexpr int kJoinWarps = 4;
template <class O>
__global__ void __launch_bounds__(32 * kJoinWarps)
attn_kv8_join_kernel(const __grid_constant__ Attn8Params p, int per_row) {
    __shared__ float4 so[kJoinWarps][32];
    __shared__ float2 sm[kJoinWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x;
    const int sub = warp % per_row, in = blockIdx.y * (kJoinWarps / per_row) + warp / per_row;
    pdl_wait();
    const int4 note = p.shared[c];
    if (note.x < 0) return;
    const int h = note.y, r = note.w * p.block_rows + in;
    const bool live = in < p.block_rows && r < p.rows;
    // parts: the second of this CTA's, then the first of the following CTAs'
    const int parts = note.z - c + 1;
    auto at = [&](int i) { return (size_t)(i == 0 ? 2 * c + 1 : 2 * (c + i)) * p.block_rows + in; };
    float M = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) {
        for (int i0 = sub; i0 < parts; i0 += 8 * per_row) {
            float4 v[8];
            float2 ml[8];
            #pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = i0 + e * per_row;
                ml[e] = make_float2(-INFINITY, 0.f);
                if (i < parts) {
                    ml[e] = __ldcg(p.part_ml + at(i));
                    v[e] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at(i) * kServeDim) + lane);
                }
            }
            float now = M;
            #pragma unroll
            for (int e = 0; e < 8; ++e) now = fmaxf(now, ml[e].x);
            const float ref = now == -INFINITY ? 0.f : now, f0 = ex2(M - ref);
            M = now;
            l *= f0;
            o.x *= f0; o.y *= f0; o.z *= f0; o.w *= f0;
            #pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (i0 + e * per_row >= parts) continue;
                const float f = ex2(ml[e].x - ref);
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
            const float now = fmaxf(M, b.x), ref = now == -INFINITY ? 0.f : now, f0 = ex2(M - ref), f1 = ex2(b.x - ref);
            M = now;
            l = __fmaf_rn(l, f0, b.y * f1);
            o.x = __fmaf_rn(o.x, f0, v.x * f1);
            o.y = __fmaf_rn(o.y, f0, v.y * f1);
            o.z = __fmaf_rn(o.z, f0, v.z * f1);
            o.w = __fmaf_rn(o.w, f0, v.w * f1);
        }
    }
    if (!live) return;
    const float inv = M == -INFINITY && l == 0.f ? 0.f : __fdiv_rn(1.f, l);
    st4(static_cast<O*>(p.out) + (((size_t)note.x * p.n_q + r / p.group) * p.n_head + (size_t)h * p.group + r % p.group) * kServeDim + 4 * lane,
        make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Rows of a CTA: 8 NT a warp, and row groups so that the four warps share them
// and the keys; beyond 64 rows a pair is read once for every 64.
struct Cut8 {
    int nt, rg, block_rows, row_blocks, ctas;
};
Cut8 cut8(int rows, int sms) {
    Cut8 x;
    x.nt = rows <= 8 ? 1 : 2;
    x.rg = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    x.block_rows = 8 * x.nt * x.rg;
    x.row_blocks = (rows + x.block_rows - 1) / x.block_rows;
    x.ctas = sms * e8_ctas(x.nt);
    return x;
}

// (rises with the rows: 8 * 3, 16 * 2, 32 * 2, 64 * 2 a SM)
size_t work8_bytes(const Cut8& x) {
    return (size_t)x.ctas * (2 * x.block_rows * (kServeDim * sizeof(float) + sizeof(float2)) + sizeof(int4));
}

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
    constexpr int kBytes = (int)sizeof(Shared8<NT>);
    const cudaError_t e = allow_smem<attn_kv8_kernel<Q, O, NT>>(kBytes);
    return e != cudaSuccess ? e : launch(attn_kv8_kernel<Q, O, NT>, dim3(ctas), dim3(kE8Threads), kBytes, st, false, tk, tv, pg, a);
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
    return work8_bytes(cut8(n_q * (n_head / p->n_head_kv), current_sms()));
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
    const Cut8 cut = cut8(n_q * (n_head / p->n_head_kv), current_sms());
    const size_t need = work8_bytes(cut);
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
    a.ksc = p->k_scale + layer * layer_scales;
    a.vsc = p->v_scale + layer * layer_scales;
    a.scale_stride = p->n_layer * layer_scales;
    a.slots = slots;
    a.n = n; a.n_q = n_q; a.n_head = n_head; a.n_kv = p->n_head_kv; a.group = n_head / p->n_head_kv;
    a.rows = n_q * a.group;
    a.rg = cut.rg; a.row_blocks = cut.row_blocks; a.block_rows = cut.block_rows;
    while ((1 << a.page_log2) < p->page_size) ++a.page_log2;
    a.wait = attn_wait_limit();
    a.status = status;
    a.part_o = static_cast<float*>(work);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)2 * cut.ctas * cut.block_rows * kServeDim);
    a.shared = reinterpret_cast<int4*>(a.part_ml + (size_t)2 * cut.ctas * cut.block_rows);
    const PagesDev pg = pages_dev(*p);
    const cudaStream_t st = (cudaStream_t)stream;
    CUtensorMap tk, tv;
    if (!encode_codes(&tk, static_cast<const int8_t*>(p->k) + layer * layer_codes, *p) ||
        !encode_codes(&tv, static_cast<const int8_t*>(p->v) + layer * layer_codes, *p))
        return fail(SLLM_CUDA_ERR_DEVICE, "attn_kv8: a tensor map could not be made");
    const bool f32 = q_type == SLLM_CUDA_KV_F32, out32 = out_type == SLLM_CUDA_KV_F32;
    cudaError_t e;
    if (cut.nt == 1)
        e = f32     ? launch8<float, float, 1>(tk, tv, pg, a, cut.ctas, st)
            : out32 ? launch8<__half, float, 1>(tk, tv, pg, a, cut.ctas, st)
                    : launch8<__half, __half, 1>(tk, tv, pg, a, cut.ctas, st);
    else
        e = f32     ? launch8<float, float, 2>(tk, tv, pg, a, cut.ctas, st)
            : out32 ? launch8<__half, float, 2>(tk, tv, pg, a, cut.ctas, st)
                    : launch8<__half, __half, 2>(tk, tv, pg, a, cut.ctas, st);
    CK(e, "attn_kv8 launch");
    const int per_row = cut.block_rows <= 8 ? 4 : cut.block_rows <= 16 ? 2 : 1;
    const dim3 grid(cut.ctas, (cut.block_rows * per_row + kJoinWarps - 1) / kJoinWarps);
    CK(out32 ? launch(attn_kv8_join_kernel<float>, grid, dim3(32 * kJoinWarps), 0, st, true, a, per_row)
             : launch(attn_kv8_join_kernel<__half>, grid, dim3(32 * kJoinWarps), 0, st, true, a, per_row),
       "attn_kv8 join");
    count_launches(2);
    return SLLM_CUDA_OK;
}
