/*
 * sllm_cuda.h -- the C ABI of the B200 (sm_100a) backend for saphira-llm's
 * I2_S ternary decode path.
 *
 * Everything here is plain C: pointers, sizes and int status codes. No CUDA,
 * torch or C++ type crosses this boundary, so saphira-llm's C11 host code can
 * include this header and link libsllm_cuda.so directly. A stream is passed as
 * `void *` (a cudaStream_t value; NULL means the legacy default stream).
 *
 * Each entry point names the reference interface it replaces, as
 * path:line inside the saphira-llm source tree.
 *
 * Conventions, held by every function below:
 *   - Status codes are numerically identical to saphira-llm's sllm_status
 *     (include/saphira_llm/status.h:26-56), so a caller can return them
 *     unchanged. Three new negative codes (-60, -61, -62) name device-side
 *     failures.
 *   - The kernel-level functions take DEVICE pointers and are asynchronous on
 *     the given stream. The model-level functions take HOST pointers and
 *     return when their results are on the host.
 *   - Once this backend is selected there is no CPU fallback. A missing or
 *     unsuitable device is reported as SLLM_CUDA_ERR_UNSUPPORTED, never
 *     silently computed on the host.
 */
#ifndef SLLM_CUDA_H
#define SLLM_CUDA_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#  define SLLM_CUDA_API __attribute__((visibility("default")))
#else
#  define SLLM_CUDA_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* the types of a KV cache (sllm_cuda_ctx_new_kv, sllm_cuda_kv_pages) */
#define SLLM_CUDA_KV_F32 0
#define SLLM_CUDA_KV_F16 1
#define SLLM_CUDA_KV_I8  2      /* paged caches only (sllm_cuda_kv_pages) */

/* ------------------------------------------------------------------ */
/* status codes                                                        */
/* ------------------------------------------------------------------ */

#define SLLM_CUDA_OK               0    /* SLLM_OK                  */
#define SLLM_CUDA_ERR_ARG         (-1)  /* SLLM_ERR_ARG             */
#define SLLM_CUDA_ERR_NOMEM       (-2)  /* SLLM_ERR_NOMEM: host or device allocation failed */
#define SLLM_CUDA_ERR_IO          (-3)  /* SLLM_ERR_IO              */
#define SLLM_CUDA_ERR_UNSUPPORTED (-4)  /* SLLM_ERR_UNSUPPORTED: no sm_100 device, or a shape this backend does not run */
#define SLLM_CUDA_ERR_TRUNCATED   (-12) /* SLLM_ERR_GGUF_TRUNCATED: a state file ends early */
#define SLLM_CUDA_ERR_KV_TYPE     (-32) /* SLLM_ERR_KV_TYPE: not a state file, or another version */
#define SLLM_CUDA_ERR_TENSOR_SHAPE (-34) /* SLLM_ERR_TENSOR_SHAPE: a state file of another geometry */
#define SLLM_CUDA_ERR_TOO_LARGE   (-36) /* SLLM_ERR_TOO_LARGE       */
#define SLLM_CUDA_ERR_DEVICE      (-60) /* a CUDA runtime call or kernel launch failed */
#define SLLM_CUDA_ERR_TIMEOUT     (-61) /* a bounded device-side wait ran out; the context stays usable */
#define SLLM_CUDA_ERR_COMM        (-62) /* a collective between devices failed */

/* Stable, human-readable name for a status. Never NULL. */
SLLM_CUDA_API const char * sllm_cuda_status_string(int status);

/* The message recorded with the most recent failure on this thread, or "". */
SLLM_CUDA_API const char * sllm_cuda_last_error(void);

/*
 * Capability probe for the dispatch row (src/dispatch.c:133
 * sllm_dispatch_resolve, src/i2s_gemm.c:315 sllm_i2s_select_auto).
 * Reports the device count and the compute capability of device 0.
 * Returns SLLM_CUDA_ERR_UNSUPPORTED when no device of compute capability
 * 10.x is visible. Any output pointer may be NULL.
 */
SLLM_CUDA_API int sllm_cuda_probe(int * n_devices, int * cc_major, int * cc_minor);

/* ------------------------------------------------------------------ */
/* kernel level: device pointers, asynchronous on `stream`             */
/* ------------------------------------------------------------------ */

/* Layout-identical to sllm_i2s_act (include/saphira_llm/i2s_gemm.h:37-40). */
typedef struct sllm_cuda_act {
    float   scale;   /* 127 / amax, or 0 for an all-zero row */
    int32_t sum;     /* sum of the quantised values          */
} sllm_cuda_act;

/*
 * Per-token int8 absmax quantisation of one row of `n` floats.
 * Replaces sllm_i2s_quant_act (include/saphira_llm/i2s_gemm.h:57,
 * src/i2s_gemm.c:45-83) with identical results: amax without a floor,
 * scale = 127/amax (IEEE division), q = clamp(roundf(x*scale)), sum of q.
 * `act_out` is one device struct. n must be >= 1 and <= 65536.
 */
SLLM_CUDA_API int sllm_cuda_i2s_quant_act(const float * x, size_t n, int8_t * q_out,
                            sllm_cuda_act * act_out, void * stream);

/*
 * Raw I2_S GEMV: rows_out[r] = sum over k of code(w, r, k) * q[k], the
 * 2-bit code (0, 1 or 2) times the int8 activation, in int32.
 * Replaces sllm_i2s_gemv (include/saphira_llm/i2s_gemm.h:81,
 * src/i2s_gemm.c:260-269) bit for bit. `w` is the packed tensor as stored in
 * the GGUF (rows of n/4 bytes, I2_S interleaved layout). Unlike the reference,
 * which silently returns 0 for n < 128, this returns SLLM_CUDA_ERR_ARG for
 * n % 128 != 0 (the loader refuses such tensors anyway, src/forward.c:306-316).
 * n above 8192 is refused with SLLM_CUDA_ERR_UNSUPPORTED (the 2B-4T model's
 * widths are 2560 and 6912; the tensor-parallel path splits wider
 * contractions into chunks of at most 8192).
 */
SLLM_CUDA_API int sllm_cuda_i2s_gemv(const uint8_t * w, size_t n_rows, size_t n,
                       const int8_t * q, int32_t * rows_out, void * stream);

/*
 * Fused float GEMV: quantise x (as sllm_cuda_i2s_quant_act), run the raw GEMV
 * and apply the epilogue y[r] = (float)(dot[r] - act.sum) * (w_scale / act.scale),
 * where w_scale is the f32 stored after the packed weights
 * (src/quant.c:102-106). This is the sequence src/forward.c:651-655 runs for
 * every projection, and the epilogue grouping is sllm_i2s_epilogue's
 * (src/i2s_gemm.c:271-290). `dots` (nullable) receives the raw int32 dots.
 */
SLLM_CUDA_API int sllm_cuda_i2s_gemv_f32(const uint8_t * w, size_t n_rows, size_t n,
                           const float * x, float * y, int32_t * dots,
                           void * stream);

/*
 * A batch of `count` (<= 256) independent float GEMVs of one shape, each as
 * sllm_cuda_i2s_gemv_f32 computes it, run as one persistent launch: GEMV i
 * reads the packed tensor w[i] (device, 16-byte aligned, scale tail after the
 * codes), input x + i * x_stride (x_stride 0: every GEMV shares x, as Q, K and
 * V share one quantised activation in src/forward.c:651-666) and writes
 * y + i * n_rows. It replaces a host loop of sllm_i2s_quant_act +
 * sllm_i2s_gemv + epilogue over tensors (src/i2s_gemm.c:45-83, :260-290;
 * bench/kernel_bench.c:62-130 times such loops). n_rows % 4 == 0. The first
 * run with given x, x_stride and y builds the launch's tables (device
 * allocation); later runs with the same buffers only launch. Results are
 * bit-identical to sllm_cuda_i2s_gemv_f32 on each tensor.
 */
typedef struct sllm_cuda_gemv_batch sllm_cuda_gemv_batch;
SLLM_CUDA_API int sllm_cuda_gemv_batch_new(const uint8_t * const * w, size_t count, size_t n_rows,
                                           size_t n, int device, sllm_cuda_gemv_batch ** out);
SLLM_CUDA_API int sllm_cuda_gemv_batch_run(sllm_cuda_gemv_batch * b, const float * x, size_t x_stride,
                                           float * y, void * stream);
SLLM_CUDA_API void sllm_cuda_gemv_batch_free(sllm_cuda_gemv_batch * b);

/* ------------------------------------------------------------------ */
/* multi-token (prefill) kernels: device pointers                      */
/* ------------------------------------------------------------------ */

/*
 * Per-token activation quantisation of a row-major [m][n] batch: row t of q
 * and acts[t] are sllm_i2s_quant_act of row t of x
 * (include/saphira_llm/i2s_gemm.h:59, src/i2s_gemm.c:45-83), the per-token
 * quantisation the prefill runs before each projection (src/forward.c:756-764).
 */
SLLM_CUDA_API int sllm_cuda_i2s_quant_act_rows(const float * x, size_t m, size_t n,
                                 int8_t * q, sllm_cuda_act * acts, void * stream);

/*
 * Prefill GEMM on the tensor cores: for every token t < m and row r <
 * n_rows, dots[t][r] = sum over k of code(w, r, k) * q[t][k] (int32), which is
 * sllm_i2s_gemv of token t (src/i2s_gemm.c:260-269) bit for bit, and
 * y[t][r] = (float)(dots[t][r] - acts[t].sum) * (w_scale / acts[t].scale),
 * the per-token epilogue of src/forward.c:653-655. The reference has no GEMM:
 * its prefill runs the GEMV once per token; this computes all of them in one
 * int8 contraction. q is row-major [m][n]; dots and y are row-major
 * [m][n_rows] and either may be NULL (not both). n % 128 == 0, n <= 65536;
 * w and q 16-byte aligned. Asynchronous on `stream`.
 */
SLLM_CUDA_API int sllm_cuda_i2s_gemm(const uint8_t * w, size_t n_rows, size_t n, size_t m,
                       const int8_t * q, const sllm_cuda_act * acts,
                       int32_t * dots, float * y, void * stream);

/*
 * The gate/up pair of the prefill FFN in one pass: h[t][r] =
 * silu(gate[t][r]) * up[t][r], each projection with the epilogue above and
 * SiLU as sllm_silu_inplace computes it (src/forward.c:756-779,
 * src/ops.c:428-461). w_gate and w_up have the same shape.
 */
SLLM_CUDA_API int sllm_cuda_i2s_gemm_silu(const uint8_t * w_gate, const uint8_t * w_up, size_t n_rows,
                            size_t n, size_t m, const int8_t * q,
                            const sllm_cuda_act * acts, float * h, void * stream);

/* ------------------------------------------------------------------ */
/* attention, paged cache and drafts: device pointers                  */
/* ------------------------------------------------------------------ */
/*
 * Operators for a caller that keeps its own device buffers and runs the
 * projections with the kernels above: what stands between Q/K/V and O
 * (attention over whole prompts, and over a paged cache while decoding), the
 * cache itself, and the choice of the next tokens when a draft is verified.
 * The reference has one contiguous cache per sequence and greedy choice only
 * (src/forward.c:466-562, :698-726, :876-883); these are additions beside it,
 * and they do not keep its summation order: results agree to the rounding of
 * 32-bit sums, not bit for bit.
 *
 * Rules for all of them:
 *   - head dim 128, as everywhere in this library; types are
 *     SLLM_CUDA_KV_F32 / _F16, and of a paged cache SLLM_CUDA_KV_I8 besides;
 *   - every array is memory of the current device (anything else is refused
 *     with SLLM_CUDA_ERR_ARG); `stream` belongs to that device;
 *   - asynchronous on `stream`, no allocation, no synchronisation: they can
 *     be captured into a CUDA graph;
 *   - a workspace is the caller's, 16-byte aligned, and holds nothing between
 *     calls. Calls (or graphs) that may overlap need workspaces of their own;
 *   - a kv_* call that names no slot (n = 0) does nothing; its lists may be NULL;
 *   - outputs and workspaces overlap no other array of the call (kv_append may
 *     write q_out, k_out and v_out exactly over contiguous f32 q, k and v);
 *   - what only the device can see to be wrong (a slot, a length or a page id
 *     out of range) is reported in `*status`, a device int that may be NULL:
 *     set to an SLLM_CUDA_ERR_* code, never cleared. Nothing outside the
 *     arrays is read or written in that case. SLLM_CUDA_ERR_TIMEOUT there is a
 *     bounded wait inside a kernel that ran out: the call's output means
 *     nothing, the device is fine.
 */

/*
 * Causal attention over packed whole prompts. Sequence s holds the tokens
 * cu_seqlens[s] .. cu_seqlens[s + 1] - 1 (n_seq + 1 ascending device ints, the
 * last at most n_tokens; empty sequences are allowed); token i of a sequence
 * sees its tokens 0 .. i:
 *     out[i][h] = sum_j softmax_j(q[i][h] . k[j][g] / sqrt(128)) v[j][g],
 * g = h / (n_head / n_head_kv). Token t's heads lie at q + t * q_stride
 * (elements; at least n_head * 128, rows 16-byte aligned), so the parts of one
 * Q/K/V array can be passed as they are. Rows of `out` behind the last
 * sequence are not written. A key that a row does not see leaves no trace in
 * it, not even as an infinity or a NaN; in a row that does see it, a value that
 * is no finite number leaves none in its dimension, a key may leave none in all
 * (in f16 a score of -inf only has weight 0). q, k and v have type `type`; out is
 * f32 or, from f16, f16. f16 inputs are multiplied on the tensor cores with
 * f32 sums and softmax; the softmax weights are rounded to f16 there (11 bits
 * down to 2^-21 of a row's largest, fewer down to 2^-31, 0 below). f32 counts as
 * infinite from 2^128 - 2^119 on.
 * The first form has no status word: wrong offsets stay inside the arrays, but
 * nobody hears of them, nor of a bounded wait that ran out. The second reports
 * both in `*status`. n_seq <= 2^20, n_tokens <= 2^24, n_head <= 1024, strides <=
 * 2^30.
 */
SLLM_CUDA_API int sllm_cuda_attn_prompt(const void * q, size_t q_stride, const void * k, size_t k_stride,
                                        const void * v, size_t v_stride, int32_t type,
                                        const int32_t * cu_seqlens, int32_t n_seq, int32_t n_tokens,
                                        int32_t n_head, int32_t n_head_kv, void * out, size_t out_stride,
                                        int32_t out_type, void * stream);
SLLM_CUDA_API int sllm_cuda_attn_prompt_checked(const void * q, size_t q_stride, const void * k, size_t k_stride,
                                                const void * v, size_t v_stride, int32_t type,
                                                const int32_t * cu_seqlens, int32_t n_seq, int32_t n_tokens,
                                                int32_t n_head, int32_t n_head_kv, void * out, size_t out_stride,
                                                int32_t out_type, int32_t * status, void * stream);

/*
 * A paged KV cache in the caller's memory. Pools are
 * [n_pages][n_layer][n_head_kv][page_size][128]; slot (sequence) s holds
 * lens[s] tokens, token t in row t % page_size of page
 * tables[s * table_width + t / page_size]. refs[p] is the number of table
 * entries that name page p; 0 means free. Entries behind a slot's last page
 * mean nothing. An empty cache is all zeros in refs and lens. Slots may share
 * pages (kv_fork); only a page with one owner is ever written. At most 2^24
 * pages, 65536 slots, 1024 layers and kv heads, 2^31 - 256 tokens a slot.
 */
typedef struct sllm_cuda_kv_pages {
    void    * k;
    void    * v;
    int32_t * refs;         /* [n_pages], 16-byte aligned */
    int32_t * tables;       /* [n_slots][table_width] */
    int32_t * lens;         /* [n_slots] */
    int32_t   n_pages, n_layer, n_head_kv;
    int32_t   page_size;    /* 16, 32, 64 or 128 tokens */
    int32_t   n_slots, table_width;
    int32_t   kv_type;      /* SLLM_CUDA_KV_F32, _F16 or _I8 */
    float   * k_scale;      /* SLLM_CUDA_KV_I8 alone (not read otherwise): */
    float   * v_scale;      /* [n_pages][n_layer][n_head_kv][page_size / 16], 16-byte aligned */
} sllm_cuda_kv_pages;

/*
 * SLLM_CUDA_KV_I8: pools of int8 codes c in [-127, 127] and one scale s for 16
 * tokens of a head (tokens 16 b .. 16 b + 15 of a sequence, a block); a value is
 * c * s. sllm_cuda_kv8_append writes such a cache, sllm_cuda_kv8_read reads it back,
 * sllm_cuda_attn_kv8 attends over it; kv_fork, kv_reserve, kv_release and kv_compact
 * take it as they take the others. kv_append and attn_prefix refuse it.
 */

/* Bytes of the workspace that the four calls below take; 0 for a bad cache. */
SLLM_CUDA_API size_t sllm_cuda_kv_work_bytes(const sllm_cuda_kv_pages * p);

/*
 * Slot dst[i] becomes a copy of what slot src[i] held before the call, for all
 * i < n at once (so a slot may be a source and a destination, as when beams
 * are reordered); what it held itself is given up. All pages are shared, none
 * is copied. A slot named twice in dst, or a wrong slot or table, is
 * SLLM_CUDA_ERR_ARG in *status, and nothing changes.
 */
SLLM_CUDA_API int sllm_cuda_kv_fork(const sllm_cuda_kv_pages * p, const int32_t * src, const int32_t * dst,
                                    int32_t n, void * work, size_t work_bytes, int32_t * status,
                                    void * stream);

/*
 * Room for n_new[i] more tokens in slots[i], whose length moves on by as many:
 * new pages are the free ones of lowest id, in the order of the slots. A
 * partly filled last page with other owners is replaced by a copy of its live
 * rows first (copy on write); of owners that are all named in the call, the
 * last keeps the page. In *status: SLLM_CUDA_ERR_NOMEM when too few pages are
 * free, SLLM_CUDA_ERR_TOO_LARGE when a table is too short, SLLM_CUDA_ERR_ARG
 * for wrong or repeated slots; nothing changes then.
 */
SLLM_CUDA_API int sllm_cuda_kv_reserve(const sllm_cuda_kv_pages * p, const int32_t * slots,
                                       const int32_t * n_new, int32_t n, void * work, size_t work_bytes,
                                       int32_t * status, void * stream);

/*
 * slots[i] keeps its first new_len[i] tokens (none where new_len is NULL); the
 * pages behind them lose an owner, and are free when they have none left.
 * SLLM_CUDA_ERR_ARG in *status, and nothing changes, for wrong or repeated
 * slots or a length above the slot's.
 */
SLLM_CUDA_API int sllm_cuda_kv_release(const sllm_cuda_kv_pages * p, const int32_t * slots,
                                       const int32_t * new_len, int32_t n, void * work, size_t work_bytes,
                                       int32_t * status, void * stream);

/*
 * Moves the live pages to the lowest ids: with L live pages, the live pages at
 * or above L, ascending, go into the free ones below L, ascending; tables and
 * counts follow. A table that names a wrong or free page is
 * SLLM_CUDA_ERR_ARG in *status, and nothing changes.
 */
SLLM_CUDA_API int sllm_cuda_kv_compact(const sllm_cuda_kv_pages * p, void * work, size_t work_bytes,
                                       int32_t * status, void * stream);

/*
 * Stores the K and V of n_tokens tokens in one layer of the cache: token t at
 * position pos[t] of slot slot[t], below the slot's length (kv_reserve first).
 * q and k are rotated (RoPE NEOX, the decode path's operations,
 * src/ops.c:529-549) with row pos[t] of the [n_ctx][64] angle tables, then q,
 * k and v are rounded to the cache's type; q_out [n_tokens][n_head][128] and
 * k_out, v_out [n_tokens][n_head_kv][128] receive them too (k_out and v_out
 * may be NULL; q and q_out may both be NULL). Strides are floats from a token
 * to the next. A token with slot[t] < 0 is padding: nothing of it is
 * written. A token whose slot, position or page is wrong, or whose
 * page has other owners, sets SLLM_CUDA_ERR_ARG in *status and is left out.
 * Two tokens for one place leave a mix of both there.
 */
SLLM_CUDA_API int sllm_cuda_kv_append(const sllm_cuda_kv_pages * p, int32_t layer, int32_t n_tokens,
                                      const int32_t * slot, const int32_t * pos, int32_t n_head,
                                      const float * q, size_t q_stride, const float * k, size_t k_stride,
                                      const float * v, size_t v_stride, const float * rope_cos,
                                      const float * rope_sin, int32_t n_ctx, void * q_out, void * k_out,
                                      void * v_out, int32_t * status, void * stream);

/*
 * The angle tables of the decode path (host arrays of n_ctx * 64 floats), by
 * the reference's recurrence on the host libm (src/ops.c:529-549).
 */
SLLM_CUDA_API int sllm_cuda_rope_table(int32_t n_ctx, float rope_freq_base, float * cos_out, float * sin_out);

/*
 * Decode attention of n sequences whose first prefix_len tokens (whole pages)
 * are the same pages, as forks of one prompt have them: the prefix is read
 * and multiplied once for all of them, from slots[0]'s table. Sequence b's
 * n_q query tokens are the last n_q tokens of slots[b]: query j sees the
 * slot's first lens - n_q + 1 + j tokens (zeros come out where that is none).
 * n_q > 1 scores drafted tokens. Every query must see the whole prefix;
 * prefix_len 0 is plain paged decode attention. q and out are
 * [n][n_q][n_head][128], q of the cache's type, out f32 or, from an f16
 * cache, f16. A sequence whose slot, length or table is wrong sets
 * SLLM_CUDA_ERR_ARG in *status and its rows of out mean nothing (all rows,
 * where the prefix's pages are wrong). n <= 4096, n_q <= 16. A workspace of
 * work_bytes(n, n_q, n_head, prefix_len) serves every call over this cache with
 * that n_head and no more sequences, query tokens and prefix.
 */
SLLM_CUDA_API size_t sllm_cuda_attn_prefix_work_bytes(const sllm_cuda_kv_pages * p, int32_t n, int32_t n_q,
                                                      int32_t n_head, int32_t prefix_len);
SLLM_CUDA_API int sllm_cuda_attn_prefix(const sllm_cuda_kv_pages * p, int32_t layer, const void * q,
                                        const int32_t * slots, int32_t n, int32_t n_q, int32_t n_head,
                                        int32_t prefix_len, void * out, int32_t out_type, void * work,
                                        size_t work_bytes, int32_t * status, void * stream);

/*
 * Stores the K and V of n_tokens tokens in one layer of an 8-bit cache, rotated
 * and placed as kv_append does it. A block's scale is the largest |value| that was
 * stored in it, divided by 127 (at least 2^-100; 0 while all are 0), and a code is
 * value / scale rounded to the nearest, ties to even. Where a token needs a larger
 * scale, the codes of the block's earlier tokens (the rows before the first that
 * this call stores there) are rounded to it: each such step costs them up to half
 * a step of the new scale. Rows behind the last token stored mean nothing
 * afterwards, so tokens go in ascending order of their positions, and a position
 * may be stored again after kv_release. The call's tokens of one block
 * stand together in its lists, in ascending order; one that does not come after
 * the token before it of the same block sets SLLM_CUDA_ERR_ARG in *status and is
 * left out of the cache, with those of the block that stand after it. A block that
 * the lists come back to later leaves a mix of both. A NaN is stored as 0, an
 * infinity as 127 times the scale of the finite values, both with
 * SLLM_CUDA_ERR_ARG in *status.
 * q_out [n_tokens][n_head][128] and k_out, v_out [n_tokens][n_head_kv][128], of
 * type out_type, receive the rotated q, k and v before quantisation (k_out and
 * v_out may be NULL; q and q_out may both be NULL). Padding, wrong tokens and
 * strides as in kv_append.
 */
SLLM_CUDA_API int sllm_cuda_kv8_append(const sllm_cuda_kv_pages * p, int32_t layer, int32_t n_tokens,
                                       const int32_t * slot, const int32_t * pos, int32_t n_head,
                                       const float * q, size_t q_stride, const float * k, size_t k_stride,
                                       const float * v, size_t v_stride, const float * rope_cos,
                                       const float * rope_sin, int32_t n_ctx, void * q_out, void * k_out,
                                       void * v_out, int32_t out_type, int32_t * status, void * stream);

/*
 * Reads n_tokens tokens of one layer of an 8-bit cache back: k_out[t], v_out[t]
 * ([n_head_kv][128] each, of type out_type; either may be NULL) are the stored
 * values of position pos[t] of slot slot[t], in any order, rounded once to
 * out_type. A token with slot[t] < 0 is padding, and its rows are left as they
 * are; so are those of a token whose slot, position or page is wrong, which sets
 * SLLM_CUDA_ERR_ARG in *status. n_tokens <= 2^24.
 */
SLLM_CUDA_API int sllm_cuda_kv8_read(const sllm_cuda_kv_pages * p, int32_t layer, int32_t n_tokens,
                                     const int32_t * slot, const int32_t * pos, void * k_out, void * v_out,
                                     int32_t out_type, int32_t * status, void * stream);

/*
 * Decode attention of n sequences over an 8-bit cache: attn_prefix without a
 * shared prefix. Sequence b's n_q query tokens are the last n_q tokens of
 * slots[b]; query j sees the slot's first lens - n_q + 1 + j tokens (zeros come
 * out where that is none). q and out are [n][n_q][n_head][128]; q is of type
 * q_type, out f32 or, from f16 queries, f16. Codes are multiplied on the tensor
 * cores exactly, in f32 sums; f16 queries are taken as they are, f32 queries and
 * their softmax weights as pairs of f16 (22 bits), the weights of f16 queries
 * rounded to f16 (11 bits down to 2^-21 of a row's largest; of more than 16 query
 * rows a kv head the weights times their keys' value scales are, or the weights
 * alone where the tables have room for little). A sequence whose slot, length or
 * table is wrong sets SLLM_CUDA_ERR_ARG in *status, and its rows of out mean
 * nothing; a wait that runs out (2 s) sets SLLM_CUDA_ERR_TIMEOUT. n <= 4096, n_q
 * <= 16, n_head <= 1024. A workspace of work_bytes(n, n_q, n_head) serves every
 * call over this cache with that n_head and no more sequences and query tokens.
 */
SLLM_CUDA_API size_t sllm_cuda_attn_kv8_work_bytes(const sllm_cuda_kv_pages * p, int32_t n, int32_t n_q,
                                                   int32_t n_head);
SLLM_CUDA_API int sllm_cuda_attn_kv8(const sllm_cuda_kv_pages * p, int32_t layer, const void * q, int32_t q_type,
                                     const int32_t * slots, int32_t n, int32_t n_q, int32_t n_head, void * out,
                                     int32_t out_type, void * work, size_t work_bytes, int32_t * status,
                                     void * stream);

/*
 * One step of n beam searches of `beams` beams each. Request i's candidates are
 * (b, x): beam b continued by word x, of value
 *     score[i][b] + logits[i][b][x] - ln sum_y exp(logits[i][b][y])
 * (64 bits; the exponentials 32, their sum 64; logits beyond 2^100 as that, those of
 * a row whose largest is beyond 2^24 counted from it); a beam with done[i][b] != 0
 * has one candidate, eos, of its own score (done NULL: none is). The `beams` best
 * come out in descending order: parent, token and score_out [n][beams]. Equal
 * values: the lower beam first, then the larger logit, then the lower word. Row
 * (i, b) of the logits lies at logits + (i * beams + b) * row_stride. A score or
 * logit of -inf makes candidates of value -inf, which are chosen, lowest (b, x)
 * first, only when there are no others; NaN and +inf count as -inf and set
 * SLLM_CUDA_ERR_ARG in *status (the logits of beams that are done, or have a score
 * of -inf, are not read). done_out[i][j] (may be NULL) is 1 when the parent was done
 * or the token is eos. src[i][j] = slots[i][parent[i][j]] (both NULL or neither):
 * with them sllm_cuda_kv_fork(src, dst = slots) lets every beam's slot hold its
 * parent's tokens. eos < 0: no such word (then done and done_out must be NULL). The
 * outputs may not overlap score or done. beams <= 16, n <= 65536, n_vocab <= 2^20.
 */
SLLM_CUDA_API int sllm_cuda_beam_select(const float * logits, size_t row_stride, const float * score,
                                        const int32_t * done, const int32_t * slots, int32_t n, int32_t beams,
                                        int32_t n_vocab, int32_t eos, float * score_out, int32_t * parent,
                                        int32_t * token, int32_t * done_out, int32_t * src, int32_t * status,
                                        void * stream);

/*
 * Verification of drafted tokens, so that what comes out is distributed as
 * the target's own samples. p [n][k + 1][n_vocab] are the target's
 * probabilities after 0 .. k drafted tokens, q [n][k][n_vocab] the draft's
 * (NULL: the draft was certain of its tokens), draft [n][k] its tokens,
 * n_draft [n] how many each sequence has (NULL: k). With uniforms in [0, 1):
 * token t is accepted while u_accept[t] * q_t(x_t) < p_t(x_t); at the first
 * refusal t the next token is drawn from max(p_t - q_t, 0) (from p_t where
 * that has no mass), after the last accepted one from p: the first index whose
 * running sum exceeds u_draw times the sum (64-bit sums; u_draw within their
 * rounding of a border may take the neighbour). Negative, NaN and infinite
 * entries count as 0. tokens [n][k + 1] receives the accepted tokens, the
 * drawn one and -1 behind it, count [n] their number; the drawn token is -1
 * where p has no mass either. A drafted id out of range is refused, a draft
 * length out of range clamped, with SLLM_CUDA_ERR_ARG in *status.
 * 1 <= k <= 64, n <= 65536, n_vocab <= 2^24.
 */
SLLM_CUDA_API int sllm_cuda_spec_verify(const float * p, const float * q, const int32_t * draft,
                                        const int32_t * n_draft, const float * u_accept, const float * u_draw,
                                        int32_t n, int32_t k, int32_t n_vocab, int32_t * tokens, int32_t * count,
                                        int32_t * status, void * stream);

/* ------------------------------------------------------------------ */
/* model level: host pointers                                          */
/* ------------------------------------------------------------------ */

/*
 * One bitnet-b1.58 layer as the reference loader records it
 * (src/forward.c:47-54, filled at src/forward.c:391-444). The I2_S pointers
 * address packed tensors INCLUDING their scale tail (rows * cols / 4 bytes of
 * codes, then the f32 scale and 28 pad bytes). All pointers are host memory
 * and are only read during sllm_cuda_model_upload.
 */
typedef struct sllm_cuda_layer_desc {
    const uint8_t * wq;        /* n_embd     x n_embd  */
    const uint8_t * wk;        /* n_embd_gqa x n_embd  */
    const uint8_t * wv;        /* n_embd_gqa x n_embd  */
    const uint8_t * wo;        /* n_embd     x n_embd  */
    const uint8_t * ffn_gate;  /* n_ff       x n_embd  */
    const uint8_t * ffn_up;    /* n_ff       x n_embd  */
    const uint8_t * ffn_down;  /* n_embd     x n_ff    */
    const float   * attn_norm;      /* n_embd */
    const float   * attn_sub_norm;  /* n_embd */
    const float   * ffn_norm;       /* n_embd */
    const float   * ffn_sub_norm;   /* n_ff   */
} sllm_cuda_layer_desc;

/*
 * The model hyperparameters and tensors (src/forward.c:56-76; metadata keys
 * read at src/forward.c:348-366). `tok_embd` is the F16 [n_vocab][n_embd]
 * embedding that is also the tied output head.
 */
typedef struct sllm_cuda_model_desc {
    int32_t n_layer;
    int32_t n_embd;
    int32_t n_ff;
    int32_t n_head;
    int32_t n_head_kv;
    int32_t n_vocab;
    int32_t n_rot;
    int32_t n_ctx_train;
    float   f_rms_eps;
    float   rope_freq_base;
    const uint16_t * tok_embd;     /* F16 bits, n_vocab * n_embd */
    const float    * output_norm;  /* n_embd */
    const sllm_cuda_layer_desc * layers;  /* n_layer entries */
} sllm_cuda_model_desc;

typedef struct sllm_cuda_model sllm_cuda_model;
typedef struct sllm_cuda_ctx   sllm_cuda_ctx;

/*
 * Copy a model to device `device` once; the device copy is immutable and may
 * be shared by several contexts. Validates the same shape rules as
 * sllm_model_load (src/forward.c:368-444): returns SLLM_CUDA_ERR_ARG for a
 * NULL desc or tensor, SLLM_CUDA_ERR_UNSUPPORTED for widths this backend does
 * not run (n_embd or n_ff not a multiple of 128 or above 8192, a head dim
 * n_embd / n_head other than 128, n_rot other than the head dim,
 * n_head % n_head_kv != 0), SLLM_CUDA_ERR_NOMEM when device memory runs out.
 * Pairs with sllm_model_load / sllm_model_free (include/saphira_llm/forward.h:32-33).
 */
SLLM_CUDA_API int  sllm_cuda_model_upload(const sllm_cuda_model_desc * desc, int device,
                            sllm_cuda_model ** out);
SLLM_CUDA_API void sllm_cuda_model_free(sllm_cuda_model * m);

/*
 * A context owns the device-resident KV cache (fp32, [layer][head_kv][pos][dim],
 * src/forward.c:81-83) and the scratch of one sequence.
 * Replaces sllm_ctx_new / sllm_ctx_free / sllm_ctx_reset
 * (include/saphira_llm/forward.h:44-48, src/forward.c:466-562).
 */
SLLM_CUDA_API int  sllm_cuda_ctx_new(const sllm_cuda_model * m, int32_t n_ctx,
                       sllm_cuda_ctx ** out);

/*
 * The same with a choice of KV cache type. SLLM_CUDA_KV_F32 is the
 * reference's cache and sllm_cuda_ctx_new's. SLLM_CUDA_KV_F16 is an option the
 * reference does not have: every cached K and V value is stored rounded to
 * the nearest half (ties to even) and read back exactly, halving the cache.
 * Everything else is computed as in the fp32 context, so the logits differ
 * from the reference's only through that rounding; the benchmark reports how
 * many greedy tokens still agree. State files stay SLKV v1 with f32 values
 * (export widens exactly, import rounds).
 */
SLLM_CUDA_API int  sllm_cuda_ctx_new_kv(const sllm_cuda_model * m, int32_t n_ctx, int32_t kv_type,
                                        sllm_cuda_ctx ** out);
SLLM_CUDA_API void sllm_cuda_ctx_free(sllm_cuda_ctx * c);
SLLM_CUDA_API void sllm_cuda_ctx_reset(sllm_cuda_ctx * c);

/* Tokens consumed so far (the reference's n_past). */
SLLM_CUDA_API int32_t sllm_cuda_ctx_n_past(const sllm_cuda_ctx * c);

/*
 * Run `n` tokens at absolute positions [base, base+n) and write n * n_vocab
 * logits to `logits_out` (host, may be NULL when only `argmax_out` is wanted).
 * `argmax_out` (host, nullable) receives the argmax of each position's logits
 * (lowest index on ties, src/forward.c:876-883). Argument rules and status
 * codes follow sllm_forward_chunk (include/saphira_llm/forward.h:107-109,
 * src/forward.c:589-609): n in [1, 256], base >= n_past, base + n <= n_ctx,
 * tokens in [0, n_vocab).
 */
SLLM_CUDA_API int sllm_cuda_forward_chunk(const sllm_cuda_model * m, sllm_cuda_ctx * c,
                            const int32_t * tokens, int32_t n, int32_t base,
                            float * logits_out, int32_t * argmax_out);

/*
 * Greedy generation, replacing sllm_generate_greedy
 * (include/saphira_llm/forward.h:136-138, src/forward.c:885-938), including
 * its BOS fallback (128000) and its continuation from the last logits when
 * n_prompt == 0. The whole loop runs on the device: one token id crosses back
 * per generated token only at the end, in `out` (n_new ids).
 */
SLLM_CUDA_API int sllm_cuda_generate_greedy(const sllm_cuda_model * m, sllm_cuda_ctx * c,
                              const int32_t * prompt, int32_t n_prompt,
                              int32_t n_new, int32_t * out);

/*
 * The projection chain of layers [layer_begin, layer_begin + n_layers) without
 * attention -- the workload the benchmark measures as "one layer's seven I2_S
 * GEMVs with RMSNorm between them": attn_norm -> quant -> Q, K, V; Q stands in
 * for the attention output -> attn_sub_norm -> quant -> O -> + x; ffn_norm ->
 * quant -> gate, up -> silu(gate) * up -> ffn_sub_norm -> quant -> down ->
 * + residual. Every step is the decode layer's own (src/forward.c:631-801),
 * with the same rounding. `x_in` / `x_out` are host arrays of n_embd floats
 * (they may alias). Uses the context's scratch and stream; it does not touch
 * the KV cache or n_past.
 */
SLLM_CUDA_API int sllm_cuda_layer_chain(const sllm_cuda_model * m, sllm_cuda_ctx * c,
                          int32_t layer_begin, int32_t n_layers,
                          const float * x_in, float * x_out);

/*
 * The same chain on a device vector `x` (n_embd floats, 16-byte aligned,
 * updated in place), asynchronous on `stream`. It uses the context's scratch
 * buffers, so it must not overlap other work on the same context.
 */
SLLM_CUDA_API int sllm_cuda_layer_chain_device(const sllm_cuda_model * m, sllm_cuda_ctx * c,
                                 int32_t layer_begin, int32_t n_layers,
                                 float * x, void * stream);

/*
 * The seven projections of layers [layer_begin, layer_begin + n_layers), each
 * on its OWN input vector -- the benchmark's configuration 1 taken literally
 * ("each uses an f32 N(0,1) activation ... with RMSNorm between them"). For
 * every layer, GEMV p normalises input p with the norm its projection uses in
 * the decode layer (Q, K, V: attn_norm; O: attn_sub_norm; gate, up: ffn_norm;
 * down: ffn_sub_norm), quantises it per token and writes f32 outputs; nothing
 * feeds one projection into another, so consecutive GEMVs overlap on the
 * device.
 *   x: 6 * n_embd + n_ff floats, inputs of Q, K, V, O, gate, up (n_embd each)
 *      and down (n_ff), shared by every layer;
 *   y: n_layers blocks of 3 * n_embd + 2 * n_embd_gqa + 2 * n_ff floats:
 *      Q (n_embd), K, V (n_embd_gqa), O (n_embd), gate, up (n_ff), down (n_embd).
 * sllm_cuda_layer_projections_sizes returns the input length and stores the
 * per-layer output length. The _device form takes 16-byte aligned device
 * vectors and is asynchronous on `stream`. The host form returns when y is on
 * the host; from 16 layers up it runs them as two launches and copies the
 * first launch's outputs back on a second stream of the context while the
 * second computes (any host memory; pinned copies faster).
 */
SLLM_CUDA_API size_t sllm_cuda_layer_projections_sizes(const sllm_cuda_model * m,
                                                       size_t * y_floats_per_layer);
SLLM_CUDA_API int sllm_cuda_layer_projections(const sllm_cuda_model * m, sllm_cuda_ctx * c,
                                              int32_t layer_begin, int32_t n_layers,
                                              const float * x_host, float * y_host);
SLLM_CUDA_API int sllm_cuda_layer_projections_device(const sllm_cuda_model * m, sllm_cuda_ctx * c,
                                                     int32_t layer_begin, int32_t n_layers,
                                                     const float * x, float * y, void * stream);

/*
 * sllm_cuda_layer_chain_device without any allocation. This entry point has
 * no counterpart in the reference: it serves callers that cannot call
 * cudaMalloc -- hosts whose own allocator already holds the device's memory
 * (a late cudaMalloc fails or fragments it), loops that cannot take
 * cudaMalloc's implicit device synchronisation -- and that hold a model but
 * no context. Same results as sllm_cuda_layer_chain_device, bit for bit. It
 * calls no cudaMalloc, cudaFree or allocating library routine.
 *
 * Its scratch (2*n_embd + 2*n_embd_gqa + n_ff floats) is a fixed 128 KB
 * device array inside the library (32768 floats), held by every device that
 * loads the library until the process exits; a larger model is refused with
 * SLLM_CUDA_ERR_TOO_LARGE. The first call on a device looks up the array's
 * address (cudaGetSymbolAddress); make that first call before any stream
 * capture. Every call on a device shares the one array, so calls that can
 * overlap on the GPU (different streams, or different threads) race: order
 * them on one stream. `x` is a device vector of n_embd floats, 16-byte
 * aligned, updated in place; asynchronous on `stream`.
 */
SLLM_CUDA_API int sllm_cuda_layer_chain_device_noalloc(const sllm_cuda_model * m,
                                                       int32_t layer_begin, int32_t n_layers,
                                                       float * x, void * stream);

/*
 * The KV cache of a context in the reference's host layout: k_out / v_out are
 * n_layer * n_head_kv * n_ctx * 128 floats each, [layer][kv head][pos][dim]
 * (src/forward.c:81-83, the layout sllm_ctx_new allocates at
 * src/forward.c:480-487). Export writes the rows of positions below n_past
 * and leaves the others untouched. Import replaces the device cache with the
 * given rows below n_past, clears every row at or above it, and sets n_past
 * and the last position's logits (n_vocab floats; NULL only when n_past is
 * 0), so that a generation without a prompt continues from them, as after
 * sllm_state_load (src/forward.c:1034-1123).
 */
SLLM_CUDA_API int sllm_cuda_ctx_kv_export(const sllm_cuda_ctx * c, float * k_out, float * v_out);
SLLM_CUDA_API int sllm_cuda_ctx_kv_import(sllm_cuda_ctx * c, const float * k_in, const float * v_in,
                                          int32_t n_past, const float * last_logits);

/*
 * Save / restore a context's state in the reference's own file format, SLKV
 * version 1 (src/forward.c:963-1123): files written here load into a CPU
 * context of the same model and back, and continue identically. Replaces
 * sllm_state_save / sllm_state_load (include/saphira_llm/forward.h:155-156),
 * with the same refusals: SLLM_CUDA_ERR_KV_TYPE for a file that is not SLKV
 * v1, SLLM_CUDA_ERR_TENSOR_SHAPE for another model or context depth,
 * SLLM_CUDA_ERR_TRUNCATED for a short file, SLLM_CUDA_ERR_IO when the file
 * cannot be opened or written.
 */
SLLM_CUDA_API int sllm_cuda_state_save(const sllm_cuda_model * m, const sllm_cuda_ctx * c, const char * path);
SLLM_CUDA_API int sllm_cuda_state_load(const sllm_cuda_model * m, sllm_cuda_ctx * c, const char * path);

/* Bytes of weights one decode step streams: every I2_S tensor with its scale
 * tail, every norm, and the F16 embedding / output head. */
SLLM_CUDA_API size_t sllm_cuda_model_weight_bytes(const sllm_cuda_model * m);

/*
 * Copy the most recent position's logits (n_vocab floats) to host memory.
 * Replaces sllm_ctx_last_logits (include/saphira_llm/forward.h:77).
 * Returns SLLM_CUDA_ERR_ARG if nothing has been forwarded yet.
 */
SLLM_CUDA_API int sllm_cuda_ctx_last_logits(const sllm_cuda_ctx * c, float * host_out);

/* ------------------------------------------------------------------ */
/* tensor-parallel decode across the GPUs of one node                  */
/* ------------------------------------------------------------------ */
/*
 * The reference decodes on one host (src/forward.c:589-835); these entry
 * points shard the same forward pass over N GPUs, one process (rank) per
 * GPU: Q/K/V and gate/up split by rows (heads, FFN rows), O and down by
 * contraction columns with an int32 all-reduce of the partial dots (exact in
 * any order), the tied f16 head by vocabulary rows. Every rank calls every
 * entry point with the same arguments (SPMD); the results equal the
 * single-GPU path's, bit for bit. NCCL carries the exchanges.
 */
#define SLLM_CUDA_TP_ID_BYTES 128

typedef struct sllm_cuda_tp_comm sllm_cuda_tp_comm;
typedef struct sllm_cuda_tp_model sllm_cuda_tp_model;
typedef struct sllm_cuda_tp_ctx sllm_cuda_tp_ctx;

/* the group's identity: rank 0 creates it and hands the bytes to the others */
SLLM_CUDA_API int sllm_cuda_tp_unique_id(uint8_t * id_out);
SLLM_CUDA_API int sllm_cuda_tp_comm_init(const uint8_t * id, int32_t n_ranks, int32_t rank,
                           int32_t device, sllm_cuda_tp_comm ** out);
SLLM_CUDA_API void sllm_cuda_tp_comm_free(sllm_cuda_tp_comm * c);

/*
 * Rank `rank`'s shard of a model given as host tensors (the same description
 * as sllm_cuda_model_upload). n_head, n_head_kv, n_embd / n_ranks and
 * n_ff / n_ranks must divide evenly (multiples of 128 for the widths); head
 * dim 128, n_embd <= 8192, n_ff <= 28672.
 */
SLLM_CUDA_API int sllm_cuda_tp_model_upload(const sllm_cuda_model_desc * d, int32_t n_ranks,
                              int32_t rank, int32_t device, sllm_cuda_tp_model ** out);

/*
 * A seeded synthetic model generated on the device, shard by shard (the
 * benchmark's configs[4]: 80 layers, 8192 / 28672, 64 / 8 heads, vocab
 * 128256): ternary codes i.i.d. over {-1, 0, 1} from a counter-based hash of
 * (seed, layer, tensor, row, column), per-tensor scales in [0.01, 0.1), norm
 * weights ~N(1, 0.02), the f16 table ~N(0, 0.02). Every shard is a slice of
 * the same model for every rank count.
 */
typedef struct sllm_cuda_tp_synth_desc {
    int32_t  n_layer, n_embd, n_ff, n_head, n_head_kv, n_vocab;
    float    f_rms_eps, rope_freq_base;
    uint64_t seed;
} sllm_cuda_tp_synth_desc;

SLLM_CUDA_API int sllm_cuda_tp_model_synth(const sllm_cuda_tp_synth_desc * d, int32_t n_ranks,
                             int32_t rank, int32_t device, sllm_cuda_tp_model ** out);
SLLM_CUDA_API void sllm_cuda_tp_model_free(sllm_cuda_tp_model * m);
SLLM_CUDA_API size_t sllm_cuda_tp_model_bytes(const sllm_cuda_tp_model * m);
/* this shard's vocabulary rows [*v0, *v0 + *n) */
SLLM_CUDA_API int sllm_cuda_tp_vocab_range(const sllm_cuda_tp_model * m, int32_t * v0, int32_t * n);

/*
 * a decode context over one shard. sllm_cuda_tp_generate_greedy needs comm
 * whenever the model has more than one rank; a context without one serves a
 * single rank, or a one-process test group.
 */
SLLM_CUDA_API int sllm_cuda_tp_ctx_new(const sllm_cuda_tp_model * m, sllm_cuda_tp_comm * comm,
                         int32_t n_ctx, sllm_cuda_tp_ctx ** out);
SLLM_CUDA_API void sllm_cuda_tp_ctx_free(sllm_cuda_tp_ctx * c);
SLLM_CUDA_API int sllm_cuda_tp_ctx_reset(sllm_cuda_tp_ctx * c);

/*
 * sllm_generate_greedy (src/forward.c:885-938) over the shards: argument
 * rules, BOS fallback and outputs as sllm_cuda_generate_greedy. A step whose
 * exchanges make no progress for 120 s aborts the communicator and returns
 * SLLM_CUDA_ERR_TIMEOUT. The exchanges are NCCL collectives, or, with the
 * environment variable SLLM_CUDA_TP_EXCHANGE=p2p at context creation, one-shot
 * kernels that store into the peers' memory over NVLink (CUDA IPC) and wait
 * on epoch flags (bounded).
 */
SLLM_CUDA_API int sllm_cuda_tp_generate_greedy(sllm_cuda_tp_ctx * c, const int32_t * prompt,
                                 int32_t n_prompt, int32_t n_new, int32_t * out);
/* the last step's logits of this shard's vocabulary rows */
SLLM_CUDA_API int sllm_cuda_tp_last_logits(const sllm_cuda_tp_ctx * c, float * host_out);

/*
 * Batch decode over one shard: n_seq <= 16 sequences, each with its own KV
 * cache of n_ctx positions, stepped together. The reference serves a batch
 * as one context per sequence (src/forward.c:78-84, :466-562); here each
 * layer GEMV of a step is one GEMM over the n_seq tokens on the tensor cores
 * (every weight byte read once per step), and each sequence's tokens and
 * logits equal, bit for bit, those of sllm_cuda_tp_generate_greedy on its own
 * context. E <= 8192 and F <= 32768 (a multiple of 32). Needs comm as a
 * context does.
 */
typedef struct sllm_cuda_tp_batch sllm_cuda_tp_batch;
SLLM_CUDA_API int sllm_cuda_tp_batch_new(const sllm_cuda_tp_model * m, sllm_cuda_tp_comm * comm,
                                         int32_t n_seq, int32_t n_ctx, sllm_cuda_tp_batch ** out);
SLLM_CUDA_API void sllm_cuda_tp_batch_free(sllm_cuda_tp_batch * b);
SLLM_CUDA_API int sllm_cuda_tp_batch_reset(sllm_cuda_tp_batch * b);
/*
 * sllm_generate_greedy (src/forward.c:885-938) for every sequence at once:
 * prompts is row-major [n_seq][n_prompt] (the same length for every
 * sequence; n_prompt may be 0 only to continue after an earlier call), out
 * receives row-major [n_seq][n_new]. Failures as sllm_cuda_tp_generate_greedy.
 */
SLLM_CUDA_API int sllm_cuda_tp_batch_generate_greedy(sllm_cuda_tp_batch * b, const int32_t * prompts,
                                                     int32_t n_prompt, int32_t n_new, int32_t * out);
/* sequence seq's last-step logits of this shard's vocabulary rows */
SLLM_CUDA_API int sllm_cuda_tp_batch_last_logits(const sllm_cuda_tp_batch * b, int32_t seq, float * host_out);

#ifdef __cplusplus
}
#endif

#endif /* SLLM_CUDA_H */
