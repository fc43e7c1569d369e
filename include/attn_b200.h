/*
 * attn_b200.h -- C ABI of the B200 causal-attention engine (libattn_b200.so).
 *
 * Drop-in boundary for pure-c-llm's attention:
 *   - attn_fwd / attn_bwd keep the exact signatures, pointer meaning and
 *     error behaviour of gpu_kernels.h:67-72 (device pointers, shapes from
 *     compile-time-style defaults, void return, exit(1) on a CUDA error like
 *     CUDA_CHECK at gpu_kernels.h:34-36), so train_kaggle.cu:155/199 link
 *     unchanged.
 *   - attn_cached_attention replaces the static cached_attention of
 *     transformer.c:203-248 (one query token against cache rows 0..pos).
 *   - the *_ex entry points take explicit shapes, a stream and a workspace
 *     and return a status instead of exiting.
 *
 * Everything here is plain C: pointers, sizes, ints.  All tensor pointers are
 * DEVICE pointers unless a comment says otherwise.  A stream argument of NULL
 * means the legacy default stream, as the reference uses.
 *
 * Layout (transformer.h:15-18): an activation is a row-major matrix with one
 * row per token; head h of a token occupies columns [h*d, (h+1)*d).  Rows are
 * `row_stride` elements apart (heads*head_dim for a dense tensor, D_MODEL in
 * the reference).  Token t of batch b is row b*T + t.
 */
#ifndef ATTN_B200_H
#define ATTN_B200_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define ATTN_API __attribute__((visibility("default")))
#else
#define ATTN_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

typedef struct CUstream_st *attn_stream_t;   /* a cudaStream_t */

/* status codes returned by every int-returning entry point */
enum {
    ATTN_OK = 0,
    ATTN_ERR_INVALID = 1,      /* bad pointer, shape, stride or alignment      */
    ATTN_ERR_UNSUPPORTED = 2,  /* valid request this build has no kernel for   */
    ATTN_ERR_CUDA = 3,         /* a CUDA runtime/driver call failed            */
    ATTN_ERR_NOMEM = 4,        /* device allocation failed                     */
    ATTN_ERR_WORKSPACE = 5,    /* caller workspace smaller than required       */
    ATTN_ERR_DEVICE = 6,       /* a kernel reported an internal error (bounded
                                  wait expired); see attn_device_error()       */
    ATTN_ERR_COMM = 7          /* a collective failed or a group wait timed
                                  out; the group has been torn down           */
};

/* element types of activations / caches */
enum {
    ATTN_F32 = 0,    /* float32 storage, float32 arithmetic (the reference's)  */
    ATTN_BF16 = 1,   /* bf16 storage, bf16 tensor-core products, fp32 accumulate */
    ATTN_I8 = 2      /* int8 KV cache codes + per-(token, head) fp32 scale      */
};

/* ------------------------------------------------------------------------
 * Errors
 * ---------------------------------------------------------------------- */
/* Text of the last failure on the calling host thread ("" if none). */
ATTN_API const char *attn_last_error(void);
/* Reads and clears the device-side error word of `device` (0 = none).  Bounded
 * waits inside kernels record a code here instead of hanging. */
ATTN_API int attn_device_error(int device, int *code_out);
/* Library version, (major << 16) | minor. */
ATTN_API int attn_version(void);

/* ------------------------------------------------------------------------
 * Training attention, drop-in (gpu_kernels.h:66-72)
 * ---------------------------------------------------------------------- */
/* A C++ translation unit that also includes the reference's gpu_kernels.h
 * (which declares attn_fwd / attn_bwd with C++ linkage) defines
 * ATTN_OMIT_MACRO_DROPINS before including this header, so the two
 * declarations do not conflict; the library exports both linkages. */
#ifndef ATTN_OMIT_MACRO_DROPINS
/* Replaces gpu_kernels.h:67 attn_fwd.  Q,K,V,att: (B*T, H*d) fp32 device.
 * `probs` is the caller's buffer (B*H*T*T floats in train_kaggle.cu:123,128).
 * In the default mode (ATTN_PROBS_LSE_OUT) this library stores the per-row
 * log-sum-exp and a copy of the output there, which attn_bwd reads back:
 * probs needs B*H*T*(1+d) floats, and T >= d+1.  In ATTN_PROBS_LSE mode it
 * stores only the log-sum-exp (B*H*T floats, any T) and attn_bwd reads the
 * output from `att` itself (see attn_set_probs_mode).  Sets att.  Exits(1)
 * with a message on failure. */
ATTN_API void attn_fwd(const float *Q, const float *K, const float *V, float *att, float *probs);

/* Replaces gpu_kernels.h:70 attn_bwd.  SETS dQ, dK, dV (like the reference's
 * cuBLAS path, beta = 0).  `scratch` is the caller's workspace (B*H*T*T
 * floats in train_kaggle.cu:138).  At head_dim 96 and 128 with T a multiple
 * of 4 the backward runs as tensor-core GEMMs over explicit score tiles: in
 * the default ATTN_PROBS_LSE_OUT mode this library fills all of `scratch`
 * with dS (as the reference's own softmax backward does) and keeps the
 * scores, P^T, dS^T, the row statistics and split operands in a library-owned
 * device buffer (2*B*H*T*(T+5d+1) floats, 654 MB at the trainer's shape); in
 * ATTN_PROBS_LSE mode dS goes to that buffer as well (B*H*T*T floats more,
 * one buffer for every layer).  Calls that use the buffer must not overlap on
 * the GPU.  Otherwise, or when the buffer cannot be allocated, it runs the
 * CUDA-core kernels and uses 2*B*H*T floats of `scratch`.  Exits(1) with a
 * message on failure. */
ATTN_API void attn_bwd(float *dQ, float *dK, float *dV, float *scratch,
              const float *dAtt, const float *Q, const float *K, const float *V,
              const float *probs);
#endif

/* Shape used by attn_fwd/attn_bwd.  Defaults are gpu_kernels.h:17-31:
 * B_SIZE 4, N_HEADS 12, T_SIZE 1024, D_HEAD 128 (DIM 1536); a build may
 * override them with -DATTN_B_SIZE= etc.  Returns ATTN_OK or an error
 * (ATTN_ERR_UNSUPPORTED for T < d+1 in ATTN_PROBS_LSE_OUT mode). */
ATTN_API int attn_set_macro_shape(int batch, int heads, int seq_len, int head_dim);

/* What attn_fwd keeps in `probs` for attn_bwd.
 *   ATTN_PROBS_LSE_OUT (default): log-sum-exp and a copy of the output,
 *     B*H*T*(1+d) floats; attn_bwd needs nothing else.
 *   ATTN_PROBS_LSE: log-sum-exp only, B*H*T floats -- the trainer's a_probs
 *     shrinks from B*H*T*T floats per layer (2.4 GB at the 343M shape) to
 *     B*H*T, and T is no longer bounded by that allocation.  attn_fwd records
 *     which `att` buffer it wrote for each `probs` buffer; attn_bwd reads the
 *     output from that `att`, which the caller must leave unchanged between
 *     the two calls (train_kaggle.cu keeps a_att[l] for the Wo gradient).
 *     attn_bwd with a `probs` that no attn_fwd of this process has filled is
 *     an error (exit(1), like any drop-in failure).
 * Returns ATTN_OK, or ATTN_ERR_INVALID for another value. */
enum { ATTN_PROBS_LSE_OUT = 0, ATTN_PROBS_LSE = 1 };
ATTN_API int attn_set_probs_mode(int mode);

/* ------------------------------------------------------------------------
 * Training attention, explicit shapes
 * ---------------------------------------------------------------------- */
typedef struct {
    int batch;                  /* B                                          */
    int heads;                  /* H (heads handled by this call)             */
    int seq_len;                /* T                                          */
    int head_dim;               /* d: 32, 64, 96 or 128                       */
    long long in_row_stride;    /* elements between rows of Q,K,V,dO (0: H*d) */
    long long out_row_stride;   /* elements between rows of O,dQ,dK,dV (0: H*d) */
} attn_shape;

/* Causal forward O = softmax(Q K^T / sqrt(d)) V per (b, h), rows j <= i.
 * dtype ATTN_F32: fp32 in/out, fp32 arithmetic (train.c:339-370 semantics).
 * dtype ATTN_BF16: bf16 in/out, tensor-core products, fp32 softmax.  At head
 * dims 32, 96 and 128 a bf16 call keeps fp32 copies of its tensors (4*B*T*H*d
 * floats) in a library-owned device buffer, grown on demand; such calls must
 * not overlap on the GPU.
 * lse (may be NULL): B*H*T floats, [b][h][t] = max + log(sum) of the scaled
 * scores of row t -- the statistic the backward recomputes P from. */
ATTN_API int attn_fwd_ex(const attn_shape *s, int dtype,
                const void *Q, const void *K, const void *V, void *O,
                float *lse, attn_stream_t stream);

/* Bytes of device workspace attn_bwd_ex needs for this shape. */
ATTN_API size_t attn_bwd_workspace_bytes(const attn_shape *s, int dtype);

/* Bytes of workspace that let attn_bwd_ex run an fp32 backward at head_dim 96
 * or 128 (T a multiple of 4, accumulate = 0) on the tensor cores, as GEMMs
 * over explicit score tiles: 2*B*H*T*(T+5d+1) + B*H*T*T floats (the scores,
 * P^T, dS^T, dS, split operands and row statistics; 855 MB at B4 H12 T1024
 * d128), rounded to 256-byte pieces.  0 for shapes without that path.  A
 * smaller workspace (at least attn_bwd_workspace_bytes) selects the CUDA-core
 * kernels. */
ATTN_API size_t attn_bwd_tc_workspace_bytes(const attn_shape *s);

/* Analytic backward (train.c:373-407): dQ, dK, dV from dO, the forward's
 * inputs, its output O and its lse.  accumulate = 1 adds into dQ/dK/dV as
 * train.c does; 0 overwrites them as gpu_kernels.cu's attn_bwd does. */
ATTN_API int attn_bwd_ex(const attn_shape *s, int dtype,
                const void *dO, const void *Q, const void *K, const void *V,
                const void *O, const float *lse,
                void *dQ, void *dK, void *dV, int accumulate,
                void *workspace, size_t workspace_bytes, attn_stream_t stream);

/* ------------------------------------------------------------------------
 * Fused QKV projection (train_kaggle.cu:152-154)
 * ---------------------------------------------------------------------- */
typedef struct {
    int rows;                   /* M: token rows of X (B*T)                    */
    int in_features;            /* columns of X = rows of each W (DIM)         */
    int out_features;           /* N: columns of each W and of each output;
                                   a multiple of 4                              */
    long long x_row_stride;     /* elements between rows of X (0: in_features) */
    long long out_row_stride;   /* elements between rows of Q, K, V
                                   (0: out_features; 3*N for the three column
                                   blocks of one (M, 3N) tensor)                */
} attn_qkv_shape;

/* Bytes of device workspace attn_qkv_proj_ex uses for this shape: the three
 * weights transposed and split, 2 * 3 * out_features * in_features floats
 * (in_features rounded up to 4). */
ATTN_API size_t attn_qkv_workspace_bytes(const attn_qkv_shape *s);

/* Q = X Wq + bq, K = X Wk + bk, V = X Wv + bv: the three gemm_nn calls of
 * train_kaggle.cu:152-154 (gemm_nn: gpu_kernels.cu:112-120, row-major fp32,
 * bias broadcast over rows) in one tensor-core launch, after one small launch
 * that splits the weights.  X (rows, in_features), each W (in_features,
 * out_features) row-major, fp32; biases may be NULL.  fp32 arithmetic (three
 * tf32 products per product, fp32 sums; results within ~1e-6 of an fp32
 * GEMM).  Outputs are SET.  Tensors 16-byte aligned.  `workspace` (256-byte
 * aligned, attn_qkv_workspace_bytes) may be NULL: the library then uses its
 * own per-device buffer, grown on demand, and calls that use it must not
 * overlap on the GPU.  Returns ATTN_OK or a status. */
ATTN_API int attn_qkv_proj_ex(const attn_qkv_shape *s, const float *x,
                const float *wq, const float *wk, const float *wv,
                const float *bq, const float *bk, const float *bv,
                float *q, float *k, float *v,
                void *workspace, size_t workspace_bytes, attn_stream_t stream);

/* The same with gemm_nn's argument style (A, B, bias, C, M, K, N): dense
 * (M, K) input, (K, N) weights, (M, N) outputs, the legacy default stream,
 * void return and exit(1) with a message on failure, like the drop-ins.
 * Replaces train_kaggle.cu:152-154's three calls with one. */
ATTN_API void attn_qkv_proj(const float *X, const float *Wq, const float *Wk, const float *Wv,
                const float *bq, const float *bk, const float *bv,
                float *Q, float *K, float *V, int M, int K_, int N);

/* ------------------------------------------------------------------------
 * KV-cached decode (transformer.c:203-248, model.h:42-45)
 * ---------------------------------------------------------------------- */
typedef struct {
    int n_seq;                  /* independent sequences (or layers) per call */
    int heads;                  /* H                                          */
    int head_dim;               /* d: 32, 64, 96 or 128                       */
    int kv_dtype;               /* ATTN_F32 or ATTN_I8                        */
    long long row_stride;       /* elements between cache rows (0: H*d)      */
    long long cap;              /* rows allocated per sequence's cache        */
    int max_len;                /* upper bound of lens[] (<= cap)             */
} attn_decode_shape;

/* Bytes of device workspace attn_decode_ex / attn_decode_ptrs_ex need. */
ATTN_API size_t attn_decode_workspace_bytes(const attn_decode_shape *s);

/* Decode one query token per sequence against that sequence's cache rows
 * 0..lens[s]-1 (lens[s] = pos+1 in transformer.c terms; lens is a DEVICE
 * int array, each in [1, max_len]; NULL means every sequence attends max_len
 * rows).
 *   q, out: n_seq x (H*d) fp32, dense.
 *   kcache/vcache: sequence s row r at base + (s*cap + r)*row_stride, fp32
 *     (ATTN_F32) or int8 codes (ATTN_I8).
 *   kscale/vscale: ATTN_I8 only, fp32 [(s*cap + r)*H + h] (NULL for fp32).
 * workspace may be NULL: the library then uses a buffer of its own per
 * device (allocated on first use); calls that use that buffer must not
 * overlap on the GPU (order them on one stream, or give each stream its own
 * workspace). */
ATTN_API int attn_decode_ex(const attn_decode_shape *s, const float *q,
                   const void *kcache, const void *vcache,
                   const float *kscale, const float *vscale,
                   const int *lens, float *out,
                   void *workspace, size_t workspace_bytes, attn_stream_t stream);

/* Same, with one cache slab per sequence: kptrs/vptrs (and kscales/vscales
 * for ATTN_I8) are DEVICE arrays of n_seq device pointers, each slab laid out
 * as cap rows of row_stride elements -- the per-layer KVCache.k[l] slabs of
 * model.h:42-45. */
ATTN_API int attn_decode_ptrs_ex(const attn_decode_shape *s, const float *q,
                        const void *const *kptrs, const void *const *vptrs,
                        const float *const *kscales, const float *const *vscales,
                        const int *lens, float *out,
                        void *workspace, size_t workspace_bytes, attn_stream_t stream);

/* No counterpart in the reference.  Same as attn_decode_ex, but it allocates
 * nothing and takes no workspace: the scratch is a fixed array of
 * ATTN_DECODE_STATIC_SCRATCH_BYTES inside the library's device image, reserved
 * on every GPU that loads the library until the process exits.  It is for
 * callers that cannot allocate device memory (memory owned by another
 * allocator, or a loop that must not let cudaMalloc synchronise the device).
 * Shapes whose scratch need (attn_decode_workspace_bytes) exceeds the array
 * are rejected with ATTN_ERR_WORKSPACE.  The first call on a device looks up
 * the array's device address (cudaGetSymbolAddress); make that first call
 * before any stream capture.  All calls share the array: calls whose kernels
 * overlap on the GPU race. */
#define ATTN_DECODE_STATIC_SCRATCH_BYTES (4u << 20)
ATTN_API int attn_decode_static_ex(const attn_decode_shape *s, const float *q,
                                   const void *kcache, const void *vcache,
                                   const float *kscale, const float *vscale,
                                   const int *lens, float *out, attn_stream_t stream);

/* cached_attention (transformer.c:203) with device pointers: one token of one
 * layer, attends rows 0..pos.  Writes out (H*d).  Uses the library's own
 * workspace, so calls must not overlap on the GPU with other calls that use
 * it.  Returns a status. */
ATTN_API int attn_cached_attention(const float *q, const float *kcache, const float *vcache,
                          float *out, int pos, int heads, int head_dim,
                          long long row_stride, attn_stream_t stream);

/* cached_attention (transformer.c:203-248) with its own argument list and
 * HOST pointers: a drop-in for the call at transformer.c:266 (forward_block).
 * q, out: H*d floats; kcache/vcache: the caller's host cache, T_MAX rows of
 * H*d floats (transformer.h:35-38 shapes, or attn_set_decode_macro_shape);
 * `scores` is accepted and unused.  The library keeps a device mirror of each
 * (kcache, vcache) pair and copies over only the rows it has not seen -- the
 * generator writes row `pos` before attending (transformer.c:256-264) -- then
 * decodes on the GPU and writes `out` before returning.  A call with a pos
 * below the mirrored length re-sends rows from pos on; rows below pos must not
 * change once sent.  Exits(1) with a message on failure. */
ATTN_API void attn_cached_attention_host(const float *q, const float *kcache, const float *vcache,
                                         float *out, float *scores, int pos);
/* Shapes of attn_cached_attention_host (defaults: transformer.h:35-38,
 * N_HEADS 16, D_HEAD 96, T_MAX 512; rows of heads*head_dim floats). */
ATTN_API int attn_set_decode_macro_shape(int heads, int head_dim, int t_max);
/* The same with explicit shapes and a status (generate.c:130-152 works with
 * run-time dims: H, DH, row stride D, BLK rows). */
ATTN_API int attn_cached_attention_host_ex(const float *q, const float *kcache, const float *vcache,
                                           float *out, int pos, int heads, int head_dim,
                                           long long row_stride, int cap);
/* Frees the device mirror of a host cache pair. */
ATTN_API int attn_host_cache_release(const float *kcache, const float *vcache);

/* INT8 quantiser for caches: the reference's symmetric absmax scheme
 * (gemm_bench.c:225-236: amax floored at 1e-8, scale = amax/127,
 * q = lroundf(x/scale) clamped to +-127) applied per (row, head).
 * x: rows x row_stride fp32; codes: same layout int8; scales: rows x heads. */
ATTN_API int attn_kv_quantize_int8(const float *x, long long rows, int heads, int head_dim,
                          long long row_stride, int8_t *codes, float *scales,
                          attn_stream_t stream);

/* ------------------------------------------------------------------------
 * Device KV cache (model.h:42-48, alloc_kv_cache at model.c:27-33 mallocs
 * host slabs; this one owns device slabs)
 * ---------------------------------------------------------------------- */
#define ATTN_MAX_LAYERS 64
typedef struct {
    int n_layers, cap, heads, head_dim, kv_dtype;
    void *k[ATTN_MAX_LAYERS];        /* cap x (heads*head_dim) per layer      */
    void *v[ATTN_MAX_LAYERS];
    float *kscale[ATTN_MAX_LAYERS];  /* cap x heads per layer (ATTN_I8 only)  */
    float *vscale[ATTN_MAX_LAYERS];
} attn_kv_cache;

ATTN_API int attn_kv_cache_alloc(attn_kv_cache *c, int n_layers, int cap, int heads,
                        int head_dim, int kv_dtype);
ATTN_API int attn_kv_cache_free(attn_kv_cache *c);
/* Writes one token's K and V rows (fp32, H*d each, device) at row `pos` of
 * `layer`, quantising on append for an ATTN_I8 cache -- the row write of
 * transformer.c:260-264. */
ATTN_API int attn_kv_cache_append(attn_kv_cache *c, int layer, int pos,
                         const float *krow, const float *vrow, attn_stream_t stream);

/* ------------------------------------------------------------------------
 * Serving over a paged cache (no counterpart in the reference, whose caches
 * are one slab per sequence): a step is attn_page_plan_ex (which cache row
 * each new token takes), attn_rope_append_ex (positions turned into Q and K,
 * K and V written to those rows) and attn_prefix_decode_ex (one query token
 * per request over the rows its group shares and its own).
 * All run on the caller's stream; none allocates, and all may be captured in a
 * graph, except attn_prefix_decode_ex without a workspace of the caller's.
 * ---------------------------------------------------------------------- */
/* A cache of `rows` token rows.  Page p of a P-token page size is rows
 * [p*P, (p+1)*P); row r of head h starts at element r*row_stride + h*d, as in
 * the other caches.  ATTN_I8 rows hold codes, with one fp32 scale per
 * (row, head) at [r*kv_heads + h]. */
typedef struct {
    int kv_dtype;               /* ATTN_F32, ATTN_BF16 or ATTN_I8              */
    long long rows;             /* token rows of k and v                       */
    long long row_stride;       /* elements between rows (0: kv_heads*head_dim) */
    void *k, *v;                /* 16-byte aligned                             */
    float *kscale, *vscale;     /* ATTN_I8 only                                */
} attn_paged_kv;

typedef struct {
    int n_seq;                  /* requests of the step, <= 16384              */
    int page_size;              /* tokens per page: a power of two, <= 1024    */
    int max_pages;              /* block_table columns                         */
    int max_tokens;             /* rows of slot_map, positions and token_seq   */
    int n_pages;                /* entries of free_pages: all pages there are
                                   (what comes back past them is lost)         */
    int table_stride;           /* ints between block_table rows (0: max_pages) */
} attn_page_shape;

/* Plans one step from the requests' lengths, on the GPU.  Request s holds
 * lens[s] tokens in pages block_table[s][0 .. ceil(lens[s]/page_size)) and
 * receives new_lens[s] more, or ends when new_lens[s] < 0: its pages go back
 * and its length becomes 0.
 *   Pages are taken from the end of one list: free_pages[0 .. *free_count),
 * then the pages of the ended requests in request and page order.  Request
 * after request takes what its tokens need beyond its last page.  A request is
 * refused, and nothing of it changes, when the list runs out at it or was run
 * out by one before it, when its length would pass max_pages*page_size, or
 * when its tokens would pass row max_tokens; one that needs no page is served
 * whatever the list holds.
 *   Written: block_table (the new entries only), free_pages (entries at and
 * past *free_count only), and
 *   lens_out[n_seq]: the lengths after the step;
 *   cu_new[n_seq+1]: request s's new tokens are rows [cu_new[s], cu_new[s+1]),
 *     refused ones included (2^31-1 where the sum passes that);
 *   slot_map[max_tokens]: the cache row of each token row, -1 for tokens of
 *     refused requests and for rows past the last token;
 *   positions[max_tokens]: pos_base[s] (0 where NULL; the length of a shared
 *     prefix, say) + the token's index in the request, 0 past the last token;
 *   token_seq[max_tokens] (may be NULL): its request, -1 past the last token;
 *   counts[4]: the free pages after the step, the tokens, the requests
 *     refused, the pages taken.
 * lens_out and counts must not overlap lens and free_count: a step's outputs
 * are the next step's inputs.  One launch, no workspace, the same result on
 * every run. */
ATTN_API int attn_page_plan_ex(const attn_page_shape *s, const int *lens, const int *new_lens,
                const int *pos_base, int *free_pages, const int *free_count, int *block_table,
                int *lens_out, int *cu_new, long long *slot_map, int *positions,
                int *token_seq, int *counts, attn_stream_t stream);

/* Frequencies of a rotary table for contexts past the trained one.  Pair i of
 * rot_dim/2 has frequency f_i = base^(-2i/rot_dim), and position p turns it by
 * p * f_i.
 *   ATTN_ROPE_PLAIN   f_i as they are
 *   ATTN_ROPE_LINEAR  f_i / factor (positions interpolated)
 *   ATTN_ROPE_BASE    base stretched to base * factor^(rot_dim/(rot_dim-2)),
 *                     so the slowest pair slows by factor and the fastest
 *                     stays (rot_dim > 2)
 *   ATTN_ROPE_RAMP    by wavelength: a pair that turns more than `fast` times
 *                     within trained_len tokens keeps f_i, one that turns less
 *                     than `slow` times takes f_i / factor, and between them
 *                     the two are mixed linearly in the pair's index, between
 *                     the indices (no whole numbers) where a pair turns just
 *                     `fast` and just `slow` times.  A checkpoint trained with
 *                     another mixture (bounds rounded to whole pairs, or linear
 *                     in the number of turns) brings its own table:
 *                     attn_rope_ex takes any
 * Every table entry is multiplied by `magnitude` (0: 1). */
enum { ATTN_ROPE_PLAIN = 0, ATTN_ROPE_LINEAR = 1, ATTN_ROPE_BASE = 2, ATTN_ROPE_RAMP = 3 };
typedef struct {
    int rot_dim;                /* even, 2 .. 128                              */
    int max_pos;                /* rows of the table                           */
    int scaling;                /* ATTN_ROPE_PLAIN ...                         */
    int trained_len;            /* ATTN_ROPE_RAMP: tokens of the trained context */
    double base;                /* 10000, say                                  */
    double factor;              /* >= 1 (unused for ATTN_ROPE_PLAIN)           */
    double fast, slow;          /* ATTN_ROPE_RAMP: turns, fast > slow > 0      */
    double magnitude;
} attn_rope_config;
/* table[max_pos][rot_dim/2][2] = cos, sin (fp32, angles in fp64). */
ATTN_API int attn_rope_table_ex(const attn_rope_config *c, float *table, attn_stream_t stream);

typedef struct {
    int tokens;
    int seq_len;                /* position of row t when positions is NULL:
                                   t % seq_len                                 */
    int heads, kv_heads, head_dim;   /* head_dim 32, 64, 96 or 128             */
    int rot_dim;                /* leading elements of each head that turn:
                                   even, 0 .. head_dim; the others are copied  */
    int interleaved;            /* pairs (2i, 2i+1); 0: (i, i + rot_dim/2)     */
    int max_pos;                /* rows of the table                           */
    long long q_row_stride, k_row_stride, v_row_stride;  /* elements (0: dense) */
    long long q_out_row_stride, k_out_row_stride;
} attn_rope_shape;

/* q_out, k_out = q, k with each pair (a, b) of a head turned by its token's
 * table row: (a cos - b sin, b cos + a sin), in fp32 from `dtype` (ATTN_F32 or
 * ATTN_BF16), rounded once.  transpose = 1 turns back ((a cos + b sin,
 * b cos - a sin)): the gradient of q and k from that of q_out and k_out.
 * positions: DEVICE ints, one per token, or NULL.  q may be q_out and k may be
 * k_out; otherwise they must not overlap.  k and k_out may both be NULL.
 * A position outside the table records 0x701 in the device error word and the
 * nearest row of the table is used. */
ATTN_API int attn_rope_ex(const attn_rope_shape *s, int dtype, const float *table,
                const int *positions, const void *q, const void *k, void *q_out, void *k_out,
                int transpose, attn_stream_t stream);

/* The serving form: q turned into q_out; k turned and v as it is written to
 * cache row slot_map[t] (a DEVICE array; a token whose slot is outside the
 * cache, -1 say, writes nothing there, and its position, which may be past the
 * table where attn_page_plan_ex refused the token, is not reported).  dtype ATTN_F32 into an ATTN_F32 or
 * ATTN_I8 cache (quantised per (token, head) as attn_kv_quantize_int8 does: a
 * NaN among a head's elements becomes a code like any other, -127),
 * ATTN_BF16 into an ATTN_BF16 cache.  Slots of a call must differ from one
 * another. */
ATTN_API int attn_rope_append_ex(const attn_rope_shape *s, const attn_paged_kv *cache, int dtype,
                const float *table, const int *positions, const long long *slot_map,
                const void *q, const void *k, const void *v, void *q_out, attn_stream_t stream);

/* Root-mean-square norm of each head of Q and K, as models with normed queries
 * and keys have it before the rotation: x becomes x * w / sqrt(mean(x^2) + eps)
 * over the head_dim elements of a head.  (Weights kept as an offset from 1 are
 * passed with the 1 added.) */
typedef struct {
    const float *q_weight, *k_weight;   /* DEVICE, head_dim floats each, shared
                                           by the heads (NULL: ones)           */
    float eps;                          /* >= 0                                */
} attn_head_norm;

/* attn_rope_ex of the normed heads, in one pass: q_out, k_out = the heads of q,
 * k normed, weighted and turned, fp32 arithmetic, rounded once.  rot_dim 0
 * norms alone.  q may be q_out and k may be k_out; k and k_out may be NULL. */
ATTN_API int attn_norm_rope_ex(const attn_rope_shape *s, const attn_head_norm *n, int dtype, const float *table,
                const int *positions, const void *q, const void *k, void *q_out, void *k_out,
                attn_stream_t stream);

/* Its gradients, from the forward's inputs q, k and the gradients dq_out,
 * dk_out of its outputs: dq, dk (SET; their rows lie as those of q and k, the
 * others as those of q_out and k_out) and, where wanted, the weights' gradients
 * dq_weight, dk_weight (head_dim floats, summed over tokens and heads; NULL:
 * not wanted; accumulate = 1 adds to them, 0 sets them; they must not overlap,
 * where one weight serves both as well).  dq may be dq_out or q
 * where the row strides of the two are the same, dk likewise; k, dk_out and dk
 * may all be NULL (a dk_weight is then as over no tokens).  The same result on
 * every run.  `workspace` (256-byte aligned) is needed when a weight's gradient
 * is wanted, and only then. */
ATTN_API size_t attn_norm_rope_bwd_workspace_bytes(const attn_rope_shape *s);
ATTN_API int attn_norm_rope_bwd_ex(const attn_rope_shape *s, const attn_head_norm *n, int dtype, const float *table,
                const int *positions, const void *q, const void *k, const void *dq_out, const void *dk_out,
                void *dq, void *dk, float *dq_weight, float *dk_weight, int accumulate,
                void *workspace, size_t workspace_bytes, attn_stream_t stream);

/* attn_rope_append_ex of the normed heads: q normed and turned into q_out, k
 * normed and turned and v as it is written to the cache. */
ATTN_API int attn_norm_rope_append_ex(const attn_rope_shape *s, const attn_head_norm *n, const attn_paged_kv *cache,
                int dtype, const float *table, const int *positions, const long long *slot_map,
                const void *q, const void *k, const void *v, void *q_out, attn_stream_t stream);

typedef struct {
    int n_seq;                  /* requests, one query token each, <= 65535    */
    int n_groups;               /* groups that share a prefix (0: none)        */
    int heads, kv_heads;        /* heads a multiple of kv_heads; query head h
                                   reads key head h / (heads / kv_heads)       */
    int head_dim;               /* 32, 64, 96 or 128                           */
    int dtype;                  /* of q and out: ATTN_BF16 with an ATTN_BF16
                                   cache, else ATTN_F32                        */
    int page_size;              /* a power of two, <= 1024                     */
    int max_prefix_pages;       /* prefix_table columns                        */
    int max_pages;              /* block_table columns                         */
    int max_prefix_len;         /* upper bounds of prefix_lens and lens        */
    int max_len;
    long long q_row_stride, out_row_stride;   /* elements (0: heads*head_dim)  */
    float scale;                /* of the scores (0: 1/sqrt(head_dim))         */
} attn_prefix_shape;

/* Bytes of device workspace attn_prefix_decode_ex needs. */
ATTN_API size_t attn_prefix_decode_workspace_bytes(const attn_prefix_shape *s, const attn_paged_kv *cache);

/* Decodes one query token per request over the rows of its group's prefix and
 * its own rows, as one softmax: out = sum_j softmax_j(scale q.k_j) v_j.  A
 * prefix is read once for each block of its group's query rows (requests x
 * heads/kv_heads), not for each request; a block has up to 4 to 256 rows, more
 * where the groups have more on average.
 *   group_begin[n_groups+1] (DEVICE, ascending): group g is requests
 *     [group_begin[g], group_begin[g+1]); a request of no group has no prefix.
 *   prefix_table[n_groups][max_prefix_pages], prefix_lens[n_groups],
 *   block_table[n_seq][max_pages], lens[n_seq]: DEVICE ints; entries past a
 *     length's pages are not read, nor are cache rows past a length.
 *   lse (may be NULL): n_seq x heads floats, the natural log of the sum of
 *     exponentials.
 * A request with no row at all gets out = 0 and lse = -inf.  A length outside
 * [0, max] is clamped and records 0x703 in the device error word; a page
 * outside the cache records 0x702 and its rows count as absent.  fp32 and INT8
 * caches: fp32 arithmetic or products of exact parts with fp32 or integer sums;
 * bf16: bf16 products, probabilities in two bf16 parts, fp32 sums and statistics.
 * A NaN in a query or a row that is read gives NaN in the outputs it reaches (in
 * an ATTN_I8 cache a NaN can be in a scale only).
 * workspace (256-byte aligned) may be NULL: the library's own per-device
 * buffer, grown on demand; calls that use it must not overlap on the GPU, and
 * while the stream is captured it is refused (ATTN_ERR_WORKSPACE), because a
 * graph would outlive the buffer. */
ATTN_API int attn_prefix_decode_ex(const attn_prefix_shape *s, const attn_paged_kv *cache,
                const void *q, const int *group_begin, const int *prefix_table,
                const int *prefix_lens, const int *block_table, const int *lens, void *out,
                float *lse, void *workspace, size_t workspace_bytes, attn_stream_t stream);

/* ------------------------------------------------------------------------
 * Drafted token trees over a paged cache (speculative decoding): a step checks
 * several drafted tokens of a request at once, of which one path is kept.
 * Draft 0 of a request is its last sampled token (or any first row), and each
 * other one descends from an earlier one, so a path's indexes ascend.  A step:
 *   attn_page_plan_ex       new_lens = the drafts: their cache rows
 *   attn_tree_plan_ex       positions by depth, and who sees whom
 *   per layer: project, attn_rope_append_ex or attn_norm_rope_append_ex,
 *   attn_tree_decode_ex     every draft over prefix, context and its ancestors
 *   (the caller compares the model's answers with the drafts)
 *   attn_tree_commit_ex     the accepted path's rows moved together, all layers;
 *                           its lens_out and counts are the next step's lens
 *                           and free_count
 * None allocates; all may be captured in a graph.
 * ---------------------------------------------------------------------- */
/* cu_rows[n_seq+1]: request s's drafts are token rows [cu_rows[s], cu_rows[s+1])
 * (the page plan's cu_new; ends are clamped to n_rows, the rows of the other
 * arrays).  parents[r]: the parent's index within the request, less than the
 * draft's own, or -1.  positions[r], as the page plan leaves them: that of each
 * request's first row is read.  Written, for the requests' rows alone:
 *   positions_out[r] (may be positions): the first row's position + the draft's
 *     depth (0 for a draft without a parent);
 *   masks[r][mask_words]: bit j % 32 of word j / 32 is set where draft j is
 *     draft r or an ancestor of it.
 * mask_words is 1 to 32, n_seq at most 65535.  A parent that is no earlier
 * draft counts as -1 and records 0x704 in the device error word; drafts past
 * 32 * mask_words get an empty mask and depth 0 and record 0x705. */
ATTN_API int attn_tree_plan_ex(int n_seq, int n_rows, int mask_words, const int *cu_rows, const int *parents,
                const int *positions, int *positions_out, uint32_t *masks, attn_stream_t stream);

typedef struct {
    int n_seq;                  /* requests, <= 65535                          */
    int n_rows;                 /* token rows of q, out, lse and masks:
                                   n_rows * heads <= 2^24                      */
    int n_groups;               /* groups that share a prefix (0: none)        */
    int heads, kv_heads;        /* as in attn_prefix_shape, and below          */
    int head_dim;
    int dtype;
    int page_size;
    int max_prefix_pages;
    int max_pages;
    int max_prefix_len;         /* upper bounds of prefix_lens and lens        */
    int max_len;
    int max_nodes;              /* upper bound of lens - ctx_lens, <= 1024     */
    int mask_words;             /* words of a row of masks, <= 32 and at least
                                   max_nodes / 32 (0 where masks is NULL)      */
    long long q_row_stride, out_row_stride;
    float scale;
} attn_tree_shape;

/* Bytes of device workspace attn_tree_decode_ex needs (by the shape, the
 * cache's type and the device's number of SMs). */
ATTN_API size_t attn_tree_decode_workspace_bytes(const attn_tree_shape *s, const attn_paged_kv *cache);

/* Each token row of request s attends, as one softmax, to the rows of its
 * group's prefix, to the first ctx_lens[s] rows of block_table[s] and to those
 * of the rows ctx_lens[s] + j, below lens[s], for which its mask has bit j
 * (masks NULL: j up to the row's index in the request).  A row that a token
 * does not see may hold anything.  lens[s] = ctx_lens[s] for a request whose
 * drafts have no rows (refused by the page plan): the page plan's lens and
 * lens_out are ctx_lens and lens.
 *   cu_rows[n_seq+1] (DEVICE, ascending): the requests' rows of q and out; ends
 *   are clamped to n_rows, and rows of no request are left as they are.
 *   group_begin[n_groups+1] (ascending): group g is requests [group_begin[g],
 *   group_begin[g+1]).  Prefixes, tables, lse, clamped lengths and error codes
 *   0x702 and 0x703, arithmetic and NaN as in attn_prefix_decode_ex.  A row that
 *   sees nothing gets out = 0 and lse = -inf.  A prefix, and a context, is read once for each
 *   block of up to 4 to 256 query rows (token rows x heads/kv_heads).
 * workspace: 256-byte aligned, of the size above; calls that may overlap on the
 * GPU need one each. */
ATTN_API int attn_tree_decode_ex(const attn_tree_shape *s, const attn_paged_kv *cache, const void *q, const int *cu_rows,
                const int *ctx_lens, const int *lens, const uint32_t *masks, const int *group_begin,
                const int *prefix_table, const int *prefix_lens, const int *block_table, void *out, float *lse,
                void *workspace, size_t workspace_bytes, attn_stream_t stream);

/* Keeps, of every request's drafts, the path that ends at draft leaf[s] (-1:
 * none): the drafts in the leaf's mask (masks NULL: drafts 0 .. leaf[s]) go, in
 * their order, to rows ctx_lens[s], ctx_lens[s] + 1, ... in each of the n_layers
 * caches (a HOST array, at most ATTN_MAX_LAYERS, all of one type; K, V and
 * scales, none of them there twice in any part, as layers that share a cache
 * pass it once), whose rows follow block_table.  Of the page shape, max_tokens is
 * the rows of masks, to which cu_rows is clamped (without masks it is not looked
 * at, nor is cu_rows clamped).  Written besides:
 *   lens_out[n_seq]: ctx_lens + the drafts kept (lens where there were none);
 *   free_pages past *free_count: the pages behind the kept rows, in request and
 *     page order (what passes n_pages entries is lost);
 *   counts[4]: the free pages after it, the drafts kept, the requests that kept
 *     none, the pages handed back.
 * A leaf that is no drafted row of its request keeps nothing and, unless the
 * request has no drafted rows, records 0x706 in the device error word; a page
 * outside a cache records 0x702 and its rows stay where they are.  lens_out and
 * counts must not overlap lens, ctx_lens, leaf, free_count and one another. */
ATTN_API int attn_tree_commit_ex(const attn_page_shape *s, int n_layers, const attn_paged_kv *caches, int kv_heads, int head_dim,
                const int *cu_rows, const int *ctx_lens, const int *lens, const int *leaf, const uint32_t *masks,
                int mask_words, const int *block_table, int *free_pages, const int *free_count, int *lens_out,
                int *counts, attn_stream_t stream);

/* ------------------------------------------------------------------------
 * Multi-GPU partitioning by (batch x head) units
 * ---------------------------------------------------------------------- */
/* Contiguous split of n_units over `world` ranks: rank gets [*begin, *end). */
ATTN_API int attn_shard_range(long long n_units, int world, int rank,
                     long long *begin, long long *end);
/* Longest-processing-time-first assignment of (seq, head) decode units whose
 * cost is the cache length: out_rank[s*heads + h] receives the rank,
 * out_load[r] (may be NULL) the summed length per rank.  Host arrays. */
ATTN_API int attn_shard_lpt(const int *lens, int n_seq, int heads, int world,
                   int *out_rank, long long *out_load);
/* After an all-gather of head shards, staging is [world][B][T][H/world][d];
 * writes out as (B*T, H*d).  dtype ATTN_F32 or ATTN_BF16. */
ATTN_API int attn_gather_permute(const void *staging, void *out, int world, int batch,
                        int seq_len, int heads, int head_dim, int dtype,
                        attn_stream_t stream);

/* ------------------------------------------------------------------------
 * Multi-GPU groups (no counterpart in the reference, whose trainer drives one
 * GPU from one host process, train_kaggle.cu:346).  NCCL over NVLink is used
 * only to gather outputs for callers that need them whole; the attention
 * itself needs no collective.  NCCL is loaded at run time (libnccl.so.2, or
 * the path in $ATTN_NCCL_LIB); NCCL_NVLS_ENABLE defaults to 0.  One group per
 * process.
 * ---------------------------------------------------------------------- */
/* One host thread drives devices 0..ngpus-1 (ncclCommInitAll); use
 * attn_fwd_multi / attn_decode_multi. */
ATTN_API int attn_init(int ngpus);
/* One process per GPU: rank 0 makes a 128-byte id, the caller hands it to
 * every rank, and each joins with attn_init_rank on `device` (-1: the current
 * device); then use the ordinary entry points on the rank's share and
 * attn_gather_split / attn_gather_rows. */
ATTN_API int attn_get_unique_id(unsigned char id[128]);
ATTN_API int attn_init_rank(int nranks, int rank, int device, const unsigned char id[128]);
/* Destroys the group's communicators (after the caller's work on them is done). */
ATTN_API int attn_finalize(void);
/* Ranks in the group, 0 when there is none. */
ATTN_API int attn_group_size(void);
/* Host-side watchdog: waits until every listed stream is idle, polling the
 * communicators' asynchronous errors.  On a communicator error, or when the
 * streams are still busy after timeout_ms, it aborts every communicator
 * (ncclCommAbort), removes the group and returns ATTN_ERR_COMM. */
ATTN_API int attn_group_sync(const attn_stream_t *streams, int n_streams, int timeout_ms);

/* A rank's share of the (batch x head) units: nb x nh ranks tile the batch and
 * head ranges evenly, with as many ranks along the batch as divide it (whole
 * batches keep a rank's rows contiguous).  Rank r holds batches
 * [batch0, batch0 + batch) and heads [head0, head0 + heads). */
typedef struct {
    int batch0, batch, head0, heads;
    int nb, nh;
} attn_split;
ATTN_API int attn_split_plan(int batch, int heads, int nranks, int rank, attn_split *out);

/* Bytes of workspace attn_gather_split / attn_fwd_multi need per rank for a
 * gather of this shape (0 when the split is by whole batches). */
ATTN_API size_t attn_gather_workspace_bytes(const attn_shape *s, int dtype, int nranks);
/* One-process-per-rank group: `local` is this rank's forward output, dense
 * (batch*T rows of heads*d, its split of `s`, the full shape); writes the
 * whole (B*T, H*d) output `out` on every rank (all-gather, then a permute
 * kernel when ranks split the heads). */
ATTN_API int attn_gather_split(const attn_shape *s, int dtype, const void *local, void *out,
                               void *workspace, size_t workspace_bytes, attn_stream_t stream);

/* Ragged decode across ranks: each rank decodes its own sequences (for
 * example by attn_shard_lpt with heads = 1) into `local`, max_local rows of
 * row_bytes (a multiple of 16).  attn_gather_rows all-gathers every rank's
 * max_local rows and writes row i of the gathered [nranks][max_local] block to
 * out row order[i] (a DEVICE array; < 0 skips padding).  order == NULL: the
 * gathered block is the output (n_out = nranks * max_local). */
ATTN_API size_t attn_gather_rows_workspace_bytes(int max_local, size_t row_bytes, int nranks);
ATTN_API int attn_gather_rows(const void *local, int max_local, size_t row_bytes, const int *order,
                              int n_out, void *out, void *workspace, size_t workspace_bytes,
                              attn_stream_t stream);

/* attn_init group, one host thread: device g holds the full-size inputs
 * q[g], k[g], v[g] (shape `s`) and runs its split (attn_split_plan with
 * rank g) into o[g] at the split's rows and columns; lse[g] (may be NULL)
 * receives its split's [batch][heads][T] statistics.  gather = 1 completes
 * o[g] on every device (NCCL all-gather on streams[g]; dense output rows
 * needed); ws[g] / ws_bytes[g] as attn_gather_workspace_bytes. */
ATTN_API int attn_fwd_multi(const attn_shape *s, int dtype, const void *const *q,
                            const void *const *k, const void *const *v, void *const *o,
                            float *const *lse, int gather, void *const *ws,
                            const size_t *ws_bytes, const attn_stream_t *streams);
/* attn_init group, one host thread: device g decodes its own sequences
 * (shapes[g], its caches and lens, out[g] with max_local rows); gather = 1
 * then writes every device's rows into out_full[g] (n_total rows, 16-byte
 * aligned) by order[g] (as attn_gather_rows), with ws[g] of
 * attn_gather_rows_workspace_bytes(max_local, H*d*4, ngpus) bytes. */
ATTN_API int attn_decode_multi(const attn_decode_shape *shapes, const float *const *q,
                               const void *const *kcache, const void *const *vcache,
                               const float *const *kscale, const float *const *vscale,
                               const int *const *lens, float *const *out, int gather,
                               int max_local, const int *const *order, int n_total,
                               float *const *out_full, void *const *ws,
                               const size_t *ws_bytes, const attn_stream_t *streams);

/* ------------------------------------------------------------------------
 * Test hook (no counterpart in the reference)
 * ---------------------------------------------------------------------- */
/* The next `launches` fp32 decode calls served by the TMA-ring decode kernel
 * (fp32 calls of up to 256 sequences and 256 MB of cache that are too large
 * for the one-CTA-per-head kernel) make one of its warps wait on a
 * barrier that nothing arrives at, bounded by `limit_cycles` SM cycles
 * (>= 1000).  The wait runs out and the kernel takes its timeout path: it
 * records code 0x32f in the device error word (attn_device_error), stops,
 * lets the copies it has in flight land, and returns; the call's output is
 * undefined and later calls run normally.  For tests of failure detection:
 * no GPU fault is involved. */
ATTN_API int attn_debug_decode_timeout(int launches, long long limit_cycles);

/* The same for the next `launches` calls of the QKV projection: the MMA
 * warp of its tensor-core kernel first waits on a barrier that nothing
 * arrives at, bounded by `limit_cycles` (>= 1000).  The kernel records 0x5ff
 * in the device error word, every role stops, and the teardown frees the
 * kernel's TMEM; the call's outputs are undefined and later calls run
 * normally. */
ATTN_API int attn_debug_qkv_timeout(int launches, long long limit_cycles);

#ifdef __cplusplus
}
#endif

#endif /* ATTN_B200_H */
