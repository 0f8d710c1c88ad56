/*
 * rac_b200.h -- extensions of the RAC C API exported by librac_b200.so.
 *
 * Four groups:
 *  1. error channel and process-wide knobs (the reference binding keeps the
 *     same knobs in rac_torch/rac_torch_bind.cpp:54-55, :205-219);
 *  2. batch forms of the _n primitives of lib/c/rac_cpu.h:110-114 and the
 *     batch helpers of lib/c/rac_cpu.h (rac_softmax_batch);
 *  3. stream-ordered device entry points: the GEMM launchers of
 *     rac_torch/rac_kernels.hip:822-909 with the same names and argument
 *     meaning, plus *_async forms of every op for callers that own device
 *     memory and a cudaStream_t (passed as void*).  These never synchronise
 *     and return a status; the PyTorch layer binds to them;
 *  4. attention over packed prompts (forward and backward), attention of new
 *     tokens over a paged key/value cache, and the pages of that cache; no
 *     counterpart in the reference, stream-ordered like group 3.
 *
 * Status codes follow lib/c/rac_cpu.h:54-59 and extend them.
 */
#ifndef RAC_B200_H
#define RAC_B200_H

#include "rac.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ── 1. status, errors, knobs ───────────────────────────────────────────── */
#define RAC_OK               0
#define RAC_ERR_NULL_PTR    -1   /* lib/c/rac_cpu.h:56 */
#define RAC_ERR_INVALID_DIM -2   /* lib/c/rac_cpu.h:57 */
#define RAC_ERR_ALLOC       -3   /* lib/c/rac_cpu.h:58 */
#define RAC_ERR_CUDA        -4   /* no usable device, or a CUDA call failed */
#define RAC_ERR_UNSUPPORTED -5   /* op/mode/layout not provided */
#define RAC_ERR_DEVICE      -6   /* a kernel's bounded loop gave up (e.g. |theta| >= 2^25) */

#define RAC_MODE_FAST     0      /* rac_kernels.hip:13 */
#define RAC_MODE_CORDIC   1      /* rac_kernels.hip:14 */
#define RAC_MODE_SHIFTADD 2      /* rac_kernels.hip:15 (integer shift-add product) */

#define RAC_ACT_NONE 0           /* rac_torch.cu:665-666 activation ids */
#define RAC_ACT_RELU 1
#define RAC_ACT_GELU 2
#define RAC_ACT_SILU 3
/* Gated FFN (SwiGLU, bench/bench_rac_transformer.c:441-453) in one GEMM: B holds
 * the gate and up weights row-interleaved (gate row c at 2c, up row c at
 * 2c+1), and C gets N/2 columns, C[m, c] = silu(v[m, 2c]) * v[m, 2c+1] with
 * v = alpha * op(A) op(B) (+ bias).  N must be even and beta 0.  The same
 * bits as a SiLU GEMM over the gate rows times a plain GEMM over the up rows,
 * multiplied elementwise.  No counterpart in the reference's extension. */
#define RAC_ACT_SWIGLU 4

/* Thread-local status of the last call made on this thread (0 = ok). */
int         rac_last_error(void);
const char *rac_last_error_string(void);
void        rac_clear_error(void);

/* Process-wide GEMM knobs used by rac_matmul and by launchers given
 * iters <= 0 / mode < 0.  iters is clamped to [1, 24]; iters <= 0 resets to
 * the default.  Defaults: iters = RAC_ITERS (env RAC_CORDIC_ITERS),
  * mode = RAC_MODE_CORDIC (env RAC_CORDIC_MODE = fast|cordic|shiftadd). */
void rac_set_cordic_iters(int iters);
int  rac_get_cordic_iters(void);
void rac_set_cordic_mode(int mode);
int  rac_get_cordic_mode(void);

/* Library and device information. */
const char *rac_b200_version(void);
int  rac_b200_device_count(void);
/* The 24 direction signs d_i of the GEMM micro-rotation sequence (see
 * rac_torch/rac_kernels.hip:176-185); for tests. */
void rac_b200_cordic_gemm_directions(int out[24]);

/* ── 2. batch forms (host or device pointers, blocking) ─────────────────── */
/* out[i] = rac_rotate_n(v[i], theta[i], iters)  (lib/c/rac_cpu.c:275-280) */
void rac_rotate_batch_n(const float2 *v, const float *theta, float2 *out, int n, int iters);
/* out[i] = rac_project_n(v[i], theta[i], iters) (lib/c/rac_cpu.c:282-288) */
void rac_project_batch_n(const float2 *v, const float *theta, float *out, int n, int iters);
void rac_exp_batch(const float *x, float *y, int n);
void rac_tanh_batch(const float *x, float *y, int n);
void rac_rsqrt_batch(const float *x, float *y, int n);
void rac_sigmoid_batch(const float *x, float *y, int n);
void rac_sincos_batch(const float *theta, float *s, float *c, int n);
/* lib/c/rac_cpu.c:459-463 */
void rac_softmax_batch(const float *x, float *out, int batch, int n);
/* rac_matmul with explicit iteration count and mode (no knob). */
void rac_matmul_ex(const float *A, const float *B, float *C, int M, int N, int K,
                   int iters, int mode);

/* ── 3. stream-ordered device entry points ──────────────────────────────── */
/* rac_kernels.hip:822-909: C = alpha * op(A) op(B) + beta * C on `stream`
 * (a cudaStream_t), device pointers, row-major, contiguous.
 *   nn: A[M,K]  B[K,N];   nt: A[M,K]  B[N,K];   tn: A[K,M]  B[K,N].
 * iters <= 0 / mode < 0 take the process-wide knobs. */
void rac_launch_nn_iters(const float *A, const float *B, float *C, int M, int N, int K,
                         float alpha, float beta, int iters, int mode, void *stream);
void rac_launch_nt_iters(const float *A, const float *B, float *C, int M, int N, int K,
                         float alpha, float beta, int iters, int mode, void *stream);
void rac_launch_tn_iters(const float *A, const float *B, float *C, int M, int N, int K,
                         float alpha, float beta, int iters, int mode, void *stream);
/* rac_kernels.hip:886-909: FAST mode, the reference's legacy entry points. */
void rac_launch_nn(const float *A, const float *B, float *C, int M, int N, int K,
                   float alpha, float beta, void *stream);
void rac_launch_nt(const float *A, const float *B, float *C, int M, int N, int K,
                   float alpha, float beta, void *stream);
void rac_launch_tn(const float *A, const float *B, float *C, int M, int N, int K,
                   float alpha, float beta, void *stream);

/* General GEMM with strides and a fused epilogue:
 *   C = act(alpha * op(A) op(B) + beta * Cin + bias)
 * layout 0/1/2 = nn/nt/tn; Cin read only when beta != 0 (may equal C);
 * bias is [N] or NULL; act is RAC_ACT_*.  Covers rac_fused_linear_kernel
 * (rac_torch.cu:705-779) and residual-add fusion.  `variant` 0 = automatic
 * tile.  Returns a status. */
int rac_gemm_async(const float *A, long long lda, const float *B, long long ldb,
                   float *C, long long ldc, const float *Cin, long long ldcin,
                   const float *bias, int M, int N, int K, int layout, int mode,
                   int iters, float alpha, float beta, int act, int variant,
                   void *stream);

/* rac_gemm_async for callers that cannot allocate device memory -- no
 * counterpart in the reference.  Same arguments and result as
 * rac_gemm_async, always split-K (`splits` K chunks; 0 = the automatic
 * count, at least 1), with the partial sums held in a 16 MiB array compiled
 * into the library instead of a workspace allocated per call: the call makes
 * no allocation at all.  Hosts that give a library a fixed device-memory
 * budget, or cannot tolerate an allocation on a latency-critical path, use
 * this form.  Limits: splits * M * N <= 4 Mi floats (else
 * RAC_ERR_INVALID_DIM with the sizes in rac_last_error_string()); every GPU
 * that loads the library holds the 16 MiB until exit; all calls share the
 * array, so calls whose kernels overlap on the GPU (two streams, two host
 * threads) race.  The first call on a device looks the array's address up
 * (make it before any stream capture on that device). */
int rac_gemm_splitk_noalloc_async(const float *A, long long lda, const float *B, long long ldb,
                                  float *C, long long ldc, const float *Cin, long long ldcin,
                                  const float *bias, int M, int N, int K, int layout, int mode,
                                  int iters, float alpha, float beta, int act, int splits,
                                  void *stream);

int rac_rotate_batch_async(const float2 *v, const float *theta, float2 *out, long long n,
                           int iters, int literal_kinv, void *stream);
int rac_project_batch_async(const float2 *v, const float *theta, float *out, long long n,
                            int iters, void *stream);
int rac_sincos_batch_async(const float *theta, float *s, float *c, long long n, void *stream);
/* op: 0 exp, 1 tanh, 2 rsqrt, 3 sigmoid */
int rac_unary_async(const float *x, float *y, long long n, int op, void *stream);
int rac_softmax_async(const float *x, float *y, long long rows, int d, void *stream);
int rac_rmsnorm_async(const float *x, float *y, const float *gamma, float eps,
                      long long rows, int d, void *stream);
int rac_layernorm_async(const float *x, float *y, const float *gamma, const float *beta,
                        float eps, long long rows, int d, void *stream);
int rac_rope_cache_async(float *cos_out, float *sin_out, int max_seq, int head_dim,
                         float base, void *stream);
/* In place on [batch_heads, seq, head_dim]; pos (optional, device int32[seq])
 * maps sequence index -> table row.  form 0 = lib/c rac_rope_apply
 * (rac_cpu.c:600-635), form 1 = torch RACRoPE (rac_torch.py:1165-1181). */
int rac_rope_apply_async(float *x, const float *cos_tab, const float *sin_tab,
                         const int *pos, long long batch_heads, int seq, int head_dim,
                         int form, void *stream);
/* Row positions[i] of the tables [table_rows, half] (dtype as in section 4) for
 * i < n, as floats: tables for rac_rope_apply_async over rows of any positions
 * (int32 or int64: pos_bytes 4 or 8).  A position outside the tables gives a row of
 * NaN, and rac_check_device_errors() reports RAC_ERR_DEVICE. */
int rac_rope_rows_async(const void *cos_tab, const void *sin_tab, int dtype, const void *positions, int pos_bytes,
                        long long n, long long table_rows, int half, float *cos_out, float *sin_out, void *stream);
/* Fused attention on `stream` (device pointers): rac_attention without the
 * [seq, seq] score tensor (lib/c/rac_cpu.c:637-703 semantics). */
int rac_attention_async(const float *q, const float *k, const float *v, const float *mask,
                        int is_causal, float *out, int batch, int n_heads, int seq,
                        int head_dim, void *stream);
/* Reads and clears the device's error word (bounded-loop overruns, pages and
 * positions that do not exist) after
 * synchronising `stream`; returns RAC_OK or RAC_ERR_DEVICE. */
int rac_check_device_errors(void *stream);

/* ── 4. packed prompts and paged caches ─────────────────────────────────── */
/* Element types.  Sums, softmax statistics and gradients are held in 32 bits
 * whatever the type.  head_dim is 32, 64 or 128; query head h reads key/value
 * head h / (heads / kv_heads).  The arguments come in a structure in host
 * memory, read before the call returns; all pointers in it are device
 * pointers, 16-byte aligned where they point to elements.  Strides count
 * elements and are multiples of 16 bytes; the last axis is contiguous. */
#define RAC_F32  0
#define RAC_F16  1
#define RAC_BF16 2

/* softmax(scale q k^T) v within each of n_seqs sequences laid end to end:
 * sequence i holds rows cu_seqlens[i] .. cu_seqlens[i+1]-1 (cu_seqlens[0] is
 * 0, n_seqs+1 rising int32), lengths of 0 allowed; its contents lead nowhere
 * outside the tensors.  q [tokens, heads, head_dim], k and v [tokens,
 * kv_heads, head_dim].  out [tokens, heads, head_dim] contiguous; lse
 * (optional) [heads, tokens], the natural logarithm of each row's sum.  Rows
 * behind the last sequence stay as they are, or become zeros where zero_rest
 * is set.
 *
 * out_low (optional, like out; 16-bit types): what rounding took from out's
 * first 128 rows of each sequence, where few keys share the weight and the
 * gradients feel it most.  With it the forward keeps the weights of those
 * rows' keys to twice the digits, and the backward, given it, takes D = do . o
 * from both.
 *
 * The backward call takes the forward's out, lse and out_low and the output's gradient
 * dout, and writes dq like q, dk and dv like k (contiguous), zeros behind the
 * last sequence.  The same inputs give the same bits.
 *
 * workspace: rac_attention_packed_workspace() bytes on the current device, 256-byte
 * aligned (may be NULL where that is 0), free again when the call's kernels are done. */
typedef struct {
    const void *q, *k, *v;
    const int *cu_seqlens;
    void *out;
    float *lse;
    void *out_low;                        /* optional, 16-bit types, see above */
    const void *dout;                     /* backward */
    void *dq, *dk, *dv;                   /* backward */
    void *workspace;
    long long strides[8];                 /* q row, q head, k row, k head, v row, v head, dout row, dout head */
    long long tokens, ws_bytes;
    int n_seqs, heads, kv_heads, head_dim, dtype, is_causal, zero_rest;
    float scale;
} rac_attention_packed_args;
long long rac_attention_packed_workspace(long long tokens, int n_seqs, int heads, int kv_heads, int head_dim,
                                         int dtype, int backward);
int rac_attention_packed_async(const rac_attention_packed_args *args, void *stream);
int rac_attention_packed_backward_async(const rac_attention_packed_args *args, void *stream);

/* Attention of new tokens over a paged cache.  Pages hold [kv_heads,
 * page_size, head_dim] each; cache row r of sequence b lies in page
 * page_table[b, r / page_size] (int32 [batch, table_width]), slot r %
 * page_size.  lengths[b] counts its rows, the new ones (the last counts[b],
 * or `nodes` where counts is NULL; at most 64) included: they are in the
 * cache already.  New row i sees every row before the new ones and the new
 * rows j whose bit is set in tree[b, i] (int64 [batch, nodes]), j <= i where
 * tree is NULL; a row that sees nothing gives zeros (the values of new rows
 * must be finite, seen or not).  q [batch, nodes, heads,
 * head_dim]; out contiguous, rows from counts[b] on as they were or zeros
 * (zero_rest).  Pages outside [0, n_pages) are not read: their rows count as
 * hidden and rac_check_device_errors() reports RAC_ERR_DEVICE.  workspace:
 * rac_attention_cached_workspace() bytes on the current device, 256-byte
 * aligned. */
typedef struct {
    const void *q, *k_pages, *v_pages;
    const int *page_table, *lengths, *counts;
    const long long *tree;
    void *out;
    void *workspace;
    long long strides[9];                 /* q batch, node, head; k page, head, row; v page, head, row */
    long long ws_bytes;
    int table_width, n_pages, page_size, batch, nodes, heads, kv_heads, head_dim, dtype, zero_rest;
    float scale;
} rac_attention_cached_args;
long long rac_attention_cached_workspace(int batch, int nodes, int heads, int kv_heads, int head_dim);
int rac_attention_cached_async(const rac_attention_cached_args *args, void *stream);

/* Page operations.  Rows and pages outside the cache are skipped and reported
 * as above. */
typedef struct {
    void *k_pages, *v_pages;
    const void *k, *v;                    /* append: new rows [tokens, kv_heads, head_dim] */
    const int *page_table, *starts, *cu_seqlens;
    const int *src, *dst;                 /* copy */
    const int *accepted, *n_accepted;     /* compact */
    long long strides[12];                /* k layer, page, head, row; v layer, page, head, row; k row, head; v row, head */
    long long tokens;
    int table_width, n_pages, page_size, batch, n, layers, kv_heads, head_dim, dtype;
} rac_cache_args;
/* Rows cu_seqlens[b] .. of k and v to cache rows starts[b] .. of sequence b. */
int rac_cache_append_async(const rac_cache_args *args, void *stream);
/* Page src[i] to page dst[i] for i < n, in every layer.  No page may be a
 * destination twice, nor a source and a destination (the copies run at once). */
int rac_cache_copy_pages_async(const rac_cache_args *args, void *stream);
/* Cache row starts[b] + accepted[b, i] to row starts[b] + i for i <
 * n_accepted[b], in every layer; accepted is [batch, n], n at most 64.  All of a
 * sequence's rows are read before the first is written. */
int rac_cache_compact_async(const rac_cache_args *args, void *stream);

/* ── op descriptors for rac_execute ─────────────────────────────────────── */
typedef struct { const float *A, *B; float *C; int M, N, K; } rac_matmul_desc;
typedef struct { const float2 *v; const float *theta; float2 *out; int n; int iters; } rac_rotate_batch_desc;
typedef struct { const float *x; float *out; int rows, n; } rac_softmax_desc;
typedef struct { const float *x; float *y; const float *gamma, *beta; float eps; int rows, d; } rac_norm_desc;
typedef struct { float *x; const float *cos_tab, *sin_tab; int batch, n_heads, seq, head_dim; } rac_rope_apply_desc;
typedef struct { float *cos_out, *sin_out; int max_seq, head_dim; float base; } rac_rope_cache_desc;
typedef struct { const float *x; float *y; int n; } rac_unary_desc;
typedef struct { const float *q, *k, *v, *mask; int is_causal; float *out;
                 int batch, n_heads, seq, head_dim; } rac_attention_desc;

#ifdef __cplusplus
}
#endif

#endif /* RAC_B200_H */
