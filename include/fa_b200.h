/*
 * fa_b200.h -- C ABI of the B200 (sm_100a) attention / MLP hot path.
 *
 * Library: libfa_b200.so (built by cs348k_fast_attention_grammar_b200/build.py).
 * All entry points are stream-ordered and asynchronous on the caller's
 * stream; none of them allocates device memory, and the caller owns every
 * buffer.  Every function returns an fa_status (0 = success); no C++
 * exception crosses this boundary.  Tensors are bf16 (raw 16-bit words)
 * unless the name says f16 or f32, pointers are device pointers, strides are
 * in elements.
 *
 * Reference interfaces replaced (paths inside nriedman/cs348k-fast-attention-grammar):
 *   fa_attn_fwd  <- the attention operator behind the kernel-module protocol
 *                   that bench.py:14-20 times: the host callable fn(KT, Q, V)
 *                   emitted at grammar/kernel_ast.py:1267-1287 (e.g.
 *                   runs/attn_full/kernels/best_it24.py:78-99), the torch
 *                   modules pytorch-naive.py:23-65 and flash-attn2-sota.py:41-63,
 *                   and the batched attention(q, k, v) of
 *                   old/kernels/old/naive.py:27-56 / old/benchmark.py:17-21.
 *   fa_attn_fwd_f32 <- the same callables at the reference's own fp32 2-D
 *                   problem (fn(KT, Q, V) with fp32 cupy arrays), staging to
 *                   bf16 on the device instead of host-side casts.
 *   fa_mlp_fwd   <- the host callable emitted for the MLP program of
 *                   run_mlp_search.py:42-127 (stages h = X@W1, a = act(h),
 *                   y = a@W2 at :58-69).
 *   fa_gemm_act  <- one matmul stage with its pointwise epilogue, the
 *                   "matmul" reduction rule grammar/kernel_ast.py:207-211
 *                   (ct.mma K-loop) followed by the relu stage of
 *                   run_mlp_search.py:62-64.
 *   *_f16        <- the same operators at the reference harnesses' default
 *                   dtype, fp16 (bench.py:32 DTYPE_MAP, old/benchmark.py:96
 *                   --dtype fp16, old/kernels/old/naive.py:27-56).
 *   fa_attn_fwd_f32_batched <- the fp32 [B, H, S, D] problem of the
 *                   reference's seeded runs (run_attention_search.py:169-181,
 *                   BASELINE cfg0), one call for all (batch, head) pairs.
 */
#ifndef FA_B200_H_
#define FA_B200_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum fa_status {
  FA_OK = 0,
  FA_ERR_NULL = 1,         /* a required pointer is NULL                        */
  FA_ERR_SHAPE = 2,        /* a dimension is <= 0 or too large                  */
  FA_ERR_HEAD_DIM = 3,     /* head dim not supported (attention: 8..128, x8)    */
  FA_ERR_ALIGN = 4,        /* pointer or stride not 16-byte aligned (TMA rule)  */
  FA_ERR_STRIDE = 5,       /* innermost stride is not 1                         */
  FA_ERR_TMA = 6,          /* cuTensorMapEncodeTiled rejected the tensor        */
  FA_ERR_LAUNCH = 7,       /* kernel launch failed (cudaGetLastError)           */
  FA_ERR_DRIVER = 8,       /* driver entry point unavailable                    */
  FA_ERR_DEVICE = 9,       /* current device is not sm_100 (B200 class)         */
  FA_ERR_ARG = 10,         /* an enum argument is out of range                  */
  FA_ERR_TIMEOUT = 11,     /* a kernel wait ran out (read by fa_device_status)  */
  FA_ERR_CUDA = 12,        /* another CUDA runtime call failed                  */
  FA_ERR_SCRATCH = 13,     /* problem exceeds fa_mlp_fwd_noalloc's fixed buffer */
  FA_ERR_PAGE = 14,        /* a block table entry or a length points outside the
                              cache (read by fa_device_status)                  */
  FA_ERR_WORKSPACE = 15    /* the workspace is missing or too small             */
} fa_status;

typedef enum fa_dtype {
  FA_BF16 = 0,
  FA_F16 = 1,
  FA_F32 = 2
} fa_dtype;

typedef enum fa_f32_precision {
  FA_F32_BF16 = 0,         /* fp32 operands rounded to bf16 (8 significant bits) */
  FA_F32_SPLIT = 1         /* bf16 hi + lo split, three products per GEMM        */
} fa_f32_precision;

typedef enum fa_activation {
  FA_ACT_NONE = 0,
  FA_ACT_RELU = 1,         /* run_mlp_search.py:62-64                           */
  FA_ACT_GELU_TANH = 2     /* 0.5x(1+tanh(sqrt(2/pi)(x+0.044715x^3)))           */
} fa_activation;

/* Human-readable text for a status code (static storage). */
const char* fa_strerror(int status);

/* Library version as major*10000 + minor*100 + patch. */
int fa_version(void);

/*
 * Fused attention forward  O = softmax(Q K^T * scale [+ causal mask]) V.
 *   q, k, v, o : [B, H, S, D] bf16, element strides
 *                strides[0..3] = q (b, h, s, d), strides[4..7] = k,
 *                strides[8..11] = v, strides[12..15] = o; every d-stride must
 *                be 1 and every other stride a multiple of 8 elements.
 *   D          : 8 .. 128, a multiple of 8 (D <= 64 runs the four-tile
 *                kernel, larger D the two-tile kernel; the head dim is
 *                zero-padded to the kernel's width on chip, never in memory).
 *   causal     : nonzero = key j visible to query i iff j <= i.
 *   scale      : softmax scale (pass 1/sqrt(D) for the reference's math).
 *   stream     : cudaStream_t (NULL = legacy default stream).
 * Computes in fp32 (tcgen05 bf16 MMAs with fp32 accumulation in TMEM).
 * With more work units (256 query rows at D = 128, 512 at D = 64; fewer
 * rows when the problem would leave most SMs idle, and at D <= 64 without a
 * causal mask a last partial wave of units split into halves) than SMs
 * the kernel runs persistent and takes units from one of 1024 library-owned
 * device counters, handed out round-robin per call and reset by the launch
 * that used it; a counter is shared only if 1024 further calls are issued
 * while a launch that holds it is still queued or running (for instance
 * replays of separately captured CUDA graphs run concurrently).
 */
int fa_attn_fwd(const void* q, const void* k, const void* v, void* o, int B, int H, int S,
                int D, const int64_t* strides, int causal, float scale, void* stream);

/*
 * fa_attn_fwd with fp16 Q, K, V and O (raw 16-bit words): the same kernels
 * with fp16 tensor-core operands (P is rounded to fp16 for O += P V),
 * fp32 accumulation and softmax.  Arguments and rules as fa_attn_fwd.
 */
int fa_attn_fwd_f16(const void* q, const void* k, const void* v, void* o, int B, int H, int S,
                    int D, const int64_t* strides, int causal, float scale, void* stream);

/*
 * The reference's own 2-D fp32 problem in one call (the kernel-module
 * callables fn(KT, Q, V) of pytorch-naive.py:23 and of every emitted module,
 * grammar/kernel_ast.py:1267-1287, and fn(K, Q, V) of flash-attn2-sota.py:41
 * on one (batch, head) pair):
 *   q [N, D], v [N, D], o [N, D] fp32, contiguous;
 *   k [N, D] fp32 (k_transposed = 0) or KT [D, N] fp32 (k_transposed = 1);
 *   ws         : bf16 workspace of 3 * N * D elements (16-byte aligned), where
 *                q, k, v are staged in bf16 (one launch) for the tensor cores;
 *   D          : as for fa_attn_fwd; causal, scale, stream as for fa_attn_fwd.
 * Two launches (staging, attention); O is written in fp32 by the attention
 * epilogue.  Inputs are rounded to bf16, accumulation is fp32.
 */
int fa_attn_fwd_f32(const void* q, const void* k, const void* v, void* o, void* ws, int N,
                    int D, int k_transposed, int causal, float scale, void* stream);

/*
 * fp32 attention for batched tensors: q, v, o contiguous [B, H, S, D] fp32,
 * k contiguous [B, H, S, D] (k_transposed = 0) or [B, H, D, S] (1).  Two
 * launches for all pairs: staging to bf16, then the attention with an fp32
 * epilogue.  precision:
 *   FA_F32_BF16  : operands rounded to bf16 (as fa_attn_fwd_f32);
 *                  ws = 3 * B * H * S * D bf16 elements;
 *   FA_F32_SPLIT : each operand x staged as hi = bf16(x) and lo = bf16(x - hi),
 *                  and S = Qh Kh^T + Qh Kl^T + Ql Kh^T, O = Ph Vh + Ph Vl + Pl Vh
 *                  accumulated in fp32 (about 16 significant bits; three times
 *                  the tensor-core work); D <= 64; ws = 3 * B * H * S * 128.
 * ws is 16-byte aligned.
 */
int fa_attn_fwd_f32_batched(const void* q, const void* k, const void* v, void* o, void* ws,
                            int B, int H, int S, int D, int k_transposed, int causal,
                            float scale, int precision, void* stream);

/*
 * C[M, N] = act(A[M, K] @ B[K, N]) in bf16 with fp32 accumulation.
 *   A row-major with row stride lda (K contiguous); B row-major [K, N] with
 *   row stride ldb (N contiguous); C row-major with row stride ldc.
 *   K and N must be multiples of 64, M any positive value; lda, ldb, ldc
 *   multiples of 8.
 */
int fa_gemm_act(const void* a, const void* b, void* c, int M, int N, int K, int64_t lda,
                int64_t ldb, int64_t ldc, int act, void* stream);

/* fa_gemm_act with fp16 A, B and C (fp32 accumulation).  Same rules. */
int fa_gemm_act_f16(const void* a, const void* b, void* c, int M, int N, int K, int64_t lda,
                    int64_t ldb, int64_t ldc, int act, void* stream);

/*
 * MLP block Y[M, K] = act(X[M, K] @ W1[K, N]) @ W2[N, K]   (all row-major bf16).
 *   hidden : caller-owned [M, N] bf16 workspace that receives act(X @ W1).
 *   K, N multiples of 64.  act = FA_ACT_GELU_TANH for the benchmark block,
 *   FA_ACT_RELU for the reference's.
 */
int fa_mlp_fwd(const void* x, const void* w1, const void* w2, void* hidden, void* y, int M,
               int K, int N, int act, void* stream);

/* fa_mlp_fwd with fp16 X, W1, W2, hidden and Y (fp32 accumulation). */
int fa_mlp_fwd_f16(const void* x, const void* w1, const void* w2, void* hidden, void* y, int M,
                   int K, int N, int act, void* stream);

/*
 * The reference's full MLP block (run_mlp_search.py:42-127, checked by its
 * verify at :138-149):
 *   hidden = relu(X @ W1)            [M, N]  caller-owned bf16 workspace
 *   resid  = hidden @ W2 + X         [M, K]  caller-owned bf16 workspace
 *                                            (residual added in GEMM 2's epilogue)
 *   out    = (resid - mean) / sqrt(var + eps) over each row (no affine)
 * K, N multiples of 64; K <= 8192 (the LayerNorm row stays in registers).
 */
int fa_mlp_ln_fwd(const void* x, const void* w1, const void* w2, void* hidden, void* resid,
                  void* out, int M, int K, int N, float eps, void* stream);

/*
 * Row LayerNorm without affine parameters: out[i, :] = (in[i, :] - mean_i) /
 * sqrt(var_i + eps), population variance, computed in fp32 (the LayerNorm
 * stage of run_mlp_search.py:76-93).  N a multiple of 8, N <= 8192; row
 * strides multiples of 8 elements.
 */
int fa_layernorm_rows(const void* in, void* out, int M, int N, int64_t ld_in, int64_t ld_out,
                      float eps, void* stream);

/*
 * fa_mlp_fwd without any device allocation: the same MLP block, with the
 * hidden activation kept in a fixed array inside the library instead of a
 * caller-provided buffer.  No counterpart in the reference.
 *   For callers that cannot call cudaMalloc or any allocator -- a plugin
 *   running inside a host whose memory pools it does not own, code that
 *   must not allocate while a CUDA graph is being built or while another
 *   component holds the device's memory budget.  They still pass X, W1, W2
 *   and Y.
 *   Limit: M * N <= 8,388,608 hidden elements (a 16 MiB bf16 array that every
 *   GPU loading the library keeps until the process exits); larger problems
 *   return FA_ERR_SCRATCH.  Other shape rules as fa_mlp_fwd.
 *   The first call on each device looks up the array's device address
 *   (cudaGetSymbolAddress); make that first call before any stream capture.
 *   All calls share the one array and it keeps the last call's contents
 *   (every element a call reads it first writes), so calls that may run at
 *   the same time on the GPU -- on different streams, or from different
 *   threads -- race and must be serialised by the caller.
 */
int fa_mlp_fwd_noalloc(const void* x, const void* w1, const void* w2, void* y, int M, int K,
                       int N, int act, void* stream);

/*
 * Rotary positions.  The first R of each head's D channels are rotated in
 * R / 2 planes (a, b):
 *     (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * inv_freq[i]
 * (t negated when `inverse`, which is also the gradient); the rest is copied.
 * Plane i is channels (i, i + R / 2), or (2i, 2i + 1) when `interleaved`.
 * Frequencies [section_end[a-1], section_end[a]) take the position of axis a
 * (images and video: time, height, width); one axis takes all of them.
 * Angles are formed in fp64 and reduced before the fp32 sine and cosine, so far
 * positions keep full precision; each value is rounded once.
 */
typedef struct fa_rotary_args {
  const void* x;           /* [B, H, S, D], D contiguous                        */
  void* out;               /* the same shape; may be x itself                   */
  const void* positions;   /* int32 or int64 [axes, B, S], strides below        */
  const void* inv_freq;    /* fp32 or fp64 [R / 2], contiguous                  */
  int64_t dtype;           /* fa_dtype of x and out                             */
  int64_t B, H, S, D, R;   /* D a multiple of 8, R a multiple of 16, R <= D     */
  int64_t x_strides[3];    /* elements: b, h, s; multiples of 16 bytes          */
  int64_t out_strides[3];
  int64_t axes;            /* 1 .. 4                                            */
  int64_t section_end[4];  /* rising; section_end[axes - 1] = R / 2             */
  int64_t pos_strides[3];  /* elements: axis, b, s (0 repeats)                  */
  int64_t pos_is_i64, freq_is_f64;
  int64_t interleaved, inverse;
} fa_rotary_args;

int fa_rotary(const fa_rotary_args* args, void* stream);

/*
 * Paged key/value cache.  Caches are [pages, page_size, Hkv, D] (any strides,
 * D contiguous); key j of sequence b is row j % page_size of page
 * block_table[b, j / page_size].  New tokens of all sequences are packed along
 * T: those of sequence b are rows [cu_seqlens[b], cu_seqlens[b + 1]) (row b
 * alone when cu_seqlens is NULL), and kv_lens[b] is the sequence's length with
 * them counted, so new token i of q_len sits at kv_lens[b] - q_len + i.
 * Borders outside [0, T] are held to it.
 *
 * fa_paged_append writes the keys, rotated as in fa_rotary when R > 0, and the
 * values of new tokens to their places, and the rotated queries, where there
 * are any, to q_out.  Without `positions` a token is rotated by its place in
 * the sequence.  Rows outside every sequence have no effect and are not written; a
 * token before its sequence's start (kv_lens[b] < q_len, as in padding
 * sequences of length 0) is not stored.  A place outside the table or a page
 * outside the cache is not written either and leaves FA_ERR_PAGE in the device
 * status word.  Two tokens with the same place leave either's values there.
 */
typedef struct fa_paged_append_args {
  const void* k;           /* [T, Hkv, D]                                       */
  const void* v;
  const void* q;           /* [T, Hq, D] or NULL                                */
  void* q_out;             /* may be q itself                                   */
  void* k_cache;
  void* v_cache;
  const int32_t* block_table;  /* [B, max_pages], row stride table_stride       */
  const int32_t* kv_lens;      /* [B]                                           */
  const int32_t* cu_seqlens;   /* [B + 1] or NULL (then T = B)                  */
  const void* positions;       /* int32 or int64 [axes, T] or NULL              */
  const void* inv_freq;        /* [R / 2]; NULL when R = 0                      */
  int64_t dtype;               /* FA_BF16 or FA_F16, all tensors alike          */
  int64_t T, B, Hq, Hkv, D, R; /* R = 0: no rotation                            */
  int64_t pages, page_size;    /* page_size a power of two, 16 .. 1024          */
  int64_t max_pages, table_stride;
  int64_t k_strides[2], v_strides[2], q_strides[2], q_out_strides[2]; /* token, head */
  int64_t k_cache_strides[3], v_cache_strides[3];                     /* page, row, head */
  int64_t axes;
  int64_t section_end[4];
  int64_t pos_strides[2];      /* axis, token                                   */
  int64_t pos_is_i64, freq_is_f64;
  int64_t interleaved;
} fa_paged_append_args;

int fa_paged_append(const fa_paged_append_args* args, void* stream);

/*
 * Attention of new tokens (one or a chunk per sequence) over the paged cache
 * that holds them:  o = softmax(q K^T * scale) V  per token and head, query
 * heads in Hkv groups that share a key/value head.  With `causal` a token sees
 * the keys up to its own place, else all kv_lens[b].  A token that sees no key,
 * or none with a score above -infinity, gets zeros; a score of +infinity or NaN
 * makes its output NaN.  Rows outside every sequence have no effect and are not written.
 * A page outside the cache reads as keys and values of zero, which have their
 * share of the weights.  Where a length goes beyond the table, tokens keep their
 * places (those fa_paged_append stores them by) and see the keys that the table
 * holds.  Both leave FA_ERR_PAGE in the device status word.  Cached values that
 * a sequence's tokens see must be finite (a value that only some of a chunk's
 * tokens see may reach the others as value * 0); rows behind kv_lens[b] may
 * hold anything.
 *   scale     : any whose product with log2(e) is finite in fp32.
 *   max_q_len : an upper bound of the tokens per sequence that only guides
 *               which kernels run (T where unknown); results hold for any value.
 *   workspace : fa_paged_attn_workspace(args) bytes, 16-byte aligned, used by
 *               this call alone until it has run (may be NULL for 0 bytes).
 */
typedef struct fa_paged_attn_args {
  const void* q;           /* [T, Hq, D]                                        */
  void* o;                 /* [T, Hq, D]                                        */
  const void* k_cache;     /* [pages, page_size, Hkv, D]                        */
  const void* v_cache;
  const int32_t* block_table;  /* [B, max_pages], row stride table_stride       */
  const int32_t* kv_lens;      /* [B]                                           */
  const int32_t* cu_seqlens;   /* [B + 1] or NULL (then T = B)                  */
  int64_t dtype;               /* FA_BF16 or FA_F16, all tensors alike          */
  int64_t T, B, Hq, Hkv, D;    /* D 8 .. 128, a multiple of 8; Hq / Hkv <= 128  */
  int64_t pages, page_size;    /* page_size a power of two, 16 .. 1024          */
  int64_t max_pages, table_stride; /* max_pages * page_size < 2^31 - 4096       */
  int64_t q_strides[2], o_strides[2];                                 /* token, head */
  int64_t k_cache_strides[3], v_cache_strides[3];                     /* page, row, head */
  int64_t max_q_len;
  int64_t causal;
  double scale;
} fa_paged_attn_args;

/* Bytes of workspace that fa_paged_attn needs for these arguments, or minus an
 * fa_status.  Depends on the sizes alone, not on what the arrays hold. */
int64_t fa_paged_attn_workspace(const fa_paged_attn_args* args);

int fa_paged_attn(const fa_paged_attn_args* args, void* workspace, int64_t workspace_bytes,
                  void* stream);

/*
 * Failure-detection self test: launches one CTA that waits on an mbarrier no
 * one ever arrives on, with a limit of limit_us microseconds (1 .. 10^6).  The
 * bounded wait gives up, records FA_ERR_TIMEOUT in the device status word and
 * the kernel returns normally (no trap, no fault), so the context stays
 * usable; read the result with fa_device_status().  Every wait inside the
 * library's kernels is bounded the same way (limit 1 s).  Reference analog:
 * the search's compile timeout (grammar/optimization.py:57-62,267-280), which
 * turns a hung compile into a recorded failure.
 */
int fa_selftest_wait_timeout(int limit_us, void* stream);

/*
 * Self test of the attention softmax's exponentials on the device: for the
 * n fp32 values x, writes out[i] = the FMA-pipe 2^x (Cody-Waite style
 * round-to-nearest range reduction, degree-3 minimax polynomial, exponent
 * add), out[n + i] = the same computed two at a time with paired fp32
 * instructions, and out[2n + i] = ex2.approx(x) (MUFU).  out holds 3n
 * floats.  These are the routines the attention kernels call.  Reference
 * analog: the exp stage that run_attention_search.py:64-67 lowers to ct.exp.
 */
int fa_selftest_exp2(const float* x, float* out, int n, void* stream);

/*
 * Reads and clears the device-side status word of the current device
 * (FA_OK, FA_ERR_TIMEOUT when a kernel's bounded wait ran out, or FA_ERR_PAGE
 * when a paged operator met a place outside the cache; a timeout outranks it).
 * Synchronises the device.
 */
int fa_device_status(void);

#ifdef __cplusplus
}
#endif

#endif /* FA_B200_H_ */
