/*
 * tritt.h - C ABI of libtritt_sm100.so: three-way ("trittention") attention for
 * NVIDIA B200 (sm_100a).
 *
 * The library replaces the device side of the reference package flash_trittention
 * (Triton kernels launched from Python); each entry point below names the reference
 * launch site it stands in for.  Host glue (argument validation, torch.autograd
 * plumbing) lives above this ABI and mirrors the reference's Python modules.
 *
 * Conventions
 *   - every tensor is row-major [B, N, T, D], innermost stride 1, base pointer 16-byte
 *     aligned, all of one dtype (TRITT_F32 / TRITT_F16 / TRITT_BF16); lse / m vectors
 *     are fp32 [B, N, T] holding the natural-log log-sum-exp of the scaled logits;
 *   - pointers are DEVICE pointers; the caller owns every buffer including `workspace`
 *     and keeps them alive until the work enqueued on `stream` has run;
 *   - calls only enqueue work on `stream` (no synchronisation, no device allocation);
 *   - return value 0 = success, negative = invalid argument, positive = cudaError_t of
 *     a failed runtime call.  tritt_last_error() gives a thread-local message;
 *   - `status_word` (an int the GPU can address: device memory or page-locked host memory; may be NULL)
 *     is OR-ed with a non-zero code by a kernel whose bounded barrier wait ran out (1 tensor-core
 *     self-test, 2 / 4 triple-dot-product forward / backward, 8 misaligned shared memory, 16 / 32
 *     soft-max attention forward / backward of the dot-product-sum path, 128 wait-expiry self-test, 1024
 *     triple-dot-product attention over a cache, or its weights) or,
 *     bit 64, by the fp16 operand conversion of an fp32 / wide-operand call that met an element beyond 65504,
 *     bit 256, by a rotation whose position its tables do not have, bit 512, by a call that met a place its cache does not have;
 *     the caller zeroes and reads it.  A non-zero word means the results of that call are invalid;
 *   - window arguments (k1_window, k2_window, kk_left, kk_right, k_diff) are distances >= 0; a value
 *     >= T means "unlimited".  Negative values are refused with an argument error when `causal` is set
 *     (the reference applies them literally, which leaves query rows with nothing to attend to);
 *   - B*N may not exceed 65535.
 */
#ifndef TRITT_H_
#define TRITT_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef void* tritt_stream_t; /* a cudaStream_t / CUstream */

enum { TRITT_F32 = 0, TRITT_F16 = 1, TRITT_BF16 = 2 };

/* operations, for tritt_workspace_bytes() */
enum { TRITT_OP_TDP_FWD = 0, TRITT_OP_TDP_BWD = 1, TRITT_OP_DPS_FWD = 2, TRITT_OP_DPS_BWD = 3 };
/* and for tritt_decode_workspace() */
enum { TRITT_OP_TDP_DECODE = 4, TRITT_OP_DPS_APPEND = 5, TRITT_OP_DPS_DECODE = 6 };

/* flags */
enum {
  TRITT_FLAG_FORCE_SIMT = 1,  /* use the plain fp32 CUDA-core kernels even where the tensor-core path applies */
  TRITT_FLAG_BWD_PARTIAL = 2, /* tritt_tdp_bwd: leave the fp32 key-side partial sums in the workspace and do not
                                 write dk1/dk2/dv1/dv2 (the caller reduces them across ranks, then calls
                                 tritt_tdp_bwd_finalize) */
  TRITT_FLAG_WIDE_OPERANDS = 4, /* triple-dot-product, bf16 inputs: form the operands with 11 significant bits (fp16
                                 copies) instead of bf16's 8, what the reference's `convert_to_float32` asks of its TF32
                                 dot products.  fp32 inputs always take that path on the tensor cores (head dimension
                                 64 / 128); fp16 inputs already have it.  Needs the larger workspace that
                                 tritt_workspace_bytes_flags() reports; an input element beyond fp16's range (65504)
                                 sets status bit 64. */
  TRITT_FLAG_BWD_CTA_PAIRS = 8  /* tritt_tdp_bwd: accepted and ignored (an earlier backward kernel could run as clusters
                                 of two CTAs; it was the slower form) */
};

/* kernel families, as reported by tritt_tdp_path() */
enum { TRITT_PATH_SIMT = 0, TRITT_PATH_TCGEN05 = 1 };

int tritt_version(void);
/* Number of kernels this library has enqueued in the calling process so far (bookkeeping for benchmarks). */
unsigned long long tritt_kernel_launches(void);
const char* tritt_last_error(void);

/* Bytes of caller-provided scratch to pass to the given operation (0 if none).  For TRITT_OP_TDP_FWD on 16-bit inputs
   the figure includes a tail behind the SiLU(V1) copy of B*N*T*D elements: up to seven floats per (batch, head), which
   let the forward bound its scores and skip the row-maximum pass, and for head dimension 64 and T > 128 up to 20 MB
   (4 * 33 KB per SM) for the kernel that serves narrow bands with small scores.  A workspace without the last part is
   accepted and runs the slower kernel there, one without the tail the two-pass soft-max.  tritt_tdp_fwd_workspace()
   gives what a call with known windows uses: calls without a narrow band have no need of the 20 MB.  For TRITT_OP_TDP_BWD on the tensor cores it includes a tail of about 1 KiB per (batch, head)
   for the largest elements behind the range shifts of fp16 products; a workspace without it is accepted and forms them
   without regard to their size, times alpha (at most 1, to a power of two) for the keys: small keys or values then lose
   bits to fp16's subnormals, and keys whose products times alpha reach 65504 overflow. */
size_t tritt_workspace_bytes(int op, int B, int N, int T, int D, int dtype);
/* The same for a call that will pass `flags` (TRITT_FLAG_WIDE_OPERANDS enlarges the triple-dot-product workspace of bf16
   inputs by the fp16 operand copies; tritt_workspace_bytes() equals flags = 0). */
size_t tritt_workspace_bytes_flags(int op, int B, int N, int T, int D, int dtype, int flags);

/* Bytes of scratch that tritt_tdp_fwd makes use of for these arguments: never more than tritt_workspace_bytes_flags(). */
size_t tritt_tdp_fwd_workspace(int B, int N, int T, int D, int dtype, int causal, int k1_window, int k2_window, int kk_left,
                               int kk_right, int q_mod, int flags);
/* Bytes of scratch tritt_tdp_fwd cannot run without for these arguments (the optional tail excluded). */
size_t tritt_tdp_fwd_min_workspace(int B, int N, int T, int D, int dtype, int causal, int k1_window, int k2_window,
                                   int kk_left, int kk_right, int flags);

/* Which kernel family a TDP call with these arguments runs on. */
int tritt_tdp_path(int op, int T, int D, int dtype, int causal, int k1_window, int k2_window, int kk_left,
                   int kk_right, int flags);
/* Which kernel family the two soft-max attentions of a DPS forward, and their row-owner / column-owner backward
   kernels, run on. */
int tritt_dps_path(int T, int D, int dtype, int k_diff, int flags);

/*
 * Triple-dot-product forward.  Replaces the launch of `_tritt_fwd` and the host-side
 * SiLU / `M + log(L)` passes around it in the reference
 * (src/flash_trittention/triple_dot_product/flash_trittention.py:61-62,92-128).
 *   S[q,j,k] = alpha * sum_h q[q,h] k1[j,h] k2[k,h];  softmax over the attended (j,k);
 *   o[q,h]   = sum_jk P[q,j,k] SiLU(v1[j,h]) v2[k,h];  lse[q] = log sum_jk exp(S).
 * (q_mod, q_rem): only query rows q with q % q_mod == q_rem are computed and written
 * (query-row sharding across devices); pass (1, 0) for all rows.
 */
int tritt_tdp_fwd(const void* q, const void* k1, const void* k2, const void* v1, const void* v2, void* o,
                  float* lse, int B, int N, int T, int D, int dtype, float alpha, int causal, int k1_window,
                  int k2_window, int kk_left, int kk_right, int q_mod, int q_rem, void* workspace,
                  size_t workspace_bytes, int* status_word, int flags, tritt_stream_t stream);

/*
 * Triple-dot-product backward.  Replaces the five launches `_tritt_bwd_dq/_dk1/_dk2/_dv1/_dv2`
 * and the host-side SiLU, D = sum(dO*O), zero-init and SiLU' passes of the reference
 * (src/flash_trittention/triple_dot_product/flash_trittention.py:158-173,191-391).
 * v1 is the RAW (pre-SiLU) tensor; dv1 is the gradient w.r.t. it.  With (q_mod, q_rem) != (1, 0)
 * only the selected rows of dq are written and the key-side gradients are partial sums.
 */
int tritt_tdp_bwd(const void* q, const void* k1, const void* k2, const void* v1, const void* v2, const void* o,
                  const void* d_o, const float* lse, void* dq, void* dk1, void* dk2, void* dv1, void* dv2, int B,
                  int N, int T, int D, int dtype, float alpha, int causal, int k1_window, int k2_window,
                  int kk_left, int kk_right, int q_mod, int q_rem, void* workspace, size_t workspace_bytes,
                  int* status_word, int flags, tritt_stream_t stream);

/*
 * Second half of a TRITT_FLAG_BWD_PARTIAL backward: converts the fp32 partial sums
 * (workspace layout: dK1 | dK2 | dSiLU(V1) | dV2, each [B,N,T,D] fp32, starting at
 * tritt_tdp_bwd_partials_offset() bytes) to the output dtype and applies SiLU'(v1) to dv1
 * (reference flash_trittention.py:390-391).  No counterpart launch in the reference: the
 * reference has no multi-device path.
 */
int tritt_tdp_bwd_finalize(const void* v1, void* dk1, void* dk2, void* dv1, void* dv2, int B, int N, int T, int D,
                           int dtype, void* workspace, size_t workspace_bytes, tritt_stream_t stream);
size_t tritt_tdp_bwd_partials_offset(int B, int N, int T, int D, int dtype);

/*
 * Dot-product-sum forward.  Replaces the launch of the reference's `_tritt_fwd`
 * (src/flash_trittention/dot_product_sum/trittention_triton.py:90-120).
 *   S[q,s,t] = alpha * (q[q].k2[t] + k1[s].k2[t]);  causal: s <= t <= q and t - s <= k_diff;
 *   o[q,h]   = sum_st P[q,s,t] SiLU(v1[s,h]) v2[t,h];  m[q] = log sum_st exp(S).
 */
int tritt_dps_fwd(const void* q, const void* k1, const void* k2, const void* v1, const void* v2, void* o, float* m,
                  int B, int N, int T, int D, int dtype, float alpha, int causal, int k_diff, void* workspace,
                  size_t workspace_bytes, int* status_word, int flags, tritt_stream_t stream);

/*
 * Dot-product-sum backward.  Replaces `_tritt_bwd_preprocess`, `_tritt_bwd_dq`, `_tritt_bwd_dk_dv`
 * and the host-side SiLU / SiLU' / dk2 merge passes of the reference
 * (src/flash_trittention/dot_product_sum/trittention_triton.py:160,183-356).
 */
int tritt_dps_bwd(const void* q, const void* k1, const void* k2, const void* v1, const void* v2, const void* o,
                  const void* d_o, const float* m, void* dq, void* dk1, void* dk2, void* dv1, void* dv2, int B,
                  int N, int T, int D, int dtype, float alpha, int causal, int k_diff, void* workspace,
                  size_t workspace_bytes, int* status_word, int flags, tritt_stream_t stream);

/*
 * The same backward for a caller that kept the forward call's workspace untouched (same inputs, same arguments):
 * the inner attention's results the forward left there (Y, its log-sum-exp, SiLU(V1), Y*V2) are read instead of being
 * computed again, which removes two launches.  `workspace` is still this call's own scratch of
 * tritt_workspace_bytes(TRITT_OP_DPS_BWD, ...) bytes.  The reference keeps no such state between its forward and
 * backward (it recomputes per query block, dot_product_sum/kernels/bwd_dq_kernel.py:28-350).
 */
int tritt_dps_bwd_saved(const void* q, const void* k1, const void* k2, const void* v1, const void* v2, const void* o,
                        const void* d_o, const float* m, void* dq, void* dk1, void* dk2, void* dv1, void* dv2, int B,
                        int N, int T, int D, int dtype, float alpha, int causal, int k_diff, void* workspace,
                        size_t workspace_bytes, const void* fwd_workspace, size_t fwd_workspace_bytes,
                        int* status_word, int flags, tritt_stream_t stream);

/*
 * Triple-dot-product forward for callers that may not allocate device memory (a plugin inside
 * another program's enqueue hook, a process whose device memory all belongs to a pool this call
 * site cannot use, a section that must avoid the allocator's device-wide synchronisation).
 * Same computation and checks as tritt_tdp_fwd for all query rows, but the scratch is an 8 MiB array
 * built into the library image (tritt_noalloc_scratch_bytes()), held by every GPU whose context has
 * loaded that image until the process exits (with CUDA's lazy module loading the driver may load it,
 * and reserve its memory, only at the first call).  Limits: 16-bit inputs on the tensor-core path
 * (head dimension 64 or 128) with B*N*T*D > 4 194 304 elements are rejected (the CUDA-core path - fp32
 * inputs, other head dimensions, TRITT_FLAG_FORCE_SIMT - needs no scratch); calls that overlap in time
 * on one GPU share the array and race; the first call on a device resolves the array's address and
 * should precede any stream capture on that device; the cached address does not survive
 * cudaDeviceReset.  It calls no allocation routine of the CUDA runtime or of any library.  This entry
 * point has no counterpart in the reference.
 */
int tritt_tdp_fwd_noalloc(const void* q, const void* k1, const void* k2, const void* v1, const void* v2, void* o,
                          float* lse, int B, int N, int T, int D, int dtype, float alpha, int causal,
                          int k1_window, int k2_window, int kk_left, int kk_right, int* status_word, int flags,
                          tritt_stream_t stream);
size_t tritt_noalloc_scratch_bytes(void);

/*
 * Self-test of the tensor-core building blocks (TMA tile loads, shared-memory operand
 * descriptors, a 16-bit operand held in tensor memory): one CTA computes
 *   C = A * Bm^T   and   C2 = round16(C) * V      (all matrices 128 x 128, row-major)
 * so that a host test can compare against a plain matmul.  No counterpart in the
 * reference (its kernels are Triton; the compiler picks the matrix instructions).
 */
int tritt_selftest_umma(const void* A, const void* Bm, const void* V, float* C, float* C2, int dtype,
                        int* status_word, tritt_stream_t stream);

/*
 * Self-test of the two bounded barrier waits that the tensor-core kernels use: a one-CTA kernel in which one
 * thread is to arrive on an mbarrier and a warp waits for it with each, giving up after `limit_ticks` clock ticks
 * (1 .. 2e9).  With skip_arrival != 0 the arrival is left out on purpose: the waits run out, the kernel ORs
 * 128 into `status_word` (1 if only one of them gave up), frees its tensor memory and returns; nothing faults and
 * the context stays usable.
 * No counterpart in the reference (Triton kernels have no hand-written waits).
 */
int tritt_selftest_wait_expiry(int skip_arrival, long long limit_ticks, int* status_word, tritt_stream_t stream);

/*
 * What tritt_tdp_bwd does with these arguments on the tensor cores, per head (host only, for tests and planning):
 *   out[0]  query rows that run in exact fp32 on the CUDA cores (of the shard, from its first)
 *   out[1]  cells (q, j, k) that the tensor-core kernel executes, masked ones among them (for a narrow band whose heads may
 *           go to the kernel that steps over diagonals: what the one over k would execute)
 *   out[2]  1 if that is the kernel that steps over queries (query shards), 0 if it steps over k
 * -12 if the call does not run on the tensor cores.  No counterpart in the reference.
 */
int tritt_tdp_bwd_plan(int T, int D, int dtype, int causal, int k1_window, int k2_window, int kk_left, int kk_right,
                       int q_mod, int q_rem, int flags, long long* out);

/*
 * Host-only self-test of the check in front of the backward kernel's launch: its warpgroups share out the registers it
 * is launched with, and a build that gives it another count per thread than the split was written for is refused
 * (0: `launched` registers per thread are what the split needs; -30: they are not).  No counterpart in the reference.
 */
int tritt_selftest_bwd_registers(int launched);

/* ------------------------------------------------------------------------------------------------------------------------
 * Around the attention: norms and rotation in front of it, and serving one or a few new tokens over a cache.  None of these
 * has a counterpart in the reference, which computes whole sequences from tensors that are normed and rotated elsewhere.
 */

/* Rows [B, N, T, D] of any of the three dtypes: element (b, n, t, d) at p + b*stride_b + n*stride_n + t*stride_t + d (strides in
   elements; the rows themselves are contiguous, 16-byte aligned). */
typedef struct {
  const void* p;
  long long stride_b, stride_n, stride_t;
} tritt_rows_t;

/*
 * Norms of queries and keys for each head, with the position rotation in the same pass.  For each row x of q, k1 and k2:
 *   u = x / sqrt(mean(x^2) + eps) * w;   of the first `rot` elements each pair (a, b) -> (a c - b s, b c + a s)
 * with c, s = cos[position], sin[position] ([positions in the tables, rot / 2] fp32, contiguous).  Pairs are (i, i + rot / 2), or
 * (2 i, 2 i + 1) if `interleaved`.  Head dimension 16, 32, 64, 128 or 256; `rot` 0 (norm alone) or a multiple of 16.
 */
typedef struct {
  tritt_rows_t x[3];          /* q, k1, k2 */
  tritt_rows_t y[3];          /* the results (forward: written); backward: their gradients (read) */
  tritt_rows_t dx[3];         /* backward: gradients of x (written) */
  const void* w[3];           /* weights [D] or, with weight_heads, [N, D]; null: 1 */
  void* dw[3];                /* backward: their gradients, in the weights' type; null: not wanted */
  const float *cos, *sin;     /* null: rot is 0 */
  const void* positions;      /* int32 or int64 (positions64), element (b, t) at b*position_stride_b + t*position_stride_t; null: t.  A position
                                 that the tables do not have sets status bit 256 and takes their nearest one */
  long long position_stride_b, position_stride_t;
  int positions64, table, rot, interleaved;   /* table: positions in the tables */
  int weight_heads, weight_dtype;             /* the weights' type is the rows' or TRITT_F32 */
  int B, N, T, D, dtype;
  float eps;
} tritt_norm_rotary_t;

int tritt_qk_norm_rotary_fwd(const tritt_norm_rotary_t* a, int* status_word, tritt_stream_t stream);
/* `workspace`: tritt_qk_norm_rotary_workspace() bytes (0 where no dw is wanted); gradients of the weights are summed in a fixed
   order, a call repeats itself bit for bit. */
int tritt_qk_norm_rotary_bwd(const tritt_norm_rotary_t* a, void* workspace, size_t workspace_bytes, int* status_word,
                             tritt_stream_t stream);
size_t tritt_qk_norm_rotary_workspace(const tritt_norm_rotary_t* a);

/* The same with positions that have several axes (time, row and column of a video's tokens): rotated pair i takes its cosine and sine from the
   position's row along axis `of`.  The position of element (b, t) along axis x stands at x*position_stride + b*position_stride_b + t*position_stride_t
   of `positions`, which must not be null. */
enum { TRITT_MAX_AXES = 4 };
typedef struct {
  long long position_stride;
  int count;                  /* axes, 1 to TRITT_MAX_AXES */
  unsigned char of[32];       /* of pair i: bits 2 (i % 4) and the next of byte i / 4 */
} tritt_axes_t;
int tritt_qk_norm_rotary_axes_fwd(const tritt_norm_rotary_t* a, const tritt_axes_t* axes, int* status_word, tritt_stream_t stream);
int tritt_qk_norm_rotary_axes_bwd(const tritt_norm_rotary_t* a, const tritt_axes_t* axes, void* workspace, size_t workspace_bytes, int* status_word,
                                  tritt_stream_t stream);

/* What an element of a cache is held in. */
enum { TRITT_CODE_F16 = 0, TRITT_CODE_E4M3 = 1, TRITT_CODE_INT8 = 2 };
enum { TRITT_MAX_ANCESTORS = 64 };

/*
 * A paged cache of rows of D elements, four of a token and head (the parts): K1, K2, SiLU(V1), and V2 (triple dot product) or
 * W (dot-product-sum: the inner attention's result times V2, whose log-sum-exp stands in `lse`).
 * An element is code * 2^(exponent - 127) with one exponent byte for a row: the least with which the row's largest element is at
 * most 448 (e4m3), at most 127 (int8) or below 2^15 (fp16), so codes are rounded once and powers of two are exact.  Elements below
 * 2^-126 count as zero.  A row with an infinite or NaN element gets the exponent 255: all of it reads as NaN, and a
 * token that attends to it gets NaN.
 * Token t of sequence b is row t % page_size of page table[b][t / page_size]; a table has at most 2^28 tokens.
 * Each call is about n new tokens of B sequences: token i of sequence b is number context[b] + i, for i < counts[b] (counts null: n).
 * It attends to the context[b] tokens before them and, of the new ones, to token m if bit m of ancestors[b][i] is set and m < i,
 * and to itself (ancestors null: to all m <= i).  Distances are counted along the tokens that it attends to: their positions are 0, 1, 2, ...
 * in order, its own is the last.  A place that the table or the cache does not have sets status bit 512 and is neither read
 * nor written; context[b] < 0 is an unused sequence: nothing of its cache is read or written, its results are those of no attended token.
 * The arrays start as zeros; a row that nobody has written reads as zeros.
 */
typedef struct {
  void* codes;                 /* [pages, 4, N, page_size, D] */
  unsigned char* exponents;    /* [pages, 4, N, page_size] */
  float* lse;                  /* [pages, N, page_size] natural-log units, or null (triple dot product) */
  int pages, page_size, N, D, code;   /* page_size: a power of two from 16 on;  D: 16, 32, 64, 128 or 256 */
  const int* table;            /* [B, table_pages] */
  long long table_stride;      /* elements between two sequences' tables */
  int table_pages;
  const int* context;          /* [B] */
  const int* counts;           /* [B] or null */
  const long long* ancestors;  /* [B, n] or null; n <= TRITT_MAX_ANCESTORS with them */
  int B, n;
} tritt_cache_t;

/* Quantises the new tokens' K1, K2, SiLU(V1) and V2 (`dtype`) into their places: of these arrays only the rows of the new tokens change.
   rows: k1, k2, raw v1, v2 [B, N, n, D]. */
int tritt_cache_write(const tritt_cache_t* c, const tritt_rows_t* rows, int dtype, int* status_word, tritt_stream_t stream);
/* Reads the new tokens' four parts back into contiguous [B, N, n, D] tensors of `dtype`, and lse into [B, N, n] (where the cache has it
   and lse is not null); zeros for i >= counts[b] and for places that there are not. */
int tritt_cache_read(const tritt_cache_t* c, void* const* parts, float* lse, int dtype, int* status_word, tritt_stream_t stream);

/*
 * Triple-dot-product attention of the n new tokens, whose rows are in the cache already (tritt_cache_write):
 *   S[q,j,k] = alpha sum_h q[q,h] K1[j,h] K2[k,h], soft-max over the attended pairs, o = sum P SiLU(V1)[j] V2[k]
 * over pairs of attended tokens within the windows (distances of positions, as for tritt_tdp_fwd: q - j <= k1_window,
 * q - k <= k2_window, k - j <= kk_left, j - k <= kk_right).  o: [B, N, n, D] contiguous; lse [B, N, n] or null.
 * A token without an attended pair (i >= counts[b], context[b] < 0) gets o = 0, lse = -infinity.  alpha is finite, here and below.
 * On the tensor cores a sequence has at most 2^30 (new token, 32 rows k of its window) groups and 2^39 products of 256 x 128 cells a head; one that has
 * more sets status bit 1024 and gets no results (o = 0, lse = -infinity).
 */
int tritt_tdp_decode(const tritt_cache_t* c, const tritt_rows_t* q, void* o, float* lse, int dtype, float alpha, int k1_window,
                     int k2_window, int kk_left, int kk_right, void* workspace, size_t workspace_bytes, int* status_word, int flags,
                     tritt_stream_t stream);
/*
 * Dot-product-sum attention of new tokens, in the two chained soft-maxes into which its score separates.  Append: writes K1, K2 and
 * SiLU(V1) of the new tokens, attends from each token t (its unrounded k2) to the tokens s with position(t) - position(s) <= k_diff,
 *   Y[t] = sum_s softmax_s(alpha K1[s].k2[t]) SiLU(V1)[s],  lse[t] = log sum_s exp(alpha K1[s].k2[t])
 * and writes W[t] = Y[t] v2[t] and lse[t].
 */
int tritt_dps_append(const tritt_cache_t* c, const tritt_rows_t* rows, int dtype, float alpha, int k_diff, void* workspace,
                     size_t workspace_bytes, int* status_word, int flags, tritt_stream_t stream);
/* Decode: o[q] = sum_t softmax_t(alpha q.K2[t] + lse[t]) W[t], m its log-sum-exp; the new tokens are in the cache already. */
int tritt_dps_decode(const tritt_cache_t* c, const tritt_rows_t* q, void* o, float* m, int dtype, float alpha, void* workspace,
                     size_t workspace_bytes, int* status_word, int flags, tritt_stream_t stream);
/* Bytes of scratch for the three calls above (op: TRITT_OP_TDP_DECODE, TRITT_OP_DPS_APPEND, TRITT_OP_DPS_DECODE); the windows of the
   triple dot product as above (0 for the others).  0: none is needed, or the description is refused.  Calls that may run at the same time need
   scratch of their own. */
size_t tritt_decode_workspace(int op, const tritt_cache_t* c, int dtype, int k1_window, int k2_window, int flags);
/* Which kernel family such a call runs on: TRITT_PATH_SIMT (fp32 arithmetic on the CUDA cores) or, for those with matrix instructions, TRITT_PATH_TCGEN05,
   which also stands for warp-level ones here (the dot-product sum, and the triple product under windows that fit in shared memory). */
int tritt_decode_path(int op, int D, int dtype, int flags);

/* ------------------------------------------------------------------------------------------------------------------------
 * Which tokens of a cache are worth keeping: the attention weight that each has got, and a cache with the heaviest ones alone.
 */

/* Weights of tokens, fp32: that of token x of sequence b and head n at before + b*before_stride_b + n*before_stride_n + x, x < before_length; the
   new ones at `after` in the same way (the same place as `before`, or another).  The weigh calls write, of every sequence with context[b] >= 0,
     after[x] = (x < context[b] ? decay * before[x] : 0) + what the call's new tokens add,   x < context[b] + (its new tokens)
   and nothing else (decay 0 does not read `before`).  A token beyond either length sets status bit 512 and is left out.  decay is finite, >= 0. */
typedef struct {
  const float* before;
  float* after;
  long long before_stride_b, before_stride_n, after_stride_b, after_stride_n;
  int before_length, after_length;
  float decay;
} tritt_weights_t;

/*
 * Triple dot product: each new token i adds sum_k P_i[x,k] + sum_j P_i[j,x] to token x, with P_i[j,k] = exp(S_i[j,k] - lse_i) over the pairs that it attends to
 * (tritt_tdp_decode; 2 in all for each token and head).  lse: [B, N, n], as tritt_tdp_decode has written it; a token whose lse is -infinity adds nothing.
 * No ancestors: drafts are weighed once they are accepted.  Sums are formed in a fixed order, a call repeats itself bit for bit.
 */
int tritt_tdp_weigh(const tritt_cache_t* c, const tritt_weights_t* w, const tritt_rows_t* q, const float* lse, int dtype, float alpha, int k1_window,
                    int k2_window, int kk_left, int kk_right, void* workspace, size_t workspace_bytes, int* status_word, tritt_stream_t stream);
/* Bytes of scratch for it: 20 (head dimensions 64 and 128) or 8 for each token that the windows and the table have room for, whatever the contexts are, for each of 148 blocks and for each head of the sequences that
   are taken at a time: as many as keep it below 2^30 bytes, one at least.  So a table of 2^17 tokens and 16 heads without windows takes 430 MB, one of 2^20 tokens 3.4 GB.  Calls that may run at the same time need scratch of their own. */
size_t tritt_tdp_weigh_workspace(const tritt_cache_t* c, int k1_window, int k2_window);
/*
 * Dot-product sum: each new token i adds exp(alpha q_i.K2[x] + lse[x] - m_i) to the tokens x that its query attends to (tritt_dps_decode), and
 * exp(alpha k2_i.K1[x] - lse[i]) to those that its k2 attends to (tritt_dps_append, whose k_diff).  k2: the unrounded rows; m: [B, N, n].  An m or lse that is
 * -infinity adds nothing.  No ancestors.
 */
int tritt_dps_weigh(const tritt_cache_t* c, const tritt_weights_t* w, const tritt_rows_t* q, const tritt_rows_t* k2, const float* m, int dtype, float alpha,
                    int k_diff, int* status_word, tritt_stream_t stream);

/*
 * Keeps `keep` tokens of each sequence and head (of c->context tokens; c->n and c->counts are not looked at): the `first` first, the `recent` last, and of the others those with
 * the largest w->before (ties: the lower number; NaN counts as the largest), first + recent <= keep.  Their rows and log-sum-exps move to the places of tokens 0, 1, 2, ...
 * in order, and their weights to w->after; kept [B, N, keep] gets their numbers, -1 behind the last, context_out [B] the tokens that are left.  A sequence that has no more than
 * `keep` tokens keeps all of them; context[b] < 0 stays as it is.
 * table_out null, or c->table itself: in place (the places behind the last kept token keep what they hold).  Else the rows go to the pages of table_out, [B, table_out_pages] with stride
 * table_out_stride, of which none may be one that the call reads, and the old ones stay as they are.  A page that several sequences share must not be written.
 * A place that there is not sets status bit 512; what it should have held, or should hold, is left out.  So does a token beyond before_length.
 * w->decay is not looked at.  w->after may be w->before (with the same strides), or must not overlap it; after_length >= keep.
 */
int tritt_cache_evict(const tritt_cache_t* c, const tritt_weights_t* w, const int* table_out, long long table_out_stride, int table_out_pages, int keep, int first,
                      int recent, int* context_out, int* kept, int* status_word, tritt_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* TRITT_H_ */
