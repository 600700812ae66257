/*
 * qrb200 -- batched Householder QR for NVIDIA B200 (sm_100a), C ABI.
 *
 * Drop-in boundary for the reference operator ``custom_kernel(data) -> (H, tau)``
 * (Raymondlol/qr-v2-b200-kernel ``submission.py:560-596``; contract of the harness that
 * calls it: ``harness/eval.py:189-211``, output checks ``harness/reference.py:175-204``).
 *
 * Layout (identical to torch.geqrf / LAPACK sgeqrf, row-major storage):
 *   A    : batch matrices, each n x n float32 row-major (row stride n), matrix b at
 *          A + b * a_batch_stride (a_batch_stride >= n*n elements). Read only.
 *   H    : batch x n x n float32 row-major, contiguous. R = triu(H); reflector j is
 *          v_j = (0,..,0, 1, H[j+1:, j]) with the unit diagonal implicit.
 *   tau  : batch x n float32, contiguous. Q = H_0 H_1 ... H_{n-1}, H_j = I - tau_j v_j v_j^T.
 * Sign convention: beta = -sign(alpha) * ||(alpha, x)||, tau = (beta - alpha)/beta,
 * tau = 0 when x == 0 (submission.py:91-107, LAPACK slarfg without rescaling).
 *
 * Execution: every call is asynchronous on ``stream`` (a cudaStream_t; NULL = legacy
 * default stream), makes no host synchronisation and allocates no memory: scratch comes
 * from the caller's ``workspace`` (size from qrb200_workspace_bytes, 256-byte aligned).
 * Two calls that share a workspace must be ordered on the same stream.
 *
 * Every entry point returns a status (QRB200_OK = 0). Device-side failures found by a
 * bounded wait are reported by qrb200_last_status() (no synchronisation) or
 * qrb200_device_status() once the work has executed.
 *
 * The first call on each device registers that device's failure word with a synchronous
 * symbol copy: make it before any stream capture on that device. The library does not
 * survive a cudaDeviceReset (its per-device set-up is not redone).
 */
#ifndef QRB200_H_
#define QRB200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
  QRB200_OK = 0,
  QRB200_ERR_ARG = 1,        /* bad shape, stride or null pointer                    */
  QRB200_ERR_WORKSPACE = 2,  /* workspace too small or not 256-byte aligned          */
  QRB200_ERR_CUDA = 3,       /* a CUDA runtime call or kernel launch failed          */
  QRB200_ERR_DEVICE = 4,     /* current device is not an sm_100 (B200-class) GPU     */
  QRB200_ERR_TIMEOUT = 5,    /* a device-side bounded wait expired (see device_status) */
  QRB200_ERR_SCRATCH_LIMIT = 6, /* qrb200_geqrf_f32_noalloc: problem needs more scratch than
                                  QRB200_NOALLOC_SCRATCH_BYTES                           */
  QRB200_ERR_INDEX = 7       /* a cache slot, block table entry or length was out of range
                                (see qrb200_last_status); it was skipped, not followed   */
};

/* Bytes of scratch that qrb200_geqrf_f32 needs for (batch, n).
 * Replaces the per-call temporaries the reference allocates through torch
 * (submission.py:177-185 H clone + tau, :453-480 V/G/M/W/Y). */
size_t qrb200_workspace_bytes(int64_t batch, int64_t n);

/* Batched QR: H, tau <- geqrf(A). Replaces custom_kernel (submission.py:560-596) and
 * its back-ends _fused_qr (:177-185), _factor_custom (:520-553) and torch.geqrf (:576, :583).
 * A is not modified (the reference clones it first, submission.py:179, :522). */
int qrb200_geqrf_f32(const float* A, float* H, float* tau, int64_t batch, int64_t n,
                     int64_t a_batch_stride, void* workspace, size_t workspace_bytes,
                     void* stream);

/* ---- using the factorisation: Q and Q^T (the reference's checker step, sorgqr/sormqr) ---- */

/* Bytes of scratch that qrb200_ormqr_f32 (nrhs columns) and qrb200_orgqr_f32 (nrhs = n) need. */
size_t qrb200_apply_workspace_bytes(int64_t batch, int64_t n, int64_t nrhs);

/* C <- Q^T C (transpose != 0) or Q C (transpose == 0), in place, for each matrix of the batch:
 * Q = H_0 H_1 ... H_{n-1} of (H, tau) in the layout qrb200_geqrf_f32 writes (H batch x n x n,
 * tau batch x n, contiguous), C batch x n x nrhs row-major contiguous. Left side only, as
 * torch.ormqr(H, tau, C, left=True, transpose=...). Blocked compact-WY on the tensor cores
 * (3xTF32). Needs n % 4 == 0, nrhs % 4 == 0, 1 <= n <= 4096, H and C 16-byte aligned
 * (QRB200_ERR_ARG otherwise). Replaces the LAPACK/cuSOLVER sormqr that a consumer of the
 * reference's (H, tau) output would call (README.md:42-50 of the reference: Q is implicit). */
int qrb200_ormqr_f32(const float* H, const float* tau, float* C, int64_t batch, int64_t n, int64_t nrhs,
                     int transpose, void* workspace, size_t workspace_bytes, void* stream);

/* Q (batch x n x n, row-major contiguous, written) = householder_product(H, tau) for square H:
 * replaces torch.linalg.householder_product, which the reference's checker calls on every
 * output (harness/reference.py:206). Same requirements as qrb200_ormqr_f32 (nrhs = n). */
int qrb200_orgqr_f32(const float* H, const float* tau, float* Q, int64_t batch, int64_t n, void* workspace,
                     size_t workspace_bytes, void* stream);

/* Human-readable text for a status code (static storage). */
const char* qrb200_status_string(int status);

/* Library version as MAJOR*10000 + MINOR*100 + PATCH. */
int qrb200_version(void);

/* Device-side failures. Every wait inside a kernel is bounded; a kernel whose wait expires
 * records the failure, skips its outputs and returns (the results of that call are invalid).
 * The record lands in a device word and in a mapped pinned host word per device.
 *
 * qrb200_last_status: QRB200_ERR_TIMEOUT (an expired wait) or QRB200_ERR_INDEX (a slot, block
 * table entry or length outside a cache) if a kernel on the current device has recorded a
 * failure since the last read, else QRB200_OK; the host word is cleared by the read. It makes
 * no CUDA call beyond cudaGetDevice and never waits, so it sees failures of work that has
 * already executed (read it after synchronising, or before the next call as the Python operator
 * does). *site_out (may be NULL) receives the wait site: 1 tensor-core mbarrier, 2 whole-matrix
 * hand-off, 3 cluster-panel exchange, 4 self-test, 5 cache index. No counterpart in the reference (its only
 * failure mechanism is the exception fallback of submission.py:572-596). */
int qrb200_last_status(int* site_out);

/* Synchronous variant: reads (and clears) the device word of the current device with a symbol
 * copy (which waits for prior work on the legacy default stream) and clears the host word;
 * *status_out = QRB200_ERR_TIMEOUT, QRB200_ERR_INDEX or QRB200_OK. */
int qrb200_device_status(int* status_out);

/* Test hook: one warp waits `polls` times on a barrier that nothing completes, so the wait runs
 * out and reports site 4 through the same path as the factorisation kernels. Asynchronous on
 * `stream`; leaves the device usable. */
int qrb200_selftest_wait_timeout(uint32_t polls, void* stream);

/* ---- allocation-free entry (no counterpart in the reference) ------------------------- */

/* Size of the library's static device scratch used by qrb200_geqrf_f32_noalloc: 32 MiB.
 * It covers every call with qrb200_workspace_bytes(batch, n) <= this: up to 1 matrix of n = 4096,
 * 3 of n = 2048, 11 of n = 1024, 29 of n = 512 or 55 of n = 256 per call; n <= 128 needs no
 * scratch at any batch size. */
#define QRB200_NOALLOC_SCRATCH_BYTES (32u << 20)

/* Same result as qrb200_geqrf_f32 (bit for bit), but the scratch is a file-scope static
 * __device__ array of the library instead of a caller workspace, so neither the caller nor the
 * library allocates device memory. For callers that cannot or should not allocate: plain C or
 * FFI code with no device allocator at hand, loops that must not call cudaMalloc/cudaFree
 * (cudaFree waits for the whole device), and processes whose device memory is already fully
 * reserved by another allocator.
 *   - Limit: returns QRB200_ERR_SCRATCH_LIMIT, launching nothing, when
 *     qrb200_workspace_bytes(batch, n) > QRB200_NOALLOC_SCRATCH_BYTES; use qrb200_geqrf_f32
 *     with a workspace for larger problems. Other errors are those of qrb200_geqrf_f32.
 *   - Set-up: the first call on each device (the current device) looks up the array's device
 *     address with cudaGetSymbolAddress, which loads the library module that holds it there;
 *     make that first call before any stream capture on that device.
 *   - Nothing needs to start at zero: every scratch word is written before it is read within
 *     a call, so the array's contents between calls do not matter.
 *   - One array per device: calls on the same device whose executions overlap (different
 *     streams, or host threads, without ordering) race on it and give wrong results. Order
 *     them on one stream, or with events. */
int qrb200_geqrf_f32_noalloc(const float* A, float* H, float* tau, int64_t batch, int64_t n,
                             int64_t a_batch_stride, void* stream);

/* ---- data in 8 and 4 bits (no counterpart in the reference) ---------------------------
 *
 * What a consumer of Q needs next to it: activations and weights rotated by an orthogonal matrix
 * hold no outlying channels, and are kept in 8 bits, keys and values in 4. All entries are
 * asynchronous on `stream`, allocate nothing, return a status, and first report (launching
 * nothing) a failure that a kernel of an earlier call has recorded, as qrb200_last_status does.
 * The first call on each device, of these or of any other entry that launches, registers its failure word for all kernels, with
 * synchronous symbol copies: make it before any stream capture on that device. */

enum { QRB200_F32 = 0, QRB200_BF16 = 1, QRB200_F16 = 2 }; /* element types */

/* Rows into 8 bits. h = x + residual (x alone when residual is NULL); t = h * weight (h alone when
 * weight is NULL); code_j = rint(t_j * 127 / a) with a = max |t_j|;
 * scale = a * (mean(h^2) + eps)^-1/2 / 127, so code * scale is the norm's output. h, rounded to
 * dtype, goes to h_out (rows x cols, contiguous; NULL exactly when residual is). Finite rows of any
 * size are normalised, through scaled squares where 32 bits do not hold theirs. h_out may be the residual itself, not
 * overlap an input otherwise (rows off 16-byte boundaries that need scaled squares are then normalised from h as stored).
 * x, residual: rows x cols of dtype with row strides in elements; weight: cols of dtype or of
 * QRB200_F32; q: row stride q_stride bytes; scale: rows. cols <= 32768. A row with a NaN or an
 * infinity gets codes 0 and a NaN scale; one whose a is below 2^-100 gets codes and scale 0. */
int qrb200_rms_norm_int8(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                         const void* weight, int weight_type, int8_t* q, int64_t q_stride, float* scale, void* h_out,
                         int64_t rows, int64_t cols, float eps, int dtype, void* stream);

/* The same without the norm: code = rint(x * 127 / max|x|), scale = max|x| / 127. */
int qrb200_quantize_int8(const void* x, int64_t x_stride, int8_t* q, int64_t q_stride, float* scale, int64_t rows,
                         int64_t cols, int dtype, void* stream);

/* out (rows x cols of dtype, contiguous) = q * scale of its row. */
int qrb200_dequantize_int8(const int8_t* q, int64_t q_stride, const float* scale, void* out, int64_t rows,
                           int64_t cols, int dtype, void* stream);

/* y[i, n] = (sum_k x[i, k] w[n, k]) x_scale[i] w_scale[n] + bias[n]: y rows x outs of dtype,
 * contiguous, 16-byte aligned; bias (may be NULL) of dtype; row strides of x and w in bytes. The sum is
 * exact in 32-bit integers for depth <= QRB200_INT8_MAX_DEPTH, and scaled in 32 bits. Operands whose rows start on 16-byte
 * boundaries are read as they lie; others are first laid out in the workspace (256-byte aligned, its
 * size from the query; 0 for the former). */
#define QRB200_INT8_MAX_DEPTH 131071
size_t qrb200_int8_linear_workspace_bytes(const int8_t* x, int64_t x_stride, const int8_t* w, int64_t w_stride,
                                          int64_t rows, int64_t outs, int64_t depth);
int qrb200_int8_linear(const int8_t* x, int64_t x_stride, const float* x_scale, const int8_t* w, int64_t w_stride,
                       const float* w_scale, const void* bias, void* y, int64_t rows, int64_t outs, int64_t depth,
                       int dtype, void* workspace, size_t workspace_bytes, void* stream);

/* A paged key/value cache in 4 bits: pages x kv_heads blocks of qrb200_kv4_block_bytes bytes,
 * contiguous, 16-byte aligned. Each group of head_dim / groups channels of a token holds 4-bit
 * codes and a step and minimum of type dtype (QRB200_BF16 or QRB200_F16). head_dim 64 or 128;
 * groups of 32, 64 or 128 channels; page_size a power of two from 16 to 1024. */
typedef struct qrb200_kv4_shape {
  int64_t pages;
  int32_t kv_heads, page_size, head_dim, groups, dtype;
} qrb200_kv4_shape;
int64_t qrb200_kv4_block_bytes(int64_t page_size, int64_t head_dim, int64_t group_size);

/* Quantises keys and values (tokens x kv_heads x head_dim of the cache's type, channels
 * contiguous, other strides in elements) into the cache at slots (page * page_size + offset). A
 * negative slot is skipped; slots of one call must differ. A group's step and minimum are its
 * range / 15 (a step less in the last place if its top would pass the type's largest number) and its
 * least entry, its codes the nearest steps; a group with a NaN or an infinity reads back as NaN. */
int qrb200_kv4_write(void* cache, const qrb200_kv4_shape* shape, const void* k, int64_t k_token_stride,
                     int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
                     const int64_t* slots, int64_t tokens, void* stream);

/* The values at slots, as tokens x kv_heads x head_dim, contiguous; zeros for a negative slot. */
int qrb200_kv4_read(const void* cache, const qrb200_kv4_shape* shape, void* k, void* v, const int64_t* slots,
                    int64_t tokens, void* stream);

/* Attention of `queries` new tokens of each sequence over the cache. q: batch x queries x q_heads x
 * head_dim of the cache's type, channels contiguous, q_strides = {batch, query, head} in elements;
 * q_heads a multiple of kv_heads (head h reads key head h / (q_heads / kv_heads)). block_table:
 * batch x max_pages pages, rows table_stride apart; entries past a sequence's length, or behind
 * every query's window, are not read.
 * lengths: batch, tokens in the cache, the queries' own among them: query i stands at position
 * lengths - queries + i. It sees the tokens up to its position (to the end when causal is 0), when
 * window > 0 only from its position - window + 1 on. out: batch x queries x q_heads x head_dim,
 * contiguous; zeros where nothing is seen (values beyond 2^100 may sum past 32 bits' range before the
 * division). scale >= 0. q_heads <= 65535, queries x q_heads / kv_heads <= 2^24, batch x queries x
 * q_heads < 2^31, (max_pages + 320) x page_size < 2^31. Workspace as the query says, 256-byte aligned. */
size_t qrb200_kv4_attention_workspace_bytes(const qrb200_kv4_shape* shape, int64_t batch, int64_t queries,
                                            int64_t q_heads, int64_t max_pages, int64_t window);
int qrb200_kv4_attention(const void* q, const int64_t* q_strides, const void* cache, const qrb200_kv4_shape* shape,
                         const int32_t* block_table, int64_t table_stride, const int32_t* lengths, void* out,
                         int64_t batch, int64_t queries, int64_t q_heads, int64_t max_pages, int64_t window,
                         int causal, float scale, void* workspace, size_t workspace_bytes, void* stream);

/* 8-bit floating point (e4m3: 448 is the largest number) with a scale for each block: 128 entries of a row
 * (tile_rows 1), or 128 rows and 128 columns (tile_rows QRB200_FP8_BLOCK); the last blocks of a row or column
 * may be smaller. scale = a / 448 with a = the block's largest magnitude; code = the number nearest to
 * 448 x / a, ties to even, as if that quotient were exact (of QRB200_F32 entries as near as 64 bits tell). A
 * block with a NaN or an infinity gets codes 0 and a NaN scale; one whose a is below 2^-100 codes and
 * scale 0. x: rows x cols of dtype, q: rows x cols bytes, row strides in elements and bytes; scale:
 * ceil(rows / tile_rows) x ceil(cols / 128), contiguous. cols <= QRB200_FP8_MAX_DEPTH. */
#define QRB200_FP8_BLOCK 128
#define QRB200_FP8_MAX_DEPTH 1048576
int qrb200_quantize_fp8(const void* x, int64_t x_stride, uint8_t* q, int64_t q_stride, float* scale, int64_t rows, int64_t cols,
                        int tile_rows, int dtype, void* stream);

/* out (rows x cols of dtype, contiguous) = q * scale of its block, rounded once. */
int qrb200_dequantize_fp8(const uint8_t* q, int64_t q_stride, const float* scale, void* out, int64_t rows, int64_t cols,
                          int tile_rows, int dtype, void* stream);

/* y[i, n] = sum_b (sum_{k in block b} x[i, k] w[n, k]) x_scale[i, b] w_scale[n / 128, b] + bias[n]: x and w of e4m3, blocks of 128
 * along the depth. y: rows x outs of dtype, contiguous, 16-byte aligned; bias (may be NULL) of dtype; row strides of x and w in
 * bytes; x_scale: rows x ceil(depth / 128), w_scale: ceil(outs / 128) x ceil(depth / 128), contiguous. Sums are in 32-bit floating point, a
 * block's before its scales and theirs. Operands whose rows start on 16-byte boundaries are read as they lie; others
 * may first be laid out in the workspace (256-byte aligned, its size from the query). */
size_t qrb200_fp8_linear_workspace_bytes(const uint8_t* x, int64_t x_stride, const uint8_t* w, int64_t w_stride, int64_t rows,
                                         int64_t outs, int64_t depth);
int qrb200_fp8_linear(const uint8_t* x, int64_t x_stride, const float* x_scale, const uint8_t* w, int64_t w_stride,
                      const float* w_scale, const void* bias, void* y, int64_t rows, int64_t outs, int64_t depth, int dtype,
                      void* workspace, size_t workspace_bytes, void* stream);

/* A paged key/value cache in 8 bits: codes, pages x kv_heads blocks of qrb200_kv8_block_bytes bytes, contiguous,
 * 16-byte aligned, and range, pages x kv_heads x 2 floats (keys, values), 8-byte aligned. A code c, from -127 to 127, of a page and head stands
 * for c range / 127. dtype QRB200_BF16 or QRB200_F16, of the keys, values and queries; head_dim 64 or 128; page_size a power
 * of two from 16 to 1024. */
typedef struct qrb200_kv8_shape {
  int64_t pages;
  int32_t kv_heads, page_size, head_dim, dtype;
} qrb200_kv8_shape;
int64_t qrb200_kv8_block_bytes(int64_t page_size, int64_t head_dim);

/* Writes keys and values (tokens x kv_heads x head_dim of the cache's type, channels contiguous, other strides in
 * elements) at slots (page * page_size + offset), in any order, each at most once; a negative slot is skipped. A page's range
 * becomes the largest of what it was and of the magnitudes written, rounded up to three significant bits (unless those pass the
 * type's largest number); codes are
 * rint(127 x / range), and those of its other tokens, where the range grew, rint(c old / range). A call that writes a page's
 * first token begins it anew, the rest of it as zeros. A NaN or an infinity makes the range NaN until
 * then. Only one call at a time may write a page. Workspace as the query says, 256-byte aligned. */
size_t qrb200_kv8_write_workspace_bytes(const qrb200_kv8_shape* shape, int64_t tokens);
int qrb200_kv8_write(void* codes, float* range, const qrb200_kv8_shape* shape, const void* k, int64_t k_token_stride,
                     int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride, const int64_t* slots,
                     int64_t tokens, void* workspace, size_t workspace_bytes, void* stream);

/* The values at slots, as tokens x kv_heads x head_dim, contiguous, 16-byte aligned; zeros for a negative slot. */
int qrb200_kv8_read(const void* codes, const float* range, const qrb200_kv8_shape* shape, void* k, void* v, const int64_t* slots,
                    int64_t tokens, void* stream);

/* qrb200_kv4_attention over this cache: operands, masks and limits as there. */
size_t qrb200_kv8_attention_workspace_bytes(const qrb200_kv8_shape* shape, int64_t batch, int64_t queries, int64_t q_heads,
                                            int64_t max_pages, int64_t window);
int qrb200_kv8_attention(const void* q, const int64_t* q_strides, const void* codes, const float* range,
                         const qrb200_kv8_shape* shape, const int32_t* block_table, int64_t table_stride, const int32_t* lengths,
                         void* out, int64_t batch, int64_t queries, int64_t q_heads, int64_t max_pages, int64_t window, int causal,
                         float scale, void* workspace, size_t workspace_bytes, void* stream);

/* ---- diagnostics (no counterpart in the reference; used by bench.py) ---------------- */

/* The three 3xTF32 tcgen05 GEMMs of the 128-wide trailing update on their own, for accuracy
 * tests: for each matrix of H (batch x n x n, contiguous, 129 <= n <= 1024, n % 4 == 0),
 * V = the unit lower trapezoid of H[:, 0:128] (entries above the diagonal of that block read as
 * zero, the diagonal as one), C = H[:, 128:n]; computes C <- C - V (Tt (V^T C)) with the
 * 128 x 128 matrix Tt given (batch x 128 x 128, row-major; the two-level schedule passes the
 * block factor T transposed), through W^T = C^T V (tc_vtc128), W'^T = W^T Tt^T (tc_tw128) and
 * C -= V W' (tc_upd128). The first 128 columns of H are left as they are. Workspace as for
 * qrb200_geqrf_f32(batch, n). */
int qrb200_diag_wide_update_f32(float* H, const float* Tt, int64_t batch, int64_t n, void* workspace,
                                size_t workspace_bytes, void* stream);

/* Number of kernels this library has launched in the process so far (all threads). */
long long qrb200_launch_count(void);

/* Per-kernel-kind totals of one profiled call. */
typedef struct qrb200_kernel_stat {
  char name[32];        /* kernel kind, e.g. "panel_factor", "wy_upd"                 */
  int32_t launches;     /* launches of this kind in the call                          */
  int32_t tensor_bound; /* 1: compute (FLOP) bound contraction, 0: memory/latency     */
  double ms;            /* summed CUDA-event duration of those launches               */
  double flops;         /* algorithmic FLOPs of those launches                         */
  double bytes;         /* algorithmic HBM bytes of those launches                     */
} qrb200_kernel_stat;

/* Same computation as qrb200_geqrf_f32, with a CUDA event pair around every launch; waits
 * for the stream, then fills up to max_stats entries (one per kernel kind that ran). */
int qrb200_profile_geqrf_f32(const float* A, float* H, float* tau, int64_t batch, int64_t n,
                             int64_t a_batch_stride, void* workspace, size_t workspace_bytes,
                             void* stream, qrb200_kernel_stat* stats, int max_stats, int* n_stats);

#ifdef __cplusplus
}
#endif

#endif /* QRB200_H_ */
