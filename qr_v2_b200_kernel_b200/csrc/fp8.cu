// C ABI of the operators on 8-bit floating point: argument checks, choice of kernel, launches.
#include "launch.h"
#include "fp8_linear.cuh"
#include "fp8_rows.cuh"

namespace qrb200 {

static bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

template <typename T, bool kAligned>
static cudaError_t launch_quantise_of(const Fp8RowsParams& p, int tile_rows, cudaStream_t s) {
  constexpr int kPer = 256 / (kFp8Block * (int)sizeof(T) / 16);  // blocks that a CTA takes at a time
  if (tile_rows == 1) {
    // Four blocks to a thread where that leaves work for every SM.
    const int64_t units = p.rows * p.blocks;
    const int items = units > 4 * kPer * 8 * (int64_t)sm_count() ? 4 : 1;
    LaunchShape l(dim3(ceil_div(units, kPer * items)), 256, 0, s);
    return items == 4 ? cudaLaunchKernelEx(&l.cfg, fp8_rows_kernel<T, kAligned, 4>, p)
                      : cudaLaunchKernelEx(&l.cfg, fp8_rows_kernel<T, kAligned, 1>, p);
  }
  LaunchShape l(dim3(ceil_div(p.rows, kFp8Block) * p.blocks), 512, 0, s);
  return cudaLaunchKernelEx(&l.cfg, fp8_tiles_kernel<T, kAligned>, p);
}

template <typename T>
static cudaError_t launch_quantise(Fp8RowsParams p, int tile_rows, cudaStream_t s) {
  constexpr int kVec = 16 / sizeof(T);
  p.q_aligned = !off16(p.q) && p.q_stride % 16 == 0;
  const bool aligned = p.cols % kVec == 0 && !off16(p.x) && p.x_stride % kVec == 0 && p.q_aligned;
  return aligned ? launch_quantise_of<T, true>(p, tile_rows, s) : launch_quantise_of<T, false>(p, tile_rows, s);
}

template <typename T>
static cudaError_t launch_values(const uint8_t* q, int64_t q_stride, const float* scale, void* out, int64_t rows, int64_t cols,
                                 int tile_rows, cudaStream_t s) {
  const bool packed = cols * sizeof(T) % 16 == 0 && q_stride % 16 == 0 && !off16(q) && !off16(out);
  const int64_t units = rows * (packed ? ceil_div(cols, 16) : cols);
  LaunchShape l(dim3(ceil_div(units, 256)), 256, 0, s);
  return cudaLaunchKernelEx(&l.cfg, packed ? fp8_values_kernel<T, true> : fp8_values_kernel<T, false>, q, (long long)q_stride, scale,
                            static_cast<T*>(out), (long long)rows, (int)cols, tile_rows);
}

template <typename T>
static cudaError_t launch_fp8(const Fp8Params& p, const Fp8Operand& x, const Fp8Operand& w, cudaStream_t s) {
  LaunchShape l(dim3(ceil_div(p.outs, 32), ceil_div(p.rows, 32)), 256, 0, s);
  return cudaLaunchKernelEx(&l.cfg, fp8_simple_kernel<T>, p, x, w);
}

static Fp8Operand fp8_operand(const uint8_t* base, int64_t rows, int64_t stride) {
  return {base, rows, stride, !off16(base) && (rows == 1 || stride % 16 == 0)};
}

}  // namespace qrb200

using namespace qrb200;

int qrb200_internal_fp8_site() { return take_site(); }

extern "C" {

int qrb200_quantize_fp8(const void* x, int64_t x_stride, uint8_t* q, int64_t q_stride, float* scale, int64_t rows, int64_t cols,
                        int tile_rows, int dtype, void* stream) {
  if (rows < 0 || cols < 0 || rows > kMaxRows || cols > QRB200_FP8_MAX_DEPTH || !type_ok(dtype)) return QRB200_ERR_ARG;
  if (tile_rows != 1 && tile_rows != QRB200_FP8_BLOCK) return QRB200_ERR_ARG;
  if (rows == 0 || cols == 0) return QRB200_OK;
  if (!x || !q || !scale || (rows > 1 && (x_stride < cols || q_stride < cols))) return QRB200_ERR_ARG;
  const int blocks = ceil_div(cols, kFp8Block);
  if (rows > ((int64_t)1 << 33) / blocks) return QRB200_ERR_ARG;
  const int st = quant_ready();
  if (st != QRB200_OK) return st;
  const Fp8RowsParams p{x, q, scale, rows, x_stride, q_stride, (int)cols, blocks, 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == QRB200_BF16  ? launch_quantise<__nv_bfloat16>(p, tile_rows, s)
                        : dtype == QRB200_F16 ? launch_quantise<__half>(p, tile_rows, s)
                                              : launch_quantise<float>(p, tile_rows, s);
  if (e != cudaSuccess) return QRB200_ERR_CUDA;
  return launched();
}

int qrb200_dequantize_fp8(const uint8_t* q, int64_t q_stride, const float* scale, void* out, int64_t rows, int64_t cols,
                          int tile_rows, int dtype, void* stream) {
  if (rows < 0 || cols < 0 || rows > kMaxRows || cols > QRB200_FP8_MAX_DEPTH || !type_ok(dtype)) return QRB200_ERR_ARG;
  if (tile_rows != 1 && tile_rows != QRB200_FP8_BLOCK) return QRB200_ERR_ARG;
  if (rows == 0 || cols == 0) return QRB200_OK;
  if (!q || !scale || !out || (rows > 1 && q_stride < cols)) return QRB200_ERR_ARG;
  if (rows > ((int64_t)1 << 38) / cols) return QRB200_ERR_ARG;
  const int st = quant_ready();
  if (st != QRB200_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == QRB200_BF16  ? launch_values<__nv_bfloat16>(q, q_stride, scale, out, rows, cols, tile_rows, s)
                        : dtype == QRB200_F16 ? launch_values<__half>(q, q_stride, scale, out, rows, cols, tile_rows, s)
                                              : launch_values<float>(q, q_stride, scale, out, rows, cols, tile_rows, s);
  if (e != cudaSuccess) return QRB200_ERR_CUDA;
  return launched();
}

size_t qrb200_fp8_linear_workspace_bytes(const uint8_t* x, int64_t x_stride, const uint8_t* w, int64_t w_stride, int64_t rows,
                                         int64_t outs, int64_t depth) {
  (void)x, (void)x_stride, (void)w, (void)w_stride, (void)rows, (void)outs, (void)depth;
  return 0;
}

int qrb200_fp8_linear(const uint8_t* x, int64_t x_stride, const float* x_scale, const uint8_t* w, int64_t w_stride,
                      const float* w_scale, const void* bias, void* y, int64_t rows, int64_t outs, int64_t depth, int dtype,
                      void* workspace, size_t workspace_bytes, void* stream) {
  if (rows < 0 || outs < 0 || depth <= 0 || depth > QRB200_FP8_MAX_DEPTH || !type_ok(dtype)) return QRB200_ERR_ARG;
  if (rows > kMaxRows / 2 || outs > kMaxRows / 2) return QRB200_ERR_ARG;
  if (rows == 0 || outs == 0) return QRB200_OK;
  if (!x || !w || !x_scale || !w_scale || !y || off16(y)) return QRB200_ERR_ARG;
  if ((rows > 1 && x_stride < depth) || (outs > 1 && w_stride < depth)) return QRB200_ERR_ARG;
  const int st = quant_ready();
  if (st != QRB200_OK) return st;
  const size_t need = qrb200_fp8_linear_workspace_bytes(x, x_stride, w, w_stride, rows, outs, depth);
  if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u)))
    return QRB200_ERR_WORKSPACE;
  const Fp8Params p{x_scale, w_scale, bias, y, (int)rows, (int)outs, (int)depth, ceil_div(depth, kFp8Block)};
  const Fp8Operand xo = fp8_operand(x, rows, x_stride), wo = fp8_operand(w, outs, w_stride);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == QRB200_BF16  ? launch_fp8<__nv_bfloat16>(p, xo, wo, s)
                        : dtype == QRB200_F16 ? launch_fp8<__half>(p, xo, wo, s)
                                              : launch_fp8<float>(p, xo, wo, s);
  if (e != cudaSuccess) return QRB200_ERR_CUDA;
  return launched();
}

}  // extern "C"
