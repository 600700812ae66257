// C ABI of the operators on 8-bit floating point: argument checks, choice of kernel, launches.
#include "codes.h"
#include "fp8_linear.cuh"
#include "fp8_rows.cuh"

namespace qrb200 {

static bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

template <typename T, bool kAligned>
static cudaError_t launch_quantise_of(Fp8RowsParams p, int tile_rows, cudaStream_t s) {
  constexpr int kPer = 256 / (kFp8Block * (int)sizeof(T) / 16);  // blocks that a CTA takes at a time
  if (tile_rows == 1) {
    // Four blocks to a thread where that leaves work for every SM.
    const int64_t units = p.rows * p.blocks;
    const int items = units > 4 * kPer * 8 * (int64_t)sm_count() ? 4 : 1;
    p.step_rows = kPer / p.blocks, p.step_blocks = kPer % p.blocks;
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
  constexpr int kVec = 16 / sizeof(T);
  const bool packed = cols % kVec == 0 && q_stride % 16 == 0 && !off16(q) && !off16(out);
  Fp8ValuesParams p{q, scale, out, rows, q_stride, (int)cols, ceil_div(cols, kFp8Block), tile_rows, packed ? (int)(cols / kVec) : ceil_div(cols, 256), 0, 0};
  p.step_rows = 256 / p.units, p.step_units = 256 % p.units;
  LaunchShape l(dim3(ceil_div(rows * p.units, packed ? 1024 : 8)), 256, 0, s);
  return cudaLaunchKernelEx(&l.cfg, packed ? fp8_values_kernel<T, true> : fp8_values_kernel<T, false>, p);
}

static I8Operand codes_operand(const uint8_t* base, int64_t rows, int64_t stride) {
  return i8_operand(reinterpret_cast<const int8_t*>(base), rows, stride);
}

template <typename T, int kBN>
static cudaError_t launch_fp8_few(const Fp8Params& p, const I8Operand& x, const I8Operand& w, unsigned split, cudaStream_t s) {
  using C = Fp8Few<kBN>;
  static OncePerDevice once;
  const cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(fp8_few_kernel<T, kBN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::smem());
  });
  if (e != cudaSuccess) return e;
  CUtensorMap tw, tx;
  if (!encode_codes(&tw, w, p.depth, 128) || !encode_codes(&tx, x, p.depth, kBN)) return cudaErrorInvalidValue;
  const int tn = ceil_div(p.outs, 128), tm = ceil_div(p.rows, kBN);
  if (tm > 65535) return cudaErrorInvalidValue;
  LaunchShape l(dim3(tn, tm, split), 192, C::smem(), s);
  if (split > 1) l.cluster(1, 1, split);
  return cudaLaunchKernelEx(&l.cfg, fp8_few_kernel<T, kBN>, p, tw, tx);
}

template <typename T>
static cudaError_t launch_fp8_wide(Fp8Params p, const I8Operand& x, const I8Operand& w, cudaStream_t s) {
  static OncePerDevice once;
  const cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(fp8_wide_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)fp8_wide_smem());
  });
  if (e != cudaSuccess) return e;
  CUtensorMap tw, tx;
  if (!encode_codes(&tw, w, p.depth, 128) || !encode_codes(&tx, x, p.depth, 128)) return cudaErrorInvalidValue;
  p.tiles_n = ceil_div(p.outs, 256);
  const int64_t tiles = (int64_t)p.tiles_n * ceil_div(p.rows, 256);
  if (tiles > (1 << 30)) return cudaErrorInvalidValue;
  p.tiles = (int)tiles;
  const int pairs = std::min(p.tiles, sm_count() / 2);
  LaunchShape l(dim3(2 * pairs), 128 + 32 * kFp8WideEpi, fp8_wide_smem(), s);
  return cudaLaunchKernelEx(&l.cfg, fp8_wide_kernel<T>, p, tx, tw);
}

// Which kernel, with how many rows a tile (`rows`) and over how many CTAs of the depth: the least
// of the estimated clocks. A CTA takes in its stages at about 40 bytes a clock; joining a split
// costs two cluster barriers (about 1500 clocks) and reading the sums at about 20 bytes a clock.
// The wide kernel's pair takes 512 clocks a stage and a tile's last epilogue is bare.
struct Fp8Plan {
  int rows;  // 16, 32, 64 or 128 (few), 256 (wide)
  unsigned split;
};
static Fp8Plan fp8_plan(int64_t rows, int64_t outs, int64_t nk) {
  const int64_t sms = sm_count();
  const int64_t pairs = (rows + 255) / 256 * ((outs + 255) / 256);
  Fp8Plan best{256, 1};
  int64_t least = (pairs + sms / 2 - 1) / (sms / 2) * (nk * 512 + 1500) + 3000;
  for (int bn = 16; bn <= 128; bn *= 2) {
    const int64_t tiles = (rows + bn - 1) / bn * ((outs + 127) / 128);
    if ((rows + bn - 1) / bn > 65535) continue;
    for (unsigned split = 1; split <= kFp8Split && split <= nk; split *= 2) {
      const int64_t clocks = (tiles * split + sms - 1) / sms *
                             ((nk + split - 1) / split * (128 + bn) * 128 / 40 + (split > 1 ? 1500 + bn * 24 : bn * 8));
      if (clocks < least) {
        least = clocks;
        best = Fp8Plan{bn, split};
      }
    }
    if (rows <= bn) break;
  }
  return best;
}

template <typename T>
static cudaError_t launch_fp8_rows(const Fp8Params& p, const I8Operand& x, const I8Operand& w, cudaStream_t s) {
  const Fp8RowsOperands r{p, x, w};
  LaunchShape l(dim3(ceil_div(p.outs, 16)), 32 * kFp8RowsWarps, 0, s);
  return cudaLaunchKernelEx(&l.cfg, x.aligned && w.aligned ? fp8_rows_linear_kernel<T, true> : fp8_rows_linear_kernel<T, false>, r);
}

// (4096 x 4096: up to eight rows 4.3-4.7 us, nine to sixteen through tcgen05 6.3-6.5.)
constexpr int kFp8Rows = 8;

template <typename T>
static cudaError_t launch_fp8(const Fp8Params& p, I8Operand x, I8Operand w, uint4* ws, cudaStream_t s) {
  if (p.rows <= kFp8Rows) return launch_fp8_rows<T>(p, x, w, s);
  const cudaError_t e = lay_out(x, w, p.depth, ws, s);
  if (e != cudaSuccess) return e;
  const Fp8Plan plan = fp8_plan(p.rows, p.outs, p.blocks);
  switch (plan.rows) {
    case 16: return launch_fp8_few<T, 16>(p, x, w, plan.split, s);
    case 32: return launch_fp8_few<T, 32>(p, x, w, plan.split, s);
    case 64: return launch_fp8_few<T, 64>(p, x, w, plan.split, s);
    case 128: return launch_fp8_few<T, 128>(p, x, w, plan.split, s);
    default: return launch_fp8_wide<T>(p, x, w, s);
  }
}

}  // namespace qrb200

using namespace qrb200;

int qrb200_internal_fp8_site() { return take_site(); }
bool qrb200_internal_fp8_register(int* word) { return register_word(word); }

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
  const Fp8RowsParams p{x, q, scale, rows, x_stride, q_stride, (int)cols, blocks, 0, 0, 0};
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
  if (rows <= 0 || outs <= 0 || depth <= 0 || depth > QRB200_FP8_MAX_DEPTH) return 0;
  const I8Operand xo = codes_operand(x, rows, x_stride), wo = codes_operand(w, outs, w_stride);
  return rows <= kFp8Rows ? 0 : layout_bytes(xo, wo, depth);
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
  const Fp8Params p{x_scale, w_scale, bias, y, (int)rows, (int)outs, (int)depth, ceil_div(depth, kFp8Block), 0, 0};
  const I8Operand xo = codes_operand(x, rows, x_stride), wo = codes_operand(w, outs, w_stride);
  uint4* ws = static_cast<uint4*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == QRB200_BF16  ? launch_fp8<__nv_bfloat16>(p, xo, wo, ws, s)
                        : dtype == QRB200_F16 ? launch_fp8<__half>(p, xo, wo, ws, s)
                                              : launch_fp8<float>(p, xo, wo, ws, s);
  if (e != cudaSuccess) return QRB200_ERR_CUDA;
  return launched();
}

}  // extern "C"
