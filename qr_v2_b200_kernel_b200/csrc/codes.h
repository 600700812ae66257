// Matrices of 8-bit codes on the host's side: their tensor maps, and laying them out for those.
#pragma once

#include "codes.cuh"
#include "launch.h"

namespace qrb200 {

// Boxes of 128 codes x `box_rows` rows, 128-byte swizzle; what lies outside the operand reads as zero.
static bool encode_codes(CUtensorMap* map, const I8Operand& o, uint64_t depth, uint32_t box_rows) {
  const PFN_cuTensorMapEncodeTiled_v12000 fn = map_encoder();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {depth, (cuuint64_t)o.rows};
  const cuuint64_t strides[1] = {o.rows > 1 ? (cuuint64_t)o.stride : (depth + 15) / 16 * 16};
  const cuuint32_t box[2] = {(cuuint32_t)kI8Depth, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(o.base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static I8Operand i8_operand(const int8_t* base, int64_t rows, int64_t stride) {
  return {base, rows, stride, (reinterpret_cast<uintptr_t>(base) & 15u) == 0 && (rows == 1 || stride % 16 == 0)};
}

// Operands that TMA cannot load as they lie are laid out in the workspace, x before w.
static cudaError_t lay_out(I8Operand& x, I8Operand& w, int depth, uint4* ws, cudaStream_t s) {
  if (x.aligned && w.aligned) return cudaSuccess;
  const int packs = ceil_div(depth, 16);
  uint4* to_x = x.aligned ? nullptr : ws;
  uint4* to_w = w.aligned ? nullptr : ws + (x.aligned ? 0 : x.rows * packs);
  const int64_t count = (to_x ? x.rows * packs : 0) + (to_w ? w.rows * packs : 0);
  LaunchShape l(dim3(ceil_div(count, 256)), 256, 0, s);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, i8_pad_kernel, x, to_x, w, to_w, depth, packs);
  if (e != cudaSuccess) return e;
  qrb200_internal_count_launch();
  if (to_x) x = {reinterpret_cast<const int8_t*>(to_x), x.rows, 16ll * packs, true};
  if (to_w) w = {reinterpret_cast<const int8_t*>(to_w), w.rows, 16ll * packs, true};
  return cudaSuccess;
}

// Bytes of the workspace that lay_out fills.
static size_t layout_bytes(const I8Operand& x, const I8Operand& w, int64_t depth) {
  const size_t pitch = (size_t)(depth + 15) / 16 * 16;
  return (x.aligned ? 0 : x.rows * pitch) + (w.aligned ? 0 : w.rows * pitch);
}

}  // namespace qrb200
