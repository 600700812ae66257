// y[i, n] = sum_b sx[i, b] sw[n / 128, b] sum_{k in block b} x[i, k] w[n, k] + bias[n] with x and w in
// 8-bit floating point (e4m3), blocks of 128 along the depth.
#pragma once

#include "fp8_rows.cuh"

namespace qrb200 {

struct Fp8Operand {
  const uint8_t* base;
  long long rows, stride;  // bytes
  bool aligned;            // base and stride are multiples of 16
};

struct Fp8Params {
  const float* sx;
  const float* sw;
  const void* bias;  // may be null; y's type
  void* y;
  int rows, outs, depth, blocks;  // blocks of the depth
};

// 32 rows x 32 channels to a CTA, the blocks of the depth one after another.
template <typename T>
__global__ void __launch_bounds__(256) fp8_simple_kernel(Fp8Params P, Fp8Operand x, Fp8Operand w) {
  __shared__ float s_x[32][kFp8Block + 1], s_w[32][kFp8Block + 1];
  griddep_launch_wait();
  const int n0 = blockIdx.x * 32, i0 = blockIdx.y * 32, tn = threadIdx.x & 31, ti = threadIdx.x >> 5;
  float acc[4] = {};
  for (int b = 0; b < P.blocks; ++b) {
    __syncthreads();
    for (int e = threadIdx.x; e < 32 * kFp8Block; e += 256) {
      const int r = e / kFp8Block, c = e % kFp8Block, k = b * kFp8Block + c;
      s_x[r][c] = i0 + r < P.rows && k < P.depth ? fp8_values(x.base[(i0 + r) * x.stride + k]).x : 0.f;
      s_w[r][c] = n0 + r < P.outs && k < P.depth ? fp8_values(w.base[(n0 + r) * w.stride + k]).x : 0.f;
    }
    __syncthreads();
    const float sw = n0 + tn < P.outs ? P.sw[(long long)((n0 + tn) / kFp8Block) * P.blocks + b] : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = ti + 8 * j;
      float part = 0.f;
      for (int c = 0; c < kFp8Block; ++c) part = fmaf(s_x[r][c], s_w[tn][c], part);
      if (i0 + r < P.rows) acc[j] = fmaf(part, P.sx[(long long)(i0 + r) * P.blocks + b] * sw, acc[j]);
    }
  }
  if (n0 + tn >= P.outs) return;
  const float bias = P.bias ? to_f32(static_cast<const T*>(P.bias)[n0 + tn]) : 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = i0 + ti + 8 * j;
    if (i < P.rows) static_cast<T*>(P.y)[(long long)i * P.outs + n0 + tn] = from_f32<T>(acc[j] + bias);
  }
}

}  // namespace qrb200
