// y[i, n] = (sum_k x[i, k] w[n, k]) sx[i] sw[n] + bias[n] with 8-bit x and w.
//
// The sum is held in 32-bit integers, so it is exact (depth <= 131071 keeps 128^2 depth below
// 2^31) and any split of the depth gives the same bits; the scales are applied in 32 bits and
// the result is rounded once.
#pragma once

#include "quant_rows.cuh"

namespace qrb200 {

struct I8Params {
  const int8_t* x;
  const int8_t* w;
  const float* sx;
  const float* sw;
  const void* bias;  // may be null; y's type
  void* y;
  long long rows, outs, x_stride, w_stride;
  int depth;
};

// 64 x 64 outputs per CTA, 16 threads a side with 4 x 4 outputs each; any alignment.
template <typename T>
__global__ void __launch_bounds__(256) i8_linear_simple_kernel(I8Params P) {
  __shared__ __align__(4) int8_t xs[64][68], ws[64][68];
  const long long i0 = (long long)blockIdx.y * 64, n0 = (long long)blockIdx.x * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < P.depth; k0 += 64) {
    for (int e = threadIdx.x; e < 64 * 64; e += 256) {
      const int r = e >> 6, c = e & 63;
      const bool k = k0 + c < P.depth;
      xs[r][c] = k && i0 + r < P.rows ? P.x[(i0 + r) * P.x_stride + k0 + c] : 0;
      ws[r][c] = k && n0 + r < P.outs ? P.w[(n0 + r) * P.w_stride + k0 + c] : 0;
    }
    __syncthreads();
    for (int c = 0; c < 64; c += 4)
      for (int a = 0; a < 4; ++a)
        for (int b = 0; b < 4; ++b)
          acc[a][b] = __dp4a(*reinterpret_cast<const int*>(&xs[4 * ty + a][c]),
                             *reinterpret_cast<const int*>(&ws[tx + 16 * b][c]), acc[a][b]);
    __syncthreads();
  }
  for (int a = 0; a < 4; ++a)
    for (int b = 0; b < 4; ++b) {
      const long long i = i0 + 4 * ty + a, n = n0 + tx + 16 * b;
      if (i >= P.rows || n >= P.outs) continue;
      float v = (float)acc[a][b] * P.sx[i] * P.sw[n];
      if (P.bias) v += to_f32(static_cast<const T*>(P.bias)[n]);
      static_cast<T*>(P.y)[i * P.outs + n] = from_f32<T>(v);
    }
}

}  // namespace qrb200
