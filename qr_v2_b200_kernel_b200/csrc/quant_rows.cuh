// Rows into 8 bits and back: root-mean-square norm with the residual's addition, plain
// quantisation, and the values that codes stand for.
//
//   h = x + residual,  t_j = h_j w_j,  a = max_j |t_j|
//   code_j = rint(t_j (127 / a)),  scale = a (mean_j h_j^2 + eps)^(-1/2) / 127
//
// 1 / rms is common to the row, so it cancels from the codes: the sum of squares and the maximum
// are two reductions of the same pass, and the codes depend on the maximum alone, which no order
// of summation changes. Everything is held in 32 bits; h is rounded once where it is stored, and
// the norm reads it before that rounding.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace qrb200 {

// 1 / a overflows or loses range below about 2^-126; a row whose largest entry is below this
// is written as zeros.
constexpr float kTinyRow = 0x1p-100f;

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return static_cast<float>(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

struct RowsParams {
  const void* x;
  const void* residual;  // may be null
  const void* weight;    // may be null
  void* h_out;           // may be null (no residual)
  int8_t* q;
  float* scale;
  long long rows, x_stride, r_stride, q_stride;
  int cols;
  float eps;
};

// One CTA per row, any alignment: the simplest form.
template <typename T, typename W, bool kNorm>
__global__ void __launch_bounds__(256) rows_int8_kernel(RowsParams P) {
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(P.x) + row * P.x_stride;
  const T* r = P.residual ? static_cast<const T*>(P.residual) + row * P.r_stride : nullptr;
  const W* w = static_cast<const W*>(P.weight);
  T* ho = P.h_out ? static_cast<T*>(P.h_out) + row * P.cols : nullptr;
  int8_t* q = P.q + row * P.q_stride;
  __shared__ float s_sum[8];
  __shared__ unsigned s_top[8];
  float sum = 0.f;
  unsigned top = 0;  // bits of the largest |t|: ordered as unsigned, with NaN above infinity
  auto value = [&](int c, float& h) {
    h = to_f32(x[c]);
    if (r) h += to_f32(r[c]);
    return w ? h * to_f32(w[c]) : h;
  };
  for (int c = threadIdx.x; c < P.cols; c += 256) {
    float h;
    const float t = value(c, h);
    if (ho) ho[c] = from_f32<T>(h);
    sum = fmaf(h, h, sum);
    top = max(top, __float_as_uint(t) & 0x7fffffffu);
  }
  top = __reduce_max_sync(kFullMask, top);
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
  if ((threadIdx.x & 31) == 0) {
    s_sum[threadIdx.x >> 5] = sum;
    s_top[threadIdx.x >> 5] = top;
  }
  __syncthreads();
  sum = 0.f;
  top = 0;
  for (int i = 0; i < 8; ++i) {
    sum += s_sum[i];
    top = max(top, s_top[i]);
  }
  const float a = __uint_as_float(top);
  const bool finite = top < 0x7f800000u, tiny = a < kTinyRow;
  const float inv = finite && !tiny ? __fmul_rn(__frcp_rn(a), 127.f) : 0.f;
  if (threadIdx.x == 0) {
    const float rms = kNorm ? rsqrtf(sum / (float)P.cols + P.eps) : 1.f;
    P.scale[row] = !finite ? __int_as_float(0x7fffffff) : tiny ? 0.f : a * rms / 127.f;
  }
  for (int c = threadIdx.x; c < P.cols; c += 256) {
    float h;
    const float t = value(c, h);
    q[c] = finite ? (int8_t)__float2int_rn(__fmul_rn(t, inv)) : 0;
  }
}

// value = code * scale of its row, rounded once.
template <typename T>
__global__ void __launch_bounds__(256) dequant_rows_kernel(const int8_t* q, long long q_stride, const float* scale,
                                                           T* out, long long rows, int cols) {
  const long long row = blockIdx.x;
  const float s = scale[row];
  for (int c = threadIdx.x; c < cols; c += 256)
    out[row * cols + c] = from_f32<T>((float)q[row * q_stride + c] * s);
}

}  // namespace qrb200
