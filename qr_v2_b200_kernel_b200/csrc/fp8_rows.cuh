// Blocks of 128 entries of a row (or of 128 rows and 128 columns) into 8-bit floating point (e4m3: a
// sign, four bits of exponent, three of mantissa) with a scale each, and back:
//
//   a = max |x| over the block,  scale = a / 448,  code = e4m3(448 x / a)
//
// 448 is the largest code. The quotient is rounded to a code as if it were exact: entries of 16 bits
// often lie midway between two codes, and a factor 448 / a rounded to 32 bits would send those either
// way.
#pragma once

#include "quant_rows.cuh"

namespace qrb200 {

constexpr int kFp8Block = 128;

struct Fp8RowsParams {
  const void* x;
  uint8_t* q;
  float* scale;  // rows of blocks x blocks, contiguous
  long long rows, x_stride, q_stride;
  int cols, blocks;  // of a row
  int q_aligned;     // rows of q start on 16-byte boundaries
};

__device__ __forceinline__ uint32_t fp8_pair(float a, float b) {  // a in the low byte
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ float2 fp8_values(uint32_t two) {  // of the low and the high byte of 16 bits
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
  return __half22float2(reinterpret_cast<const __half2&>(h));
}

// What a block's entries are divided by: a / 512 and its reciprocal (a from 2^-100 on, so both are normal).
struct Fp8Block {
  float div, inv;
};

// An entry for which 32 bits leave open on which side of a border between codes 448 x / a lies: the
// quotient in 64 bits, rounded to 32 with its last bit standing for all that is cut off.
static __device__ __noinline__ float fp8_next_to_border(float x, float div) {
  const double q = (double)x * 0.875 / (double)div;
  const float r = __double2float_rz(q);
  return (double)r == q ? r : __uint_as_float(__float_as_uint(r) | 1u);
}

// 448 x / a, as a 32-bit number that rounds to the code that the exact quotient does.
template <typename T>
__device__ __forceinline__ float fp8_quotient(T x, const Fp8Block& b) {
  const float v = to_f32(x), p = v * 0.875f;
  const float q = p * b.inv;
  if constexpr (sizeof(T) == 2) {
    // p is exact, and the remainder's correction makes the quotient the nearest of 32 bits: a border is
    // one of those, and no other quotient of 16-bit numbers is near enough to round to one.
    return fmaf(fmaf(-q, b.div, p), b.inv, q);
  } else {
    // A border has four bits and a half: of the 20 behind them only the first is set. From 2^-11 to 2^-6
    // the codes lie 2^-9 apart, and borders elsewhere; below, there is nothing but 0.
    const uint32_t bits = __float_as_uint(q);
    const bool near = ((bits - 0x80000u + 8) & 0xfffffu) <= 16u || (bits & 0x7fffffffu) - 0x3a000000u < 0x02800010u;
    return near ? fp8_next_to_border(v, b.div) : q;
  }
}

// A block's largest magnitude (as bits: NaN above infinity) to its scale; whether it has codes at all.
__device__ __forceinline__ bool fp8_scale(unsigned top, float* scale) {
  const float a = __uint_as_float(top);
  if (top >= 0x7f800000u) *scale = __int_as_float(0x7fffffff);
  else *scale = a < kTinyRow ? 0.f : a / 448.f;
  return top < 0x7f800000u && a >= kTinyRow;
}

template <typename T, int kVec>
__device__ __forceinline__ void fp8_codes(uint32_t (&word)[kVec / 4], const T (&x)[kVec], unsigned top) {
  const float div = __uint_as_float(top) * 0x1p-9f;
  const Fp8Block b{div, __frcp_rn(div)};
#pragma unroll
  for (int i = 0; i < kVec / 4; ++i)
    word[i] = fp8_pair(fp8_quotient(x[4 * i], b), fp8_quotient(x[4 * i + 1], b)) |
              fp8_pair(fp8_quotient(x[4 * i + 2], b), fp8_quotient(x[4 * i + 3], b)) << 16;
}

template <bool kAligned, typename T, int kVec>
__device__ __forceinline__ void fp8_store(uint8_t* q, const uint32_t (&word)[kVec / 4], int left, bool q_aligned) {
  if (kAligned || (q_aligned && left >= kVec)) {
    if constexpr (kVec == 8) *reinterpret_cast<uint2*>(q) = make_uint2(word[0], word[1]);
    else *reinterpret_cast<uint32_t*>(q) = word[0];
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (i < left) q[i] = (uint8_t)(word[i / 4] >> (8 * (i & 3)));
  }
}

// Blocks of a row: a pack (16 bytes) to a thread, so 16 (32-bit entries: 32) threads to a block, kItems
// blocks to a thread, all asked for before the first is used.
template <typename T, bool kAligned, int kItems>
__global__ void __launch_bounds__(256) fp8_rows_kernel(Fp8RowsParams P) {
  constexpr int kVec = 16 / sizeof(T), kSpan = kFp8Block / kVec, kPer = 256 / kSpan;  // threads of a block; blocks at a time
  griddep_launch_wait();
  const int lane = threadIdx.x % kSpan;
  const long long total = P.rows * P.blocks, first = (long long)blockIdx.x * (kPer * kItems) + threadIdx.x / kSpan;
  const char* lo = static_cast<const char*>(P.x);
  const Span in{lo, lo + ((P.rows - 1) * P.x_stride + P.cols) * (long long)sizeof(T)};
  alignas(16) T x[kItems][kVec];
  const auto place = [&](int i, long long& row, int& col) {
    const long long at = first + i * kPer;
    row = total <= 0xffffffffll ? (long long)((uint32_t)at / (uint32_t)P.blocks) : at / P.blocks;
    col = (int)(at - row * P.blocks) * kFp8Block + lane * kVec;
    return at < total && col < P.cols;
  };
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    long long row;
    int col;
    const bool mine = place(i, row, col);
    if (mine) load_pack<kAligned>(x[i], static_cast<const T*>(P.x) + row * P.x_stride + col, P.cols - col, in);
    else
#pragma unroll
      for (int e = 0; e < kVec; ++e) x[i][e] = from_f32<T>(0.f);
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    long long row;
    int col;
    const bool mine = place(i, row, col);
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < kVec; ++e) top = max(top, __float_as_uint(to_f32(x[i][e])) & 0x7fffffffu);
#pragma unroll
    for (int o = kSpan / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(kFullMask, top, o));
    float scale;
    const bool codes = fp8_scale(top, &scale);
    if (!mine) continue;
    if (lane == 0) P.scale[first + i * kPer] = scale;
    uint32_t word[kVec / 4] = {};
    if (codes) fp8_codes<T, kVec>(word, x[i], top);
    fp8_store<kAligned, T, kVec>(P.q + row * P.q_stride + col, word, P.cols - col, P.q_aligned);
  }
}

// Blocks of 128 rows and 128 columns, one to a CTA, held in registers between the maximum and the codes.
template <typename T, bool kAligned>
__global__ void __launch_bounds__(512) fp8_tiles_kernel(Fp8RowsParams P) {
  constexpr int kVec = 16 / sizeof(T), kSpan = kFp8Block / kVec, kStep = 512 / kSpan, kItems = kFp8Block / kStep;
  __shared__ unsigned s_top[16];
  griddep_launch_wait();
  const long long tile = blockIdx.x, tile_row = tile / P.blocks;
  const int col = (int)(tile % P.blocks) * kFp8Block + threadIdx.x % kSpan * kVec;
  const long long row0 = tile_row * kFp8Block + threadIdx.x / kSpan;
  const char* lo = static_cast<const char*>(P.x);
  const Span in{lo, lo + ((P.rows - 1) * P.x_stride + P.cols) * (long long)sizeof(T)};
  alignas(16) T x[kItems][kVec];
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const long long row = row0 + i * kStep;
    if (row < P.rows && col < P.cols) load_pack<kAligned>(x[i], static_cast<const T*>(P.x) + row * P.x_stride + col, P.cols - col, in);
    else
#pragma unroll
      for (int e = 0; e < kVec; ++e) x[i][e] = from_f32<T>(0.f);
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i)
#pragma unroll
    for (int e = 0; e < kVec; ++e) top = max(top, __float_as_uint(to_f32(x[i][e])) & 0x7fffffffu);
  top = __reduce_max_sync(kFullMask, top);
  if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
  __syncthreads();
  top = __reduce_max_sync(kFullMask, s_top[threadIdx.x & 15]);
  float scale;
  const bool codes = fp8_scale(top, &scale);
  if (threadIdx.x == 0) P.scale[tile] = scale;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const long long row = row0 + i * kStep;
    if (row >= P.rows || col >= P.cols) continue;
    uint32_t word[kVec / 4] = {};
    if (codes) fp8_codes<T, kVec>(word, x[i], top);
    fp8_store<kAligned, T, kVec>(P.q + row * P.q_stride + col, word, P.cols - col, P.q_aligned);
  }
}

// value = code * scale of its block, rounded once: sixteen codes to a thread where both sides' rows start on
// 16-byte boundaries (kPacked), else one, a warp's side by side.
template <typename T, bool kPacked>
__global__ void __launch_bounds__(256) fp8_values_kernel(const uint8_t* q, long long q_stride, const float* scale, T* out,
                                                         long long rows, int cols, int tile_rows) {
  constexpr int kSpan = kPacked ? 16 : 1;
  griddep_launch_wait();
  const int spans = (cols + kSpan - 1) / kSpan, blocks = (cols + kFp8Block - 1) / kFp8Block;
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = at <= 0xffffffffll ? (long long)((uint32_t)at / (uint32_t)spans) : at / spans;
  if (row >= rows) return;
  const int c = (int)(at - row * spans) * kSpan;
  const float s = scale[(tile_rows == 1 ? row : row / kFp8Block) * blocks + c / kFp8Block];
  q += row * q_stride + c;
  out += row * cols + c;
  if constexpr (kPacked) {
    const int n = cols - c;  // a multiple of a pack of the values
    uint32_t word[4] = {};
    if (n >= 16) *reinterpret_cast<uint4*>(word) = __ldg(reinterpret_cast<const uint4*>(q));
    else
#pragma unroll
      for (int e = 0; e < 16; ++e) word[e / 4] |= e < n ? (uint32_t)q[e] << (8 * (e & 3)) : 0u;
    constexpr int kPart = 16 / sizeof(T);
#pragma unroll
    for (int h = 0; h < 16; h += kPart) {
      alignas(16) T v[kPart];
#pragma unroll
      for (int e = 0; e < kPart; e += 2) {
        const float2 two = fp8_values(word[(h + e) / 4] >> (8 * ((h + e) & 2)));
        put2(&v[e], two.x * s, two.y * s);
      }
      if (h < n) store_pack<true>(out + h, v, kPart);
    }
  } else {
    *out = from_f32<T>(fp8_values(*q).x * s);
  }
}

}  // namespace qrb200
