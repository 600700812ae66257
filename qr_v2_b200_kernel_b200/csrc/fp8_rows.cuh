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
  int step_rows, step_blocks;  // rows and blocks from a thread's block to its next
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

// What a block's entries are divided by: a / 512 and its reciprocal, to within two units in the last place (a from
// 2^-100 on, so both are normal).
struct Fp8Block {
  float div, inv;
};
__device__ __forceinline__ Fp8Block fp8_block(unsigned top) {
  Fp8Block b;
  b.div = __uint_as_float(top) * 0x1p-9f;
  asm("rcp.approx.f32 %0, %1;" : "=f"(b.inv) : "f"(b.div));
  return b;
}

// An entry for which 32 bits leave open on which side of a border between codes 448 x / a lies: the
// quotient in 64 bits, rounded to 32 with its last bit standing for all that is cut off.
static __device__ __noinline__ float fp8_next_to_border(float x, float div) {
  const double q = (double)x * 0.875 / (double)div;
  const float r = __double2float_rz(q);
  return (double)r == q ? r : __uint_as_float(__float_as_uint(r) | 1u);
}

// 448 x / a of two entries, as 32-bit numbers that round to the codes that the exact quotients do.
template <typename T>
__device__ __forceinline__ float2 fp8_quotients(float2 v, const Fp8Block& b) {
  const float2 div = make_float2(-b.div, -b.div), inv = make_float2(b.inv, b.inv);
  const float2 p = __fmul2_rn(v, make_float2(0.875f, 0.875f));
  float2 q = __fmul2_rn(p, inv);
  if constexpr (sizeof(T) == 2) {
    // p is exact, and the remainder's correction makes the quotient right to some 2^-44 before it is rounded: a
    // quotient of 16-bit numbers that lies on a border becomes that border, and no other is near enough to round to one.
    return __ffma2_rn(__ffma2_rn(q, div, p), inv, q);
  } else {
    // A border has four bits and a half: of the 20 behind them only the first is set. From 2^-11 to 2^-6
    // the codes lie 2^-9 apart, and borders elsewhere; below, there is nothing but 0.
    const auto near = [](float x) {
      const uint32_t bits = __float_as_uint(x);
      return ((bits - 0x80000u + 8) & 0xfffffu) <= 16u || (bits & 0x7fffffffu) - 0x3a000000u < 0x02800010u;
    };
    if (near(q.x)) q.x = fp8_next_to_border(v.x, b.div);
    if (near(q.y)) q.y = fp8_next_to_border(v.y, b.div);
    return q;
  }
}

// The largest magnitude of a pack, as the bits of a 32-bit float: ordered as whole numbers, NaN above infinity.
template <typename T, int kVec>
__device__ __forceinline__ unsigned fp8_top(const T (&x)[kVec]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(x);
  if constexpr (sizeof(T) == 2) {
    const uint32_t top = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
    const uint16_t most = (uint16_t)max(top & 0xffffu, top >> 16);
    return __float_as_uint(to_f32(reinterpret_cast<const T&>(most)));
  } else {
    return max(max(w[0] & 0x7fffffffu, w[1] & 0x7fffffffu), max(w[2] & 0x7fffffffu, w[3] & 0x7fffffffu));
  }
}
// a / 448, rounded once (the remainder's correction of a product with 1 / 448).
__device__ __forceinline__ float fp8_scale(unsigned top) {
  const float a = __uint_as_float(top), q = a * (1.f / 448.f);
  const float scale = fmaf(fmaf(-q, 448.f, a), 1.f / 448.f, q);
  return top >= 0x7f800000u ? __int_as_float(0x7fffffff) : a < kTinyRow ? 0.f : scale;
}
__device__ __forceinline__ bool fp8_has_codes(unsigned top) { return top < 0x7f800000u && __uint_as_float(top) >= kTinyRow; }

template <typename T, int kVec>
__device__ __forceinline__ void fp8_codes(uint32_t (&word)[kVec / 4], const T (&x)[kVec], unsigned top) {
  const Fp8Block b = fp8_block(top);
#pragma unroll
  for (int i = 0; i < kVec / 4; ++i) {
    const float2 lo = fp8_quotients<T>(make_float2(to_f32(x[4 * i]), to_f32(x[4 * i + 1])), b);
    const float2 hi = fp8_quotients<T>(make_float2(to_f32(x[4 * i + 2]), to_f32(x[4 * i + 3])), b);
    word[i] = fp8_pair(lo.x, lo.y) | fp8_pair(hi.x, hi.y) << 16;
  }
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
// blocks to a thread, all asked for before the first is used. 16384 x 4096 bf16: 40 us, 5.0 TB/s, fp32 80, 4.2. In
// bf16 instructions bound it (issue slots 75 % busy, ALU 65 %, memory 50 %).
template <typename T, bool kAligned, int kItems>
__global__ void __launch_bounds__(256) fp8_rows_kernel(Fp8RowsParams P) {
  constexpr int kVec = 16 / sizeof(T), kSpan = kFp8Block / kVec, kPer = 256 / kSpan;  // threads of a block; blocks at a time
  griddep_launch_wait();
  const int lane = threadIdx.x % kSpan;
  const long long first = (long long)blockIdx.x * (kPer * kItems) + threadIdx.x / kSpan;
  const char* lo = static_cast<const char*>(P.x);
  const Span in{lo, lo + ((P.rows - 1) * P.x_stride + P.cols) * (long long)sizeof(T)};
  alignas(16) T x[kItems][kVec];
  // A thread's block and, step_rows rows and step_blocks blocks on, its next.
  const long long row0 = first <= 0xffffffffll ? (long long)((uint32_t)first / (uint32_t)P.blocks) : first / P.blocks;
  const int block0 = (int)(first - row0 * P.blocks);
  long long row = row0;
  int block = block0;
  const auto advance = [&]() {
    row += P.step_rows, block += P.step_blocks;
    if (block >= P.blocks) block -= P.blocks, ++row;
  };
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int col = block * kFp8Block + lane * kVec;
    if (row < P.rows && col < P.cols) load_pack<kAligned>(x[i], static_cast<const T*>(P.x) + row * P.x_stride + col, P.cols - col, in);
    else
#pragma unroll
      for (int e = 0; e < kVec; ++e) x[i][e] = from_f32<T>(0.f);
    advance();
  }
  row = row0, block = block0;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int col = block * kFp8Block + lane * kVec;
    unsigned top = fp8_top(x[i]);
#pragma unroll
    for (int o = kSpan / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(kFullMask, top, o));
    if (row < P.rows && col < P.cols) {
      if (lane == 0) P.scale[first + i * kPer] = fp8_scale(top);
      uint32_t word[kVec / 4] = {};
      if (fp8_has_codes(top)) fp8_codes<T, kVec>(word, x[i], top);
      fp8_store<kAligned, T, kVec>(P.q + row * P.q_stride + col, word, P.cols - col, P.q_aligned);
    }
    advance();
  }
}

// Blocks of 128 rows and 128 columns, one to a CTA, held in registers between the maximum and the codes, three CTAs an SM. 5000 x 2040 fp32:
// 13.4 us, 3.8 TB/s, 640 CTAs in 1.4 waves (issue slots 60 % busy); 16384 x 4096 bf16 37.5, 5.4.
template <typename T, bool kAligned>
__global__ void __launch_bounds__(512, 3) fp8_tiles_kernel(Fp8RowsParams P) {
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
    top = max(top, fp8_top(x[i]));
  top = __reduce_max_sync(kFullMask, top);
  if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
  __syncthreads();
  top = __reduce_max_sync(kFullMask, s_top[threadIdx.x & 15]);
  const bool codes = fp8_has_codes(top);
  if (threadIdx.x == 0) P.scale[tile] = fp8_scale(top);
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const long long row = row0 + i * kStep;
    if (row >= P.rows || col >= P.cols) continue;
    uint32_t word[kVec / 4] = {};
    if (codes) fp8_codes<T, kVec>(word, x[i], top);
    fp8_store<kAligned, T, kVec>(P.q + row * P.q_stride + col, word, P.cols - col, P.q_aligned);
  }
}

// value = code * scale of its block, rounded once: four packs of 16 bytes of values to a thread, a CTA's width apart,
// where both sides' rows start on 16-byte boundaries (kPacked), else eight values, a warp on 256 neighbouring ones. 16384 x 4096
// to bf16 32 us, 6.3 TB/s; 8192 x 2047 to fp16 14 us, 3.6.
struct Fp8ValuesParams {
  const uint8_t* q;
  const float* scale;
  void* out;
  long long rows, q_stride;
  int cols, blocks, tile_rows;
  int units;                  // packs of a row, or its spans of 256
  int step_rows, step_units;  // from a thread's pack to its next
};
template <typename T, bool kPacked>
__global__ void __launch_bounds__(256) fp8_values_kernel(Fp8ValuesParams P) {
  griddep_launch_wait();
  const auto scale_at = [&](long long row, int c) {
    return __ldg(P.scale + (P.tile_rows == 1 ? row : row / kFp8Block) * P.blocks + c / kFp8Block);
  };
  const auto split = [&](long long at, long long& row, int& unit) {
    row = at <= 0xffffffffll ? (long long)((uint32_t)at / (uint32_t)P.units) : at / P.units;
    unit = (int)(at - row * P.units);
  };
  if constexpr (kPacked) {
    constexpr int kVec = 16 / sizeof(T), kItems = 4;
    long long row[kItems];
    int unit[kItems];
    uint32_t word[kItems][kVec / 4];
    float s[kItems];
    split((long long)blockIdx.x * (256 * kItems) + threadIdx.x, row[0], unit[0]);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (i > 0) {
        row[i] = row[i - 1] + P.step_rows, unit[i] = unit[i - 1] + P.step_units;
        if (unit[i] >= P.units) unit[i] -= P.units, ++row[i];
      }
      if (row[i] >= P.rows) continue;
      const uint8_t* q = P.q + row[i] * P.q_stride + unit[i] * kVec;
      if constexpr (kVec == 8) *reinterpret_cast<uint2*>(word[i]) = __ldg(reinterpret_cast<const uint2*>(q));
      else word[i][0] = __ldg(reinterpret_cast<const uint32_t*>(q));
      s[i] = scale_at(row[i], unit[i] * kVec);
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (row[i] >= P.rows) continue;
      alignas(16) T v[kVec];
#pragma unroll
      for (int e = 0; e < kVec; e += 2) {
        const float2 two = fp8_values(word[i][e / 4] >> (8 * (e & 2)));
        put2(&v[e], two.x * s[i], two.y * s[i]);
      }
      *reinterpret_cast<uint4*>(static_cast<T*>(P.out) + row[i] * P.cols + unit[i] * kVec) = *reinterpret_cast<const uint4*>(v);
    }
  } else {
    const int lane = threadIdx.x & 31;
    long long row;
    int unit;
    split((long long)blockIdx.x * 8 + (threadIdx.x >> 5), row, unit);
    if (row >= P.rows) return;
    const int c = unit * 256;
    const uint8_t* q = P.q + row * P.q_stride + c;
    T* out = static_cast<T*>(P.out) + row * P.cols + c;
    uint32_t code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) code[i] = c + lane + 32 * i < P.cols ? __ldg(q + lane + 32 * i) : 0;
    const float s[2] = {scale_at(row, c), c + kFp8Block < P.cols ? scale_at(row, c + kFp8Block) : 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + lane + 32 * i < P.cols) out[lane + 32 * i] = from_f32<T>(fp8_values(code[i]).x * s[i / 4]);
  }
}

}  // namespace qrb200
