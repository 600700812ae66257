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

// Two neighbouring results, rounded by one instruction where T has 16 bits.
__device__ __forceinline__ void put2(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
__device__ __forceinline__ void put2(__nv_bfloat16* p, float a, float b) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b);
}
__device__ __forceinline__ void put2(__half* p, float a, float b) { *reinterpret_cast<__half2*>(p) = __floats2half2_rn(a, b); }

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
  int q_aligned;  // rows of q start on 16-byte boundaries
};

// A pack is 16 bytes of consecutive elements. Where all rows start on 16-byte boundaries and hold
// whole packs (kAligned) it is one load or store. Elsewhere a load takes the two aligned blocks
// around it and shifts, if both lie within the operand ([lo, hi)), else it goes element by element;
// elements from n on read as zero. A store goes by aligned pairs.
struct Span {
  const char* lo;
  const char* hi;
};
template <bool kAligned, typename T, int kVec>
__device__ __forceinline__ void load_pack(T (&v)[kVec], const T* p, int n, Span in) {
  static_assert(kVec * sizeof(T) == 16, "a pack");
  if constexpr (kAligned) {
    *reinterpret_cast<uint4*>(v) = __ldg(reinterpret_cast<const uint4*>(p));
  } else {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const uint4* block = reinterpret_cast<const uint4*>(at & ~(uintptr_t)15);
    const int off = (int)(at & 15);
    if (reinterpret_cast<const char*>(block) >= in.lo && reinterpret_cast<const char*>(block + (off ? 2 : 1)) <= in.hi) {
      uint32_t w[8] = {};
      *reinterpret_cast<uint4*>(w) = __ldg(block);
      if (off) *reinterpret_cast<uint4*>(w + 4) = __ldg(block + 1);
      if (off & 8) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
      }
      if (off & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(v)[i] = __funnelshift_r(w[i], w[i + 1], 8 * (off & 3));
      if (n < kVec) {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          if (i >= n) v[i] = from_f32<T>(0.f);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) v[i] = i < n ? __ldg(p + i) : from_f32<T>(0.f);
    }
  }
}
template <bool kAligned, typename T, int kVec>
__device__ __forceinline__ void store_pack(T* p, const T (&v)[kVec], int n) {
  if constexpr (kAligned) {
    static_assert(kVec * sizeof(T) == 16, "a pack");
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
  } else {
    if constexpr (sizeof(T) == 2) {
      if (n >= kVec) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
        if (reinterpret_cast<uintptr_t>(p) & 2) {  // the first and the last element stand alone
          p[0] = v[0];
#pragma unroll
          for (int i = 0; i + 1 < kVec / 2; ++i) *reinterpret_cast<uint32_t*>(p + 2 * i + 1) = __funnelshift_r(w[i], w[i + 1], 16);
          p[kVec - 1] = v[kVec - 1];
        } else {
#pragma unroll
          for (int i = 0; i < kVec / 2; ++i) *reinterpret_cast<uint32_t*>(p + 2 * i) = w[i];
        }
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (i < n) p[i] = v[i];
  }
}

// A row of finite numbers whose squares' sum left 32 bits' range, or whose h w did (top: infinity):
// the same formulas on h 2^-k, with 2^k above both the largest |h| and sqrt(eps), which the scale
// takes back. Out of line, from memory and element by element: the hot path keeps a branch to the end that
// ordinary rows never take. All threads of the row come here; each takes what it holds there.
// h_out (null: h is x, or stored already) is written last, as it may be the residual.
template <typename T, typename W>
__device__ __noinline__ void rows_outside(const T* x, const T* residual, T* h_out, const W* w, int8_t* q, float* scale, int cols,
                                          float eps, bool over) {
  constexpr int kVec = 16 / sizeof(T);
  __shared__ float s_sum[32];
  __shared__ unsigned s_top[32];
  const int tid = threadIdx.x, threads = blockDim.x;
  const auto each = [&](auto f) {
#pragma unroll 1
    for (int c = tid * kVec; c < cols; c += threads * kVec)
#pragma unroll 1
      for (int j = c; j < min(c + kVec, cols); ++j) f(j, residual ? to_f32(x[j]) + to_f32(residual[j]) : to_f32(x[j]));
  };
  float sum = 0.f;
  unsigned top = 0;
  const auto join = [&]() {
    top = __reduce_max_sync(kFullMask, top);
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
    if (threads == 32) return;
    __syncthreads();  // what was joined before has been read
    if ((tid & 31) == 0) {
      s_sum[tid >> 5] = sum;
      s_top[tid >> 5] = top;
    }
    __syncthreads();
    const bool mine = (tid & 31) < threads >> 5;
    sum = mine ? s_sum[tid & 31] : 0.f;
    top = __reduce_max_sync(kFullMask, mine ? s_top[tid & 31] : 0u);
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
  };
  each([&](int, float h) { top = max(top, __float_as_uint(h) & 0x7fffffffu); });
  join();
  bool finite = top < 0x7f800000u;
  // 2^-k in two factors that are both normal numbers.
  const int k = max(1, (int)(__float_as_uint(fmaxf(__uint_as_float(top), sqrtf(eps))) >> 23)) - 126;
  const float down = __int_as_float((127 - (k >> 1)) << 23), rest = __int_as_float((127 - (k - (k >> 1))) << 23);
  top = 0;
  each([&](int j, float h) {
    const float v = h * down * rest, t = w ? (over ? v : h) * to_f32(w[j]) : over ? v : h;
    sum = fmaf(v, v, sum);
    top = max(top, __float_as_uint(t) & 0x7fffffffu);
  });
  join();
  finite = finite && top < 0x7f800000u;
  const float a = __uint_as_float(top), inv = finite ? __fmul_rn(__frcp_rn(a), 127.f) : 0.f;
  if (tid == 0) {
    const float rms = rsqrtf(sum / (float)cols + eps * down * down * rest * rest) / 127.f;
    *scale = finite ? (over ? a * rms : a * down * rms * rest) : __int_as_float(0x7fffffff);
  }
  each([&](int j, float h) {
    const float t = (over ? h * down * rest : h) * (w ? to_f32(w[j]) : 1.f);
    q[j] = finite ? (int8_t)__float2int_rn(__fmul_rn(t, inv)) : (int8_t)0;
    if (h_out) h_out[j] = from_f32<T>(h);
  });
}

// A row lives in the registers of blockDim.x threads, kItems packs each, a block's y rows beside
// one another: memory is read once and written once, and bounds it. (16384 x 4096 bf16: 71 us, 6.6
// TB/s; rows off 16-byte boundaries cost twice that, 16384 x 2047 77 us with gain and residual;
// storing those through shared memory, element beside element, lost.) Every load of the row is asked for before
// the first is used. Which thread holds which element depends on the row's length alone, so a row's
// result, bit for bit, depends on neither its neighbours, their number nor anybody's alignment.
// (Short rows, one pack a thread, go two blocks' worth of threads to an SM: 16384 x 64 5.3 us for 5.7.)
template <typename T, typename W, bool kNorm, bool kAligned, int kItems>
__global__ void __launch_bounds__(1024, kItems == 1 ? 2 : 1) rows_int8_kernel(RowsParams P) {
  constexpr int kVec = 16 / sizeof(T);
  // h_out may be the residual, so h is stored once nobody needs that any more (which is also faster:
  // 71.4 us for 77.5), in 32 bits, where what is stored is h, and off 16-byte boundaries (77 us for 85) at once.
  constexpr bool kLate = sizeof(T) == 2 && kAligned;
  __shared__ float s_sum[32];
  __shared__ unsigned s_top[32];
  griddep_launch_wait();
  const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const bool in = row < P.rows;
  const int packs = (P.cols + kVec - 1) / kVec, tid = threadIdx.x, threads = blockDim.x;
  const T* x = static_cast<const T*>(P.x) + row * P.x_stride;
  const T* r = static_cast<const T*>(P.residual) + row * P.r_stride;
  const W* w = static_cast<const W*>(P.weight);
  T* h_out = static_cast<T*>(P.h_out) + row * P.cols;
  // The operands' extents, for loads off 16-byte boundaries.
  const auto extent = [&](const void* base, long long stride) {
    const char* lo = static_cast<const char*>(base);
    return Span{lo, lo + ((P.rows - 1) * stride + P.cols) * (long long)sizeof(T)};
  };
  const Span xs = extent(P.x, P.x_stride), rs = extent(P.residual, P.r_stride);
  const Span ws{static_cast<const char*>(P.weight), static_cast<const char*>(P.weight) + P.cols * sizeof(W)};
  alignas(16) T xv[kItems][kVec], rv[kItems][kVec];
  float t[kItems][kVec];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int c = tid + i * threads;
    if (!in || c >= packs) continue;
    load_pack<kAligned>(xv[i], x + c * kVec, P.cols - c * kVec, xs);
    if (kNorm && P.residual) load_pack<kAligned>(rv[i], r + c * kVec, P.cols - c * kVec, rs);
  }
  float sum = 0.f;
  unsigned top = 0;  // bits of the largest |t|: ordered as unsigned, with NaN above infinity
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int c = tid + i * threads;
    if (!in || c >= packs) continue;
#pragma unroll
    for (int e = 0; e < kVec; ++e) t[i][e] = to_f32(xv[i][e]);
    if constexpr (kNorm) {
      if (P.residual) {
#pragma unroll
        for (int e = 0; e < kVec; e += 2) {
          t[i][e] += to_f32(rv[i][e]);
          t[i][e + 1] += to_f32(rv[i][e + 1]);
          put2(&rv[i][e], t[i][e], t[i][e + 1]);
        }
        if constexpr (!kLate) store_pack<kAligned>(h_out + c * kVec, rv[i], P.cols - c * kVec);
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) sum = fmaf(t[i][e], t[i][e], sum);
      if (w) {
        constexpr int kPart = 16 / sizeof(W);  // a 32-bit weight beside 16-bit rows takes two packs
#pragma unroll
        for (int h = 0; h < kVec; h += kPart) {
          alignas(16) W wv[kPart];
          load_pack<kAligned>(wv, w + c * kVec + h, P.cols - c * kVec - h, ws);
#pragma unroll
          for (int e = 0; e < kPart; ++e) t[i][h + e] *= to_f32(wv[e]);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) top = max(top, __float_as_uint(t[i][e]) & 0x7fffffffu);
  }
  top = __reduce_max_sync(kFullMask, top);
  if constexpr (kNorm)
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
  if (threads > 32) {  // one row to the block
    const int warps = threads >> 5;
    if ((tid & 31) == 0) {
      s_sum[tid >> 5] = sum;
      s_top[tid >> 5] = top;
    }
    __syncthreads();
    sum = (tid & 31) < warps ? s_sum[tid & 31] : 0.f;
    top = __reduce_max_sync(kFullMask, (tid & 31) < warps ? s_top[tid & 31] : 0u);
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
  }
  if (!in) return;
  const float a = __uint_as_float(top);
  const bool finite = top < 0x7f800000u, tiny = a < kTinyRow;
  if constexpr (kNorm) {
    // NaN in the sum is one in the row; a mean from 2^-100 on has lost nothing to squares below 2^-126.
    if (!tiny && (sum > 0x1.fffffep127f || fmaf((float)P.cols, P.eps, sum) < 0x1p-100f * (float)P.cols || (!finite && sum == sum))) {
      const bool stored = !kLate && P.residual && (sizeof(T) == 4 || r == h_out);
      rows_outside<T, W>(stored ? h_out : x, P.residual && !stored ? r : nullptr, kLate && P.residual ? h_out : nullptr, w,
                         P.q + row * P.q_stride, P.scale + row, P.cols, P.eps, !finite);
      return;
    }
    if (kLate && P.residual) {
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int c = tid + i * threads;
        if (c < packs) store_pack<kAligned>(h_out + c * kVec, rv[i], P.cols - c * kVec);
      }
    }
  }
  const float inv = finite && !tiny ? __fmul_rn(__frcp_rn(a), 127.f) : 0.f;
  if (tid == 0) {
    const float rms = kNorm ? rsqrtf(sum / (float)P.cols + P.eps) : 1.f;
    P.scale[row] = !finite ? __int_as_float(0x7fffffff) : tiny ? 0.f : a * rms / 127.f;
  }
  int8_t* q = P.q + row * P.q_stride;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int c = tid + i * threads;
    if (c >= packs) continue;
    uint32_t word[kVec / 4] = {};
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const int code = finite ? __float2int_rn(__fmul_rn(t[i][e], inv)) : 0;
      word[e / 4] |= (uint32_t)(code & 255) << (8 * (e & 3));
    }
    if (kAligned || (P.q_aligned && (c + 1) * kVec <= P.cols)) {
      if constexpr (kVec == 8) *reinterpret_cast<uint2*>(q + c * 8) = make_uint2(word[0], word[1]);
      else *reinterpret_cast<uint32_t*>(q + c * 4) = word[0];
    } else {
      store_pack<false>(q + c * kVec, reinterpret_cast<const int8_t(&)[kVec]>(word), P.cols - c * kVec);
    }
  }
}

// value = code * scale of its row, rounded once: sixteen codes of a row to a thread (kPacked: their
// rows start on 16-byte boundaries, and the values'; kTail: the last of a row may be fewer), or
// eight, 32 apart, with a warp on 256 neighbouring ones.
// 16384 x 4096 into bf16: 33 us, 6.1 TB/s.
template <typename T, bool kPacked, bool kTail>
__global__ void __launch_bounds__(256) dequant_rows_kernel(const int8_t* q, long long q_stride, const float* scale,
                                                           T* out, long long rows, int cols) {
  constexpr int kSpan = kPacked ? 16 : 256;
  griddep_launch_wait();
  const int spans = (cols + kSpan - 1) / kSpan;
  const long long at = ((long long)blockIdx.x * 256 + threadIdx.x) / (kPacked ? 1 : 32);
  // The division is in 32 bits where the index fits it.
  const long long row = at <= 0xffffffffll ? (long long)((uint32_t)at / (uint32_t)spans) : at / spans;
  if (row >= rows) return;
  const int c = (int)(at - row * spans) * kSpan;
  const float s = scale[row];
  q += row * q_stride + c;
  out += row * cols + c;
  if constexpr (kPacked) {
    const int n = kTail ? cols - c : 16;
    uint32_t word[4] = {};
    if (n >= 16) {
      *reinterpret_cast<uint4*>(word) = __ldg(reinterpret_cast<const uint4*>(q));
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) word[e / 4] |= e < n ? (uint32_t)(uint8_t)q[e] << (8 * (e & 3)) : 0u;
    }
    constexpr int kPart = 16 / sizeof(T);
#pragma unroll
    for (int h = 0; h < 16; h += kPart) {
      alignas(16) T v[kPart];
#pragma unroll
      for (int e = 0; e < kPart; e += 2) {
        // A byte plus 128, under the exponent of 2^23: exact, and cheaper than a conversion.
        const auto value = [&](int i) {
          const uint32_t bits = __byte_perm(word[i / 4] ^ 0x80808080u, 0x4b000000u, 0x7440 + (i & 3));
          return (__uint_as_float(bits) - 8388736.f) * s;
        };
        put2(&v[e], value(h + e), value(h + e + 1));
      }
      if (!kTail || h < n) store_pack<true>(out + h, v, kPart);  // n is a multiple of a pack
    }
  } else {
    const int lane = threadIdx.x & 31, n = cols - c;
    int code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) code[i] = lane + 32 * i < n ? __ldg(q + lane + 32 * i) : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < n) out[lane + 32 * i] = from_f32<T>((float)code[i] * s);
  }
}

}  // namespace qrb200
