// A key/value cache in 8 bits with a range for each page and head: its layout, its writer and its reader.
//
// Keys and values of a page and head have a range R each, and a code stands for code R / 127. Tokens come
// a few at a time, so R grows as they do: with a = the largest magnitude written,
//   R = max(R, a rounded up to three significant bits),   code = rint(127 x / R)   (a half to the larger magnitude),
// and where R grew from R' the codes of the page's other tokens become rint(code R' / R). (Rounded up, R
// takes at most four steps to double, so a token is seldom rounded again; that costs at most a quarter
// of the range, 9 % on average. It also makes the quotients safe: 127 x / R is midway between two
// codes only for x = R / 2, and no other 16-bit x comes nearer than 2^-17 of it.) The call that writes a page's first token begins
// it anew: R from what the call writes, zeros for the rest of the page. A NaN or an infinity makes R NaN
// until then. A largest magnitude below 2^-100 counts as zero.
//
// Layout. One block per (page, head): P / 16 runs of 16 tokens, [key codes 16 D B][value codes 16 D B], a code
// c as the byte c + 128. The bytes lie the way the 16 x 8 x 16 matrix instruction's left operand wants them,
// so that what the attention copies is already in the order of its registers, 16 bytes at a time.
// Lane (g, t) = (lane / 4, lane % 4) of that operand holds rows g and g + 8, columns {2t, 2t+1, 2t+8, 2t+9}:
//   keys: rows are tokens, columns channels (their order is free: queries are permuted alike). Tokens 0
//     to 7, then 8 to 15; of each, pieces of 64 channels; of each, 16 bytes for every lane: word w holds channels 16 w +
//     4 t + e of the piece, e = 0..3;
//   values: rows are channels, columns tokens. Pieces of 32 channels; of each, 16 bytes for every lane: word w
//     holds channel 16 (w / 2) + 8 (w % 2) + g, its bytes tokens 2t, 2t+1, 2t+8, 2t+9.
#pragma once

#include <type_traits>

#include "quant_rows.cuh"
#include "tc.cuh"

namespace qrb200 {

struct Kv8Shape {
  int heads, page, dim, shift;  // page = 2^shift
  long long pages;
  __host__ __device__ int block_bytes() const { return 2 * page * dim; }
};

struct Kv8IoParams {
  unsigned char* codes;
  float* range;  // [page][head][2]: keys, values
  const void* k;
  const void* v;
  void* k_out;
  void* v_out;
  const long long* slots;
  int* rows;  // workspace: a slot's row of this call, where there are many
  long long tokens, k_ts, k_hs, v_ts, v_hs;  // strides in elements
  Kv8Shape sh;
  int chunk;  // rows of a CTA
};

// Offsets of a token's code within its block: of channel c, as a key and as a value.
__device__ __forceinline__ int kv8_key_at(int dim, int token, int c) {
  return token / 16 * (32 * dim) + (token >> 3 & 1) * (8 * dim) + (c >> 6) * 512 + (token & 7) * 64 + (c >> 2 & 3) * 16 +
         (c >> 4 & 3) * 4 + (c & 3);
}
__device__ __forceinline__ int kv8_value_at(int dim, int token, int c) {
  return token / 16 * (32 * dim) + 16 * dim + (c >> 5) * 512 + (c & 7) * 64 + (token >> 1 & 3) * 16 + (c >> 3 & 3) * 4 +
         (token & 1) + (token >> 2 & 2);
}

constexpr uint32_t kKv8Zeros = 0x80808080u;
constexpr int kKv8Few = 1024;  // rows up to which a CTA looks a page's rows up among all of them

// Three significant bits, rounded up, of a magnitude's bits (the magnitude itself where that would pass the type's
// largest number, so that no value reads back as infinity); NaN for what is not finite.
template <typename T>
__device__ __forceinline__ float kv8_range(unsigned top) {
  if (top >= 0x7f800000u) return __int_as_float(0x7fffffff);
  if (__uint_as_float(top) < kTinyRow) return 0.f;
  const unsigned up = (top + 0x1fffffu) & ~0x1fffffu;
  constexpr unsigned kMost = std::is_same<T, __half>::value ? 0x477fe000u : 0x7f7f0000u;  // 65504; 255 2^120
  return __uint_as_float(up <= kMost ? up : top);
}
__device__ __forceinline__ float kv8_step(float range) { return range / 127.f; }
// 127 / R, a little up: the one x between two codes, R / 2, goes to the upper one, and nothing else moves.
__device__ __forceinline__ float kv8_inverse(float range) { return 127.f / range * (1.f + 0x1p-20f); }

// What page a row writes, or -1.
__device__ __forceinline__ long long kv8_page(const Kv8IoParams& P, long long slot) {
  const long long page = slot >> P.sh.shift;
  return slot < 0 || page >= P.sh.pages ? -1 : page;
}

__global__ void __launch_bounds__(256) kv8_rows_kernel(Kv8IoParams P) {
  griddep_launch_wait();
  const long long r = (long long)blockIdx.x * 256 + threadIdx.x;
  if (r < P.tokens && kv8_page(P, P.slots[r]) >= 0) P.rows[P.slots[r]] = (int)r;
}

// A CTA takes a stretch of rows and a head. Rows of one page are written by one CTA, whichever holds the
// lowest of them, so that nothing is shared: it finds all of the page's rows (s_row: the row of each
// slot), their largest magnitude, moves the older codes if the range grew, and writes the new ones.
template <typename T, int kDim>
__global__ void __launch_bounds__(256) kv8_write_kernel(Kv8IoParams P) {
  constexpr int kSpan = kDim / 8, kAtOnce = 256 / kSpan;  // threads of a token, tokens at a time
  __shared__ int s_row[1024];
  __shared__ unsigned s_low[8], s_top[2][8];
  griddep_launch_wait();
  const int head = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, c0 = 8 * (tid % kSpan);
  const long long row0 = (long long)blockIdx.x * P.chunk, row1 = min(P.tokens, row0 + P.chunk);
  for (long long r = row0; r < row1;) {
    const long long page = kv8_page(P, P.slots[r]);
    if (page < 0) {
      if (P.slots[r] >= 0 && tid == 0) report_device_failure(kSiteIndex);
      ++r;
      continue;
    }
    long long end = r + 1;
    while (end < row1 && kv8_page(P, P.slots[end]) == page) ++end;
    // The rows of the page's slots, and the lowest of them.
    __syncthreads();  // the page before is done
    unsigned low = 0xffffffffu;
    if (P.rows) {
      for (int j = tid; j < P.sh.page; j += 256) {
        const long long slot = (page << P.sh.shift) + j;
        const int at = P.rows[slot];  // whatever it held before, unless the row says so too
        const bool is = at >= 0 && at < P.tokens && P.slots[at] == slot;
        s_row[j] = is ? at : -1;
        if (is) low = min(low, (unsigned)at);
      }
    } else {
      for (int j = tid; j < P.sh.page; j += 256) s_row[j] = -1;
      __syncthreads();
      for (int at = tid; at < P.tokens; at += 256)
        if (kv8_page(P, P.slots[at]) == page) {
          atomicMax(&s_row[(int)P.slots[at] & (P.sh.page - 1)], at);
          low = min(low, (unsigned)at);
        }
    }
    low = __reduce_min_sync(kFullMask, low);
    if ((tid & 31) == 0) s_low[warp] = low;
    __syncthreads();
    low = __reduce_min_sync(kFullMask, s_low[tid & 7]);
    const bool leads = low >= r && low < end;
    r = end;
    if (!leads) continue;
    unsigned top[2] = {0, 0};
    const auto each = [&](auto f) {
      for (int j = tid / kSpan; j < P.sh.page; j += kAtOnce) {
        const int row = s_row[j];
        if (row < 0) continue;
        const T* from[2] = {static_cast<const T*>(P.k) + row * P.k_ts + head * P.k_hs + c0,
                            static_cast<const T*>(P.v) + row * P.v_ts + head * P.v_hs + c0};
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int e = 0; e < 8; ++e) f(part, j, e, to_f32(from[part][e]));
      }
    };
    each([&](int part, int, int, float x) { top[part] = max(top[part], __float_as_uint(x) & 0x7fffffffu); });
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      top[part] = __reduce_max_sync(kFullMask, top[part]);
      if ((tid & 31) == 0) s_top[part][warp] = top[part];
    }
    __syncthreads();
    float* range = P.range + (page * P.sh.heads + head) * 2;
    unsigned char* block = P.codes + (page * P.sh.heads + head) * P.sh.block_bytes();
    const bool fresh = s_row[0] >= 0;
    float old[2], now[2];
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const float grown = kv8_range<T>(__reduce_max_sync(kFullMask, s_top[part][tid & 7]));
      old[part] = fresh ? 0.f : range[part];
      now[part] = grown == grown && old[part] == old[part] ? fmaxf(grown, old[part]) : __int_as_float(0x7fffffff);
    }
    __syncthreads();  // every thread has read the older range
    if (tid < 2) range[tid] = now[tid];
    // Older codes to the new range (its quotient with the ranges 2^-8 of theirs, whose product with a code
    // is finite, and exact): 16 bytes at a time, keys and values in runs of 16 tokens.
    for (int at = tid; at < P.sh.block_bytes() / 16; at += 256) {
      const int part = at / kDim & 1;
      if (now[part] != now[part] || (!fresh && now[part] == old[part])) continue;
      uint4 w = make_uint4(kKv8Zeros, kKv8Zeros, kKv8Zeros, kKv8Zeros);
      if (old[part] > 0.f) {
        w = reinterpret_cast<const uint4*>(block)[at];
        uint32_t* word = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t next = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = (int)(word[i] >> (8 * e) & 255) - 128;
            next |= (uint32_t)(__float2int_rn(__fdiv_rn((float)c * (old[part] * 0x1p-8f), now[part] * 0x1p-8f)) + 128) << (8 * e);
          }
          word[i] = next;
        }
      }
      reinterpret_cast<uint4*>(block)[at] = w;
    }
    __syncthreads();  // before the new codes go into the same words
    const float inv[2] = {now[0] > 0.f ? kv8_inverse(now[0]) : 0.f, now[1] > 0.f ? kv8_inverse(now[1]) : 0.f};
    each([&](int part, int j, int e, float x) {
      const int code = inv[part] > 0.f ? __float2int_rn(x * inv[part]) : 0;
      block[part ? kv8_value_at(kDim, j, c0 + e) : kv8_key_at(kDim, j, c0 + e)] = (unsigned char)(code + 128);
    });
  }
}

// The values at slots; a negative slot reads as zeros. Eight channels to a thread.
template <typename T, int kDim>
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8IoParams P) {
  constexpr int kSpan = kDim / 8, kAtOnce = 256 / kSpan;
  griddep_launch_wait();
  const long long row = (long long)blockIdx.x * kAtOnce + threadIdx.x / kSpan;
  const int head = blockIdx.y, c0 = 8 * (threadIdx.x % kSpan);
  if (row >= P.tokens) return;
  const long long slot = P.slots[row], page = kv8_page(P, slot);
  if (page < 0 && slot >= 0 && head == 0 && c0 == 0) report_device_failure(kSiteIndex);
  const int j = (int)slot & (P.sh.page - 1);
  const long long at = page < 0 ? 0 : page * P.sh.heads + head;
  const unsigned char* block = P.codes + at * P.sh.block_bytes();
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    alignas(16) T out[8];
    const float step = page < 0 ? 0.f : kv8_step(P.range[at * 2 + part]);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      float c[2] = {0.f, 0.f};
      if (page >= 0)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          c[i] = (float)((int)block[part ? kv8_value_at(kDim, j, c0 + e + i) : kv8_key_at(kDim, j, c0 + e + i)] - 128);
      put2(out + e, c[0] * step, c[1] * step);
    }
    *reinterpret_cast<uint4*>(static_cast<T*>(part ? P.v_out : P.k_out) + (row * P.sh.heads + head) * kDim + c0) =
        *reinterpret_cast<const uint4*>(out);
  }
}

}  // namespace qrb200
