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
  // Workspace, where there are many rows: how many pages get few of them and how many more, a row of each page (the first kind
  // from the list's front, the second from its end), and the row of each slot.
  int *pages, *list, *rows;
  long long tokens, k_ts, k_hs, v_ts, v_hs;  // strides in elements
  Kv8Shape sh;
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
constexpr int kKv8Few = 1024;  // rows up to which a page's are looked up among all of them
constexpr int kKv8Thin = 8;    // rows of a page up to which a warp takes a head, else a CTA

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

// Many rows: which row a slot has (whichever was stored last where a slot is given twice), and, once that is known, the
// pages: each by the lowest of its rows, in any order.
__global__ void __launch_bounds__(256) kv8_rows_kernel(Kv8IoParams P) {
  griddep_launch_wait();
  const long long r = (long long)blockIdx.x * 256 + threadIdx.x;
  if (r < 2) P.pages[r] = 0;
  if (r >= P.tokens) return;
  const long long slot = P.slots[r];
  if (kv8_page(P, slot) >= 0) P.rows[slot] = (int)r;
  else if (slot >= 0) report_device_failure(kSiteIndex);
}
// The row of a slot, or -1; P.rows holds anything where this call gives none.
__device__ __forceinline__ int kv8_row(const Kv8IoParams& P, long long slot) {
  const int at = P.rows[slot];
  return at >= 0 && at < P.tokens && P.slots[at] == slot ? at : -1;
}
constexpr int kKv8Seek = 4;  // rows of a warp, so that their look-ups wait together
__global__ void __launch_bounds__(256) kv8_pages_kernel(Kv8IoParams P) {
  griddep_launch_wait();
  const int lane = threadIdx.x & 31;
  const long long first = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * kKv8Seek;
  long long page[kKv8Seek];
  unsigned low[kKv8Seek];
  int rows[kKv8Seek] = {};
#pragma unroll
  for (int i = 0; i < kKv8Seek; ++i) {
    const long long r = first + i;
    page[i] = r < P.tokens ? kv8_page(P, P.slots[r]) : -1;
    low[i] = 0xffffffffu;
    // The row before is lower, where it is the one that its slot has.
    if (r > 0 && page[i] >= 0 && kv8_page(P, P.slots[r - 1]) == page[i] && P.rows[P.slots[r - 1]] == r - 1) page[i] = -1;
  }
  for (int j = lane; j < P.sh.page; j += 32)
#pragma unroll
    for (int i = 0; i < kKv8Seek; ++i)
      if (page[i] >= 0) {
        const int at = kv8_row(P, (page[i] << P.sh.shift) + j);
        low[i] = min(low[i], (unsigned)at);  // (-1 is the largest)
        rows[i] += at >= 0;
      }
#pragma unroll
  for (int i = 0; i < kKv8Seek; ++i)
    if (page[i] >= 0 && __reduce_min_sync(kFullMask, low[i]) == first + i) {
      const bool thin = __reduce_add_sync(kFullMask, rows[i]) <= kKv8Thin;
      if (lane == 0) {
        const int at = atomicAdd(P.pages + !thin, 1);
        P.list[thin ? at : P.tokens - 1 - at] = (int)(first + i);
      }
    }
}

// Threads and bytes. In a run of 16 tokens thread (chunk, t) holds channels 8 chunk to 8 chunk + 7 of tokens 2t, 2t + 1,
// 2t + 8, 2t + 9: of the values whole words then, one a channel, 64 bytes apart, and of each key two words, 16 bytes apart.
__device__ __forceinline__ int kv8_token(int t, int i) { return 2 * t + (i & 1) + 8 * (i >> 1); }

// The largest magnitude of sixteen-bit numbers, as their bits: ordered as whole numbers, NaN above infinity.
__device__ __forceinline__ uint32_t kv8_top(uint32_t top, const uint4& x) {
  top = __vmaxu2(__vmaxu2(top, x.x & 0x7fff7fffu), x.y & 0x7fff7fffu);
  return __vmaxu2(__vmaxu2(top, x.z & 0x7fff7fffu), x.w & 0x7fff7fffu);
}
template <typename T>
__device__ __forceinline__ unsigned kv8_top_bits(uint32_t pair) {  // of a 32-bit float
  const uint16_t top = (uint16_t)max(pair & 0xffffu, pair >> 16);
  return __float_as_uint(to_f32(reinterpret_cast<const T&>(top)));
}
// Eight numbers to bytes code + 128, in the low bytes of floats: x inv + 128, under the exponent of 2^23, rounded once.
template <typename T>
__device__ __forceinline__ void kv8_bytes(uint32_t (&f)[8], const uint4& x, float inv) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 two = make_float2(to_f32(reinterpret_cast<const T*>(&w[i])[0]), to_f32(reinterpret_cast<const T*>(&w[i])[1]));
    f[2 * i] = __float_as_uint(fmaf(two.x, inv, 0x1.8p23f + 128.f));
    f[2 * i + 1] = __float_as_uint(fmaf(two.y, inv, 0x1.8p23f + 128.f));
  }
}
__device__ __forceinline__ uint32_t kv8_word(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {  // of low bytes
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// The older codes of a page and head to a new range: their quotient with the ranges 2^-8 of theirs, whose product with
// a code is finite, and exact.
__device__ __forceinline__ uint32_t kv8_moved(uint32_t word, float old, float now) {
  uint32_t next = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = (int)(word >> (8 * e) & 255) - 128;
    next |= (uint32_t)(__float2int_rn(__fdiv_rn((float)c * (old * 0x1p-8f), now * 0x1p-8f)) + 128) << (8 * e);
  }
  return next;
}

// A page's head whose new rows are few, by a warp or (kTeam) a CTA of eight, four rows at a time to each: tokens one by one, four
// channels (64: two) to a lane, and bytes stored where they belong, since a step of decoding brings a page one.
template <typename T, int kDim, bool kVec, bool kTeam>
__device__ __forceinline__ void kv8_write_thin(const Kv8IoParams& P, const int* s_row, unsigned (*s_top)[2], long long page, int head) {
  constexpr int kPer = kDim / 32;  // channels of a lane
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const auto sync = [&]() {
    if (kTeam) __syncthreads();
    else __syncwarp();
  };
  const int c0 = kPer * lane;
  const auto load = [&](T(&x)[2][kPer], int row) {
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const T* from = (part ? static_cast<const T*>(P.v) + row * P.v_ts + head * P.v_hs : static_cast<const T*>(P.k) + row * P.k_ts + head * P.k_hs) + c0;
      if constexpr (kVec && kPer == 4) {
        *reinterpret_cast<uint2*>(x[part]) = __ldg(reinterpret_cast<const uint2*>(from));
      } else if constexpr (kVec) {
        *reinterpret_cast<uint32_t*>(x[part]) = __ldg(reinterpret_cast<const uint32_t*>(from));
      } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[part][e] = from[e];
      }
    }
  };
  // f(token, row) for the page's new tokens, loaded four at a time (eight change nothing).
  const auto each = [&](auto f) {
    for (int base = 0; base < P.sh.page; base += 32) {
      const int mine = base + lane < P.sh.page ? s_row[base + lane] : -1;
      unsigned have = __ballot_sync(kFullMask, mine >= 0 && (!kTeam || ((base + lane) >> 2 & 7) == warp));
      while (have) {
        alignas(8) T x[4][2][kPer];
        int token[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          token[i] = have ? __ffs(have) - 1 : -1;
          have &= have - 1;
          if (token[i] >= 0) load(x[i], __shfl_sync(kFullMask, mine, token[i]));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (token[i] >= 0) f(base + token[i], x[i]);
      }
    }
  };
  unsigned top[2] = {0, 0};
  each([&](int, const T(&x)[2][kPer]) {
#pragma unroll
    for (int part = 0; part < 2; ++part)
#pragma unroll
      for (int e = 0; e < kPer; ++e) top[part] = max(top[part], __float_as_uint(to_f32(x[part][e])) & 0x7fffffffu);
  });
  for (int part = 0; part < 2; ++part) top[part] = __reduce_max_sync(kFullMask, top[part]);
  if constexpr (kTeam) {
    if (lane == 0) s_top[warp][0] = top[0], s_top[warp][1] = top[1];
    __syncthreads();
    for (int part = 0; part < 2; ++part) top[part] = __reduce_max_sync(kFullMask, s_top[lane & 7][part]);
  }
  float* range = P.range + (page * P.sh.heads + head) * 2;
  unsigned char* block = P.codes + (page * P.sh.heads + head) * P.sh.block_bytes();
  const bool fresh = s_row[0] >= 0;
  float old[2], now[2], inv[2];
  bool move[2];
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const float grown = kv8_range<T>(top[part]);
    old[part] = fresh ? 0.f : range[part];
    now[part] = grown == grown && old[part] == old[part] ? fmaxf(grown, old[part]) : __int_as_float(0x7fffffff);
    inv[part] = now[part] > 0.f ? kv8_inverse(now[part]) : 0.f;
    move[part] = now[part] == now[part] && (fresh || now[part] != old[part]);
  }
  sync();  // every lane has read the older range
  if (lane < 2 && (!kTeam || warp == 0)) range[lane] = now[lane];
  if (move[0] || move[1]) {
#pragma unroll 4
    for (int at = kTeam ? threadIdx.x : lane; at < P.sh.block_bytes() / 16; at += kTeam ? 256 : 32) {
      const int part = at / kDim & 1;
      if (!move[part]) continue;
      uint4 w = make_uint4(kKv8Zeros, kKv8Zeros, kKv8Zeros, kKv8Zeros);
      if (old[part] > 0.f) {
        w = reinterpret_cast<const uint4*>(block)[at];
        w = make_uint4(kv8_moved(w.x, old[part], now[part]), kv8_moved(w.y, old[part], now[part]), kv8_moved(w.z, old[part], now[part]),
                       kv8_moved(w.w, old[part], now[part]));
      }
      reinterpret_cast<uint4*>(block)[at] = w;
    }
    sync();  // before the new codes go into the same words
  }
  each([&](int token, const T(&x)[2][kPer]) {
    uint32_t f[2][kPer];
#pragma unroll
    for (int part = 0; part < 2; ++part)
#pragma unroll
      for (int e = 0; e < kPer; ++e) f[part][e] = __float_as_uint(fmaf(to_f32(x[part][e]), inv[part], 0x1.8p23f + 128.f));
    unsigned char* key = block + kv8_key_at(kDim, token, c0);
    if constexpr (kPer == 4) *reinterpret_cast<uint32_t*>(key) = kv8_word(f[0][0], f[0][1], f[0][2], f[0][3]);
    else *reinterpret_cast<uint16_t*>(key) = (uint16_t)__byte_perm(f[0][0], f[0][1], 0x0040);
#pragma unroll
    for (int e = 0; e < kPer; ++e) block[kv8_value_at(kDim, token, c0 + e)] = (unsigned char)f[1][e];
  });
}

// Up to kKv8Few rows, in one launch: a CTA to a row and eight heads. It finds the page's other rows among all, and the CTAs of a
// page's rows share the heads, by their rows' order: a warp to a head where they are few, a CTA to a head where there are as many
// CTAs. Few and light CTAs, so that this kernel and the next overlap. (8 heads x 128 channels: single tokens of 16 sequences 3.6 us,
// of 256 5.1, of 1024 9.2; 12 tokens of one 3.8, 64 6.1, 500 10.9, 1000 14.9. Through the lists below: 14 for 256 single
// tokens, 23 for 1024; 12 and 18 for 128 and 500 of one sequence.)
template <typename T, int kDim, bool kVec>
__global__ void __launch_bounds__(256) kv8_write_few_kernel(Kv8IoParams P) {
  __shared__ int s_row[1024];
  __shared__ unsigned s_count[8], s_top[8][2];
  griddep_launch_wait();
  const int tid = threadIdx.x, warp = tid >> 5, r = blockIdx.x;
  const long long page = kv8_page(P, P.slots[r]);
  if (page < 0) {
    if (P.slots[r] >= 0 && tid == 0) report_device_failure(kSiteIndex);
    return;
  }
  for (int j = tid; j < P.sh.page; j += 256) s_row[j] = -1;
  __syncthreads();
  unsigned count = 0;  // the page's rows, and above 2^16 those before this one
  for (int at = tid; at < P.tokens; at += 256) {
    const long long slot = P.slots[at];
    if (kv8_page(P, slot) == page) {
      atomicMax(&s_row[(int)slot & (P.sh.page - 1)], at);
      count += at < r ? 0x10001u : 1u;
    }
  }
  count = __reduce_add_sync(kFullMask, count);
  if ((tid & 31) == 0) s_count[warp] = count;
  __syncthreads();
  count = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) count += s_count[i];
  const int rows = count & 0xffff, rank = count >> 16, head0 = 8 * blockIdx.y, heads = min(8, P.sh.heads - head0);
  if (rows < 8) {
    if (rank + rows * warp < heads) kv8_write_thin<T, kDim, kVec, false>(P, s_row, s_top, page, head0 + rank + rows * warp);
  } else if (rank < heads) {
    kv8_write_thin<T, kDim, kVec, true>(P, s_row, s_top, page, head0 + rank);
  }
}

// Some heads of a page with more new rows, by the CTA: their largest magnitude, then the runs that change, put together in
// shared memory, 64 tokens at a time: the older codes, moved if the range grew, and the new ones over them. Up to 64
// tokens a page, everything is read once.
template <int kDim>
struct Kv8Thick {
  static constexpr int kChunks = kDim / 8, kRunThreads = 4 * kChunks;  // threads of a run
  static constexpr int kRuns = 4, kThreads = kRuns * kRunThreads;      // runs at a time
  uint4 image[kRuns * 2 * kDim];
  unsigned top[2][kThreads / 32];
  unsigned char has[2][kThreads / 32];
};
template <typename T, int kDim, bool kVec>
__device__ __forceinline__ void kv8_write_thick(const Kv8IoParams& P, Kv8Thick<kDim>& S, const int* s_row, long long page, int head0, int heads) {
  using K = Kv8Thick<kDim>;
  constexpr int kRuns = K::kRuns, kThreads = K::kThreads, kRunWarps = K::kRunThreads / 32, kRun = 32 * kDim;
  const int tid = threadIdx.x, warp = tid >> 5;
  const int t = tid & 3, chunk = (tid >> 2) % K::kChunks, mine = tid / K::kRunThreads;  // this thread's run of those at a time
  const int runs = P.sh.page / 16;
  uint4 x[2][4];  // this thread's tokens of a run: keys, values
  int rows[4];
  const auto fetch = [&](int head, int run) {
#pragma unroll
    for (int i = 0; i < 4; ++i) rows[i] = run < runs ? s_row[16 * run + kv8_token(t, i)] : -1;
#pragma unroll
    for (int part = 0; part < 2; ++part)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[part][i] = make_uint4(0, 0, 0, 0);
        if (rows[i] >= 0) {
          const T* from = part ? static_cast<const T*>(P.v) + rows[i] * P.v_ts + head * P.v_hs : static_cast<const T*>(P.k) + rows[i] * P.k_ts + head * P.k_hs;
          if constexpr (kVec) {
            x[part][i] = __ldg(reinterpret_cast<const uint4*>(from + 8 * chunk));
          } else {
            alignas(16) T y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = from[8 * chunk + e];
            x[part][i] = *reinterpret_cast<const uint4*>(y);
          }
        }
      }
  };
  unsigned char* image = reinterpret_cast<unsigned char*>(S.image);
  if (runs <= kRuns) fetch(head0, mine);
  for (int head = head0; head < head0 + heads; ++head) {
    uint32_t top[2] = {0, 0};
    for (int base = 0; base < runs; base += kRuns) {
      if (runs > kRuns) fetch(head, base + mine);
#pragma unroll
      for (int i = 0; i < 4; ++i) top[0] = kv8_top(top[0], x[0][i]), top[1] = kv8_top(top[1], x[1][i]);
    }
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const unsigned most = __reduce_max_sync(kFullMask, kv8_top_bits<T>(top[part]));
      if ((tid & 31) == 0) S.top[part][warp] = most;
    }
    __syncthreads();
    float* range = P.range + (page * P.sh.heads + head) * 2;
    unsigned char* block = P.codes + (page * P.sh.heads + head) * P.sh.block_bytes();
    const bool fresh = s_row[0] >= 0;
    float old[2], now[2], inv[2];
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const float grown = kv8_range<T>(__reduce_max_sync(kFullMask, S.top[part][tid & (kThreads / 32 - 1)]));
      old[part] = fresh ? 0.f : range[part];
      now[part] = grown == grown && old[part] == old[part] ? fmaxf(grown, old[part]) : __int_as_float(0x7fffffff);
      inv[part] = now[part] > 0.f ? kv8_inverse(now[part]) : 0.f;
    }
    const bool move[2] = {now[0] == now[0] && (fresh || now[0] != old[0]), now[1] == now[1] && (fresh || now[1] != old[1])};
    __syncthreads();  // every thread has read the older range
    if (tid < 2) range[tid] = now[tid];
    for (int base = 0; base < runs; base += kRuns) {
      if (runs > kRuns) fetch(head, base + mine);
      const bool any = rows[0] >= 0 || rows[1] >= 0 || rows[2] >= 0 || rows[3] >= 0;
      const bool all = rows[0] >= 0 && rows[1] >= 0 && rows[2] >= 0 && rows[3] >= 0;
      // Of each run, whether anything is written and whether it is filled (a run's threads are whole warps).
      const bool some = __any_sync(kFullMask, any), whole = __all_sync(kFullMask, all);
      unsigned char* has = S.has[base / kRuns & 1];
      if ((tid & 31) == 0) has[warp] = (some ? 1 : 0) | (whole ? 2 : 0);
      __syncthreads();
      unsigned changed = 0, filled = 0;
#pragma unroll
      for (int i = 0; i < kRuns; ++i) {
        unsigned either = has[i * kRunWarps], both = either;
        if (kRunWarps == 2) either |= has[2 * i + 1], both &= has[2 * i + 1];
        if (base + i < runs) changed |= ((either & 1) || move[0] || move[1] ? 1u : 0u) << i;
        filled |= (both >> 1) << i;
      }
      if (changed == 0) continue;  // (never where the page is taken at once)
      if (changed & ~filled) {
        // The older codes first, moved to the new range, or zeros.
#pragma unroll 4
        for (int at = tid; at < kRuns * kRun / 16; at += kThreads) {
          if (!((changed & ~filled) >> (at * 16 / kRun) & 1)) continue;
          const int part = at / kDim & 1;
          uint4 w = make_uint4(kKv8Zeros, kKv8Zeros, kKv8Zeros, kKv8Zeros);
          if (!move[part] || old[part] > 0.f) w = reinterpret_cast<const uint4*>(block + (long long)base * kRun)[at];
          if (move[part] && old[part] > 0.f)
            w = make_uint4(kv8_moved(w.x, old[part], now[part]), kv8_moved(w.y, old[part], now[part]), kv8_moved(w.z, old[part], now[part]),
                           kv8_moved(w.w, old[part], now[part]));
          S.image[at] = w;
        }
        __syncthreads();
      }
      if (any) {
        unsigned char* run = image + mine * kRun;
        uint32_t f[4][8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          kv8_bytes<T>(f[i], x[0][i], inv[0]);
          if (rows[i] >= 0) {
            uint32_t* to = reinterpret_cast<uint32_t*>(run + kv8_key_at(kDim, kv8_token(t, i), 8 * chunk));
            to[0] = kv8_word(f[i][0], f[i][1], f[i][2], f[i][3]);
            to[4] = kv8_word(f[i][4], f[i][5], f[i][6], f[i][7]);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) kv8_bytes<T>(f[i], x[1][i], inv[1]);
        unsigned char* to = run + kv8_value_at(kDim, 2 * t, 8 * chunk);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (all) {
            *reinterpret_cast<uint32_t*>(to + 64 * e) = kv8_word(f[0][e], f[1][e], f[2][e], f[3][e]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (rows[i] >= 0) to[64 * e + i] = (unsigned char)f[i][e];
          }
        }
      }
      __syncthreads();
      if (runs <= kRuns && head + 1 < head0 + heads) fetch(head + 1, mine);  // under way while this head's bytes leave
      for (int at = tid; at < kRuns * kRun / 16; at += kThreads) {
        if (changed >> (at * 16 / kRun) & 1) reinterpret_cast<uint4*>(block + (long long)base * kRun)[at] = S.image[at];
      }
      __syncthreads();  // the image is free
    }
  }
}

// More: of the pages with few rows, unless they are so few themselves that the next kernel does them by the way (the ends of
// sequences), each warp takes as many heads, in order, as any other, (2048 single tokens x 8 heads x 128 channels 33 us;
// by CTAs, as below, 202)
constexpr int kKv8ThinWarps = 4;
// (Up to 256 of their heads: two sequences' 936 tokens x 4 heads 19.3 -> 12.1 us, sixteen's 512 x 8 37.6 -> 28.6.)
__device__ __forceinline__ int kv8_thin_pages(const Kv8IoParams& P) { return (long long)P.pages[0] * P.sh.heads > 256 ? P.pages[0] : 0; }
template <typename T, int kDim, bool kVec>
__global__ void __launch_bounds__(32 * kKv8ThinWarps) kv8_write_thin_kernel(Kv8IoParams P) {
  __shared__ int s_row[kKv8ThinWarps][1024];
  griddep_launch_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long units = (long long)kv8_thin_pages(P) * P.sh.heads, warps = gridDim.x * (long long)kKv8ThinWarps, per = (units + warps - 1) / warps;
  const long long first = (blockIdx.x * (long long)kKv8ThinWarps + warp) * per, end = min(units, first + per);
  for (long long unit = first; unit < end; ++unit) {
    const int head = (int)(unit % P.sh.heads);
    const long long page = kv8_page(P, P.slots[P.list[unit / P.sh.heads]]);
    if (unit == first || head == 0) {
      __syncwarp();  // the page before is done
      for (int j = lane; j < P.sh.page; j += 32) s_row[warp][j] = kv8_row(P, (page << P.sh.shift) + j);
      __syncwarp();
    }
    kv8_write_thin<T, kDim, kVec, false>(P, s_row[warp], nullptr, page, head);
  }
}
// and each CTA. 32768 tokens x 8 heads x 128 channels, bf16: 69 us from a page's first token, 71 from within one, 3.0 TB/s of
// keys, values and codes, the three kernels before it 8 of them. No pipe is full (issue slots 41 %, memory 31 %): a head's loads,
// maximum, packing and stores follow one another, and 128 registers leave sixteen warps an SM.
template <typename T, int kDim, bool kVec>
__global__ void __launch_bounds__(2 * kDim) kv8_write_kernel(Kv8IoParams P) {
  __shared__ Kv8Thick<kDim> s_thick;
  __shared__ int s_row[1024];
  griddep_launch_wait();
  const int thick = P.pages[1], pages = thick + P.pages[0] - kv8_thin_pages(P);
  const long long units = (long long)pages * P.sh.heads, per = (units + gridDim.x - 1) / gridDim.x, end = min(units, (blockIdx.x + 1) * per);
  for (long long unit = blockIdx.x * per; unit < end;) {
    const int head0 = (int)(unit % P.sh.heads), heads = (int)min((long long)(P.sh.heads - head0), end - unit);
    const int at = (int)(unit / P.sh.heads);
    const long long page = kv8_page(P, P.slots[P.list[at < thick ? P.tokens - 1 - at : at - thick]]);
    unit += heads;
    __syncthreads();  // the page before is done
    for (int j = threadIdx.x; j < P.sh.page; j += 2 * kDim) s_row[j] = kv8_row(P, (page << P.sh.shift) + j);
    __syncthreads();
    kv8_write_thick<T, kDim, kVec>(P, s_thick, s_row, page, head0, heads);
  }
}

// The values at slots; a negative slot reads as zeros. A warp takes 16 rows of a head: a whole run, as sequences are read, goes
// through shared memory, other rows come as they lie. 32768 tokens x 8 heads x 128 channels in whole runs 36 us, 5.6 TB/s.
template <typename T, int kDim>
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8IoParams P) {
  constexpr int kRun = 32 * kDim;
  __shared__ uint4 s_run[8][kRun / 16];
  griddep_launch_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = lane & 3;
  const long long unit = (long long)blockIdx.x * 8 + warp, first = unit / P.sh.heads * 16;
  const int head = (int)(unit % P.sh.heads);
  if (first >= P.tokens) return;
  const long long slot = lane < 16 && first + lane < P.tokens ? P.slots[first + lane] : -1, slot0 = __shfl_sync(kFullMask, slot, 0);
  if (slot >= 0 && kv8_page(P, slot) < 0 && head == 0) report_device_failure(kSiteIndex);
  const bool whole = __all_sync(kFullMask, lane >= 16 || slot == slot0 + lane) && (slot0 & 15) == 0 && kv8_page(P, slot0) >= 0;
  const auto place = [&](long long s, float2& step) {  // the run that holds a slot
    const long long page = kv8_page(P, s);
    if (page < 0) return static_cast<const unsigned char*>(nullptr);
    const float2 r = __ldg(reinterpret_cast<const float2*>(P.range) + page * P.sh.heads + head);
    step = make_float2(kv8_step(r.x), kv8_step(r.y));
    return static_cast<const unsigned char*>(P.codes) + (page * P.sh.heads + head) * P.sh.block_bytes() + ((int)s & (P.sh.page - 1)) / 16 * kRun;
  };
  const auto value = [&](uint32_t w, int e) {  // of byte e
    return __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + e)) - 8388736.f;
  };
  if (whole) {
    float2 step;
    const unsigned char* run = place(slot0, step);
#pragma unroll
    for (int i = 0; i < kRun / 512; ++i) s_run[warp][32 * i + lane] = __ldg(reinterpret_cast<const uint4*>(run) + 32 * i + lane);
    __syncwarp();
    const unsigned char* bytes = reinterpret_cast<const unsigned char*>(s_run[warp]);
#pragma unroll
    for (int chunk = lane >> 2; chunk < kDim / 8; chunk += 8) {
      uint32_t v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = *reinterpret_cast<const uint32_t*>(bytes + kv8_value_at(kDim, 2 * t, 8 * chunk) + 64 * e);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int token = kv8_token(t, i);
        const uint32_t* from = reinterpret_cast<const uint32_t*>(bytes + kv8_key_at(kDim, token, 8 * chunk));
        const uint32_t k[2] = {from[0], from[4]};
        alignas(16) T out[8];
        const long long at = ((first + token) * P.sh.heads + head) * kDim + 8 * chunk;
#pragma unroll
        for (int e = 0; e < 8; e += 2) put2(out + e, value(k[e >> 2], e & 3) * step.x, value(k[e >> 2], (e & 3) + 1) * step.x);
        *reinterpret_cast<uint4*>(static_cast<T*>(P.k_out) + at) = *reinterpret_cast<const uint4*>(out);
#pragma unroll
        for (int e = 0; e < 8; e += 2) put2(out + e, value(v[e], i) * step.y, value(v[e + 1], i) * step.y);
        *reinterpret_cast<uint4*>(static_cast<T*>(P.v_out) + at) = *reinterpret_cast<const uint4*>(out);
      }
    }
    return;
  }
  // Each row's place and steps at once, then eight channels of a row to a lane.
  float2 step = make_float2(0.f, 0.f);
  const unsigned char* run = place(slot, step);
  constexpr int kSpan = kDim / 8;
#pragma unroll 4
  for (int i = 0; i < 16 * kSpan / 32; ++i) {
    const int token = (32 * i + lane) / kSpan, c0 = 8 * (lane % kSpan);
    const int j = __shfl_sync(kFullMask, (int)slot & 15, token);
    const unsigned char* from = reinterpret_cast<const unsigned char*>(__shfl_sync(kFullMask, reinterpret_cast<unsigned long long>(run), token));
    const float key = __shfl_sync(kFullMask, step.x, token), other = __shfl_sync(kFullMask, step.y, token);
    uint32_t k[2] = {kKv8Zeros, kKv8Zeros}, v[8];
    if (from) {
      const uint32_t* keys = reinterpret_cast<const uint32_t*>(from + kv8_key_at(kDim, j, c0));
      k[0] = __ldg(keys), k[1] = __ldg(keys + 4);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = from ? (uint32_t)__ldg(from + kv8_value_at(kDim, j, c0) + 64 * e) : 128u;
    if (first + token >= P.tokens) continue;
    alignas(16) T out[8];
    const long long at = ((first + token) * P.sh.heads + head) * kDim + c0;
#pragma unroll
    for (int e = 0; e < 8; e += 2) put2(out + e, value(k[e >> 2], e & 3) * key, value(k[e >> 2], (e & 3) + 1) * key);
    *reinterpret_cast<uint4*>(static_cast<T*>(P.k_out) + at) = *reinterpret_cast<const uint4*>(out);
#pragma unroll
    for (int e = 0; e < 8; e += 2) put2(out + e, value(v[e], 0) * other, value(v[e + 1], 0) * other);
    *reinterpret_cast<uint4*>(static_cast<T*>(P.v_out) + at) = *reinterpret_cast<const uint4*>(out);
  }
}

}  // namespace qrb200
