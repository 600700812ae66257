// A key/value cache in 4 bits: its layout, its quantisation as it is written, its reader, and
// the attention of a few queries over it.
//
// Per token, head and group of G channels, with lo and hi the group's ends:
//   s = hi/15 - lo/15 rounded to the cache's type (the next lower number if m + 15 s would round to
//   infinity there),  m = lo,
//   code = min(15, max(0, rint((x - m) (1/s)))),  value = m + s code.
// m is exact (it is one of the inputs) and the codes are taken against the rounded s, so the
// reader sees what the writer meant. s < 2^-126 has no reciprocal: codes 0. A group that holds a
// NaN or an infinity reads back as NaN.
//
// Layout. One block per (page, head): P / 16 runs of 16 tokens, D channels, NG = D / G groups. A run is
//   [key codes 8 D B][value codes 8 D B][key (s, m) 64 NG B][value (s, m) 64 NG B]
// so that a run's loads share one address, and what is read together lies together (a multiple of
// 128 bytes). The codes lie the way the 16 x 8 x 16 matrix instruction's left operand wants them,
// so that what the attention copies into shared memory is already in the order of its registers,
// 16 bytes at a time, with nothing to transpose or unpack on the way.
// Lane (g, t) = (lane / 4, lane % 4) of that operand holds rows g and g + 8, columns
// {2t, 2t+1, 2t+8, 2t+9}:
//   keys: rows are tokens, columns channels (their order is free: queries are permuted alike).
//     A token's D/2 bytes are four parts, one for each t; word w of a part holds the steps
//     j = 2w, 2w + 1, channels 16 j + 4 t + e, e = 0..3, at nibble 2 (j & 1) + (e >> 1) + 4 (e & 1);
//   values: rows are channels, columns tokens. The run is D/16 tiles of 32 words, one for
//     each lane, stored as [tile / 4][lane][tile % 4]; word bytes 0, 2, 1, 3 are tokens 2t, 2t+1,
//     2t+8, 2t+9, low nibble channel 16 tile + g, high nibble + 8. A byte belongs to one token:
//     tokens written at the same time by different threads never share one.
#pragma once

#include <type_traits>

#include "quant_rows.cuh"
#include "tc.cuh"

namespace qrb200 {

struct Kv4Shape {
  int heads, page, dim, groups, shift;  // groups per head; page = 2^shift
  long long pages;
  __host__ __device__ int run_bytes() const { return 16 * dim + 128 * groups; }
  __host__ __device__ int block_bytes() const { return page / 16 * run_bytes(); }
};

template <typename T>
struct Pair16 {
  T s, m;
};

template <typename T>
struct Two;
template <>
struct Two<__nv_bfloat16> {
  using type = __nv_bfloat162;
};
template <>
struct Two<__half> {
  using type = __half2;
};
// (least, -greatest) of eight numbers, NaN if one is.
template <typename T>
__device__ __forceinline__ typename Two<T>::type kv4_ends(const T (&x)[8]) {
  using T2 = typename Two<T>::type;
  const T2* p = reinterpret_cast<const T2*>(x);
  const T2 lo = __hmin2_nan(__hmin2_nan(p[0], p[1]), __hmin2_nan(p[2], p[3]));
  const T2 hi = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3]));
  T2 r;
  r.x = __hmin_nan(lo.x, lo.y);
  r.y = __hneg(__hmax_nan(hi.x, hi.y));
  return r;
}
// Nibble codes at bits 0 and 16 of w as two numbers.
__device__ __forceinline__ float2 kv4_codes(uint32_t w) {
  const uint32_t x = (w & 0x000f000fu) | 0x64006400u;
  return __half22float2(__hsub2(reinterpret_cast<const __half2&>(x), __floats2half2_rn(1024.f, 1024.f)));
}

struct Kv4IoParams {
  unsigned char* cache;
  const void* k;
  const void* v;
  void* k_out;
  void* v_out;
  const long long* slots;
  long long tokens, k_ts, k_hs, v_ts, v_hs;  // strides in elements
  Kv4Shape sh;
  int span;  // heads to a CTA
};

// Where a token's run lies, or null for a slot that is skipped; an index past the cache is reported.
__device__ __forceinline__ unsigned char* kv4_run(const Kv4IoParams& P, long long slot, int head, bool report) {
  if (slot < 0) return nullptr;
  const long long page = slot >> P.sh.shift;
  if (page >= P.sh.pages) {
    if (report) report_device_failure(kSiteIndex);
    return nullptr;
  }
  return P.cache + (page * P.sh.heads + head) * P.sh.block_bytes() + ((int)slot & (P.sh.page - 1)) / 16 * P.sh.run_bytes();
}

// Sixteen tokens to a CTA, kDim / 8 threads to a token, 8 channels (16 bytes) to a thread, head
// after head of P.span of them; the next head's loads are under way while one is quantised. When
// the sixteen fill a run, as prompts do, the run is put together in shared memory and stored whole;
// otherwise each thread stores its words (keys) and bytes (values). Long prompts are bound by
// instructions: codes come out of the 32-bit floating sum's bits, packed as they lie.
// 32768 tokens x 8 heads x 128 channels, bf16: 54 us (2.8 TB/s; 320 instructions of a warp for its
// 512 elements, issue slots 77 % busy). Walking several heads took it from 63, registers for 40
// warps an SM in place of 32 from 56 (48 warps would spill: 56).
template <typename T, int kDim, int kGroups, bool kVec>
__global__ void __launch_bounds__(2 * kDim, kVec ? 640 / kDim : 1) kv4_write_kernel(Kv4IoParams P) {
  constexpr int kChunks = kDim / 8, kSpan = kChunks / kGroups;  // threads of a token, of a group
  constexpr int kRunBytes = 16 * kDim + 128 * kGroups;
  __shared__ uint4 s_run[2][kRunBytes / 16];
  griddep_launch_wait();
  const int chunk = threadIdx.x % kChunks, mine = threadIdx.x / kChunks;
  const int head0 = blockIdx.y * P.span, heads = min(P.span, P.sh.heads - head0);
  const long long first = (long long)blockIdx.x * 16, tok = first + mine;
  const bool in = tok < P.tokens;
  const T* k = static_cast<const T*>(P.k) + tok * P.k_ts + head0 * P.k_hs + 8 * chunk;
  const T* v = static_cast<const T*>(P.v) + tok * P.v_ts + head0 * P.v_hs + 8 * chunk;
  const auto load = [&](T(&x)[8], const T* src) {
    if constexpr (kVec) {
      *reinterpret_cast<uint4*>(x) = in ? __ldg(reinterpret_cast<const uint4*>(src)) : uint4{};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = in ? src[i] : from_f32<T>(0.f);
    }
  };
  alignas(16) T x[2][8];
  load(x[0], k);
  load(x[1], v);
  const long long slot = in ? P.slots[tok] : -1, slot0 = P.slots[first];
  const bool whole = __syncthreads_and(in && slot == slot0 + mine && (slot0 & 15) == 0);
  unsigned char* run = kv4_run(P, whole ? slot0 : slot, head0, chunk == 0);
  const int block = P.sh.block_bytes();
  // Quantises both parts into the run at `out` (null: nowhere), as its token `at`.
  const auto quantise = [&](unsigned char* out, int at) {
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      // The group's ends, exact in 16 bits: this thread's eight channels two at a time, then (lo,
      // -hi) over the group's threads. NaN carries through; infinity shows at an end.
      typename Two<T>::type ends = kv4_ends(x[part]);
#pragma unroll
      for (int o = kSpan >> 1; o; o >>= 1) {
        const uint32_t other = __shfl_xor_sync(kFullMask, reinterpret_cast<const uint32_t&>(ends), o);
        ends = __hmin2_nan(ends, reinterpret_cast<const typename Two<T>::type&>(other));
      }
      const float lo = to_f32(ends.x), hi = -to_f32(ends.y);
      constexpr float kFifteenth = 1.f / 15.f;
      Pair16<T> pr;
      pr.s = from_f32<T>(__fsub_rn(__fmul_rn(hi, kFifteenth), __fmul_rn(lo, kFifteenth)));
      pr.m = from_f32<T>(lo);
      // Not finite, or near the top of the type, where a step rounded up may put the group's top past the
      // largest number: then the next lower step.
      constexpr float kNear = std::is_same<T, __half>::value ? 65000.f : 0x1.f8p127f;
      constexpr float kBeyond = std::is_same<T, __half>::value ? 65520.f : 0x1.ffp127f;  // rounds to infinity
      if (!(lo > -__int_as_float(0x7f800000) && hi < kNear)) {
        if (!(fabsf(lo) < __int_as_float(0x7f800000) && fabsf(hi) < __int_as_float(0x7f800000)))
          pr.s = pr.m = from_f32<T>(__int_as_float(0x7fffffff));
        else if (fmaf(15.f, to_f32(pr.s), lo) >= kBeyond)
          --reinterpret_cast<uint16_t&>(pr.s);
      }
      const float s = to_f32(pr.s), m = to_f32(pr.m);
      // bf16 ends may be further apart than 32 bits reach: such a group is quantised at half its size.
      const float part_of = std::is_same<T, __nv_bfloat16>::value && hi - lo > 0x1.fffffep127f ? 0.5f : 1.f;
      const float inv = s >= 0x1p-126f ? __frcp_rn(s * part_of) : 0.f, least = -m * part_of;
      // x - m is never negative. Added to 1.5 2^23, a number below 2^22 leaves its nearest whole
      // number (ties to even) in the low bits, above a constant that the packing takes off. Where s
      // is normal, its rounding keeps every code below 15.5. (In a group that is not finite the
      // codes come out as anything: they share no byte or word with another group's.)
      uint32_t code[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // Difference, product and sum are each rounded: (x - m) / s often lies midway between two
        // codes, all being short numbers, and one rounding less would break such ties another way.
        // (The paired forms of these operations are fused by the compiler. The difference's own
        // fused form only halves both, which is exact.)
        float steps = __fmul_rn(__fmaf_rn(to_f32(x[part][i]), part_of, least), inv);
        if constexpr (std::is_same<T, __half>::value) steps = fminf(steps, 15.f);  // subnormal s
        code[i] = __float_as_uint(__fadd_rn(steps, 0x1.8p23f));
      }
      constexpr uint32_t kBits = 0x4b400000u;
      if (part == 0) {
        // Step j = chunk / 2, t = 2 (chunk & 1) and the next; the other half of each word, step j ^
        // 1, is chunk ^ 2's.
        const int up = (chunk & 2) ? 8 : 0;
        constexpr uint32_t kAll = kBits + (kBits << 16) + (kBits << 4) + (kBits << 20);
        const uint32_t a = (code[0] + (code[1] << 16) + (code[2] << 4) + (code[3] << 20) - kAll) << up;
        const uint32_t b = (code[4] + (code[5] << 16) + (code[6] << 4) + (code[7] << 20) - kAll) << up;
        const uint32_t got = __shfl_xor_sync(kFullMask, up ? a : b, 2), word = (up ? b : a) | got;
        const int t = 2 * (chunk & 1) + (up ? 1 : 0);
        if (out) *reinterpret_cast<uint32_t*>(out + at * (kDim / 2) + t * (kDim / 8) + (chunk >> 2) * 4) = word;
      } else {
        // Tile chunk / 2; an even chunk has the low nibbles of its 8 bytes, its odd neighbour the
        // high ones.
        const bool odd = chunk & 1;
        constexpr uint32_t kAll = kBits + (kBits << 8) + (kBits << 16) + (kBits << 24);
        const uint32_t a = code[0] + (code[1] << 8) + (code[2] << 16) + (code[3] << 24) - kAll;
        const uint32_t b = code[4] + (code[5] << 8) + (code[6] << 16) + (code[7] << 24) - kAll;
        const uint32_t got = __shfl_xor_sync(kFullMask, odd ? a : b, 1), bytes = odd ? got | b << 4 : a | got << 4;
        const int tile = chunk >> 1, byte = 2 * (at & 1) + (at >> 3), lane = (odd ? 16 : 0) + ((at & 7) >> 1);
        if (out) {
          unsigned char* to = out + 8 * kDim + (tile >> 2) * 512 + lane * 16 + (tile & 3) * 4 + byte;
#pragma unroll
          for (int i = 0; i < 4; ++i) to[64 * i] = (unsigned char)(bytes >> (8 * i));
        }
      }
      if (out && chunk % kSpan == 0)
        reinterpret_cast<Pair16<T>*>(out + 16 * kDim + part * 64 * kGroups)[at * kGroups + chunk / kSpan] = pr;
    }
  };
  for (int h = 0; h < heads; ++h) {
    alignas(16) T next[2][8];
    if (h + 1 < heads) {
      load(next[0], k + (h + 1) * P.k_hs);
      load(next[1], v + (h + 1) * P.v_hs);
    }
    if (whole) {
      quantise(reinterpret_cast<unsigned char*>(s_run[h & 1]), mine);
      __syncthreads();  // also: the other buffer has been stored
      if (run)
        for (int i = threadIdx.x; i < kRunBytes / 16; i += 2 * kDim) reinterpret_cast<uint4*>(run)[i] = s_run[h & 1][i];
    } else {
      quantise(run, (int)(slot & 15));
    }
    if (run) run += block;
#pragma unroll
    for (int part = 0; part < 2; ++part)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[part][i] = next[part][i];
  }
}

// The values at slots, as kv4_write_kernel cuts them; a negative slot reads as zeros. A whole run
// goes through shared memory.
// 32768 tokens x 8 heads x 128 channels, bf16: 30 us, 5.7 TB/s.
template <typename T, int kDim, int kGroups>
__global__ void __launch_bounds__(2 * kDim) kv4_read_kernel(Kv4IoParams P) {
  constexpr int kChunks = kDim / 8, kSpan = kChunks / kGroups;  // threads of a token, of a group
  constexpr int kRunBytes = 16 * kDim + 128 * kGroups;
  __shared__ uint4 s_run[2][kRunBytes / 16];
  griddep_launch_wait();
  const int chunk = threadIdx.x % kChunks, mine = threadIdx.x / kChunks;
  const int head0 = blockIdx.y * P.span, heads = min(P.span, P.sh.heads - head0);
  const long long first = (long long)blockIdx.x * 16, tok = first + mine;
  const bool in = tok < P.tokens;
  const long long slot = in ? P.slots[tok] : -1, slot0 = P.slots[first];
  const bool whole = __syncthreads_and(in && slot == slot0 + mine && (slot0 & 15) == 0);
  const unsigned char* run = kv4_run(P, whole ? slot0 : slot, head0, chunk == 0);
  const int block = P.sh.block_bytes();
  T* k = static_cast<T*>(P.k_out) + (tok * P.sh.heads + head0) * kDim + 8 * chunk;
  T* v = static_cast<T*>(P.v_out) + (tok * P.sh.heads + head0) * kDim + 8 * chunk;
  // Both parts of token `at` of the run at `from` (null: zeros).
  const auto values = [&](const unsigned char* from, int at) {
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      float2 code[4];
      alignas(16) T out[8];
      if (from) {
        if (part == 0) {
          const unsigned char* w = from + at * (kDim / 2) + 2 * (chunk & 1) * (kDim / 8) + (chunk >> 2) * 4;
          const int up = (chunk & 2) ? 8 : 0;
          const uint32_t a = *reinterpret_cast<const uint32_t*>(w) >> up, b = *reinterpret_cast<const uint32_t*>(w + kDim / 8) >> up;
          code[0] = kv4_codes(a), code[1] = kv4_codes(a >> 4), code[2] = kv4_codes(b), code[3] = kv4_codes(b >> 4);
        } else {
          const int tile = chunk >> 1, byte = 2 * (at & 1) + (at >> 3), shift = 4 * (chunk & 1);
          const unsigned char* c = from + 8 * kDim + (tile >> 2) * 512 + ((at & 7) >> 1) * 16 + (tile & 3) * 4 + byte;
#pragma unroll
          for (int i = 0; i < 4; ++i) code[i] = kv4_codes((c[128 * i] | (uint32_t)c[128 * i + 64] << 16) >> shift);
        }
        const Pair16<T> pr =
            reinterpret_cast<const Pair16<T>*>(from + 16 * kDim + part * 64 * kGroups)[at * kGroups + chunk / kSpan];
        const float s = to_f32(pr.s), m = to_f32(pr.m);
#pragma unroll
        for (int i = 0; i < 4; ++i) put2(out + 2 * i, fmaf(s, code[i].x, m), fmaf(s, code[i].y, m));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = from_f32<T>(0.f);
      }
      if (in) *reinterpret_cast<uint4*>(part ? v : k) = *reinterpret_cast<uint4*>(out);
    }
    k += kDim;
    v += kDim;
  };
  if (!whole || !run) {
    for (int h = 0; h < heads; ++h) {
      values(run, (int)(slot & 15));
      if (run) run += block;
    }
    return;
  }
  constexpr int kPieces = kRunBytes / 16, kThreads = 2 * kDim;  // at most two pieces a thread
  static_assert(kPieces <= 2 * kThreads, "");
  uint4 piece[2];
  const auto fetch = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (threadIdx.x + i * kThreads < kPieces) piece[i] = __ldg(reinterpret_cast<const uint4*>(run) + threadIdx.x + i * kThreads);
    run += block;
  };
  fetch();
  for (int h = 0; h < heads; ++h) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (threadIdx.x + i * kThreads < kPieces) s_run[h & 1][threadIdx.x + i * kThreads] = piece[i];
    __syncthreads();  // also: the other buffer has been read
    if (h + 1 < heads) fetch();
    values(reinterpret_cast<const unsigned char*>(s_run[h & 1]), mine);
  }
}

}  // namespace qrb200
