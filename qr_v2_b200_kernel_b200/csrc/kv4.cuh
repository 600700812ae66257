// A key/value cache in 4 bits: its layout, its quantisation as it is written, its reader, and
// the attention of a few queries over it.
//
// Per token, head and group of G channels, with lo and hi the group's ends:
//   s = hi/15 - lo/15 rounded to the cache's type,  m = lo,
//   code = min(15, max(0, rint((x - m) (1/s)))),  value = m + s code.
// m is exact (it is one of the inputs) and the codes are taken against the rounded s, so the
// reader sees what the writer meant. s < 2^-126 has no reciprocal: codes 0. A group that holds a
// NaN or an infinity reads back as NaN.
//
// Layout. One block per (page, head), P tokens of D channels, NG = D / G groups:
//   [key codes P D/2 B][value codes P D/2 B][key (s, m) P NG 4 B][value (s, m) P NG 4 B]
// The codes lie the way the 16 x 8 x 16 matrix instruction's left operand wants them, so that
// the attention loads them straight into registers, 16 bytes at a time, and no shared memory or
// transposition stands between the cache and the product. Lane (g, t) = (lane / 4, lane % 4) of
// that operand holds rows g and g + 8, columns {2t, 2t+1, 2t+8, 2t+9}:
//   keys: rows are tokens, columns channels (their order is free: queries are permuted alike).
//     A token's D/2 bytes are four runs, one for each t; word w of a run holds the steps
//     j = 2w, 2w + 1, channels 16 j + 4 t + e, e = 0..3, at nibble 2 (j & 1) + (e >> 1) + 4 (e & 1);
//   values: rows are channels, columns tokens. Each 16 tokens are D/16 tiles of 32 words, one for
//     each lane, stored as [tile / 4][lane][tile % 4]; word bytes 0, 2, 1, 3 are tokens 2t, 2t+1,
//     2t+8, 2t+9, low nibble channel 16 tile + g, high nibble + 8. A byte belongs to one token:
//     tokens written at the same time by different threads never share one.
#pragma once

#include "quant_rows.cuh"
#include "tc.cuh"

namespace qrb200 {

struct Kv4Shape {
  int heads, page, dim, groups;  // groups per head
  long long pages;
  __host__ __device__ int block_bytes() const { return page * (dim + 8 * groups); }
  __host__ __device__ int v_codes() const { return page * dim / 2; }
  __host__ __device__ int k_pairs() const { return page * dim; }
  __host__ __device__ int v_pairs() const { return page * (dim + 4 * groups); }
};

// Byte and shift of a key's and a value's code inside its block's code section.
__device__ __forceinline__ int kv4_key_byte(int dim, int tok, int d, int* shift) {
  const int j = d >> 4, t = (d >> 2) & 3, e = d & 3;
  const int nib = 2 * (j & 1) + (e >> 1) + 4 * (e & 1);
  *shift = 4 * (nib & 1);
  return tok * (dim / 2) + t * (dim / 8) + (j >> 1) * 4 + (nib >> 1);
}
__device__ __forceinline__ int kv4_value_byte(int dim, int tok, int d, int* shift) {
  const int kk = tok & 15, tile = d >> 4, r = d & 15;
  const int lane = (r & 7) * 4 + ((kk & 7) >> 1);
  const int byte = 2 * (kk & 1) + (kk >> 3);
  *shift = 4 * (r >> 3);
  return (tok >> 4) * 8 * dim + (tile >> 2) * 512 + lane * 16 + (tile & 3) * 4 + byte;
}

template <typename T>
struct Pair16 {
  T s, m;
};

struct Kv4IoParams {
  unsigned char* cache;
  const void* k;
  const void* v;
  void* k_out;
  void* v_out;
  const long long* slots;
  long long tokens, k_ts, k_hs, v_ts, v_hs;  // strides in elements
  Kv4Shape sh;
};

// One warp quantises one token's key or value of one head: kN = D / 32 channels to a lane, neighbouring
// ones, so a group is a run of G / kN lanes.
template <typename T, int kN>
__global__ void __launch_bounds__(128) kv4_write_kernel(Kv4IoParams P) {
  const int lane = threadIdx.x & 31;
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const long long tok = unit / P.sh.heads;
  const int head = (int)(unit % P.sh.heads);
  if (tok >= P.tokens) return;
  const long long slot = P.slots[tok];
  if (slot < 0) return;
  const long long page = slot / P.sh.page;
  if (page >= P.sh.pages) {
    if (lane == 0) report_device_failure(kSiteIndex);
    return;
  }
  const int at = (int)(slot % P.sh.page);
  unsigned char* block = P.cache + (page * P.sh.heads + head) * (long long)P.sh.block_bytes();
  const int span = 32 / P.sh.groups;  // lanes of a group
  for (int part = 0; part < 2; ++part) {
    const T* src = part ? static_cast<const T*>(P.v) + tok * P.v_ts + head * P.v_hs
                        : static_cast<const T*>(P.k) + tok * P.k_ts + head * P.k_hs;
    float x[kN];
    float lo = __int_as_float(0x7f800000), hi = -lo;
    bool fine = true;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      x[i] = to_f32(src[lane * kN + i]);
      fine = fine && fabsf(x[i]) < __int_as_float(0x7f800000);
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
    }
    for (int o = span >> 1; o; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(kFullMask, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(kFullMask, hi, o));
      fine = __shfl_xor_sync(kFullMask, (int)fine, o) && fine;
    }
    constexpr float kFifteenth = 1.f / 15.f;
    const float nan = __int_as_float(0x7fffffff);
    Pair16<T> pr;
    pr.s = from_f32<T>(fine ? __fsub_rn(__fmul_rn(hi, kFifteenth), __fmul_rn(lo, kFifteenth)) : nan);
    pr.m = from_f32<T>(fine ? lo : nan);
    const float s = to_f32(pr.s), m = to_f32(pr.m);
    const float inv = s >= 0x1p-126f ? __frcp_rn(s) : 0.f;
    if (lane % span == 0)
      reinterpret_cast<Pair16<T>*>(block + (part ? P.sh.v_pairs() : P.sh.k_pairs()))[at * P.sh.groups + lane / span] = pr;
    int code[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i)
      code[i] = fine ? (int)fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[i], m), inv)), 0.f), 15.f) : 0;
    // Each byte is put together and stored by the lane that holds its low nibble.
    unsigned char* codes = block + (part ? P.sh.v_codes() : 0);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int d = lane * kN + i;
      const int partner = part ? d + 8 : (d & 2 ? -1 : d + 2);  // the channel of the byte's high nibble
      const int pl = (partner < 0 ? 0 : partner / kN) & 31;
      int high = 0;
#pragma unroll
      for (int q = 0; q < kN; ++q) {
        const int got = __shfl_sync(kFullMask, code[q], pl);
        if (partner >= 0 && partner % kN == q) high = got;
      }
      int shift;
      const int byte = part ? kv4_value_byte(P.sh.dim, at, d, &shift) : kv4_key_byte(P.sh.dim, at, d, &shift);
      if (shift == 0) codes[byte] = (unsigned char)(code[i] | high << 4);
    }
  }
}

// Values at slots; a negative slot reads as zeros. One thread per channel of a token and head.
template <typename T>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4IoParams P) {
  const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
  const int dim = P.sh.dim;
  const long long unit = e / dim, tok = unit / P.sh.heads;
  if (tok >= P.tokens) return;
  const int d = (int)(e % dim), head = (int)(unit % P.sh.heads);
  const long long slot = P.slots[tok], page = slot / P.sh.page;
  const bool there = slot >= 0 && page < P.sh.pages;
  if (slot >= 0 && !there && d == 0) report_device_failure(kSiteIndex);
  float out[2] = {0.f, 0.f};
  if (there) {
    const int at = (int)(slot % P.sh.page), g = d / (dim / P.sh.groups);
    const unsigned char* block = P.cache + (page * P.sh.heads + head) * (long long)P.sh.block_bytes();
    for (int part = 0; part < 2; ++part) {
      int shift;
      const int byte = part ? kv4_value_byte(dim, at, d, &shift) : kv4_key_byte(dim, at, d, &shift);
      const int code = (block[(part ? P.sh.v_codes() : 0) + byte] >> shift) & 15;
      const Pair16<T> pr =
          reinterpret_cast<const Pair16<T>*>(block + (part ? P.sh.v_pairs() : P.sh.k_pairs()))[at * P.sh.groups + g];
      out[part] = fmaf(to_f32(pr.s), (float)code, to_f32(pr.m));
    }
  }
  static_cast<T*>(P.k_out)[e] = from_f32<T>(out[0]);
  static_cast<T*>(P.v_out)[e] = from_f32<T>(out[1]);
}

}  // namespace qrb200
