// Attention over the 8-bit cache (layout and formulas: kv8.cuh).
#pragma once

#include "kv8.cuh"

namespace qrb200 {

struct Kv8AttnParams {
  const unsigned char* codes;
  const float* range;
  const void* q;
  void* out;
  const int* table;
  const int* lengths;
  long long q_bs, q_ts, q_hs, table_stride;  // strides in elements
  int batch, queries, q_heads, share, max_pages, window, causal;
  float scale;
  Kv8Shape sh;
};

// A warp to a query row: token after token, its channels over the lanes.
template <typename T, int kDim>
__global__ void __launch_bounds__(128) kv8_simple_kernel(Kv8AttnParams P) {
  constexpr int kPer = kDim / 32;
  griddep_launch_wait();
  const int lane = threadIdx.x & 31, head = blockIdx.y, b = blockIdx.z;
  const long long query = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (query >= P.queries) return;
  int len = P.lengths[b];
  if (len < 0 || len > (long long)P.max_pages * P.sh.page || (len > 0 && P.sh.pages == 0)) {
    if (lane == 0) report_device_failure(kSiteIndex);
    len = 0;
  }
  const T* q = static_cast<const T*>(P.q) + b * P.q_bs + query * P.q_ts + head * P.q_hs;
  float qv[kPer], o[kPer] = {}, m = -INFINITY, l = 0.f;
  for (int i = 0; i < kPer; ++i) qv[i] = to_f32(q[32 * i + lane]) * P.scale;
  const int pos = len - P.queries + (int)query, hi = P.causal ? max(0, pos + 1) : len;
  const int lo = P.window > 0 ? max(0, pos - P.window + 1) : 0;
  for (int tok = lo; tok < hi; ++tok) {
    const int page = P.table[b * P.table_stride + (tok >> P.sh.shift)], j = tok & (P.sh.page - 1);
    if (page < 0 || page >= P.sh.pages) {
      if (lane == 0) report_device_failure(kSiteIndex);
      continue;
    }
    const long long at = (long long)page * P.sh.heads + head / P.share;
    const unsigned char* block = P.codes + at * P.sh.block_bytes();
    float s = 0.f;
    for (int i = 0; i < kPer; ++i) s = fmaf(qv[i], (float)((int)block[kv8_key_at(kDim, j, 32 * i + lane)] - 128), s);
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(kFullMask, s, x);
    s *= kv8_step(P.range[at * 2]);
    const float step = kv8_step(P.range[at * 2 + 1]), next = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.f : expf(m - next), p = expf(s - next);
    l = fmaf(l, keep, p);
    for (int i = 0; i < kPer; ++i) o[i] = fmaf(o[i], keep, p * step * (float)((int)block[kv8_value_at(kDim, j, 32 * i + lane)] - 128));
    m = next;
  }
  T* out = static_cast<T*>(P.out) + (((long long)b * P.queries + query) * P.q_heads + head) * kDim;
  for (int i = 0; i < kPer; ++i) out[32 * i + lane] = from_f32<T>(l == 0.f ? 0.f : o[i] / l);
}

}  // namespace qrb200
