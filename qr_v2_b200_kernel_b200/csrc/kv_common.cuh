// What attention over either cache shares: warp-level products, copies, weights, and the join of a long
// token range's parts.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cluster.cuh"
#include "quant_rows.cuh"

namespace qrb200 {

constexpr int kKvWarps = 4;
constexpr int kKvCluster = 8;  // the most CTAs that join their parts within a cluster (the portable size)

template <typename T>
__device__ __forceinline__ void kv_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void kv_mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void kv_mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float kv_power(int e) { return __int_as_float((max(-126, min(127, e)) + 127) << 23); }
__device__ __forceinline__ uint32_t kv_pack(float2 x) {
  const __half2 r = __float22half2_rn(x);
  return reinterpret_cast<const uint32_t&>(r);
}
__device__ __forceinline__ uint32_t kv_transpose(uint32_t x) {  // an 8 x 8 matrix of 16-bit numbers over the warp
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// 2^x to within 2 units in the last place of 32 bits, which is what the scores are good for.
__device__ __forceinline__ float kv_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// What a part with this (maximum, sum) counts against the maximum m of all: nothing where it saw
// nothing, NaN where its scores were. (A part is added even if its weight underflows to 0: a value that is
// NaN makes the result NaN, wherever the parts are cut. One that saw nothing holds zeros.)
__device__ __forceinline__ float kv_part_weight(float2 ml, float m) {
  return ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : ml.y) : kv_exp2(ml.x - m);
}
template <int kWords>
__device__ __forceinline__ void kv_load(uint32_t (&w)[kWords], const unsigned char* p) {  // from shared memory
  if constexpr (kWords == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (kWords == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}
__device__ __forceinline__ void kv_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t mbar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(mbar)
               : "memory");
}
constexpr float kKvLazy = 4.f;      // powers of two that a score may stand above the reference

__device__ __forceinline__ void mbar_expect(uint32_t mbar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(mbar), "r"(bytes) : "memory");
}

// The end of a CTA's work: its warps' parts of each row (s_o, unnormalised) against their common maximum, and the CTAs' of a
// split through the cluster's shared memory, or into memory for kv_join_kernel. spare: shared memory for
// kRows x (kKvCluster + 1) floats.
template <typename T, int kDim, int kRows, typename Params>
__device__ __forceinline__ void kv_join_warps(const Params& P, float (*s_o)[kRows][kDim + 4], float2 (*s_ml)[kRows], float* spare,
                                              const int* s_bad, int split, int tile, int head, int b, int rows, int row0) {
  constexpr int kLanesRow = 32 * kKvWarps / kRows;  // threads of a row
  const int r = threadIdx.x / kLanesRow, d0 = threadIdx.x % kLanesRow;
  float m = -INFINITY, l = 0.f, f[kKvWarps];
#pragma unroll
  for (int w = 0; w < kKvWarps; ++w) m = fmaxf(m, s_ml[w][r].x);
#pragma unroll
  for (int w = 0; w < kKvWarps; ++w) {
    f[w] = kv_part_weight(s_ml[w][r], m);
    l = fmaf(f[w], s_ml[w][r].y, l);
  }
  const auto out_row = [&](int row) {
    return static_cast<T*>(P.out) +
           (((long long)b * P.queries + (row0 + row) / P.share) * P.q_heads + head * P.share + (row0 + row) % P.share) * kDim;
  };
  const auto joined = [&](int d) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kKvWarps; ++w) x = fmaf(f[w], s_o[w][r][d], x);
    return x;
  };
  if (P.splits == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;  // nothing seen: zeros
    if (row0 + r < rows && !*s_bad)
      for (int d = d0; d < kDim; d += kLanesRow) out_row(r)[d] = from_f32<T>(joined(d) * inv);
  } else if (!P.part_ml) {
    // The CTA's part takes its first warp's place; each CTA then joins every splits-th row of all
    // of them.
    for (int d = d0; d < kDim; d += kLanesRow) s_o[0][r][d] = joined(d);
    __syncthreads();  // every warp's (maximum, sum) has been read
    if (d0 == 0) s_ml[0][r] = make_float2(m, l);
    cluster_sync();
    // What each CTA's part of a row counts, and the whole row's sum: a thread to a row.
    float(*s_w)[kKvCluster + 1] = reinterpret_cast<float(*)[kKvCluster + 1]>(spare);
    bool bad = false;
    for (int c = 0; c < P.splits; ++c) bad = ld_cluster(smem_u32(s_bad), c) != 0 || bad;
    if (threadIdx.x < kRows) {
      float2 ml[kKvCluster];
      float top = -INFINITY, total = 0.f;
#pragma unroll
      for (int c = 0; c < kKvCluster; ++c) {
        ml[c] = make_float2(-INFINITY, 0.f);
        if (c < P.splits) {
          ml[c].x = __int_as_float(ld_cluster(smem_u32(&s_ml[0][threadIdx.x].x), c));
          ml[c].y = __int_as_float(ld_cluster(smem_u32(&s_ml[0][threadIdx.x].y), c));
        }
        top = fmaxf(top, ml[c].x);
      }
#pragma unroll
      for (int c = 0; c < kKvCluster; ++c) {
        const float w = kv_part_weight(ml[c], top);
        total = fmaf(w, ml[c].y, total);
        s_w[threadIdx.x][c] = w;
      }
      s_w[threadIdx.x][kKvCluster] = total == 0.f ? 0.f : 1.f / total;
    }
    __syncthreads();
    const int own = bad ? 0 : (min(kRows, rows - row0) - split + P.splits - 1) / P.splits;  // rows split, split + splits, ...
    for (int e = threadIdx.x; e < own * kDim; e += 32 * kKvWarps) {
      const int row = split + e / kDim * P.splits, d = e % kDim;
      float v[kKvCluster], x = 0.f;
#pragma unroll
      for (int c = 0; c < kKvCluster; ++c) v[c] = c < P.splits ? __int_as_float(ld_cluster(smem_u32(&s_o[0][row][d]), c)) : 0.f;
#pragma unroll
      for (int c = 0; c < kKvCluster; ++c) x = fmaf(s_w[row][c], v[c], x);
      out_row(row)[d] = from_f32<T>(x * s_w[row][kKvCluster]);
    }
    cluster_sync();  // nobody leaves while its part is being read
  } else if (row0 + r < rows && !*s_bad) {
    const long long part = (((long long)b * P.sh.heads + head) * P.tiles + tile) * P.splits + split;
    for (int d = d0; d < kDim; d += kLanesRow) P.part_o[(part * kRows + r) * kDim + d] = joined(d);
    if (d0 == 0) P.part_ml[part * kRows + r] = make_float2(m, l);
  }
}

// One CTA per query row: the splits' parts against their common maximum, a warp every eighth, then
// the warps' sums in order.
constexpr int kKvJoinWarps = 8;
template <typename T, int kDim, typename Params>
__global__ void __launch_bounds__(32 * kKvJoinWarps) kv_join_kernel(Params P, int tile_rows) {
  __shared__ float s_x[kKvJoinWarps][kDim], s_l[kKvJoinWarps];
  griddep_launch_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rows = P.queries * P.share;
  const int unit = blockIdx.x, r = unit % rows, head = unit / rows % P.sh.heads, b = unit / rows / P.sh.heads;
  const long long part =
      (((long long)b * P.sh.heads + head) * P.tiles + r / tile_rows) * P.splits * tile_rows + r % tile_rows;
  float m = -INFINITY, l = 0.f, x[kDim / 32] = {};
  int end = 0;  // of the parts that saw something: a table wider than the sequence leaves the last ones empty
  for (int s = lane; s < P.splits; s += 32) {
    const float2 ml = P.part_ml[part + (long long)s * tile_rows];
    m = fmaxf(m, ml.x);
    if (!(ml.x == -INFINITY && ml.y == 0.f)) end = s + 1;
  }
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, o));
  end = __reduce_max_sync(kFullMask, end);
#pragma unroll 8
  for (int s = warp; s < end; s += kKvJoinWarps) {
    const float2 ml = P.part_ml[part + (long long)s * tile_rows];
    const float* o = P.part_o + (part + (long long)s * tile_rows) * kDim;
    const float f = kv_part_weight(ml, m);
    l = fmaf(f, ml.y, l);
#pragma unroll
    for (int i = 0; i < kDim / 32; ++i) {
      const float v = o[32 * i + lane];
      x[i] = fmaf(f, v, x[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kDim / 32; ++i) s_x[warp][32 * i + lane] = x[i];
  if (lane == 0) s_l[warp] = l;
  __syncthreads();
  if (threadIdx.x >= kDim) return;
  l = 0.f;
  float y = 0.f;
#pragma unroll
  for (int w = 0; w < kKvJoinWarps; ++w) {
    l += s_l[w];
    y += s_x[w][threadIdx.x];
  }
  static_cast<T*>(P.out)[(((long long)b * P.queries + r / P.share) * P.q_heads + head * P.share + r % P.share) * kDim + threadIdx.x] =
      from_f32<T>(l == 0.f ? 0.f : y * (1.f / l));
}

}  // namespace qrb200
