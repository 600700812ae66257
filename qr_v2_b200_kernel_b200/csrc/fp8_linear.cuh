// y[i, n] = sum_b sx[i, b] sw[n / 128, b] sum_{k in block b} x[i, k] w[n, k] + bias[n] with x and w in
// 8-bit floating point (e4m3), blocks of 128 along the depth.
//
// A block's products are the matrix instructions'; what joins the blocks is 32-bit arithmetic outside them,
// since the scales differ: a tensor-core accumulator holds one block of the depth only, and is added,
// scaled, to sums in registers while the next block is multiplied into another one.
#pragma once

#include "codes.cuh"
#include "fp8_rows.cuh"

namespace qrb200 {

struct Fp8Params {
  const float* sx;  // rows x blocks
  const float* sw;  // (outs / 128) x blocks
  const void* bias;  // may be null; y's type
  void* y;
  int rows, outs, depth, blocks;  // blocks of the depth
  int tiles_n, tiles;             // wide kernel: channel tiles, all tiles
};

// kind::f8f6f4: e4m3 operands, both K-major, 32-bit floating accumulator.
__host__ __device__ constexpr uint32_t fp8_idesc(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void fp8_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
      :
      : "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void fp8_mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
      :
      : "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}

// ---- up to eight rows -----------------------------------------------------------------------
//
// The time is that of reading the weights once, and at these sizes mostly latency. A CTA takes 16 channels, a warp every
// sixteenth block of the depth: weights, straight from memory, are the 16-row operand of the warp-level matrix instruction and
// rows of x its columns; the order of a block's products is free, so a lane's 32 bytes of a row are two wide loads. Many warps
// with a block each in flight: 1 x 4096 x 4096 4.3 us, 3.9 TB/s of weights.
struct Fp8RowsOperands {
  Fp8Params p;
  I8Operand x, w;
};
constexpr int kFp8RowsWarps = 16;

__device__ __forceinline__ void fp8_mma_warp(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T, bool kAligned>
__global__ void __launch_bounds__(32 * kFp8RowsWarps, 2) fp8_rows_linear_kernel(Fp8RowsOperands R) {
  __shared__ float s_sum[kFp8RowsWarps][8][17];
  griddep_launch_wait();
  const Fp8Params& P = R.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16;
  const float* sw = P.sw + (long long)(n0 / kFp8Block) * P.blocks;
  const long long wr[2] = {min(n0 + g, P.outs - 1), min(n0 + g + 8, P.outs - 1)};
  float acc[4] = {};
  for (int b = warp; b < P.blocks; b += kFp8RowsWarps) {
    uint4 w[2][2], x[2];
    const bool whole = kAligned && (b + 1) * kFp8Block <= P.depth;
    const auto get = [&](const I8Operand& o, long long row, int k) {
      return whole         ? __ldg(reinterpret_cast<const uint4*>(o.base + row * o.stride + k))
             : k < P.depth ? i8_codes16<kAligned>(o, row, k, P.depth)
                           : make_uint4(0, 0, 0, 0);
    };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = b * kFp8Block + 64 * h + 16 * t;
#pragma unroll
      for (int r = 0; r < 2; ++r) w[r][h] = get(R.w, wr[r], k);
      x[h] = g < P.rows ? get(R.x, g, k) : make_uint4(0, 0, 0, 0);
    }
    const float ws = __ldg(sw + b);
    float s[2], d[4] = {};
#pragma unroll
    for (int c = 0; c < 2; ++c) s[c] = 2 * t + c < P.rows ? __ldg(P.sx + (long long)(2 * t + c) * P.blocks + b) * ws : 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      fp8_mma_warp(d, w[0][h].x, w[1][h].x, w[0][h].y, w[1][h].y, x[h].x, x[h].y);
      fp8_mma_warp(d, w[0][h].z, w[1][h].z, w[0][h].w, w[1][h].w, x[h].z, x[h].w);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(d[e], s[e & 1], acc[e]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) s_sum[warp][2 * t + (e & 1)][g + 8 * (e >> 1)] = acc[e];
  __syncthreads();
  const int row = threadIdx.x >> 4, n = n0 + (threadIdx.x & 15);
  if (row >= P.rows || n >= P.outs) return;
  float sum = P.bias ? to_f32(static_cast<const T*>(P.bias)[n]) : 0.f;
#pragma unroll
  for (int i = 0; i < kFp8RowsWarps; ++i) sum += s_sum[i][row][threadIdx.x & 15];
  static_cast<T*>(P.y)[(long long)row * P.outs + n] = from_f32<T>(sum);
}

// ---- few rows ------------------------------------------------------------------------------
//
// The weights are the traffic, so they are the 128-row operand (M = output channels) and the rows of x
// the narrow one (N = kBN). The depth is cut over the cluster's CTAs so that every SM streams weights; each
// CTA then adds all the CTAs' sums of some rows of x, in their order, through distributed shared memory.
//
// Warp 0 issues the loads, warp 1 the MMAs into two accumulators in turn, warps 2-5 hold one output
// channel a lane and kBN sums each. 4096 x 4096: 9 to 16 rows 6.3-6.5 us, 64 8.4, 128 10.7, that is 2.6 to 1.6 TB/s of weights: the
// set-up, the first loads and the join of the cut depth, one after another (issue slots 16 % busy, tensor pipe 11 %; 333 x 1000 x 2000 8.4).
constexpr int kFp8Split = 4;  // the most CTAs that share a tile's depth
constexpr int kFp8Scales = 8;  // blocks whose scales are held at a time
template <int kBN>
struct Fp8Few {
  static constexpr int kStage = 128 * kI8Depth + kBN * kI8Depth;
  static constexpr int kStages = kBN <= 32 ? 6 : kBN == 64 ? 5 : 6;
  static constexpr int kCols = 2 * kBN;  // TMEM columns
  static constexpr size_t smem() { return 1024 + (size_t)kStages * kStage; }
  static_assert(kBN * 128 * 4 <= kStages * kStage, "the sums take the ring's place");
};

template <typename T, int kBN>
__global__ void __launch_bounds__(192) fp8_few_kernel(Fp8Params P, const __grid_constant__ CUtensorMap tm_w,
                                                      const __grid_constant__ CUtensorMap tm_x) {
  using C = Fp8Few<kBN>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ uint64_t full[C::kStages], empty[C::kStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_bad;
  __shared__ __align__(16) float s_scale[2][kFp8Scales][kBN];
  unsigned char* ring = align1024(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * 128, i0 = blockIdx.y * kBN;
  const int split = gridDim.z, part = blockIdx.z;
  const int k_lo = (int)((long long)P.blocks * part / split), k_hi = (int)((long long)P.blocks * (part + 1) / split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], 4);
    }
    s_bad = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
    prefetch_map(&tm_w);
    prefetch_map(&tm_x);
  }
  griddep_launch_wait();  // before TMEM is taken: a kernel still running may need it
  if (warp == 1) tmem_alloc(&s_tmem, C::kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  const int ch = ((warp & 3) << 5) + lane;  // the channel, and the TMEM lane, of warps 2-5
  const bool epi = warp >= 2;
  const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  float acc[kBN];
#pragma unroll
  for (int j = 0; j < kBN; ++j) acc[j] = 0.f;

  if (warp == 0 && lane == 0) {
    int issued = 0;
    for (int k = k_lo; k < k_hi; ++k, ++issued) {
      const int s = issued % C::kStages, turn = issued / C::kStages;
      if (turn > 0 && !mbar_wait_quick(&empty[s], (turn - 1) & 1)) {
        s_bad = 1;
        break;
      }
      const uint32_t at = smem_u32(ring) + s * C::kStage, bar = smem_u32(&full[s]);
      i8_expect(bar, C::kStage);
      i8_load(at, &tm_w, bar, k * kI8Depth, n0);
      i8_load(at + 128 * kI8Depth, &tm_x, bar, k * kI8Depth, i0);
    }
    // Whatever happened, no load is in flight when this CTA ends.
    for (int j = max(0, issued - C::kStages); j < issued; ++j)
      if (!mbar_wait_quick(&full[j % C::kStages], (j / C::kStages) & 1)) s_bad = 1;
  } else if (warp == 1) {
    constexpr uint32_t idesc = fp8_idesc(128, kBN);
    const uint64_t w0 = i8_sdesc(smem_u32(ring)), x0 = i8_sdesc(smem_u32(ring) + 128 * kI8Depth);
    uint32_t s = 0, turn = 0;
    for (int j = 0; j < k_hi - k_lo; ++j) {
      const uint32_t buf = j & 1;
      if (!__all_sync(kFullMask, (j < 2 || mbar_wait_quick(&acc_empty[buf], ((j >> 1) - 1) & 1)) && mbar_wait_quick(&full[s], turn))) {
        s_bad = 1;
        break;
      }
      tc_fence_after();
      const uint64_t at = s * (C::kStage >> 4);
      if (elect_one()) {
#pragma unroll
        for (int c = 0; c < kI8Depth / 32; ++c) fp8_mma(tmem + buf * kBN, w0 + at + 2 * c, x0 + at + 2 * c, idesc, c > 0);
        mma_commit(&empty[s]);
        mma_commit(&acc_full[buf]);
      }
      __syncwarp();
      if (++s == C::kStages) s = 0, turn ^= 1;
    }
    // The last products are over before anybody reuses the ring (the accumulators say so) or TMEM is freed.
  } else if (epi) {
    // Both scales' products for some blocks at a time: a row and four of those blocks, or fewer, to a thread.
    const float* sw = P.sw + (long long)blockIdx.x * P.blocks;
    constexpr int kMine = (kFp8Scales * kBN + 127) / 128;
    float next[kMine];
    const int tid = threadIdx.x - 64;
    const auto ask = [&](int k0) {
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int at = tid + 128 * i, k = k0 + at % kFp8Scales, row = i0 + at / kFp8Scales;
        next[i] = at < kFp8Scales * kBN && k < k_hi && row < P.rows ? P.sx[(long long)row * P.blocks + k] * sw[k] : 0.f;
      }
    };
    ask(k_lo);
    bool ok = true;
    for (int k0 = k_lo, j = 0; k0 < k_hi; k0 += kFp8Scales) {
      float(*scale)[kBN] = s_scale[(j / kFp8Scales) & 1];
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int at = tid + 128 * i;
        if (at < kFp8Scales * kBN) scale[at % kFp8Scales][at / kFp8Scales] = next[i];
      }
      named_sync(1, 128);  // also: what the other buffer held has been used
      ask(k0 + kFp8Scales);
      for (int k = k0; k < min(k_hi, k0 + kFp8Scales); ++k, ++j) {
        const int buf = j & 1;
        ok = ok && warp_wait_quick(&acc_full[buf], (j >> 1) & 1);
        if (!ok) continue;
        tc_fence_after();
        float v[2][16];
        tmem_ask16(lanes + buf * kBN, v[0]);
#pragma unroll
        for (int c = 0; c < kBN / 16; ++c) {
          tmem_arrived(v[c & 1]);
          if (c + 1 < kBN / 16) tmem_ask16(lanes + buf * kBN + 16 * (c + 1), v[(c + 1) & 1]);
          if (c + 1 == kBN / 16) {  // every sum of this warp is in registers
            tc_fence_before();
            if (lane == 0) mbar_arrive(&acc_empty[buf]);
          }
#pragma unroll
          for (int q = 0; q < 16; q += 4) {
            const float4 s4 = *reinterpret_cast<const float4*>(&scale[k - k0][16 * c + q]);
            acc[16 * c + q] = fmaf(v[c & 1][q], s4.x, acc[16 * c + q]);
            acc[16 * c + q + 1] = fmaf(v[c & 1][q + 1], s4.y, acc[16 * c + q + 1]);
            acc[16 * c + q + 2] = fmaf(v[c & 1][q + 2], s4.z, acc[16 * c + q + 2]);
            acc[16 * c + q + 3] = fmaf(v[c & 1][q + 3], s4.w, acc[16 * c + q + 3]);
          }
        }
      }
    }
    if (!ok) s_bad = 1;
  }
  __syncwarp();
  // Four channels a lane for the way out.
  const int c4 = 4 * lane;
  float b4[4] = {};
  if (epi && P.bias) {
#pragma unroll
    for (int c = 0; c < 4; ++c) b4[c] = n0 + c4 + c < P.outs ? to_f32(static_cast<const T*>(P.bias)[n0 + c4 + c]) : 0.f;
  }
  tc_fence_before();
  __syncthreads();
  // The ring is free (every load has landed, every MMA is done): sums as [row][channel]. Row j is
  // CTA j % split's to add and to write, a warp to a row.
  float* sums = reinterpret_cast<float*>(ring);
  if (epi)
#pragma unroll
    for (int j = 0; j < kBN; ++j) sums[j * 128 + ch] = acc[j];
  bool bad = false;
  if (split > 1) {
    cluster_sync();
    for (int r = 0; r < split; ++r) bad = ld_cluster(smem_u32(&s_bad), r) != 0 || bad;
  } else {
    __syncthreads();
    bad = s_bad != 0;
  }
  if (epi && !bad) {
    T* y = static_cast<T*>(P.y);
    const bool whole = P.outs % 4 == 0;
    for (int j = part + split * (warp - 2); j < kBN && i0 + j < P.rows; j += 4 * split) {
      float4 sum = make_float4(b4[0], b4[1], b4[2], b4[3]);
#pragma unroll
      for (int r = 0; r < kFp8Split; ++r)
        if (r < split) {
          float4 v;
          if (split == 1) {
            v = *reinterpret_cast<const float4*>(&sums[j * 128 + c4]);
          } else {
            const int4 i = ld_cluster4(smem_u32(&sums[j * 128 + c4]), r);
            v = make_float4(__int_as_float(i.x), __int_as_float(i.y), __int_as_float(i.z), __int_as_float(i.w));
          }
          sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
      alignas(16) T out[4];
      put2(out, sum.x, sum.y);
      put2(out + 2, sum.z, sum.w);
      T* to = y + (long long)(i0 + j) * P.outs + n0 + c4;
      if (whole) {
        if (n0 + c4 < P.outs) {
          if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(out);
          else *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(out);
        }
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (n0 + c4 + c < P.outs) to[c] = out[c];
      }
    }
  }
  if (split > 1) cluster_sync();  // nobody leaves while its sums are being read
  tc_fence_after();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, C::kCols);
}

// ---- many rows -----------------------------------------------------------------------------
//
// 256 rows x 256 channels per pair of CTAs (cta_group::2: each CTA holds 128 rows of x, 128 of the
// channels' weights and its rows' 128 x 256 sums), persistent. Warp 0 loads its CTA's halves, warp 1 of the
// pair's first CTA issues the MMAs, a block of the depth into each of two accumulators in TMEM in turn; warps
// 4-11 add each block, scaled, to the 128 sums a lane that they hold in registers: a row to a lane, and the
// 128 channels of one block of the weights to a warp, so that both scales are one factor. They take the
// registers that warps 0-3 have no use for.
//
// A block's products take 512 clocks, and its accumulator must be free again 512 later. Between lie the
// commit, the epilogue's loads and the other CTA's word, so what those wait for is kept short:
// * one warp of a CTA asks the memory barriers for the eight, and passes the word on by named barriers.
//   On each of those the same nine warps wait for one another, block after block, so that they stay in step where a wait for the memory ran
//   out and nothing else holds them back;
// * half of a block's sums are loaded at once, and the accumulator is free before the last half is added;
// * the scales of four blocks come in one load (32 lines a warp's load, it holds up the barriers behind it).
// 8192 x 8192 x 4096: 239 us, 2.3 P op/s; without the additions (one accumulator over the depth, one scale a row
// and channel) the same products take 207 us under the power cap.
constexpr int kFp8WideStage = 2 * 128 * kI8Depth;  // bytes per CTA and stage
constexpr int kFp8WideStages = 5;
constexpr int kFp8WideEpi = 8;  // epilogue warps
constexpr int kFp8Hand = 32 * kFp8WideEpi + 32;  // threads of a named barrier between them and warp 2 or 3
constexpr int kFp8Pitch = 144;  // bytes of a staged output row (128 and 16 to spread the banks)
constexpr size_t fp8_wide_smem() { return 1024 + (size_t)kFp8WideStages * kFp8WideStage + kFp8WideEpi * 32 * kFp8Pitch; }

template <typename T>
__global__ void __launch_bounds__(128 + 32 * kFp8WideEpi, 1) __cluster_dims__(2, 1, 1)
    fp8_wide_kernel(Fp8Params P, const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ uint64_t full[kFp8WideStages], done[kFp8WideStages], acc_empty[2];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_bad;  // a wait ran out: keep to the barriers, write nothing
  unsigned char* ring = align1024(smem_raw);
  unsigned char* staged = ring + kFp8WideStages * kFp8WideStage;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1, nk = P.blocks;

  if (threadIdx.x == 0) {
    s_bad = 0;
    for (int s = 0; s < kFp8WideStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&done[s], 1);
    }
    for (int s = 0; s < 2; ++s) mbar_init(&acc_empty[s], 2);  // both CTAs
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
    prefetch_map(&tm_w);
    prefetch_map(&tm_x);
  }
  griddep_launch_wait();  // before TMEM is taken: a kernel still running may need it
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are initialised
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  // Tiles run down the rows within bands of kBand channel tiles, so that the tiles in flight share
  // both operands in L2.
  constexpr int kBand = 8;
  const int tiles_m = P.tiles / P.tiles_n;
  auto place = [&](int tile, int& m, int& n) {
    const int band = tile / (kBand * tiles_m), in = tile - band * kBand * tiles_m;
    const int width = min(kBand, P.tiles_n - band * kBand);
    m = in / width;
    n = band * kBand + in % width;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");  // 128 x 40 + 256 x 232 = the launch's 384 x 168
    if (warp == 0 && lane == 0) {
      int issued = 0;
      bool ok = true;
      for (int tile = pair; tile < P.tiles && ok; tile += pairs) {
        int m, n;
        place(tile, m, n);
        for (int k = 0; k < nk; ++k, ++issued) {
          const int s = issued % kFp8WideStages, turn = issued / kFp8WideStages;
          if (turn > 0 && !mbar_wait_quick(&done[s], (turn - 1) & 1)) {
            ok = false;
            break;
          }
          const uint32_t at = smem_u32(ring) + s * kFp8WideStage, bar = pair_leader(smem_u32(&full[s]));
          if (rank == 0) i8_expect(smem_u32(&full[s]), 2 * kFp8WideStage);
          i8_load_pair(at, &tm_x, bar, k * kI8Depth, m * 256 + (int)rank * 128);
          i8_load_pair(at + 128 * kI8Depth, &tm_w, bar, k * kI8Depth, n * 256 + (int)rank * 128);
        }
      }
      // No load is in flight when the pair ends: the loads of both CTAs land on the leader's
      // barriers, and `done` says that the last use of each stage is over.
      for (int j = max(0, issued - kFp8WideStages); j < issued; ++j)
        mbar_wait_quick(&done[j % kFp8WideStages], (j / kFp8WideStages) & 1);
    } else if (warp == 1 && rank == 0) {
      constexpr uint32_t idesc = fp8_idesc(256, 256);
      const uint64_t x0 = i8_sdesc(smem_u32(ring)), w0 = i8_sdesc(smem_u32(ring) + 128 * kI8Depth);
      uint32_t s = 0, turn = 0, j = 0;
      bool ok = true;
      for (int tile = pair; tile < P.tiles && ok; tile += pairs)
        for (int k = 0; k < nk; ++k, ++j) {
          const uint32_t buf = j & 1;
          ok = __all_sync(kFullMask, mbar_wait_quick(&full[s], turn) && (j < 2 || mbar_wait_quick(&acc_empty[buf], ((j >> 1) - 1) & 1)));
          if (!ok) break;
          tc_fence_after();
          const uint64_t at = s * (kFp8WideStage >> 4);
          if (elect_one()) {
#pragma unroll
            for (int c = 0; c < kI8Depth / 32; ++c) fp8_mma_pair(tmem + buf * 256, x0 + at + 2 * c, w0 + at + 2 * c, idesc, c > 0);
            commit_pair(&done[s]);
          }
          __syncwarp();
          if (++s == kFp8WideStages) s = 0, turn ^= 1;
        }
    } else if (warp == 2) {
      // Tells the epilogue warps that a block is done: one warp asks the barrier in their stead.
      uint32_t s = 0, turn = 0, j = 0;
      for (int tile = pair; tile < P.tiles; tile += pairs)
        for (int k = 0; k < nk; ++k, ++j) {
          if (!s_bad && !mbar_wait_quick(&done[s], turn)) s_bad = 1;
          __syncwarp();
          named_sync(1 + (j & 1), kFp8Hand);
          if (++s == kFp8WideStages) s = 0, turn ^= 1;
        }
    } else if (warp == 3) {
      // Tells the MMAs' warp that the epilogue warps hold a block's sums. (Relaxed: nothing in memory hangs on it, and a
      // release would wait for what has been asked for.)
      uint32_t j = 0;
      for (int tile = pair; tile < P.tiles; tile += pairs)
        for (int k = 0; k < nk; ++k, ++j) {
          named_sync(3 + (j & 1), kFp8Hand);
          if (lane == 0)
            asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(pair_leader(smem_u32(&acc_empty[j & 1])))
                         : "memory");
        }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    constexpr int kPer = 128 / sizeof(T);  // outputs in a staged row of 128 bytes
    const int ew = warp & 3, half = (warp - 4) >> 2;
    unsigned char* mine = staged + (warp - 4) * 32 * kFp8Pitch;
    const uint32_t lanes = tmem + ((uint32_t)(ew * 32) << 16) + 128 * half;
    const bool wide = P.outs % (16 / (int)sizeof(T)) == 0;  // 16-byte rows of y (y itself is 16-byte aligned)
    const bool fours = nk % 4 == 0 && ((reinterpret_cast<uintptr_t>(P.sx) | reinterpret_cast<uintptr_t>(P.sw)) & 15u) == 0;
    T* y = static_cast<T*>(P.y);
    uint32_t j = 0;
    for (int tile = pair; tile < P.tiles; tile += pairs) {
      int m, n;
      place(tile, m, n);
      const int n0 = n * 256 + 128 * half, row0 = m * 256 + (int)rank * 128 + ew * 32;
      const bool real = row0 + lane < P.rows && n0 < P.outs;
      const float* sx = P.sx + (long long)(real ? row0 + lane : 0) * nk;
      const float* sw = P.sw + (long long)(real ? n0 / kFp8Block : 0) * nk;
      // The scales of four blocks at a time, asked for four ahead.
      alignas(16) float scale[4] = {}, next_x[4] = {}, next_w[4] = {};
      const auto ask = [&](int k) {
        if (fours) {
          if (k < nk) {
            *reinterpret_cast<float4*>(next_x) = __ldg(reinterpret_cast<const float4*>(sx + k));
            *reinterpret_cast<float4*>(next_w) = __ldg(reinterpret_cast<const float4*>(sw + k));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (k + i < nk) next_x[i] = __ldg(sx + k + i), next_w[i] = __ldg(sw + k + i);
        }
      };
      ask(0);
      float2 acc[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i] = make_float2(0.f, 0.f);
      for (int k = 0; k < nk; ++k, ++j) {
        const int buf = j & 1;
        if ((k & 3) == 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) scale[i] = next_x[i] * next_w[i];
          ask(k + 4);
        }
        const float both = (k & 2) ? (k & 1) ? scale[3] : scale[2] : (k & 1) ? scale[1] : scale[0];
        named_sync(1 + buf, kFp8Hand);
        tc_fence_after();
        // Half of the columns are asked for at once and the others as those are added, so that the accumulator
        // is free before the last half is.
        float v[4][16];
        const auto add = [&](int c) {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            acc[8 * c + q] = __ffma2_rn(make_float2(v[c & 3][2 * q], v[c & 3][2 * q + 1]), make_float2(both, both), acc[8 * c + q]);
        };
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ask16(lanes + buf * 256 + 16 * c, v[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_arrived(v[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          add(c);
          tmem_ask16(lanes + buf * 256 + 16 * (c + 4), v[c]);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_arrived(v[c]);
        tc_fence_before();
        named_sync(3 + buf, kFp8Hand);
#pragma unroll
        for (int c = 4; c < 8; ++c) add(c);
      }
      if (s_bad) continue;
#pragma unroll
      for (int c0 = 0; c0 < 128; c0 += kPer) {
        __syncwarp();
#pragma unroll
        for (int q = 0; q < kPer; q += 16 / (int)sizeof(T)) {
          alignas(16) T out[16 / sizeof(T)];
#pragma unroll
          for (int e = 0; e < 16 / (int)sizeof(T); e += 2) {
            float2 sum = acc[(c0 + q + e) / 2];
            if (P.bias) {
              const int c = n0 + c0 + q + e;
              if (c < P.outs) sum.x += to_f32(static_cast<const T*>(P.bias)[c]);
              if (c + 1 < P.outs) sum.y += to_f32(static_cast<const T*>(P.bias)[c + 1]);
            }
            put2(out + e, sum.x, sum.y);
          }
          *reinterpret_cast<uint4*>(mine + lane * kFp8Pitch + q * sizeof(T)) = *reinterpret_cast<const uint4*>(out);
        }
        __syncwarp();
        const int left = P.outs - n0 - c0;  // columns of this chunk that exist
        if (left <= 0) continue;
        if (wide) {
          const int piece = lane & 7, col = piece * (16 / (int)sizeof(T));
#pragma unroll
          for (int r = lane >> 3; r < 32; r += 4)
            if (row0 + r < P.rows && col < left)
              *reinterpret_cast<uint4*>(y + (long long)(row0 + r) * P.outs + n0 + c0 + col) =
                  *reinterpret_cast<const uint4*>(mine + r * kFp8Pitch + 16 * piece);
        } else {
          // Rows off 16-byte boundaries: a row's chunk by aligned pairs (16-bit results), or
          // element beside element.
          const int count = min(kPer, left);
#pragma unroll 4
          for (int r = 0; r < 32 && row0 + r < P.rows; ++r) {
            const T* from = reinterpret_cast<const T*>(mine + r * kFp8Pitch);
            T* to = y + (long long)(row0 + r) * P.outs + n0 + c0;
            if constexpr (sizeof(T) == 2) {
              const int odd = (int)(reinterpret_cast<uintptr_t>(to) >> 1 & 1), c = 2 * lane + odd;
              if (odd && lane == 0) to[0] = from[0];
              if (c + 1 < count) {
                alignas(4) const T two[2] = {from[c], from[c + 1]};
                *reinterpret_cast<uint32_t*>(to + c) = *reinterpret_cast<const uint32_t*>(two);
              } else if (c < count) {
                to[c] = from[c];
              }
            } else if (lane < count) {
              to[lane] = from[lane];
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the pair's products, loads and arrivals are over in both CTAs
  if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

}  // namespace qrb200
