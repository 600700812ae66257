// y[i, n] = (sum_k x[i, k] w[n, k]) sx[i] sw[n] + bias[n] with 8-bit x and w.
//
// The sum is held in 32-bit integers, so it is exact (depth <= 131071 keeps 128^2 depth below
// 2^31) and any split of the depth gives the same bits; the scales are applied in 32 bits and
// the result is rounded once.
#pragma once

#include "codes.cuh"
#include "quant_rows.cuh"

namespace qrb200 {

struct I8Params {
  const float* sx;
  const float* sw;
  const void* bias;  // may be null; y's type
  void* y;
  int rows, outs, depth;
  int tiles_n, tiles;  // wide kernel: channel tiles, all tiles
};

// kind::i8: signed 8-bit operands, both K-major, 32-bit integer accumulator.
__host__ __device__ constexpr uint32_t i8_idesc(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void i8_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n"
      :
      : "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, int (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld32i(uint32_t taddr, int (&v)[32]) {
  float f[32];
  tmem_ld32(taddr, f);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __float_as_int(f[i]);
}

// ---- one to four rows ----------------------------------------------------------------------
//
// The time is that of reading the weights once, and at these sizes mostly latency: no tiles,
// barriers or tensor memory, just wide loads into four-way dot products, and operands as they lie.
// A warp takes two channels, a lane 16 codes of each 512; sums are joined by the warp's integer
// reduction. (1 x 4096 x 4096: 6.6 us through the tensor cores, 3.2 us here, 5.2 TB/s of weights
// that L2 holds.)
struct I8RowsParams {
  I8Params p;
  I8Operand x, w;
};

template <typename T, int kM, bool kAligned>  // kM rows, or fewer of four
__global__ void __launch_bounds__(128) i8_rows_kernel(I8RowsParams R) {
  constexpr int kUnroll = kM <= 2 ? 4 : 2;
  griddep_launch_wait();
  const I8Params& P = R.p;
  const int lane = threadIdx.x & 31, n = (blockIdx.x * 4 + (threadIdx.x >> 5)) * 2;
  if (n >= P.outs) return;
  const int n1 = min(n + 1, P.outs - 1);
  const int8_t* w0 = R.w.base + n * R.w.stride;
  const int8_t* w1 = R.w.base + n1 * R.w.stride;
  int acc[kM][2] = {};
  for (int k0 = 16 * lane; k0 < P.depth; k0 += 512 * kUnroll) {
    uint4 w[kUnroll][2], x[kUnroll][kM];
    if (kAligned && k0 - 16 * lane + 512 * kUnroll <= P.depth) {  // all in range: every load is asked for at once
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        w[u][0] = __ldg(reinterpret_cast<const uint4*>(w0 + k0 + 512 * u));
        w[u][1] = __ldg(reinterpret_cast<const uint4*>(w1 + k0 + 512 * u));
#pragma unroll
        for (int m = 0; m < kM; ++m)
          x[u][m] = __ldg(reinterpret_cast<const uint4*>(R.x.base + (kM <= 2 ? m : min(m, P.rows - 1)) * R.x.stride + k0 + 512 * u));
      }
    } else {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int k = k0 + 512 * u;
        const bool in = k < P.depth;
        w[u][0] = in ? i8_codes16<kAligned>(R.w, n, k, P.depth) : make_uint4(0, 0, 0, 0);
        w[u][1] = in ? i8_codes16<kAligned>(R.w, n1, k, P.depth) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < kM; ++m) x[u][m] = in && m < P.rows ? i8_codes16<kAligned>(R.x, m, k, P.depth) : make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int m = 0; m < kM; ++m)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          acc[m][c] = __dp4a((int)w[u][c].x, (int)x[u][m].x, acc[m][c]);
          acc[m][c] = __dp4a((int)w[u][c].y, (int)x[u][m].y, acc[m][c]);
          acc[m][c] = __dp4a((int)w[u][c].z, (int)x[u][m].z, acc[m][c]);
          acc[m][c] = __dp4a((int)w[u][c].w, (int)x[u][m].w, acc[m][c]);
        }
  }
#pragma unroll
  for (int m = 0; m < kM; ++m)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int sum = __reduce_add_sync(kFullMask, acc[m][c]);
      if (lane == 2 * m + c && m < P.rows && n + c < P.outs) {
        const float b = P.bias ? to_f32(static_cast<const T*>(P.bias)[n + c]) : 0.f;
        static_cast<T*>(P.y)[(long long)m * P.outs + n + c] = from_f32<T>(fmaf((float)sum * P.sx[m], P.sw[n + c], b));
      }
    }
}

// ---- few rows ------------------------------------------------------------------------------
//
// With few rows the weights are the traffic, so they are the 128-row operand (M = output channels)
// and the rows of x the narrow one (N = kBN): no tensor-core row is wasted on padding. The depth is
// cut over the cluster's CTAs so that every SM streams weights; each CTA then adds all the CTAs'
// integer sums of some rows of x, exactly, through distributed shared memory, in the one launch.
//
// Warp 0 issues the loads, warp 1 the MMAs, warps 2-5 hold one output channel a lane.
// 16 x 4096 x 4096: 5.9 us, 2.9 TB/s of weights; 128 rows 8.7 us; 333 x 1000 x 2048 7.1 us. Some
// 4 us of each are set-up, the first loads, the join and the way out.
constexpr int kI8Split = 4;  // the most CTAs that share a tile's depth
template <int kBN>
struct I8Few {
  static constexpr int kStage = 128 * kI8Depth + kBN * kI8Depth;
  // Loads in flight hide their latency: about 100 KB, which leaves room for the next kernel's
  // set-up, or, for the largest tile, what one CTA can have.
  static constexpr int kStages = kBN <= 32 ? 6 : kBN == 64 ? 5 : 6;
  static constexpr int kCols = kBN < 32 ? 32 : kBN;  // TMEM columns
  static constexpr size_t smem() { return 1024 + (size_t)kStages * kStage; }
  static_assert(kBN * 128 * 4 <= kStages * kStage, "the sums take the ring's place");
};

template <typename T, int kBN>
__global__ void __launch_bounds__(192) i8_few_kernel(I8Params P, const __grid_constant__ CUtensorMap tm_w,
                                                     const __grid_constant__ CUtensorMap tm_x) {
  using C = I8Few<kBN>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ uint64_t full[C::kStages], empty[C::kStages], done;
  __shared__ uint32_t s_tmem;
  __shared__ int s_bad;
  __shared__ float s_sx[kBN];
  unsigned char* ring = align1024(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * 128, i0 = blockIdx.y * kBN;
  const int split = gridDim.z, part = blockIdx.z;
  const int nk = (P.depth + kI8Depth - 1) / kI8Depth;
  const int k_lo = (int)((long long)nk * part / split), k_hi = (int)((long long)nk * (part + 1) / split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
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

  if (warp == 0 && lane == 0) {
    int issued = 0;
    for (int k = k_lo; k < k_hi; ++k, ++issued) {
      const int s = issued % C::kStages, turn = issued / C::kStages;
      if (turn > 0 && !mbar_wait(&empty[s], (turn - 1) & 1)) {
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
      if (!mbar_wait(&full[j % C::kStages], (j / C::kStages) & 1)) s_bad = 1;
  } else if (warp == 1 && lane == 0) {
    constexpr uint32_t idesc = i8_idesc(128, kBN);
    int j = 0;
    for (int k = k_lo; k < k_hi; ++k, ++j) {
      const int s = j % C::kStages;
      if (!mbar_wait(&full[s], (j / C::kStages) & 1)) {
        s_bad = 1;
        break;
      }
      tc_fence_after();
      const uint32_t at = smem_u32(ring) + s * C::kStage;
#pragma unroll
      for (int c = 0; c < kI8Depth / 32; ++c)
        i8_mma(tmem, i8_sdesc(at + 32 * c), i8_sdesc(at + 128 * kI8Depth + 32 * c), idesc, j > 0 || c > 0);
      mma_commit(&empty[s]);
    }
    mma_commit(&done);
  }
  __syncwarp();
  const int ch = ((warp & 3) << 5) + lane;  // the channel, and the TMEM lane, of warps 2-5
  const bool epi = warp >= 2;
  const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  // Four channels a lane for the way out, their scales and bias asked for while the products run.
  const int c4 = 4 * lane;
  float w4[4] = {}, b4[4] = {};
  if (epi) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const bool in = n0 + c4 + c < P.outs;
      w4[c] = in ? P.sw[n0 + c4 + c] : 0.f;
      b4[c] = in && P.bias ? to_f32(static_cast<const T*>(P.bias)[n0 + c4 + c]) : 0.f;
    }
    for (int j = threadIdx.x - 64; j < kBN; j += 128) s_sx[j] = i0 + j < P.rows ? P.sx[i0 + j] : 0.f;
    if (!mbar_wait(&done, 0)) s_bad = 1;
  }
  tc_fence_after();
  __syncthreads();
  // The ring is free (every load has landed, every MMA is done): sums as [row][channel]. Row j is
  // CTA j % split's to add and to write, a warp to a row.
  int* sums = reinterpret_cast<int*>(ring);
  if (epi)
#pragma unroll 1
    for (int j = 0; j < kBN && i0 + j < P.rows; j += 16) {
      int v[16];
      tmem_ld16(lanes + j, v);
#pragma unroll
      for (int q = 0; q < 16; ++q) sums[(j + q) * 128 + ch] = v[q];
    }
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
      int4 acc = make_int4(0, 0, 0, 0);
      if (split == 1) {
        acc = *reinterpret_cast<const int4*>(&sums[j * 128 + c4]);
      } else {
#pragma unroll
        for (int r = 0; r < kI8Split; ++r)
          if (r < split) {
            const int4 v = ld_cluster4(smem_u32(&sums[j * 128 + c4]), r);
            acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
          }
      }
      const float sx = s_sx[j];
      alignas(16) T out[4];
      put2(out, fmaf((float)acc.x * sx, w4[0], b4[0]), fmaf((float)acc.y * sx, w4[1], b4[1]));
      put2(out + 2, fmaf((float)acc.z * sx, w4[2], b4[2]), fmaf((float)acc.w * sx, w4[3], b4[3]));
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
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, C::kCols);
}

// ---- many rows -----------------------------------------------------------------------------
//
// 256 rows x 256 channels per pair of CTAs (cta_group::2: each CTA holds 128 rows of x, 128 of the
// channels' weights and its rows' 128 x 256 sums), persistent, with two accumulators in TMEM so
// that a tile's epilogue runs under the next tile's products. Warp 0 loads its CTA's halves, warp 1
// of the pair's first CTA issues the MMAs, warps 4-11 scale, round and store, half of a tile's
// channels each four.
// 8192 x 8192 x 4096: 187 us, 2.95 P op/s, the tensor pipe 76 % active under the power cap;
// 4096 x 4096 x 512 16.5 us, bound by the epilogue.
constexpr int kI8WideStage = 2 * 128 * kI8Depth;  // bytes per CTA and stage
constexpr int kI8WideStages = 5;
constexpr int kI8WideEpi = 8;  // epilogue warps
constexpr int kI8Pitch = 144;  // bytes of a staged output row (128 and 16 to spread the banks)
constexpr size_t i8_wide_smem() { return 1024 + (size_t)kI8WideStages * kI8WideStage + kI8WideEpi * 32 * kI8Pitch; }

__device__ __forceinline__ void i8_mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n"
      :
      : "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
template <typename T>
__global__ void __launch_bounds__(128 + 32 * kI8WideEpi, 1) __cluster_dims__(2, 1, 1)
    i8_wide_kernel(I8Params P, const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ uint64_t full[kI8WideStages], empty[kI8WideStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t s_tmem;
  __shared__ __align__(16) float s_sw[2][256], s_b[2][256];
  unsigned char* ring = align1024(smem_raw);
  unsigned char* staged = ring + kI8WideStages * kI8WideStage;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int nk = (P.depth + kI8Depth - 1) / kI8Depth;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kI8WideStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], 2 * kI8WideEpi);  // the epilogue warps of both CTAs
    }
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

  if (warp == 0 && lane == 0) {
    int issued = 0;
    bool ok = true;
    for (int tile = pair; tile < P.tiles && ok; tile += pairs) {
      int m, n;
      place(tile, m, n);
      for (int k = 0; k < nk; ++k, ++issued) {
        const int s = issued % kI8WideStages, turn = issued / kI8WideStages;
        if (turn > 0 && !mbar_wait(&empty[s], (turn - 1) & 1)) {
          ok = false;
          break;
        }
        const uint32_t at = smem_u32(ring) + s * kI8WideStage, bar = pair_leader(smem_u32(&full[s]));
        if (rank == 0) i8_expect(smem_u32(&full[s]), 2 * kI8WideStage);
        i8_load_pair(at, &tm_x, bar, k * kI8Depth, m * 256 + (int)rank * 128);
        i8_load_pair(at + 128 * kI8Depth, &tm_w, bar, k * kI8Depth, n * 256 + (int)rank * 128);
      }
    }
    // No load is in flight when the pair ends: the loads of both CTAs land on the leader's
    // barriers, and `empty` says that the last use of each stage is over.
    for (int j = max(0, issued - kI8WideStages); j < issued; ++j)
      mbar_wait(&empty[j % kI8WideStages], (j / kI8WideStages) & 1);
  } else if (warp == 1 && lane == 0 && rank == 0) {
    constexpr uint32_t idesc = i8_idesc(256, 256);
    int j = 0, t = 0;
    bool ok = true;
    for (int tile = pair; tile < P.tiles && ok; tile += pairs, ++t) {
      const int buf = t & 1;
      if (t >= 2 && !mbar_wait(&acc_empty[buf], ((t >> 1) - 1) & 1)) break;
      tc_fence_after();
      for (int k = 0; k < nk; ++k, ++j) {
        const int s = j % kI8WideStages;
        if (!mbar_wait(&full[s], (j / kI8WideStages) & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t at = smem_u32(ring) + s * kI8WideStage;
#pragma unroll
        for (int c = 0; c < kI8Depth / 32; ++c)
          i8_mma_pair(tmem + buf * 256, i8_sdesc(at + 32 * c), i8_sdesc(at + 128 * kI8Depth + 32 * c), idesc,
                      k > 0 || c > 0);
        commit_pair(&empty[s]);
      }
      if (ok) commit_pair(&acc_full[buf]);
    }
  } else if (warp >= 4) {
    constexpr int kPer = 128 / sizeof(T);  // outputs in a staged row of 128 bytes
    const int ew = warp & 3, half = (warp - 4) >> 2, et = threadIdx.x - 128;
    unsigned char* mine = staged + (warp - 4) * 32 * kI8Pitch;
    const uint32_t lanes = tmem + ((uint32_t)(ew * 32) << 16);
    const bool wide = P.outs % (16 / (int)sizeof(T)) == 0;  // 16-byte rows of y (y itself is 16-byte aligned)
    T* y = static_cast<T*>(P.y);
    int t = 0;
    bool bad = false;  // a wait ran out: keep to the barriers, touch nothing
    // A tile's scales are asked for while the tile before it is scaled: a channel's to each thread,
    // its own row's to each lane.
    float next_sw = 0.f, next_b = 0.f, next_sx = 0.f;
    const auto ask = [&](int tile) {
      if (tile >= P.tiles) return;
      int m, n;
      place(tile, m, n);
      const int c = n * 256 + et, r = m * 256 + (int)rank * 128 + ew * 32 + lane;
      next_sw = c < P.outs ? P.sw[c] : 0.f;
      next_b = c < P.outs && P.bias ? to_f32(static_cast<const T*>(P.bias)[c]) : 0.f;
      next_sx = r < P.rows ? P.sx[r] : 0.f;
    };
    static_assert(32 * kI8WideEpi == 256, "a channel to a thread");
    ask(pair);
    for (int tile = pair; tile < P.tiles; tile += pairs, ++t) {
      int m, n;
      place(tile, m, n);
      const int n0 = n * 256, row0 = m * 256 + (int)rank * 128 + ew * 32;
      const float* sw = s_sw[t & 1];
      const float* sb = s_b[t & 1];
      s_sw[t & 1][et] = next_sw;
      s_b[t & 1][et] = next_b;
      const float sx = next_sx;
      named_sync(1, 32 * kI8WideEpi);  // also: the tile before the last has been scaled, so the other buffer is free
      ask(tile + pairs);
      bad = bad || !__all_sync(kFullMask, mbar_wait(&acc_full[t & 1], (t >> 1) & 1));
      tc_fence_after();
      if (bad) continue;
#pragma unroll 1
      for (int c0 = 128 * half; c0 < 128 * half + 128; c0 += kPer) {
        __syncwarp();
#pragma unroll
        for (int h = 0; h < kPer; h += 32) {
          int v[32];
          tmem_ld32i(lanes + (t & 1) * 256 + c0 + h, v);
          alignas(16) T out[32];
#pragma unroll
          for (int q = 0; q < 32; q += 4) {
            const float4 w4 = *reinterpret_cast<const float4*>(&sw[c0 + h + q]);
            const float4 b4 = *reinterpret_cast<const float4*>(&sb[c0 + h + q]);
            put2(out + q, fmaf((float)v[q] * sx, w4.x, b4.x), fmaf((float)v[q + 1] * sx, w4.y, b4.y));
            put2(out + q + 2, fmaf((float)v[q + 2] * sx, w4.z, b4.z), fmaf((float)v[q + 3] * sx, w4.w, b4.w));
          }
#pragma unroll
          for (int q = 0; q < 32 * (int)sizeof(T) / 16; ++q)
            *reinterpret_cast<uint4*>(mine + lane * kI8Pitch + h * sizeof(T) + 16 * q) = reinterpret_cast<uint4*>(out)[q];
        }
        if (c0 + kPer >= 128 * half + 128) {  // every sum of this warp is in registers: the accumulator is free
          tc_fence_before();
          if (lane == 0)
            asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                             pair_leader(smem_u32(&acc_empty[t & 1])))
                         : "memory");
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
                  *reinterpret_cast<const uint4*>(mine + r * kI8Pitch + 16 * piece);
        } else {
          // Rows off 16-byte boundaries: a row's chunk by aligned pairs (16-bit results), or
          // element beside element.
          const int count = min(kPer, left);
#pragma unroll 4
          for (int r = 0; r < 32 && row0 + r < P.rows; ++r) {
            const T* from = reinterpret_cast<const T*>(mine + r * kI8Pitch);
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
