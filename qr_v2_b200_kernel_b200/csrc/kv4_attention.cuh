// Attention of a few queries over the 4-bit cache (layout and formulas: kv4.cuh).
//
// With m_t and s_t a token's minimum and step, c_t its codes:
//   q . k_t = sum_groups s_t (q . c_t) + m_t sum(q),     o = sum_t (p_t s_t) c_t + sum_t p_t m_t.
// So the codes themselves are the matrix operands, exact in 16 bits: no key or value is ever
// rounded, steps and minima are applied in 32 bits. Keys (and values transposed) are the 16-row
// left operand, 8 query rows that share the key head the right one, so a head with few query rows
// wastes little of the matrix instruction.
//
// Instructions bound it before the memory does, so the inner loop is kept short:
// * a key's nibble needs one logical operation: left in place in an otherwise empty 16-bit number
//   it is a subnormal (or the first normal binade, which continues them), worth code 2^-133 in bf16, 16
//   times that four bits higher. The factors are powers of two: 1/16 goes to the queries of those channels;
//   each query row is brought by another to the top of its type's range, where neither it nor the
//   products lose bits; the scores take both back.
// * the instruction adds its products on a grid set by their operands' exponent fields, and a subnormal's
//   field is that of a larger number: at bits 0 to 3 of a bf16 8 to 128 times (code 15 to 1), of an fp16 64 to
//   1024 times, so that what is much smaller than the largest product loses bits. fp16 keys, and all values, which are fp16 here,
//   are therefore shifted to bits 4 to 7 (code 2^-20), two operations more of each eight nibbles (keys: 123 ->
//   128 us, and with one channel of the queries 256 times the others an error of 3e-6 for 2.4e-5, that of
//   32-bit operations being 6e-7 and the result's rounding 1.8e-5; values: 119 -> 122 us).
// * sums of codes do not drift: tokens 8 to 15 of a run count down from the group's top, k = (m + 15 s)
//   - s (15 - c), for nothing (the complement is part of the mask, the sign of the step), so
//   that what is summed has no common sign. The instruction still cuts off where it adds, so every
//   eighth step the sums are set aside: added, rounded to nearest, to sums in shared memory. The
//   result's error is then some units of 2^-24 of the values at any length (of fp16 outputs over 8192
//   tokens 0.7 % are not the nearest, 0.3 % of those of 32-bit operations throughout; 20 %
//   with codes counted up and half the bits cut), for the same time.
// * the weights p_t s_t are the only rounded operand: two fp16 numbers each, high and low, 22 bits
//   in all (one alone would add an error the size of the result's own rounding). They are scaled by
//   a power of two that puts the largest step near 2^11, so that a weight keeps its leading bits
//   down to 2^-25 of the largest.
// * the running maximum and that scale move only when a score exceeds the reference by 2^4 or a
//   step its bound, so that the output is rarely rescaled and the warp rarely reduces.
// * a lane's two query rows go through paired 32-bit operations (127 -> 123 us).
// Each warp walks its own stretch of tokens, a step of 32 or 64 at a time, through a ring of two
// or three steps in shared memory that bulk asynchronous copies fill: a run's bytes are already in the order
// of the operand's registers. The token range is cut over CTAs (blockIdx.x % splits) and over a CTA's four
// warps; the parts are joined through shared memory and, between CTAs, through the cluster's shared
// memory (up to eight) or by kv4_join_kernel, always in a fixed order.
// 64 sequences x 8192 tokens, 64 heads on 8: 123 us, 4.7 TB/s of cache; 1 x 65536 30 us; one of
// 513 tokens 6.5 us, which is latency from end to end.
#pragma once

#include <type_traits>

#include "cluster.cuh"
#include "kv4.cuh"

namespace qrb200 {

struct Kv4AttnParams {
  const unsigned char* cache;
  const void* q;
  void* out;
  float* part_o;       // [batch][head][tile][split][rows of a tile][dim], unnormalised, when splits > kKvCluster
  float2* part_ml;     // [...][rows of a tile]: maximum (base 2) and sum
  const int* table;
  const int* lengths;
  long long q_bs, q_ts, q_hs, table_stride;  // strides in elements
  int batch, queries, q_heads, share, max_pages, window, causal, splits, tiles;
  int q_wide;  // four channels of q lie on an 8-byte boundary
  float scale2;  // scale times log2(e)
  Kv4Shape sh;
};

constexpr int kKvWarps = 4;
constexpr int kKvCluster = 8;  // the most CTAs that join their parts within a cluster (the portable size)
// Runs of 16 tokens in a warp's step: as many as the registers hold beside the output (twice the
// channels, half the runs). With 64 channels a warp that has no more than two such steps takes them
// in halves: its time is that of code running for the first time, and there is half as much (12 x
// 2047 tokens, five drafts, window 1000: 12.2 against 10.0 us; 64 x 8192 tokens in halves would
// take 58 against 51 us; with 128 channels halves lose, 6.8 against 6.4 us for one sequence of
// 513).
__host__ __device__ constexpr int kv_runs(int dim, bool brief) { return dim == 64 && !brief ? 4 : 2; }

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

// Nibbles p and p + 4 of a word of keys as a pair of 16-bit numbers, the code as a subnormal (or the first
// normal binade): in bf16 left where they stand, at bits 0 to 3 or, times 16, 4 to 7; in fp16 all at bits 4 to 7.
template <typename T>
__device__ __forceinline__ uint32_t kv_key_pair(uint32_t w, int p) {
  if constexpr (std::is_same<T, __half>::value) return (p == 0 ? w << 4 : w >> (4 * p - 4)) & 0x00f000f0u;
  if (p & 2) w >>= 8;
  return w & (p & 1 ? 0x00f000f0u : 0x000f000fu);
}
// A lane's word of values as the left operand: sixteen times the code of tokens 0 to 7 (channels g,
// then g + 8), sixteen times 15 - code of tokens 8 to 15.
__device__ __forceinline__ void kv_values(uint32_t (&a)[4], uint32_t w) {
  constexpr uint32_t kMask = 0x00f000f0u;
  a[0] = w << 4 & kMask, a[1] = w & kMask, a[2] = ~(w >> 4) & kMask, a[3] = ~(w >> 8) & kMask;
}
// Where a query row's largest entry is put (its exponent), what its type makes of the code 1 (the
// negative exponent), and the factor of the queries that meet nibbles 1 and 3. Scores are built from
// queries brought to 2^-kKvSpare, so that keys of any size give finite ones, and multiplied by what
// takes that back, the scale included, as the last step.
constexpr int kKvSpare = 8;
template <typename T>
struct KvKey;
template <>
struct KvKey<__nv_bfloat16> {
  static constexpr int kTop = 100, kOne = 133;
  static constexpr float kOdd = 0.0625f;
};
template <>
struct KvKey<__half> {
  static constexpr int kTop = 13, kOne = 20;
  static constexpr float kOdd = 1.f;
};
__device__ __forceinline__ float kv_power(int e) { return __int_as_float((max(-126, min(127, e)) + 127) << 23); }
// The power of two that brings a row whose largest entry has these bits (32-bit float, no sign) to
// kTop, as far as it and what takes it back, scale2 2^(kTop + kKvSpare - lift), are normal numbers.
template <typename T>
__device__ __forceinline__ int kv_lift(unsigned top, float scale2) {
  const int least = KvKey<T>::kTop + kKvSpare - 126 + max(0, (__float_as_int(scale2) >> 23) - 126);
  return max(least, min(120, KvKey<T>::kTop + 127 - (int)(top >> 23)));
}

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
// A (step, minimum) word.
template <typename T>
__device__ __forceinline__ float2 kv_step_low(uint32_t w) {
  const Pair16<T> pr = reinterpret_cast<const Pair16<T>&>(w);
  return make_float2(to_f32(pr.s), to_f32(pr.m));
}
constexpr float kKvLazy = 4.f;      // powers of two that a score may stand above the reference
constexpr int kKvStepExp = 11;      // the largest step's place: weights stay below 2^(11 + 4) in fp16

__device__ __forceinline__ void mbar_expect(uint32_t mbar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(mbar), "r"(bytes) : "memory");
}

// Steps in a warp's ring. With eight query rows two leave room for the sums set aside of four CTAs
// an SM, and cost nothing (64 x 8192 tokens 121.3 us, with three 122.1).
__host__ __device__ constexpr int kv_stages(int nt) { return nt == 1 ? 2 : 3; }
constexpr int kKvAside = 8;  // steps between settings-aside (every fourth: 1.8 us more of 123)
// CTAs to an SM that registers are kept for. Four (128 registers) beat three wherever little spills
// (64 x 8192 tokens, one group: 126 against 138 us); four groups of steps would (125 against 111
// us).
__host__ __device__ constexpr int kv_ctas(int groups, int nt) { return nt > 1 ? 2 : groups < 4 ? 4 : 3; }
// Dynamic shared memory: the warps' rings, reused at the end for their parts of the output, and
// behind them the sums set aside.
__host__ __device__ constexpr int kv_stage_bytes(int dim, int groups, bool brief) {
  return kv_runs(dim, brief) * (16 * dim + 128 * groups);
}
__host__ __device__ constexpr int kv_ring_bytes(int dim, int groups, int nt, bool brief) {
  const int ring = kKvWarps * kv_stages(nt) * kv_stage_bytes(dim, groups, brief), parts = kKvWarps * 8 * nt * (dim + 4) * 4;
  return ring > parts ? ring : parts;
}
__host__ __device__ constexpr int kv_smem_bytes(int dim, int groups, int nt, bool brief) {
  return kv_ring_bytes(dim, groups, nt, brief) + kKvWarps * 8 * nt * dim * 4;
}

template <typename T, int kDim, int kGroups, int kNT, bool kBrief>
__global__ void __launch_bounds__(32 * kKvWarps, kv_ctas(kGroups, kNT)) kv4_attention_kernel(Kv4AttnParams P) {
  constexpr int kRows = 8 * kNT;           // query rows of a tile
  constexpr int kSteps = kDim / 16;        // 16-channel steps of q . k; also 16-channel tiles of the output
  constexpr int kPer = kSteps / kGroups;   // steps of a group
  constexpr int kKW = kDim / 32;           // words of a lane's key codes, for one token
  constexpr int kVC = kDim / 64;           // 16-byte pieces of a lane's value codes, for 16 tokens
  constexpr int kRuns = kv_runs(kDim, kBrief), kUnit = 16 * kRuns;
  constexpr int kRunBytes = 16 * kDim + 128 * kGroups, kStage = kRuns * kRunBytes;
  constexpr int kStages = kv_stages(kNT);
  const float unbare = kv_power(KvKey<T>::kOne - KvKey<T>::kTop - kKvSpare);  // q . c from the product with bare codes
  constexpr float kNone = -INFINITY;
  extern __shared__ __align__(128) unsigned char s_ring[];
  __shared__ uint2 s_q[kNT][kSteps][32];
  __shared__ float s_qsum[kKvWarps][kNT][8][kGroups];
  __shared__ unsigned s_qtop[kKvWarps][kNT][8];
  __shared__ float2 s_ml[kKvWarps][kRows];
  __shared__ uint64_t s_full[kKvWarps][kStages];
  __shared__ int s_bad;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % P.splits, tile = blockIdx.x / P.splits, head = blockIdx.y, b = blockIdx.z;
  const int rows = P.queries * P.share, row0 = tile * kRows;

  if (threadIdx.x == 0) s_bad = 0;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&s_full[warp][i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  __syncwarp();
  griddep_launch_wait();
  int len = P.lengths[b];
  // The queries, asked for before anything waits: step j wants channels 16 j + 4 t + {0, 1} and {2,
  // 3} of row g.
  T qv[kNT][kSteps / kKvWarps][4];
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
    const int r = row0 + 8 * n + g;
    const T* q = static_cast<const T*>(P.q) + b * P.q_bs + (long long)(r / P.share) * P.q_ts +
                 (head * P.share + r % P.share) * P.q_hs + 4 * t;
#pragma unroll
    for (int i = 0; i < kSteps / kKvWarps; ++i) {
      const T* at = q + 16 * (i * kKvWarps + warp);
      if (P.q_wide) {
        *reinterpret_cast<uint2*>(qv[n][i]) = r < rows ? __ldg(reinterpret_cast<const uint2*>(at)) : make_uint2(0, 0);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) qv[n][i][e] = r < rows ? at[e] : from_f32<T>(0.f);
      }
    }
  }
  if (len < 0 || len > (long long)P.max_pages * P.sh.page || (len > 0 && P.sh.pages == 0)) {
    if (threadIdx.x == 0) report_device_failure(kSiteIndex);
    len = 0;
  }
  // Tokens [lo, hi) that each row sees (lane r holds row r's), all rows together, and every row.
  int my_lo = 0, my_hi = 0;
  const bool real = lane < kRows && row0 + lane < rows;
  if (real) {
    const int pos = len - P.queries + (row0 + lane) / P.share;
    my_hi = P.causal ? max(0, pos + 1) : len;
    my_lo = P.window > 0 ? max(0, pos - P.window + 1) : 0;
  }
  const bool sees = my_hi > my_lo;
  const int all_lo = __reduce_min_sync(kFullMask, sees ? my_lo : 0x7fffffff);
  const int all_hi = __reduce_max_sync(kFullMask, sees ? my_hi : 0);
  const int in_lo = __reduce_max_sync(kFullMask, my_lo), in_hi = __reduce_min_sync(kFullMask, real ? my_hi : 0x7fffffff);
  // This warp's steps [u, u_hi) of its CTA's share of the range.
  const int u0 = all_hi > 0 ? all_lo / kUnit : 0, u1 = (all_hi + kUnit - 1) / kUnit;
  const int per = (u1 - u0 + P.splits - 1) / P.splits;
  const int cta_lo = min(u1, u0 + split * per), cta_hi = min(u1, cta_lo + per);
  const int per_warp = (cta_hi - cta_lo + kKvWarps - 1) / kKvWarps;
  int u = min(cta_hi, cta_lo + warp * per_warp);
  const int u_hi = min(cta_hi, u + per_warp);

  // The ring. Lane i of `page` holds the page of run `page_base` + i, -1 outside the range, before
  // which pages may be gone from the table, or where the table is wrong.
  unsigned char* ring = s_ring + warp * (kStages * kStage);
  const int page_runs = P.sh.page / 16, page_shift = P.sh.shift - 4;
  const int first_run = all_lo / 16, last_run = min(u_hi * kRuns, (len + 15) / 16);
  int page_base = u * kRuns, page = -1;
  auto look_up = [&]() {
    page = -1;
    if (page_base + lane >= first_run && page_base + lane < last_run) {
      page = __ldg(P.table + b * P.table_stride + ((page_base + lane) >> page_shift));
      if (page < 0 || page >= P.sh.pages) {
        report_device_failure(kSiteIndex);
        page = -1;
      }
    }
  };
  unsigned missing = 0;  // kRuns bits a stage: its runs without a page
  auto issue = [&](int unit, int stage) {
    if (unit * kRuns >= page_base + 32) {
      page_base = unit * kRuns;
      look_up();
    }
    const uint32_t bar = smem_u32(&s_full[warp][stage]), dst = smem_u32(ring + stage * kStage);
    const auto at = [&](int pg, int run) {
      return P.cache + ((long long)pg * P.sh.heads + head) * P.sh.block_bytes() + (run & (page_runs - 1)) * kRunBytes;
    };
    unsigned gone = 0;
    if (page_runs >= kRuns && (unit + 1) * kRuns <= last_run) {  // one page, the last run's, holds the step: one copy
      const int run = unit * kRuns, pg = __shfl_sync(kFullMask, page, run + kRuns - 1 - page_base);
      if (pg < 0) gone = (1u << kRuns) - 1;
      if (lane == 0) {
        mbar_expect(bar, pg < 0 ? 0 : kStage);
        if (pg >= 0) kv_copy(dst, at(pg, run), kStage, bar);
      }
    } else {
      for (int i = 0; i < kRuns; ++i) gone |= __shfl_sync(kFullMask, page, unit * kRuns + i - page_base) < 0 ? 1u << i : 0u;
      if (lane == 0) mbar_expect(bar, (kRuns - __popc(gone)) * kRunBytes);
      for (int i = 0; i < kRuns; ++i) {
        const int run = unit * kRuns + i, pg = __shfl_sync(kFullMask, page, run - page_base);
        if (lane == 0 && pg >= 0) kv_copy(dst + i * kRunBytes, at(pg, run), kRunBytes, bar);
      }
    }
    missing = (missing & ~(((1u << kRuns) - 1) << (8 * stage))) | gone << (8 * stage);
  };
  const int count = u_hi - u;
  if (count > 0) look_up();
  for (int i = 0; i < kStages && i < count; ++i) issue(u + i, i);

  // Queries as the right operand. The warps share the work; first each row's largest entry and each
  // group's sum.
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
    float part[kGroups] = {};
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < kSteps / kKvWarps; ++i) {
      const int j = i * kKvWarps + warp;
      float add = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = to_f32(qv[n][i][e]);
        add = fmaf(v, 0x1p-8f, add);  // (a sum of 128 may leave the range that one is in)
        top = max(top, __float_as_uint(v) & 0x7fffffffu);
      }
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) part[gr] += j / kPer == gr ? add : 0.f;
    }
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      top = max(top, __shfl_xor_sync(kFullMask, top, x));
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) part[gr] += __shfl_xor_sync(kFullMask, part[gr], x);
    }
    if (t == 0) {
      s_qtop[warp][n][g] = top;
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) s_qsum[warp][n][g][gr] = part[gr];
    }
  }
  __syncthreads();
  const auto lift = [&](int n, int row) {
    unsigned top = 0;
    for (int w = 0; w < kKvWarps; ++w) top = max(top, s_qtop[w][n][row]);
    return kv_lift<T>(top, P.scale2);
  };
  // qsum: a group's sum at the size that scores are built from; back: what takes that size back, into
  // the exponent's units (base 2), so that the largest score less itself is 0 and its weight 1, exactly.
  float2 qsum[kNT][kGroups], back[kNT];
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
    const float up = kv_power(lift(n, g));
#pragma unroll
    for (int i = 0; i < kSteps / kKvWarps; ++i) {
      alignas(8) T x[4];
      put2(x, to_f32(qv[n][i][0]) * up, to_f32(qv[n][i][1]) * up);
      put2(x + 2, to_f32(qv[n][i][2]) * (up * KvKey<T>::kOdd), to_f32(qv[n][i][3]) * (up * KvKey<T>::kOdd));
      s_q[n][i * kKvWarps + warp][lane] = *reinterpret_cast<uint2*>(x);
    }
    const int lift0 = lift(n, 2 * t) - KvKey<T>::kTop, lift1 = lift(n, 2 * t + 1) - KvKey<T>::kTop;
    back[n] = make_float2(kv_power(kKvSpare - lift0) * P.scale2, kv_power(kKvSpare - lift1) * P.scale2);
#pragma unroll
    for (int gr = 0; gr < kGroups; ++gr) {
      qsum[n][gr] = make_float2(0.f, 0.f);
      for (int w = 0; w < kKvWarps; ++w) {
        qsum[n][gr].x += s_qsum[w][n][2 * t][gr];
        qsum[n][gr].y += s_qsum[w][n][2 * t + 1][gr];
      }
      // 2^8 of the sums' and 2^-kKvSpare cancel.
      qsum[n][gr] = make_float2(qsum[n][gr].x * kv_power(lift0), qsum[n][gr].y * kv_power(lift1));
    }
  }
  __syncthreads();

  float o[kNT][kSteps][4] = {};  // scaled by `unit`
  float2 sum[kNT] = {}, lows[kNT][kGroups] = {};
  // Weights are 2^(score + less), the reference being -less; bound is where a score moves it: 4
  // above, rounded down where scores are so large (so the reference cannot be had back from it), and
  // -inf while nothing has been seen. cap bounds the steps, unit scales them.
  float2 less[kNT] = {};
  float bound[kNT][2], cap = 0.f, unit = 1.f;
#pragma unroll
  for (int n = 0; n < kNT; ++n) bound[n][0] = bound[n][1] = kNone;
  const auto reference = [&](int n, int c) { return bound[n][c] == kNone ? kNone : -(c ? less[n].y : less[n].x); };

  // This lane's sums set aside, 32 lanes apart; `aside` once there are some.
  float4* apart = reinterpret_cast<float4*>(s_ring + kv_ring_bytes(kDim, kGroups, kNT, kBrief)) + warp * (kRows * kDim / 4) + lane;
  bool ok = true, aside = false;
  int stage = 0, turn = 0;
  for (int k = 0; ok && k < count;) {
    const int pause = min(count, k + kKvAside);
    for (; k < pause; ++k, ++u) {
      const int tok0 = u * kUnit;
      const unsigned char* runs = ring + stage * kStage;
      const unsigned gone = missing >> (8 * stage) & ((1u << kRuns) - 1);
      ok = ok && __all_sync(kFullMask, mbar_wait(&s_full[warp][stage], turn));
      if (!ok) break;
      // Scores: s[i][n][h] holds token tok0 + 16 i + 8 h + g against rows 8 n + 2 t
      // and the next.
      float2 s[kRuns][kNT][2];
      {
        float acc[kRuns][kNT][4];
        uint32_t kc[kRuns][2][kKW];
#pragma unroll
        for (int i = 0; i < kRuns; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) kv_load(kc[i][h], runs + i * kRunBytes + h * (4 * kDim) + lane * (kDim / 8));
#pragma unroll
        for (int gr = 0; gr < kGroups; ++gr) {
#pragma unroll
          for (int i = 0; i < kRuns; ++i)
#pragma unroll
            for (int n = 0; n < kNT; ++n) acc[i][n][0] = acc[i][n][1] = acc[i][n][2] = acc[i][n][3] = 0.f;
#pragma unroll
          for (int j = gr * kPer; j < (gr + 1) * kPer; ++j) {
            const int p = 2 * (j & 1);
            uint2 q[kNT];
#pragma unroll
            for (int n = 0; n < kNT; ++n) q[n] = s_q[n][j][lane];
#pragma unroll
            for (int i = 0; i < kRuns; ++i) {
              const uint32_t a[4] = {kv_key_pair<T>(kc[i][0][j >> 1], p), kv_key_pair<T>(kc[i][1][j >> 1], p),
                                     kv_key_pair<T>(kc[i][0][j >> 1], p + 1), kv_key_pair<T>(kc[i][1][j >> 1], p + 1)};
#pragma unroll
              for (int n = 0; n < kNT; ++n) kv_mma<T>(acc[i][n], a, q[n].x, q[n].y);
            }
          }
#pragma unroll
          for (int i = 0; i < kRuns; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float2 k = kv_step_low<T>(
                  *reinterpret_cast<const uint32_t*>(runs + i * kRunBytes + 16 * kDim + ((g + 8 * h) * kGroups + gr) * 4));
#pragma unroll
              for (int n = 0; n < kNT; ++n) {
                const float2 kx = make_float2(k.x, k.x), ky = make_float2(k.y, k.y);
                const float2 low = gr ? __ffma2_rn(ky, qsum[n][gr], s[i][n][h]) : __fmul2_rn(ky, qsum[n][gr]);
                const float2 dot = __fmul2_rn(make_float2(acc[i][n][2 * h], acc[i][n][2 * h + 1]), make_float2(unbare, unbare));
                s[i][n][h] = __ffma2_rn(kx, dot, low);
                if (gr == kGroups - 1) s[i][n][h] = __fmul2_rn(s[i][n][h], back[n]);
              }
            }
        }
      }
      uint32_t vp[kRuns][2][kGroups];
#pragma unroll
      for (int i = 0; i < kRuns; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) kv_load(vp[i][h], runs + i * kRunBytes + 16 * kDim + 64 * kGroups + (g + 8 * h) * (4 * kGroups));
      const bool full = !gone && tok0 >= in_lo && tok0 + kUnit <= in_hi;  // every row sees every token
      uint32_t seen[kNT];
      if (!full) {
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          int lo[2], hi[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            lo[c] = __shfl_sync(kFullMask, my_lo, 8 * n + 2 * t + c);
            hi[c] = __shfl_sync(kFullMask, my_hi, 8 * n + 2 * t + c);
          }
          seen[n] = 0;
#pragma unroll
          for (int i = 0; i < kRuns; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int tok = tok0 + 16 * i + 8 * h + g;
              const bool x = tok >= lo[0] && tok < hi[0] && !(gone >> i & 1);
              const bool y = tok >= lo[1] && tok < hi[1] && !(gone >> i & 1);
              seen[n] |= (x ? 1u : 0u) << (4 * i + 2 * h) | (y ? 2u : 0u) << (4 * i + 2 * h);
              if (!x) s[i][n][h].x = kNone;
              if (!y) s[i][n][h].y = kNone;
              if (n == 0 && (tok < all_lo || tok >= all_hi || (gone >> i & 1)))
#pragma unroll
                for (int gr = 0; gr < kGroups; ++gr) vp[i][h][gr] = 0;  // seen by no row: may hold anything
            }
        }
      }
      float2 val[kRuns][2][kGroups];  // step and minimum
      float up[kNT][2], steps = 0.f;
#pragma unroll
      for (int i = 0; i < kRuns; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int gr = 0; gr < kGroups; ++gr) {
            val[i][h][gr] = kv_step_low<T>(vp[i][h][gr]);
            steps = fmaxf(steps, val[i][h][gr].x);
            if (h) val[i][h][gr].y = fmaf(15.f, val[i][h][gr].x, val[i][h][gr].y);  // codes count down from here
          }
      bool move = steps > cap;
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        up[n][0] = s[0][n][0].x;
        up[n][1] = s[0][n][0].y;
#pragma unroll
        for (int i = 0; i < kRuns; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            up[n][0] = fmaxf(up[n][0], s[i][n][h].x);
            up[n][1] = fmaxf(up[n][1], s[i][n][h].y);
          }
        move = move || up[n][0] > bound[n][0] || up[n][1] > bound[n][1];
      }
      if (__any_sync(kFullMask, move)) {
        steps = fmaxf(steps, cap);
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) steps = fmaxf(steps, __shfl_xor_sync(kFullMask, steps, x));
        float ratio = 1.f;
        if (steps > cap) {  // the power of two above the largest step, and the scale that puts it at 2^11
          const int e = max(-100, min(126, (int)(__float_as_uint(steps) >> 23) - 126));
          cap = __int_as_float((e + 127) << 23);
          const float fresh = __int_as_float((kKvStepExp - e + 127) << 23);
          ratio = fresh / unit;
          unit = fresh;
        }
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          float keep[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) up[n][c] = fmaxf(up[n][c], __shfl_xor_sync(kFullMask, up[n][c], x));
            const float last = reference(n, c), next = fmaxf(up[n][c], last);
            keep[c] = next == kNone ? 0.f : kv_exp2(last - next);
            bound[n][c] = __fadd_rd(next, kKvLazy);
            // A row that has seen nothing has the reference -inf: its weights, 2^-inf, come from any
            // finite one.
            (c ? less[n].y : less[n].x) = next == kNone ? 0.f : -next;
          }
          sum[n] = make_float2(sum[n].x * keep[0], sum[n].y * keep[1]);
#pragma unroll
          for (int gr = 0; gr < kGroups; ++gr) lows[n][gr] = make_float2(lows[n][gr].x * keep[0], lows[n][gr].y * keep[1]);
#pragma unroll
          for (int j = 0; j < kSteps; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][j][e] *= keep[e & 1] * ratio;
          if (aside) {
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
              float4 a = apart[32 * (n * kSteps + j)];
              a.x *= keep[0] * ratio, a.y *= keep[1] * ratio, a.z *= keep[0] * ratio, a.w *= keep[1] * ratio;
              apart[32 * (n * kSteps + j)] = a;
            }
          }
        }
      }
      // Weights and output; kAll: every row sees every token (no tests in the common case).
      auto finish = [&](auto all) {
        constexpr bool kAll = decltype(all)::value;
#pragma unroll
        for (int i = 0; i < kRuns; ++i) {
          uint32_t vc[kVC][4];
#pragma unroll
          for (int c = 0; c < kVC; ++c) kv_load(vc[c], runs + i * kRunBytes + 8 * kDim + c * 512 + lane * 16);
#pragma unroll
          for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float2 e = __fadd2_rn(s[i][n][h], less[n]), p = make_float2(kv_exp2(e.x), kv_exp2(e.y));
              sum[n] = __fadd2_rn(sum[n], p);
              s[i][n][h] = p;
            }
#pragma unroll
          for (int gr = 0; gr < kGroups; ++gr) {
            uint32_t w[2][kNT][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float scaled = val[i][h][gr].x * (h ? -unit : unit);
#pragma unroll
              for (int n = 0; n < kNT; ++n) {
                const float2 p = s[i][n][h];
                float2 x = __fmul2_rn(p, make_float2(scaled, scaled));
                if constexpr (kAll) {
                  lows[n][gr] = __ffma2_rn(p, make_float2(val[i][h][gr].y, val[i][h][gr].y), lows[n][gr]);
                } else {  // what a row does not see may be NaN
                  if (seen[n] >> (4 * i + 2 * h) & 1) lows[n][gr].x = fmaf(p.x, val[i][h][gr].y, lows[n][gr].x);
                  else x.x = 0.f;
                  if (seen[n] >> (4 * i + 2 * h) & 2) lows[n][gr].y = fmaf(p.y, val[i][h][gr].y, lows[n][gr].y);
                  else x.y = 0.f;
                }
                const uint32_t high = kv_pack(x);
                w[0][n][h] = kv_transpose(high);
                const float2 top = __half22float2(__hneg2(reinterpret_cast<const __half2&>(high)));
                w[1][n][h] = kv_transpose(kv_pack(__fadd2_rn(x, top)));
              }
            }
#pragma unroll
            for (int j = gr * kPer; j < (gr + 1) * kPer; ++j) {
              const uint32_t word = vc[j >> 2][j & 3];
              uint32_t a[4];
              kv_values(a, word);
#pragma unroll
              for (int n = 0; n < kNT; ++n)
#pragma unroll
                for (int half = 0; half < 2; ++half) kv_mma<__half>(o[n][j], a, w[half][n][0], w[half][n][1]);
            }
          }
        }
      };
      if (full) finish(std::true_type{});
      else finish(std::false_type{});
      __syncwarp();  // every lane has read this stage
      if (k + kStages < count) issue(u + kStages, stage);
      if (++stage == kStages) {
        stage = 0;
        turn ^= 1;
      }
    }
    if (ok && k < count) {  // set the sums aside
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
          if (aside) a = apart[32 * (n * kSteps + j)];
          a.x += o[n][j][0], a.y += o[n][j][1], a.z += o[n][j][2], a.w += o[n][j][3];
          apart[32 * (n * kSteps + j)] = a;
          o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
        }
      aside = true;
    }
  }
  if (!ok) {
    // A copy did not arrive in time: nothing is written, and what is under way is waited for (with
    // a limit) first.
    for (int i = 0; i < kStages; ++i) mbar_wait(&s_full[warp][i], i < stage ? turn ^ 1 : turn);
    s_bad = 1;
  }
  if (aside) {
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        const float4 a = apart[32 * (n * kSteps + j)];
        o[n][j][0] += a.x, o[n][j][1] += a.y, o[n][j][2] += a.z, o[n][j][3] += a.w;
      }
  }
  __syncthreads();  // the rings are free
  float(*s_o)[kRows][kDim + 4] = reinterpret_cast<float(*)[kRows][kDim + 4]>(s_ring);

  const float lower = 1.f / unit;
  constexpr float kOne = 0x1p20f;  // what a code's unit counts less in the operand
  // The warps' parts: o[n][j][e] is channel 16 j + g + 8 (e / 2) of row 8 n + 2 t + e % 2.
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float l = c ? sum[n].y : sum[n].x, add[kGroups];
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) add[gr] = c ? lows[n][gr].y : lows[n][gr].x;
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        l += __shfl_xor_sync(kFullMask, l, x);
#pragma unroll
        for (int gr = 0; gr < kGroups; ++gr) add[gr] += __shfl_xor_sync(kFullMask, add[gr], x);
      }
      if (g == 0) s_ml[warp][8 * n + 2 * t + c] = make_float2(reference(n, c), l);
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        s_o[warp][8 * n + 2 * t + c][16 * j + g] = fmaf(o[n][j][c] * kOne, lower, add[j / kPer]);
        s_o[warp][8 * n + 2 * t + c][16 * j + g + 8] = fmaf(o[n][j][2 + c] * kOne, lower, add[j / kPer]);
      }
    }
  __syncthreads();
  constexpr int kLanesRow = 32 * kKvWarps / kRows;  // threads of a row
  const int r = threadIdx.x / kLanesRow, d0 = threadIdx.x % kLanesRow;
  float m = kNone, l = 0.f, f[kKvWarps];
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
    if (row0 + r < rows && !s_bad)
      for (int d = d0; d < kDim; d += kLanesRow) out_row(r)[d] = from_f32<T>(joined(d) * inv);
  } else if (P.splits <= kKvCluster) {
    // The CTA's part takes its first warp's place; each CTA then joins every splits-th row of all
    // of them.
    for (int d = d0; d < kDim; d += kLanesRow) s_o[0][r][d] = joined(d);
    __syncthreads();  // every warp's (maximum, sum) has been read
    if (d0 == 0) s_ml[0][r] = make_float2(m, l);
    cluster_sync();
    // What each CTA's part of a row counts, and the whole row's sum: a thread to a row.
    float(*s_w)[kKvCluster + 1] = reinterpret_cast<float(*)[kKvCluster + 1]>(s_q);
    bool bad = false;
    for (int c = 0; c < P.splits; ++c) bad = ld_cluster(smem_u32(&s_bad), c) != 0 || bad;
    if (threadIdx.x < kRows) {
      float2 ml[kKvCluster];
      float top = kNone, total = 0.f;
#pragma unroll
      for (int c = 0; c < kKvCluster; ++c) {
        ml[c] = make_float2(kNone, 0.f);
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
  } else if (row0 + r < rows && !s_bad) {
    const long long part = (((long long)b * P.sh.heads + head) * P.tiles + tile) * P.splits + split;
    for (int d = d0; d < kDim; d += kLanesRow) P.part_o[(part * kRows + r) * kDim + d] = joined(d);
    if (d0 == 0) P.part_ml[part * kRows + r] = make_float2(m, l);
  }
}

// One CTA per query row: the splits' parts against their common maximum, a warp every eighth, then
// the warps' sums in order.
constexpr int kKvJoinWarps = 8;
template <typename T, int kDim>
__global__ void __launch_bounds__(32 * kKvJoinWarps) kv4_join_kernel(Kv4AttnParams P, int tile_rows) {
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
