// Attention over the 8-bit cache (layout and formulas: kv8.cuh).
//
// With r_t and w_t the steps (range / 127) of token t's page for keys and values, c_t its codes:
//   q . k_t = r_t (q . c_t),     o = sum_t (p_t w_t) c_t.
// So the codes are the matrix operands, exact in 16 bits: a byte c + 128 under the exponent of 1024 is the fp16 number
// 1152 + c, one addition away from c. No key or value is ever rounded; steps are applied in 32 bits.
//
// 64 sequences of 8192 tokens, 8 heads of 128 channels with 8 query rows each, bf16: 176 us for 1.07 GB, 6.1 TB/s (under the power
// cap, 213). The bytes bound it there, with issue slots 65 % busy; fewer or shorter sequences wait for a chain of latencies (one
// of 513 tokens 7.2 us). A CTA's four warps take a quarter of its tokens each, so nothing is shared until the end.
#pragma once

#include <type_traits>

#include "kv8.cuh"
#include "kv_common.cuh"

namespace qrb200 {

struct Kv8AttnParams {
  const unsigned char* codes;
  const float* range;
  const void* q;
  void* out;
  float* part_o;   // [batch][head][tile][split][rows of a tile][dim], unnormalised, where parts go through memory;
                   // of prompts, a CTA's sums set aside; else null
  float2* part_ml;  // [...][rows of a tile]: maximum (base 2) and sum; null where a cluster joins them
  const int* table;
  const int* lengths;
  long long q_bs, q_ts, q_hs, table_stride;  // strides in elements
  int batch, queries, q_heads, share, max_pages, window, causal, splits, tiles;
  int q_wide;    // four channels of q lie on an 8-byte boundary
  float scale_part;  // the scale's significand times log2(e)
  int scale_power;   // and its power of two
  Kv8Shape sh;
};

// Two codes of a word (bytes 0 and 1, or 2 and 3) as fp16 numbers.
template <int kHigh>
__device__ __forceinline__ uint32_t kv8_codes(uint32_t w) {
  const uint32_t x = __byte_perm(w, 0x64646464u, kHigh ? 0x4342 : 0x4140);
  const __half2 c = __hsub2(reinterpret_cast<const __half2&>(x), __half2half2(__ushort_as_half(0x6480)));  // 1152
  return reinterpret_cast<const uint32_t&>(c);
}
// An 8-bit number's significand in [1, 2), and its power of two.
__device__ __forceinline__ float kv8_part(float x) { return __uint_as_float((__float_as_uint(x) & 0x807fffffu) | 0x3f800000u); }
__device__ __forceinline__ int kv8_power(float x) { return (int)(__float_as_uint(x) >> 23 & 255) - 127; }

// The power of two above a step, as its exponent.
__device__ __forceinline__ float kv8_above(float step) { return __uint_as_float(__float_as_uint(step) >> 23 | 0x4b000000u) - (8388608.f + 126.f); }
// A value's step times a row's unit. (Beyond 2^100 only where weights are below 2^-100: bounded, so that none of them times
// this is infinite. NaN stays.)
__device__ __forceinline__ float kv8_scaled(float step, float unit) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(step * unit), "f"(0x1p100f));
  return r;
}

constexpr int kKv8Top = 14;      // where a query row's largest entry is put (its exponent)
constexpr int kKv8StepExp = 10;  // a row's largest weight times step is put below this power of two, and stays below 2^(10 + 4)
constexpr int kKv8Aside = 8;     // steps between settings-aside

// Bytes of a warp's step, 4 KB or 8: a step costs some 1000 clocks of instructions that wait for one another and 500 for each
// 4 KB, so long steps suit few warps, and short ones leave shared memory for twice as many (four CTAs an SM for two,
// at 128 registers for 168). With sixteen query rows, which take the registers of two CTAs anyway, long ones.
// (64 x 8192 tokens, 8 heads: short 172 us, long 180; 1 x 8192 13.8, 10.7.)
__host__ __device__ constexpr int kv8_runs(int dim, bool brief) { return (brief ? 128 : 256) / dim; }
constexpr int kKv8Stages = 2;  // steps in a warp's ring
__host__ __device__ constexpr int kv8_ctas(bool brief) { return brief ? 4 : 2; }
__host__ __device__ constexpr int kv8_ring_bytes(int dim, int nt, bool brief) {
  const int ring = kKvWarps * kKv8Stages * kv8_runs(dim, brief) * 32 * dim, parts = kKvWarps * 8 * nt * (dim + 4) * 4;
  return ring > parts ? ring : parts;
}
// Dynamic shared memory: the warps' rings, reused at the end for their parts of the output, and
// behind them the sums set aside.
__host__ __device__ constexpr int kv8_smem_bytes(int dim, int nt, bool brief) {
  return kv8_ring_bytes(dim, nt, brief) + kKvWarps * 8 * nt * dim * 4;
}

template <typename T, int kDim, int kNT, bool kBrief>
__global__ void __launch_bounds__(32 * kKvWarps, kv8_ctas(kBrief)) kv8_attention_kernel(Kv8AttnParams P) {
  constexpr int kRows = 8 * kNT;      // query rows of a tile
  constexpr int kSteps = kDim / 16;   // 16-channel steps of q . k; also 16-channel tiles of the output
  constexpr int kRuns = kv8_runs(kDim, kBrief), kUnit = 16 * kRuns;
  constexpr int kRunBytes = 32 * kDim, kStage = kRuns * kRunBytes;
  constexpr int kStages = kKv8Stages;
  constexpr float kNone = -INFINITY;
  extern __shared__ __align__(128) unsigned char s_ring[];
  __shared__ uint2 s_q[kNT][kSteps][32];
  __shared__ unsigned s_qtop[kKvWarps][kNT][8];
  __shared__ float4 s_step[kKvWarps][kStages][kRuns];  // a run's key and value steps, and the power of two above the latter
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
    my_lo = P.window > 0 && pos >= P.window ? pos - P.window + 1 : 0;
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
  // which pages may be gone from the table, or where the table is wrong; `steps` its steps.
  unsigned char* ring = s_ring + warp * (kStages * kStage);
  const int page_runs = P.sh.page / 16, page_shift = P.sh.shift - 4;
  const int first_run = all_lo / 16, last_run = min(u_hi * kRuns, (len + 15) / 16);
  int page_base = u * kRuns, page = -1;
  float2 step = make_float2(0.f, 0.f);
  auto look_up = [&]() {
    page = -1;
    step = make_float2(0.f, 0.f);
    if (page_base + lane >= first_run && page_base + lane < last_run) {
      page = __ldg(P.table + b * P.table_stride + ((page_base + lane) >> page_shift));
      if (page < 0 || page >= P.sh.pages) {
        report_device_failure(kSiteIndex);
        page = -1;
      } else {
        step = __ldg(reinterpret_cast<const float2*>(P.range) + (long long)page * P.sh.heads + head);
        step.x = kv8_step(step.x), step.y = kv8_step(step.y);
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
    const int mine = page_base + lane - unit * kRuns;
    if (mine >= 0 && mine < kRuns) s_step[warp][stage][mine] = make_float4(step.x, step.y, kv8_above(step.y), 0.f);
    const auto at = [&](int pg, int run) {
      return P.codes + ((long long)pg * P.sh.heads + head) * P.sh.block_bytes() + (run & (page_runs - 1)) * kRunBytes;
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

  // Queries as the right operand, in fp16: each row brought by a power of two to the top of its range, where
  // what the largest entry leaves of the others is 2^-38 of it. The warps share the work; first each row's
  // largest entry.
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < kSteps / kKvWarps; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(to_f32(qv[n][i][e])) & 0x7fffffffu);
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) top = max(top, __shfl_xor_sync(kFullMask, top, x));
    if (t == 0) s_qtop[warp][n][g] = top;
  }
  __syncthreads();
  const auto power = [&](int n, int row) {  // of the row's largest entry; a row of zeros or of no numbers has any
    unsigned top = 0;
    for (int w = 0; w < kKvWarps; ++w) top = max(top, s_qtop[w][n][row]);
    return max(1, min(254, (int)(top >> 23))) - 127;
  };
  // back: the power of two that takes a row's size and the scale's back, into the exponent's units (base 2).
  int back[kNT][2];
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
    const int lift = kKv8Top - power(n, g);  // up to 140: in two factors
    const float up = kv_power(lift / 2), more = kv_power(lift - lift / 2);
#pragma unroll
    for (int i = 0; i < kSteps / kKvWarps; ++i) {
      alignas(8) __half x[4];
      put2(x, to_f32(qv[n][i][0]) * up * more, to_f32(qv[n][i][1]) * up * more);
      put2(x + 2, to_f32(qv[n][i][2]) * up * more, to_f32(qv[n][i][3]) * up * more);
      s_q[n][i * kKvWarps + warp][lane] = *reinterpret_cast<uint2*>(x);
    }
    back[n][0] = power(n, 2 * t) - kKv8Top + P.scale_power;
    back[n][1] = power(n, 2 * t + 1) - kKv8Top + P.scale_power;
  }
  __syncthreads();

  float o[kNT][kSteps][4] = {};  // scaled by `unit`
  float2 sum[kNT] = {};
  // Weights are 2^(score + less), the reference being -less; bound is where a score moves it: 4
  // above, rounded down where scores are so large (so the reference cannot be had back from it), and
  // -inf while nothing has been seen. With their steps weights are held times `unit`, which puts the largest that the row has met
  // at 2^kKv8StepExp; reach is where a weight with the power of two above its value's step, in exponents, moves it, 4 above. A row's numbers hang on
  // nothing but what the row sees.
  float2 less[kNT] = {}, unit[kNT];
  float bound[kNT][2], reach[kNT][2];
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
    bound[n][0] = bound[n][1] = reach[n][0] = reach[n][1] = kNone;
    unit[n] = make_float2(1.f, 1.f);
  }
  const auto reference = [&](int n, int c) { return bound[n][c] == kNone ? kNone : -(c ? less[n].y : less[n].x); };

  // This lane's sums set aside, 32 lanes apart; `aside` once there are some.
  float4* apart = reinterpret_cast<float4*>(s_ring + kv8_ring_bytes(kDim, kNT, kBrief)) + warp * (kRows * kDim / 4) + lane;
  bool ok = true, aside = false;
  int stage = 0, turn = 0;
  for (int k = 0; ok && k < count;) {
    const int pause = min(count, k + kKv8Aside);
    for (; k < pause; ++k, ++u) {
      const int tok0 = u * kUnit;
      const unsigned char* runs = ring + stage * kStage;
      const unsigned gone = missing >> (8 * stage) & ((1u << kRuns) - 1);
      ok = ok && warp_wait_quick(&s_full[warp][stage], turn);
      if (!ok) break;
      // Scores: s[i][n][h] holds token tok0 + 16 i + 8 h + g against rows 8 n + 2 t
      // and the next.
      float2 s[kRuns][kNT][2];
      float2 steps[kRuns];
      float above = kNone;  // of all of them
      {
        float acc[kRuns][kNT][4] = {};
#pragma unroll
        for (int c = 0; c < kDim / 64; ++c) {
          uint32_t kc[kRuns][2][4];
#pragma unroll
          for (int i = 0; i < kRuns; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) kv_load(kc[i][h], runs + i * kRunBytes + h * (8 * kDim) + c * 512 + lane * 16);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint2 q[kNT];
#pragma unroll
            for (int n = 0; n < kNT; ++n) q[n] = s_q[n][4 * c + w][lane];
#pragma unroll
            for (int i = 0; i < kRuns; ++i) {
              const uint32_t a[4] = {kv8_codes<0>(kc[i][0][w]), kv8_codes<0>(kc[i][1][w]), kv8_codes<1>(kc[i][0][w]), kv8_codes<1>(kc[i][1][w])};
#pragma unroll
              for (int n = 0; n < kNT; ++n) kv_mma<__half>(acc[i][n], a, q[n].x, q[n].y);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < kRuns; ++i) {
          const float4 of_run = s_step[warp][stage][i];
          steps[i] = make_float2(of_run.x, of_run.y);
          above = fmaxf(above, of_run.z);
          const float keys = steps[i].x > 0.f ? kv8_part(steps[i].x) * P.scale_part : steps[i].x;  // 0 and NaN as they are
          const int e = kv8_power(steps[i].x);  // (factors below 2^97, products below 2^29: no score is infinite, nor 0 times one NaN)
#pragma unroll
          for (int n = 0; n < kNT; ++n) {
            const float2 f = make_float2(keys * kv_power(min(94, e + back[n][0])), keys * kv_power(min(94, e + back[n][1])));
#pragma unroll
            for (int h = 0; h < 2; ++h) s[i][n][h] = __fmul2_rn(make_float2(acc[i][n][2 * h], acc[i][n][2 * h + 1]), f);
          }
        }
      }
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
            }
        }
      }
      // The largest score, and whether a weight with the power of two above its value's step may be further up than any before. (That is
      // added to the difference: next to a large score it would be lost.)
      float up[kNT][2];
      bool move = false;
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        up[n][0] = up[n][1] = kNone;
#pragma unroll
        for (int i = 0; i < kRuns; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            up[n][0] = fmaxf(up[n][0], s[i][n][h].x);
            up[n][1] = fmaxf(up[n][1], s[i][n][h].y);
          }
        move = move || up[n][0] > bound[n][0] || up[n][1] > bound[n][1] || up[n][0] + less[n].x + above > reach[n][0] || up[n][1] + less[n].y + above > reach[n][1];
      }
      if (__any_sync(kFullMask, move)) {
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          float keep[2], all[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            // The row's largest score in each run. (Shuffles by the whole warp, whatever its rows need; all of a row's lanes decide alike.)
            float high[kRuns];
#pragma unroll
            for (int i = 0; i < kRuns; ++i) {
              high[i] = c ? fmaxf(s[i][n][0].y, s[i][n][1].y) : fmaxf(s[i][n][0].x, s[i][n][1].x);
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) high[i] = fmaxf(high[i], __shfl_xor_sync(kFullMask, high[i], x));
            }
            const float last = reference(n, c), was = c ? unit[n].y : unit[n].x;
            float next = last;
#pragma unroll
            for (int i = 0; i < kRuns; ++i) next = fmaxf(next, high[i]);
            // The largest weight with the power of two above its value's step, in exponents, against a reference.
            const auto furthest = [&](float base) {
              float x = kNone;
#pragma unroll
              for (int i = 0; i < kRuns; ++i) x = fmaxf(x, high[i] - base + kv8_above(steps[i].y));
              return x;
            };
            const bool mine = next > bound[n][c] || furthest(last) > reach[n][c];
            const float top = fmaxf(furthest(next), reach[n][c] - kKvLazy - (next - last));
            keep[c] = all[c] = 1.f;
            if (mine) {
              const int power = min(100, max(-126, kKv8StepExp - (int)ceilf(fmaxf(top, -200.f)))), by = power - kv8_power(was);
              keep[c] = kv_exp2(last - next);
              all[c] = keep[c] * (by < -126 ? 0.f : kv_power(by));
              bound[n][c] = __fadd_rd(next, kKvLazy);
              reach[n][c] = top + kKvLazy;
              (c ? less[n].y : less[n].x) = -next;
              (c ? unit[n].y : unit[n].x) = kv_power(power);
            }
          }
          sum[n] = make_float2(sum[n].x * keep[0], sum[n].y * keep[1]);
#pragma unroll
          for (int j = 0; j < kSteps; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][j][e] *= all[e & 1];
          if (aside) {
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
              float4 a = apart[32 * (n * kSteps + j)];
              a.x *= all[0], a.y *= all[1], a.z *= all[0], a.w *= all[1];
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
          uint32_t w[2][kNT][2];
#pragma unroll
          for (int n = 0; n < kNT; ++n) {
            const float2 scaled = make_float2(kv8_scaled(steps[i].y, unit[n].x), kv8_scaled(steps[i].y, unit[n].y));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float2 e = __fadd2_rn(s[i][n][h], less[n]), p = make_float2(kv_exp2(e.x), kv_exp2(e.y));
              sum[n] = __fadd2_rn(sum[n], p);
              float2 x = __fmul2_rn(p, scaled);
              if constexpr (!kAll) {  // what a row does not see may be NaN
                if (!(seen[n] >> (4 * i + 2 * h) & 1)) x.x = 0.f;
                if (!(seen[n] >> (4 * i + 2 * h) & 2)) x.y = 0.f;
              }
              const uint32_t high = kv_pack(x);
              w[0][n][h] = kv_transpose(high);
              const float2 top = __half22float2(__hneg2(reinterpret_cast<const __half2&>(high)));
              w[1][n][h] = kv_transpose(kv_pack(__fadd2_rn(x, top)));
            }
          }
#pragma unroll
          for (int c = 0; c < kDim / 32; ++c) {
            uint32_t vc[4];
            kv_load(vc, runs + i * kRunBytes + 16 * kDim + c * 512 + lane * 16);
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const uint32_t a[4] = {kv8_codes<0>(vc[2 * z]), kv8_codes<0>(vc[2 * z + 1]), kv8_codes<1>(vc[2 * z]), kv8_codes<1>(vc[2 * z + 1])};
#pragma unroll
              for (int n = 0; n < kNT; ++n)
#pragma unroll
                for (int half = 0; half < 2; ++half) kv_mma<__half>(o[n][2 * c + z], a, w[half][n][0], w[half][n][1]);
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

  // The warps' parts: o[n][j][e] is channel 16 j + g + 8 (e / 2) of row 8 n + 2 t + e % 2. With their sums of weights they are
  // held times 2^-24, so that many of the type's largest values add up to a number still.
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float l = c ? sum[n].y : sum[n].x;
      const float lower = kv_power(-24 - kv8_power(c ? unit[n].y : unit[n].x));
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(kFullMask, l, x);
      if (g == 0) s_ml[warp][8 * n + 2 * t + c] = make_float2(reference(n, c), l * 0x1p-24f);
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        s_o[warp][8 * n + 2 * t + c][16 * j + g] = o[n][j][c] * lower;
        s_o[warp][8 * n + 2 * t + c][16 * j + g + 8] = o[n][j][2 + c] * lower;
      }
    }
  __syncthreads();
  kv_join_warps<T, kDim, kRows>(P, s_o, s_ml, reinterpret_cast<float*>(s_q), &s_bad, split, tile, head, b, rows, row0);
}

}  // namespace qrb200
