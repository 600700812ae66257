// Attention of a few queries over the 4-bit cache (layout and formulas: kv4.cuh).
//
// With c the centred code (code - 8, exact in 16 bits) and mid = m + 8 s:
//   q . k_t = sum_groups s_t (q . c_t) + mid_t sum(q),     o = sum_t (p_t s_t) c_t + sum_t p_t mid_t.
// So the codes themselves are the matrix operands: no key or value is ever rounded to 16 bits, steps and
// minima are applied in 32. Keys (and values transposed) are the 16-row left operand, 8 query rows that share the key
// head the right one, so a head with few query rows wastes little of the matrix instruction. The weights p_t s_t are the
// only rounded operand: each is two bf16 halves, high and low, 16 bits of significand in all.
//
// A warp takes 32 or 64 tokens at a time: scores, running maximum (base 2), weights, output. Codes go from global memory
// straight to registers; the next tokens' keys load while the current ones' softmax and output run.
// The token range is cut over CTAs (blockIdx.x) and over a CTA's four warps; the parts are joined through shared memory and,
// between CTAs, by kv4_join_kernel, in a fixed order.
#pragma once

#include "kv4.cuh"

namespace qrb200 {

struct Kv4AttnParams {
  const unsigned char* cache;
  const void* q;
  void* out;
  float* part_o;       // [batch][head][tile][split][rows of a tile][dim], unnormalised, when splits > 1
  float2* part_ml;     // [...][rows of a tile]: maximum (base 2) and sum
  const int* table;
  const int* lengths;
  long long q_bs, q_ts, q_hs, table_stride;  // strides in elements
  int batch, queries, q_heads, share, max_pages, window, causal, splits, tiles;
  float scale2;  // scale times log2(e)
  Kv4Shape sh;
};

constexpr int kKvWarps = 4;
// Runs of 16 tokens in a warp's step: as many as the registers hold beside the output (twice the channels, half the runs).
__host__ __device__ constexpr int kv_runs(int dim) { return dim == 64 ? 4 : 2; }

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

// Nibbles p and p + 4 of w as a pair of 16-bit numbers, less 8. Placed under an exponent whose unit is
// 1 (128 in bf16, 1024 in fp16), a nibble is that power of two plus its code, exactly; the subtraction is exact too.
template <typename T>
__device__ __forceinline__ uint32_t kv_pair(uint32_t w, int p);
template <>
__device__ __forceinline__ uint32_t kv_pair<__nv_bfloat16>(uint32_t w, int p) {
  const uint32_t x = ((w >> (4 * p)) & 0x000f000fu) | 0x43004300u;
  const __nv_bfloat162 r = __hsub2(reinterpret_cast<const __nv_bfloat162&>(x), __floats2bfloat162_rn(136.f, 136.f));
  return reinterpret_cast<const uint32_t&>(r);
}
template <>
__device__ __forceinline__ uint32_t kv_pair<__half>(uint32_t w, int p) {
  const uint32_t x = ((w >> (4 * p)) & 0x000f000fu) | 0x64006400u;
  const __half2 r = __hsub2(reinterpret_cast<const __half2&>(x), __floats2half2_rn(1032.f, 1032.f));
  return reinterpret_cast<const uint32_t&>(r);
}

__device__ __forceinline__ uint32_t kv_pack_bf16(float lo, float hi) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(r);
}
__device__ __forceinline__ uint32_t kv_transpose(uint32_t x) {  // an 8 x 8 matrix of 16-bit numbers over the warp
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float kv_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <int kWords>
__device__ __forceinline__ void kv_load(uint32_t (&w)[kWords], const unsigned char* p) {
  if constexpr (kWords == 4) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (kWords == 2) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
}
// A (step, minimum) word as (step, minimum + 8 steps).
template <typename T>
__device__ __forceinline__ float2 kv_step_mid(uint32_t w) {
  const Pair16<T> pr = reinterpret_cast<const Pair16<T>&>(w);
  const float s = to_f32(pr.s);
  return make_float2(s, fmaf(8.f, s, to_f32(pr.m)));
}

template <typename T, int kDim, int kGroups, int kNT>
__global__ void __launch_bounds__(32 * kKvWarps, kNT == 1 ? 3 : 2) kv4_attention_kernel(Kv4AttnParams P) {
  constexpr int kRows = 8 * kNT;           // query rows of a tile
  constexpr int kSteps = kDim / 16;        // 16-channel steps of q . k; also 16-channel tiles of the output
  constexpr int kPer = kSteps / kGroups;   // steps of a group
  constexpr int kKW = kDim / 32;           // words of a lane's key codes, for one token
  constexpr int kVC = kDim / 64;           // 16-byte pieces of a lane's value codes, for 16 tokens
  constexpr int kRuns = kv_runs(kDim), kUnit = 16 * kRuns;
  constexpr float kNone = -INFINITY;
  __shared__ float s_o[kKvWarps][kRows][kDim + 4];
  __shared__ float2 s_ml[kKvWarps][kRows];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x, head = blockIdx.y % P.sh.heads, tile = blockIdx.y / P.sh.heads, b = blockIdx.z;
  const int rows = P.queries * P.share, row0 = tile * kRows;
  const int block_bytes = P.sh.block_bytes();

  griddep_launch_wait();
  int len = P.lengths[b];
  if (len < 0 || len > (long long)P.max_pages * P.sh.page) {
    if (threadIdx.x == 0) report_device_failure(kSiteIndex);
    len = 0;
  }
  // Tokens [lo, hi) that a query row sees; those of this thread's two columns of each 8.
  auto range = [&](int r, int& lo, int& hi) {
    const int pos = len - P.queries + r / P.share;
    hi = r >= rows ? 0 : P.causal ? max(0, pos + 1) : len;
    lo = P.window > 0 ? max(0, pos - P.window + 1) : 0;
  };
  int lo[kNT][2], hi[kNT][2], all_lo = 0x7fffffff, all_hi = 0, in_lo = 0, in_hi = 0x7fffffff;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    int l, h;
    range(row0 + r, l, h);
    if (h > l) {
      all_lo = min(all_lo, l);
      all_hi = max(all_hi, h);
    }
    if (row0 + r < rows) {
      in_lo = max(in_lo, l);
      in_hi = min(in_hi, h);
    }
  }
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) range(row0 + 8 * n + 2 * t + c, lo[n][c], hi[n][c]);
  const int u0 = all_hi > 0 ? all_lo / kUnit : 0, u1 = (all_hi + kUnit - 1) / kUnit;
  const int per = (u1 - u0 + P.splits - 1) / P.splits;
  const int u_lo = u0 + split * per, u_hi = min(u1, u_lo + per);

  // Queries as the right operand: step j wants channels 16 j + 4 t + {0, 1} and {2, 3} of row g.
  uint32_t qf[kNT][kSteps][2];
  float qsum[kNT][kGroups][2];
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
    const int r = row0 + 8 * n + g;
    const T* q = static_cast<const T*>(P.q) + b * P.q_bs + (long long)(r / P.share) * P.q_ts +
                 (head * P.share + r % P.share) * P.q_hs + 4 * t;
#pragma unroll
    for (int gr = 0; gr < kGroups; ++gr) {
      float sum = 0.f;
#pragma unroll
      for (int j = gr * kPer; j < (gr + 1) * kPer; ++j) {
        T x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = r < rows ? q[16 * j + e] : from_f32<T>(0.f);
          sum += to_f32(x[e]);
        }
        qf[n][j][0] = reinterpret_cast<uint32_t*>(x)[0];
        qf[n][j][1] = reinterpret_cast<uint32_t*>(x)[1];
      }
      sum += __shfl_xor_sync(kFullMask, sum, 1);
      sum += __shfl_xor_sync(kFullMask, sum, 2);  // row g's sum, in its four lanes
      qsum[n][gr][0] = __shfl_sync(kFullMask, sum, 8 * t);
      qsum[n][gr][1] = __shfl_sync(kFullMask, sum, 8 * t + 4);
    }
  }

  float o[kNT][kSteps][4] = {};
  float top[kNT][2], sum[kNT][2] = {}, mids[kNT][kGroups][2] = {};
#pragma unroll
  for (int n = 0; n < kNT; ++n) top[n][0] = top[n][1] = kNone;

  // Where a unit's runs of 16 tokens lie: the block of each run's page, or null past the range.
  const unsigned char* blocks[kRuns];
  auto locate = [&](int u) {
    const int tok = u * kUnit + 16 * (t & (kRuns - 1));
    int page = -1;
    if (u < u_hi && tok < len) {
      page = __ldg(P.table + b * P.table_stride + tok / P.sh.page);
      if (page < 0 || page >= P.sh.pages) {
        if (g == 0 && t < kRuns) report_device_failure(kSiteIndex);
        page = -1;
      }
    }
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const int pg = __shfl_sync(kFullMask, page, i);
      blocks[i] = pg < 0 ? nullptr : P.cache + ((long long)pg * P.sh.heads + head) * block_bytes;
    }
  };
  uint32_t kc[kRuns][2][kKW], kp[kRuns][2][kGroups];
  auto load_keys = [&](int u) {
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const int at = (u * kUnit + 16 * i) & (P.sh.page - 1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (blocks[i]) {
          const int tok = at + g + 8 * h;
          kv_load(kc[i][h], blocks[i] + tok * (kDim / 2) + t * (kDim / 8));
          kv_load(kp[i][h], blocks[i] + P.sh.k_pairs() + tok * (4 * kGroups));
        } else {
#pragma unroll
          for (int w = 0; w < kKW; ++w) kc[i][h][w] = 0;
#pragma unroll
          for (int w = 0; w < kGroups; ++w) kp[i][h][w] = 0;
        }
      }
    }
  };

  int u = u_lo + warp;
  locate(u);
  load_keys(u);
  for (; u < u_hi; u += kKvWarps) {
    const int tok0 = u * kUnit;
    uint32_t vc[kRuns][kVC][4], vp[kRuns][2][kGroups];
    bool there = true;
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const int at = (tok0 + 16 * i) & (P.sh.page - 1);
      there = there && blocks[i];
#pragma unroll
      for (int c = 0; c < kVC; ++c) {
        if (blocks[i]) kv_load(vc[i][c], blocks[i] + P.sh.v_codes() + (at >> 4) * (8 * kDim) + c * 512 + lane * 16);
        else vc[i][c][0] = vc[i][c][1] = vc[i][c][2] = vc[i][c][3] = 0;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (blocks[i]) kv_load(vp[i][h], blocks[i] + P.sh.v_pairs() + (at + g + 8 * h) * (4 * kGroups));
        else
#pragma unroll
          for (int w = 0; w < kGroups; ++w) vp[i][h][w] = 0;
      }
    }
    // Scores, in base 2: s[i][n][2 h + c] is token tok0 + 16 i + 8 h + g against row 8 n + 2 t + c.
    float s[kRuns][kNT][4];
    unsigned gone = 0;  // runs whose page is missing
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      gone |= blocks[i] ? 0u : 1u << i;
#pragma unroll
      for (int n = 0; n < kNT; ++n) s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.f;
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) {
        float acc[kNT][4] = {};
#pragma unroll
        for (int j = gr * kPer; j < (gr + 1) * kPer; ++j) {
          const int p = 2 * (j & 1);
          const uint32_t a[4] = {kv_pair<T>(kc[i][0][j >> 1], p), kv_pair<T>(kc[i][1][j >> 1], p),
                                 kv_pair<T>(kc[i][0][j >> 1], p + 1), kv_pair<T>(kc[i][1][j >> 1], p + 1)};
#pragma unroll
          for (int n = 0; n < kNT; ++n) kv_mma<T>(acc[n], a, qf[n][j][0], qf[n][j][1]);
        }
        const float2 k0 = kv_step_mid<T>(kp[i][0][gr]), k1 = kv_step_mid<T>(kp[i][1][gr]);
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          s[i][n][0] += fmaf(k0.x, acc[n][0], k0.y * qsum[n][gr][0]);
          s[i][n][1] += fmaf(k0.x, acc[n][1], k0.y * qsum[n][gr][1]);
          s[i][n][2] += fmaf(k1.x, acc[n][2], k1.y * qsum[n][gr][0]);
          s[i][n][3] += fmaf(k1.x, acc[n][3], k1.y * qsum[n][gr][1]);
        }
      }
    }
    locate(u + kKvWarps);  // the next unit's keys are under way while this one's softmax and output run
    load_keys(u + kKvWarps);

    const bool full = !gone && tok0 >= in_lo && tok0 + kUnit <= in_hi;  // every row sees every token
    uint32_t seen[kNT];
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      seen[n] = 0xffffu;
      if (!full) {
#pragma unroll
        for (int i = 0; i < kRuns; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int tok = tok0 + 16 * i + 8 * (e >> 1) + g;
            if (tok < lo[n][e & 1] || tok >= hi[n][e & 1] || (gone >> i & 1)) seen[n] &= ~(1u << (4 * i + e));
          }
      }
    }
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      float up[2] = {top[n][0], top[n][1]}, ref[2], keep[2];
#pragma unroll
      for (int i = 0; i < kRuns; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i][n][e] = (seen[n] >> (4 * i + e) & 1) ? s[i][n][e] * P.scale2 : kNone;
          up[e & 1] = fmaxf(up[e & 1], s[i][n][e]);
        }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) up[c] = fmaxf(up[c], __shfl_xor_sync(kFullMask, up[c], x));
        ref[c] = up[c] == kNone ? 0.f : up[c];  // nothing seen yet: every weight is 2^-inf
        keep[c] = kv_exp2(top[n][c] - ref[c]);
        sum[n][c] *= keep[c];
      }
      if (__any_sync(kFullMask, up[0] != top[n][0] || up[1] != top[n][1])) {
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][j][e] *= keep[e & 1];
#pragma unroll
        for (int gr = 0; gr < kGroups; ++gr) {
          mids[n][gr][0] *= keep[0];
          mids[n][gr][1] *= keep[1];
        }
      }
      top[n][0] = up[0];
      top[n][1] = up[1];
#pragma unroll
      for (int i = 0; i < kRuns; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i][n][e] = kv_exp2(s[i][n][e] - ref[e & 1]);
          sum[n][e & 1] += s[i][n][e];
        }
    }
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) {
        const float2 v0 = kv_step_mid<T>(vp[i][0][gr]), v1 = kv_step_mid<T>(vp[i][1][gr]);
        uint32_t high[kNT][2], low[kNT][2];
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          float w[4], m[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[e] = s[i][n][e] * (e < 2 ? v0.x : v1.x);
            m[e] = s[i][n][e] * (e < 2 ? v0.y : v1.y);
            if (!full && !(seen[n] >> (4 * i + e) & 1)) w[e] = m[e] = 0.f;  // what is masked may be NaN
          }
          mids[n][gr][0] += m[0] + m[2];
          mids[n][gr][1] += m[1] + m[3];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t hw = kv_pack_bf16(w[2 * h], w[2 * h + 1]);
            const float r0 = w[2 * h] - __uint_as_float(hw << 16), r1 = w[2 * h + 1] - __uint_as_float(hw & 0xffff0000u);
            high[n][h] = kv_transpose(hw);
            low[n][h] = kv_transpose(kv_pack_bf16(r0, r1));
          }
        }
#pragma unroll
        for (int j = gr * kPer; j < (gr + 1) * kPer; ++j) {
          const uint32_t word = vc[i][j >> 2][j & 3];
          const uint32_t a[4] = {kv_pair<__nv_bfloat16>(word, 0), kv_pair<__nv_bfloat16>(word, 1),
                                 kv_pair<__nv_bfloat16>(word, 2), kv_pair<__nv_bfloat16>(word, 3)};
#pragma unroll
          for (int n = 0; n < kNT; ++n) {
            kv_mma<__nv_bfloat16>(o[n][j], a, high[n][0], high[n][1]);
            kv_mma<__nv_bfloat16>(o[n][j], a, low[n][0], low[n][1]);
          }
        }
      }
    }
  }

  // The warps' parts: o[n][j][e] is channel 16 j + g + 8 (e / 2) of row 8 n + 2 t + e % 2.
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        sum[n][c] += __shfl_xor_sync(kFullMask, sum[n][c], x);
#pragma unroll
        for (int gr = 0; gr < kGroups; ++gr) mids[n][gr][c] += __shfl_xor_sync(kFullMask, mids[n][gr][c], x);
      }
      if (g == 0) s_ml[warp][8 * n + 2 * t + c] = make_float2(top[n][c], sum[n][c]);
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        s_o[warp][8 * n + 2 * t + c][16 * j + g] = o[n][j][c] + mids[n][j / kPer][c];
        s_o[warp][8 * n + 2 * t + c][16 * j + g + 8] = o[n][j][2 + c] + mids[n][j / kPer][c];
      }
    }
  __syncthreads();
  constexpr int kLanesRow = 32 * kKvWarps / kRows;  // threads of a row
  const int r = threadIdx.x / kLanesRow, d0 = threadIdx.x % kLanesRow;
  if (row0 + r >= rows) return;
  float m = kNone, l = 0.f, f[kKvWarps];
#pragma unroll
  for (int w = 0; w < kKvWarps; ++w) m = fmaxf(m, s_ml[w][r].x);
#pragma unroll
  for (int w = 0; w < kKvWarps; ++w) {
    f[w] = s_ml[w][r].x == kNone ? (s_ml[w][r].y == 0.f ? 0.f : s_ml[w][r].y) : kv_exp2(s_ml[w][r].x - m);
    l = fmaf(f[w], s_ml[w][r].y, l);
  }
  const long long part = (((long long)b * P.sh.heads + head) * P.tiles + tile) * P.splits + split;
  T* out = static_cast<T*>(P.out) +
           (((long long)b * P.queries + (row0 + r) / P.share) * P.q_heads + head * P.share + (row0 + r) % P.share) * kDim;
  const float inv = l == 0.f ? 0.f : 1.f / l;  // nothing seen: zeros
  for (int d = d0; d < kDim; d += kLanesRow) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kKvWarps; ++w) x = f[w] == 0.f ? x : fmaf(f[w], s_o[w][r][d], x);
    if (P.splits == 1) out[d] = from_f32<T>(x * inv);
    else P.part_o[(part * kRows + r) * kDim + d] = x;
  }
  if (P.splits > 1 && d0 == 0) P.part_ml[part * kRows + r] = make_float2(m, l);
}

// One warp per query row: the splits' parts against their common maximum, in order.
template <typename T, int kDim>
__global__ void __launch_bounds__(128) kv4_join_kernel(Kv4AttnParams P, int tile_rows) {
  griddep_launch_wait();
  const int lane = threadIdx.x & 31, rows = P.queries * P.share;
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (unit >= (long long)P.batch * P.sh.heads * rows) return;
  const int r = (int)(unit % rows), head = (int)(unit / rows % P.sh.heads), b = (int)(unit / rows / P.sh.heads);
  const long long part =
      (((long long)b * P.sh.heads + head) * P.tiles + r / tile_rows) * P.splits * tile_rows + r % tile_rows;
  float m = -INFINITY, l = 0.f, x[kDim / 32] = {};
  for (int s = lane; s < P.splits; s += 32) m = fmaxf(m, P.part_ml[part + (long long)s * tile_rows].x);
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, o));
#pragma unroll 4
  for (int s = 0; s < P.splits; ++s) {
    const float2 ml = P.part_ml[part + (long long)s * tile_rows];
    const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : ml.y) : kv_exp2(ml.x - m);
    l = fmaf(f, ml.y, l);
    const float* o = P.part_o + (part + (long long)s * tile_rows) * kDim;
#pragma unroll
    for (int i = 0; i < kDim / 32; ++i) {
      const float v = o[32 * i + lane];
      x[i] = f == 0.f ? x[i] : fmaf(f, v, x[i]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* out = static_cast<T*>(P.out) +
           (((long long)b * P.queries + r / P.share) * P.q_heads + head * P.share + r % P.share) * kDim;
#pragma unroll
  for (int i = 0; i < kDim / 32; ++i) out[32 * i + lane] = from_f32<T>(x[i] * inv);
}

}  // namespace qrb200
