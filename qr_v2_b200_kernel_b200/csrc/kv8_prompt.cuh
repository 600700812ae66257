// Attention of many queries (prompts, chunks of them) over the 8-bit cache (layout and formulas: kv8.cuh).
//
// Up to 256 query rows that share a key head to a CTA, as two tiles of 128. In steps of 64 tokens:
//   S = Q K^T (fp16 x fp16, Q brought by a power of two to the top of fp16's range, K's codes exact),
//   P = 2^(S r - reference) w,  O += P V  (V's codes exact; r and w the steps of the tokens' pages),
// S, P and O in tensor memory (P takes S's place), the softmax of a row in one thread. Each tile has two S, so that
// the scores of the next step are there when a softmax ends.
//
// Two sequences' 2048 queries over 4096 tokens, 16 heads on 4 of 128 channels, bf16: 172 us, 0.60 PFLOP/s (fp16 192, 64 channels
// 143). No pipe is full (tensor 46 %, exponentials 31 %, issue slots 49 %): a tile's step is a chain of its products, the
// loads of its scores, its softmax and its stores, which two tiles and two S fill by half.
//
// Warps 0-3 and 4-7: the softmax of the first and the second tile. Warp 14: bulk copies of the cache's bytes. Warps 8-11:
// these into fp16 operands (16-bit numbers in memory are twice the traffic, and what the cache saves), K-major in the 128-byte
// swizzle, values transposed, which is how their bytes lie. (Loads straight into these warps' registers are waited
// for by the fence that the operands need.) Warps 12 and 13: a tile's MMAs each (their issue takes some 45
// clocks, as long as the smallest of them run).
//
// A matrix instruction cuts off what it adds, so a sum over many tokens comes out small (over 131072 by 2^-10). So O is added in 32 bits
// to sums in global memory every 32 steps, every 16 for fp16 results: of 2 x 2048 queries over 4096 tokens 0.2 % of the bf16
// and 0.7 % of the fp16 results are then not the nearest (of elementary 32-bit operations 0.1 % of the bf16 ones).
//
// P is two fp16 numbers, high and low, 22 bits. (One would do for bf16 results but for a tenth of them, which then are
// not the nearest.) It is scaled, a row at a time, by a power of two that puts the largest weight times step that the row has met
// at 2^11, so weights keep their leading bits down to 2^-25 of the largest, whatever pages the row does not see or has no weight for.
#pragma once

#include "codes.cuh"
#include "kv8_attention.cuh"

namespace qrb200 {

constexpr int kPromptRows = 256, kPromptTokens = 64;
constexpr int kPromptStages = 3, kPromptRaw = 2;  // steps of operands, and of bytes, in shared memory
constexpr int kPromptThreads = 32 * 15;
constexpr int kPromptTop = 11;  // a row's largest weight times step is put below this power of two, and stays below 2^(11 + 4)
// Steps between settings-aside, a power of two. (Both types, 2 x 2048 queries over 4096 tokens: never 158 us, 32 166, 16 183, 8 209.)
__host__ __device__ constexpr int prompt_aside(bool half) { return half ? 16 : 32; }
__host__ __device__ constexpr int prompt_tile(int dim) { return 128 * dim * 2; }  // bytes of 128 rows of fp16
__host__ __device__ constexpr int prompt_smem_bytes(int dim) { return 1024 + (2 + kPromptStages) * prompt_tile(dim) + kPromptRaw * prompt_tile(dim) / 2; }

// kind::f16: fp16 operands, both K-major, 32-bit accumulator.
__host__ __device__ constexpr uint32_t f16_idesc(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }
// The operands' descriptors by their lower words, which hold the addresses; the upper word is the same for all.
__device__ __forceinline__ void f16_mma(uint32_t d, uint32_t a, uint32_t b, uint32_t upper, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %3};\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}\n"
      :
      : "r"(d), "r"(a), "r"(b), "r"(upper), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void f16_mma_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t upper, uint32_t idesc, bool accumulate) {  // A in tensor memory
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}\n"
      :
      : "r"(d), "r"(a), "r"(b), "r"(upper), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void tmem_put16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      :
      : "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_put_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// What turns a row's products with a run's codes into scores. (Products are 2^-24 to 2^29, if not 0: bounded, so that none of them
// times this is infinite, nor 0 times it NaN. NaN stays.)
__device__ __forceinline__ float kv8_factor(float step, float2 back) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(step * back.x * back.y), "f"(0x1p97f));
  return r;
}

// Sums set aside in global memory, by one thread each: added to where they lie, so that nothing waits for them.
__device__ __forceinline__ void aside_store(float4* to, const float4& x) {
  asm volatile("st.relaxed.gpu.global.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(to), "f"(x.x), "f"(x.y), "f"(x.z), "f"(x.w) : "memory");
}
__device__ __forceinline__ void aside_add(float4* to, const float4& x) {
  asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(to), "f"(x.x), "f"(x.y), "f"(x.z), "f"(x.w) : "memory");
}
__device__ __forceinline__ float4 aside_load(const float4* from) {
  float4 x;
  asm volatile("ld.relaxed.gpu.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "l"(from) : "memory");
  return x;
}

// Columns of S (rows of K in shared memory) in their order. Of a step's 64 tokens, four runs of 16, column c holds token
// prompt_token(c): the order that the values' bytes give a lane sixteen neighbours in.
__host__ __device__ constexpr int prompt_run(int c) { return c >> 2 & 3; }
__host__ __device__ constexpr int prompt_token(int c) { return 16 * prompt_run(c) + 2 * (c >> 4) + (c & 1) + 8 * (c >> 1 & 1); }
// A row's 16-byte piece in the 128-byte swizzle.
__device__ __forceinline__ uint32_t swizzled(int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }

// A row's sums join those set aside. Out of line: the loop around it has no registers to spare.
template <int kDim>
static __device__ __noinline__ void prompt_set_aside(uint32_t o_at, float4* to, float lag, bool first) {
  const bool moved = __any_sync(kFullMask, lag != 1.f);
#pragma unroll 1
  for (int c = 0; c < kDim; c += 32) {
    float o[2][16];
    tmem_ask16(o_at + c, o[0]);
    tmem_ask16(o_at + c + 16, o[1]);
    tmem_arrived(o[0]);
    tmem_arrived(o[1]);
#pragma unroll
    for (int i = 0; i < 8; ++i, to += kPromptRows) {
      const float* x = &o[i >> 2][4 * (i & 3)];
      float4 y = make_float4(x[0], x[1], x[2], x[3]);
      if (first || moved) {
        if (!first) {
          const float4 a = aside_load(to);
          y = make_float4(fmaf(a.x, lag, y.x), fmaf(a.y, lag, y.y), fmaf(a.z, lag, y.z), fmaf(a.w, lag, y.w));
        }
        aside_store(to, y);
      } else {
        aside_add(to, y);
      }
    }
  }
}

template <typename T, int kDim>
__global__ void __launch_bounds__(kPromptThreads, 1) kv8_prompt_kernel(Kv8AttnParams P) {
  constexpr int kTile = prompt_tile(kDim), kAtoms = kDim / 64;
  constexpr float kNone = -INFINITY;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ uint64_t raw_full[kPromptRaw], raw_empty[kPromptRaw], kv_full[kPromptStages], kv_empty[kPromptStages], s_full[2][2], p_full[2][2], o_full[2][2];  // [tile][odd steps]
  // (A softmax may be two steps ahead of the products with the values, and a barrier tells a phase only from the one before it:
  // so each step waits for a barrier whose last phase but one is known to be over.)
  __shared__ uint32_t s_tmem;
  __shared__ float4 s_key[kPromptStages], s_value[kPromptStages];  // steps of a stage's runs, the keys' scaled
  __shared__ float s_above[kPromptStages];  // the power of two above the largest of the values' steps
  __shared__ int s_gone[kPromptStages];      // bits: runs without a page
  __shared__ float2 s_step[kPromptRaw][4];
  __shared__ int s_missing[kPromptRaw];
  __shared__ volatile int s_bad;  // a wait ran out: keep to the barriers, write nothing
  unsigned char* sq = align1024(smem_raw);
  unsigned char* sk = sq + 2 * kTile;  // stages of [keys][values], half a tile each
  unsigned char* raw = sk + kPromptStages * kTile;  // steps of the cache's bytes
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = P.batch * P.sh.heads;
  // The last queries, which see most, first.
  const int tile = P.tiles - 1 - (int)(blockIdx.x / units), unit = blockIdx.x % units, head = unit % P.sh.heads, b = unit / P.sh.heads;
  const int rows = P.queries * P.share, row0 = tile * kPromptRows;
  const int both = row0 + 128 < rows ? 2 : 1;  // tiles with rows

  if (threadIdx.x == 0) {
    for (int i = 0; i < kPromptRaw; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], 4);
    }
    for (int i = 0; i < kPromptStages; ++i) {
      mbar_init(&kv_full[i], 4);
      mbar_init(&kv_empty[i], both);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i][0], 1);
      mbar_init(&s_full[i][1], 1);
      mbar_init(&p_full[i][0], 4);
      mbar_init(&p_full[i][1], 4);
      mbar_init(&o_full[i][0], 1);
      mbar_init(&o_full[i][1], 1);
    }
    s_bad = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  griddep_launch_wait();  // before TMEM is taken: a kernel still running may need it
  if (warp == 12) tmem_alloc(&s_tmem, 512);
  int len = P.lengths[b];
  if (len < 0 || len > (long long)P.max_pages * P.sh.page || (len > 0 && P.sh.pages == 0)) {
    if (threadIdx.x == 0) report_device_failure(kSiteIndex);
    len = 0;
  }
  // Tokens [lo, hi) that a row sees, and those of the CTA's rows together.
  const auto range_of = [&](int row, int& lo, int& hi) {
    const int pos = len - P.queries + row / P.share;
    hi = P.causal ? max(0, pos + 1) : len;
    lo = P.window > 0 && pos >= P.window ? pos - P.window + 1 : 0;
    if (lo > hi) lo = hi;
  };
  int all_lo, all_hi, last_lo, last_hi;
  range_of(row0, all_lo, all_hi);
  const int last = min(rows, row0 + kPromptRows) - 1;
  range_of(last, last_lo, last_hi);
  // Positions grow with the row, and so do both ends; rows before the sequence's start see nothing.
  if (all_hi <= all_lo) {
    const int first = P.queries - len;  // the first query at a position
    all_lo = last_lo;
    if (first >= 0 && last >= first * P.share) {
      int hi;
      range_of(max(row0, first * P.share), all_lo, hi);
    }
  }
  all_hi = last_hi;
  const int block0 = all_lo / kPromptTokens, count = all_hi > all_lo ? (all_hi + kPromptTokens - 1) / kPromptTokens - block0 : 0;
  const int first_run = all_lo / 16, last_run = (all_hi + 15) / 16;
  // A run's page, -1 outside the range or where the table is wrong.
  const auto page_of = [&](int run) {
    if (run < first_run || run >= last_run) return -1;
    const int page = __ldg(P.table + b * P.table_stride + (run >> (P.sh.shift - 4)));
    if (page < 0 || page >= P.sh.pages) {
      report_device_failure(kSiteIndex);
      return -1;
    }
    return page;
  };
  const float2* steps = reinterpret_cast<const float2*>(P.range);
  const int page_runs = P.sh.page / 16;

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const auto gave_up = [&]() { return __any_sync(kFullMask, s_bad) != 0; };  // the same to a whole warp, whenever its lanes look
  const int aside_every = P.part_o ? prompt_aside(std::is_same<T, __half>::value) : 1 << 30;

  if (warp < 8) {
    // ---- the softmax of a tile, a row to a thread ----
    const int mine = warp >> 2, in_tile = threadIdx.x & 127, row = row0 + 128 * mine + in_tile;
    const bool real = row < rows;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), o_at = lanes + 256 + 128 * mine;
    int lo = 0, hi = 0;
    float2 back;  // two powers of two that take a row's size and the scale's back, into the exponent's units (base 2)
    if (real) range_of(row, lo, hi);
    {
      // The row's query, permuted as the keys' bytes are: piece k of 64 channels holds channels 16 w + 4 t + e with t =
      // k / 2 and w = 2 (k & 1), 2 (k & 1) + 1.
      const T* q = static_cast<const T*>(P.q) + b * P.q_bs + (long long)(row / P.share) * P.q_ts + (head * P.share + row % P.share) * P.q_hs;
      const auto four = [&](T(&x)[4], int c) {
        if (!real) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = from_f32<T>(0.f);
        } else if (P.q_wide) {
          *reinterpret_cast<uint2*>(x) = __ldg(reinterpret_cast<const uint2*>(q + c));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = q[c + e];
        }
      };
      unsigned top = 0;
#pragma unroll 8
      for (int c = 0; c < kDim; c += 4) {
        alignas(8) T x[4];
        four(x, c);
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(to_f32(x[e])) & 0x7fffffffu);
      }
      const int power = max(1, min(254, (int)(top >> 23))) - 127, lift = kKv8Top - power;
      const float up = kv_power(lift / 2), more = kv_power(lift - lift / 2);
      const int by = power - kKv8Top + P.scale_power;
      back = make_float2(kv_power(by / 2), kv_power(by - by / 2));
#pragma unroll 1
      for (int a = 0; a < kAtoms; ++a)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          alignas(16) __half y[8];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            alignas(8) T x[4];
            four(x, 64 * a + 16 * (2 * (k & 1) + i) + 4 * (k >> 1));
            put2(y + 4 * i, to_f32(x[0]) * up * more, to_f32(x[1]) * up * more);
            put2(y + 4 * i + 2, to_f32(x[2]) * up * more, to_f32(x[3]) * up * more);
          }
          *reinterpret_cast<uint4*>(sq + mine * kTile + a * (128 * 128) + swizzled(in_tile, k)) = *reinterpret_cast<const uint4*>(y);
        }
    }
    fence_async_smem();
    named_sync(1 + mine, 160);  // with the MMAs' warp: the tile's queries are there
    if (mine < both) {
      // What every row of the warp sees.
      const int in_lo = __reduce_max_sync(kFullMask, lo), in_hi = __reduce_min_sync(kFullMask, real ? hi : 0x7fffffff);
      // Weights are 2^(score - ref); with their steps they are held times `unit`, which puts the largest that the row has met, 2^reach
      // at most, at 2^kPromptTop. A row's numbers hang on nothing but what the row sees.
      float ref = kNone, sum = 0.f, reach = kNone, unit = 1.f;
      bool calm = true;  // no row's reference in the warp is so large that its rounding matters
      // Set aside, four channels of a row beside the next row's: the sums of earlier steps, against the reference of then, which `lag`
      // brings to the present one.
      const auto set_aside = [&]() {
        return reinterpret_cast<float4*>(P.part_o) + (long long)blockIdx.x * (kDim / 4 * kPromptRows) + 128 * (threadIdx.x >> 7) + (threadIdx.x & 127);
      };
      float lag = 1.f;
      bool ok = true;
      for (int j = 0; j < count;) {
        const int pause = min(count, j + aside_every);
        for (; j < pause; ++j) {
          const int st = j % kPromptStages, tok0 = (block0 + j) * kPromptTokens;
          const uint32_t s_at = lanes + 128 * mine + 64 * (j & 1);
          ok = ok && mbar_wait_quick(&s_full[mine][j & 1], (j >> 1) & 1);
          __syncwarp();
          tc_fence_after();
          float v[4][16];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ask16(s_at + 16 * c, v[c]);
          const float4 k4 = s_key[st], w4 = s_value[st];
          const float f[4] = {kv8_factor(k4.x, back), kv8_factor(k4.y, back), kv8_factor(k4.z, back), kv8_factor(k4.w, back)}, w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_arrived(v[c]);
          const int gone = s_gone[st];
          const bool full = tok0 >= in_lo && tok0 + kPromptTokens <= in_hi && gone == 0;
          // The largest score of each run. (Factors are not negative, so the largest product gives it.)
          float score[4];
          const auto largest = [&](auto all) {
            constexpr bool kAll = decltype(all)::value;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float m = kNone;
#pragma unroll
              for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int at = tok0 + prompt_token(16 * c + 4 * r + i);
                  const float x = v[c][4 * r + i];
                  m = kAll || (at >= lo && at < hi && !(gone >> r & 1)) ? fmaxf(m, x) : m;
                }
              score[r] = kAll || m > kNone ? __fmul_rn(m, f[r]) : kNone;  // (rounded before anything is taken from it)
            }
          };
          if (full) largest(std::true_type{});
          else largest(std::false_type{});
          // Of all, and with the power of two above its value's step, which is added to the difference: next to a large score it would be lost.
          const float top = fmaxf(fmaxf(score[0], score[1]), fmaxf(score[2], score[3])), base = ref == kNone ? top : ref;
          // (First with the largest of the steps, which the row need not see.)
          if (__any_sync(kFullMask, top > __fadd_rd(ref, kKvLazy) || top - base + s_above[st] > reach + kKvLazy || (ref == kNone && top > kNone))) {
            float far = kNone;
#pragma unroll
            for (int r = 0; r < 4; ++r) far = fmaxf(far, score[r] - base + kv8_above(w[r]));
            const bool move = top > __fadd_rd(ref, kKvLazy) || far > reach + kKvLazy || (ref == kNone && top > kNone);
            float keep = 1.f, ratio = 1.f;
            const bool none = ref == kNone;
            if (move) {
              const float next = fmaxf(ref, top);
              reach = fmaxf(reach, far) - (next - base);
              const int power = min(100, max(-126, kPromptTop - (int)ceilf(fmaxf(reach, -200.f)))), by = power - kv8_power(unit);
              keep = none ? 0.f : kv_exp2(ref - next);
              ratio = by < -126 ? 0.f : kv_power(by);
              unit = kv_power(power);
              ref = next;
            }
            if ((j & (aside_every - 1)) != 0) {  // once the products before are over
              ok = ok && mbar_wait_quick(&o_full[mine][(j - 1) & 1], ((j - 1) >> 1) & 1);
              __syncwarp();
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < kDim; c += 16) {
                float o[16];
                tmem_ask16(o_at + c, o);
                tmem_arrived(o);
                uint32_t kept[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) kept[i] = __float_as_uint(none ? 0.f : o[i] * (keep * ratio));
                tmem_put16(o_at + c, kept);
              }
              tmem_put_wait();
            }
            sum *= keep;
            lag *= keep * ratio;
            calm = __all_sync(kFullMask, ref == kNone || fabsf(ref) < 0x1p20f);
          }
          const float scaled[4] = {kv8_scaled(w[0], unit), kv8_scaled(w[1], unit), kv8_scaled(w[2], unit), kv8_scaled(w[3], unit)};
          const float less = ref == kNone ? 0.f : -ref;
          const float2 less2 = make_float2(less, less);
          float2 sums = make_float2(0.f, 0.f);
          const auto weights = [&](auto all) {
            constexpr bool kAll = decltype(all)::value;
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
              uint32_t high[16], low[16];
#pragma unroll
              for (int d = 0; d < 2; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const float2 f2 = make_float2(f[r], f[r]), w2 = make_float2(scaled[r], scaled[r]);
#pragma unroll
                  for (int i = 0; i < 4; i += 2) {
                    // (In one operation the difference from a large reference is that of the unrounded score, which may be far above 0;
                    // paired products and sums would be made one.)
                    const float2 v2 = make_float2(v[c + d][4 * r + i], v[c + d][4 * r + i + 1]);
                    const float2 x = kAll ? __ffma2_rn(v2, f2, less2) : make_float2(__fmul_rn(v2.x, f[r]) + less, __fmul_rn(v2.y, f[r]) + less);
                    const int at = tok0 + prompt_token(16 * (c + d) + 4 * r + i);  // and the next
                    const bool one = kAll || (at >= lo && at < hi && !(gone >> r & 1)), two = kAll || (at + 1 >= lo && at + 1 < hi && !(gone >> r & 1));
                    float2 p = make_float2(one ? kv_exp2(x.x) : 0.f, two ? kv_exp2(x.y) : 0.f);
                    sums = __fadd2_rn(sums, p);
                    p = __fmul2_rn(p, w2);
                    if constexpr (!kAll) {  // what a row does not see may be NaN
                      if (!one) p.x = 0.f;
                      if (!two) p.y = 0.f;
                    }
                    high[8 * d + 2 * r + i / 2] = kv_pack(p);
                    const float2 back2 = __half22float2(__hneg2(reinterpret_cast<const __half2&>(high[8 * d + 2 * r + i / 2])));
                    low[8 * d + 2 * r + i / 2] = kv_pack(__fadd2_rn(p, back2));
                  }
                }
              tmem_put16(s_at + 16 * c, high);
              tmem_put16(s_at + 16 * c + 16, low);
            }
          };
          if (full && calm) weights(std::true_type{});
          else weights(std::false_type{});
          sum += sums.x + sums.y;
          tmem_put_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[mine][j & 1]);
        }
        if (j < count) {  // the next product with the values begins new sums
          ok = ok && mbar_wait_quick(&o_full[mine][(j - 1) & 1], ((j - 1) >> 1) & 1);
          __syncwarp();
          tc_fence_after();
          prompt_set_aside<kDim>(o_at, set_aside(), lag, j == aside_every);
          lag = 1.f;
        }
      }
      if (count > 0) ok = ok && mbar_wait_quick(&o_full[mine][(count - 1) & 1], ((count - 1) >> 1) & 1);
      if (!ok) s_bad = 1;
      __syncwarp();
      tc_fence_after();
      const float inv = sum == 0.f ? 0.f : kv_power(-kv8_power(unit)) / sum;  // nothing seen: zeros
      T* out = static_cast<T*>(P.out) + (((long long)b * P.queries + row / P.share) * P.q_heads + head * P.share + row % P.share) * kDim;
      const bool apart = count > aside_every;
      float4 a[2][8];
      const auto ask = [&](int c) {
        if (apart && c < kDim)
#pragma unroll
          for (int i = 0; i < 8; ++i) a[c >> 5 & 1][i] = aside_load(set_aside() + (c / 4 + i) * kPromptRows);
      };
      ask(0);
#pragma unroll
      for (int c = 0; c < kDim; c += 16) {
        if ((c & 31) == 0) ask(c + 32);
        float o[16] = {};
        if (count > 0) {
          tmem_ask16(o_at + c, o);
          tmem_arrived(o);
        }
        if (apart) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 x = a[c >> 5 & 1][(c >> 2 & 4) + i];
            o[4 * i] = fmaf(x.x, lag, o[4 * i]), o[4 * i + 1] = fmaf(x.y, lag, o[4 * i + 1]);
            o[4 * i + 2] = fmaf(x.z, lag, o[4 * i + 2]), o[4 * i + 3] = fmaf(x.w, lag, o[4 * i + 3]);
          }
        }
        alignas(16) T y[16];
#pragma unroll
        for (int i = 0; i < 16; i += 2) put2(y + i, sum == 0.f ? 0.f : o[i] * inv, sum == 0.f ? 0.f : o[i + 1] * inv);
        if (real && !s_bad) {
          *reinterpret_cast<uint4*>(out + c) = *reinterpret_cast<const uint4*>(y);
          *reinterpret_cast<uint4*>(out + c + 8) = *reinterpret_cast<const uint4*>(y + 8);
        }
      }
    }
  } else if (warp < 12) {
    // ---- keys and values to operands ----
    // 64 channels: two warps take two runs of keys each, two 32 channels of values. 128: each takes a run and 32 channels.
    const int cw = warp - 8, g = lane >> 2, t = lane & 3;
    constexpr bool kBoth = kAtoms == 2;
    constexpr int kRun = 32 * kDim;
    for (int j = 0; j < count; ++j) {
      const int st = j % kPromptStages, rs = j % kPromptRaw;
      unsigned char* keys = sk + st * kTile;
      unsigned char* values = keys + kTile / 2;
      const unsigned char* from = raw + rs * (kTile / 2) + lane * 16;
      bool bad = gave_up() || !warp_wait_quick(&raw_full[rs], (j / kPromptRaw) & 1);
      bad = bad || (j >= kPromptStages && !warp_wait_quick(&kv_empty[st], (j / kPromptStages - 1) & 1));
      if (bad) s_bad = 1;
      if (kBoth || cw < 2)
#pragma unroll
        for (int l = 0; l < 4; ++l) {
          const int run = kBoth ? cw : 2 * cw + (l >> 1), h = kBoth ? l >> 1 : l & 1, a = kBoth ? l & 1 : 0;
          const int row = 16 * (g >> 1) + 4 * run + 2 * h + (g & 1);
          const uint4 w = *reinterpret_cast<const uint4*>(from + run * kRun + h * (8 * kDim) + a * 512);
          unsigned char* to = keys + a * (64 * 128);
          *reinterpret_cast<uint4*>(to + swizzled(row, 2 * t)) = make_uint4(kv8_codes<0>(w.x), kv8_codes<1>(w.x), kv8_codes<0>(w.y), kv8_codes<1>(w.y));
          *reinterpret_cast<uint4*>(to + swizzled(row, 2 * t + 1)) = make_uint4(kv8_codes<0>(w.z), kv8_codes<1>(w.z), kv8_codes<0>(w.w), kv8_codes<1>(w.w));
        }
      if (kBoth || cw >= 2) {
        const int piece = kBoth ? cw : cw - 2;
        uint4 w[4];
#pragma unroll
        for (int l = 0; l < 4; ++l) w[l] = *reinterpret_cast<const uint4*>(from + l * kRun + 16 * kDim + piece * 512);
        const auto put = [&](int i, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
          const int row = 32 * piece + 8 * i + g;
          *reinterpret_cast<uint4*>(values + swizzled(row, 2 * t)) = make_uint4(kv8_codes<0>(w0), kv8_codes<1>(w0), kv8_codes<0>(w1), kv8_codes<1>(w1));
          *reinterpret_cast<uint4*>(values + swizzled(row, 2 * t + 1)) = make_uint4(kv8_codes<0>(w2), kv8_codes<1>(w2), kv8_codes<0>(w3), kv8_codes<1>(w3));
        };
        put(0, w[0].x, w[1].x, w[2].x, w[3].x);
        put(1, w[0].y, w[1].y, w[2].y, w[3].y);
        put(2, w[0].z, w[1].z, w[2].z, w[3].z);
        put(3, w[0].w, w[1].w, w[2].w, w[3].w);
      }
      if (cw == 0 && lane < 4) {
        const float2 step = s_step[rs][lane];
        reinterpret_cast<float*>(&s_key[st])[lane] = step.x * P.scale_part;  // (steps are 2^-107 to 2^121, the scale's part below 3)
        reinterpret_cast<float*>(&s_value[st])[lane] = step.y;
        const float above = kv8_above(step.y), other = fmaxf(above, __shfl_xor_sync(15u, above, 1));
        const float most = fmaxf(other, __shfl_xor_sync(15u, other, 2));
        if (lane == 0) s_gone[st] = s_missing[rs], s_above[st] = most;
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&kv_full[st]);
        mbar_arrive(&raw_empty[rs]);
      }
    }
  } else if (warp == 14) {
    // ---- bulk copies, a run of 16 tokens to each of four lanes ----
    const auto look_up = [&](int j) { return j < count ? page_of((block0 + j) * 4 + (lane & 3)) : -1; };
    constexpr int kRun = 32 * kDim;
    int page = look_up(0);
    for (int j = 0; j < count && !gave_up(); ++j) {
      const int rs = j % kPromptRaw, next = look_up(j + 1);
      float2 step = make_float2(0.f, 0.f);
      if (page >= 0) step = __ldg(steps + (long long)page * P.sh.heads + head);
      const unsigned here = __ballot_sync(kFullMask, page >= 0) & 15u;
      if (j >= kPromptRaw && !warp_wait_quick(&raw_empty[rs], (j / kPromptRaw - 1) & 1)) {
        s_bad = 1;
        break;
      }
      if (lane < 4) s_step[rs][lane] = make_float2(kv8_step(step.x), kv8_step(step.y));
      if (lane == 0) s_missing[rs] = 15 & ~here;
      __syncwarp();
      const uint32_t bar = smem_u32(&raw_full[rs]);
      if (lane == 0) mbar_expect(bar, __popc(here) * kRun);
      __syncwarp();
      if (lane < 4 && page >= 0)
        kv_copy(smem_u32(raw + rs * (kTile / 2) + lane * kRun),
                P.codes + ((long long)page * P.sh.heads + head) * P.sh.block_bytes() + (((block0 + j) * 4 + lane) & (page_runs - 1)) * kRun,
                kRun, bar);
      page = next;
    }
    // Every copy is waited for by those who convert it; should they have given up, here, with a limit.
    if (s_bad)
      for (int rs = 0; rs < kPromptRaw; ++rs) mbar_wait_limit(&raw_full[rs], 0, 1u << 16, kSiteMbarrier), mbar_wait_limit(&raw_full[rs], 1, 1u << 16, kSiteMbarrier);
  } else {
    // ---- a tile's MMAs ----
    constexpr uint32_t to_s = f16_idesc(128, kPromptTokens), to_o = f16_idesc(128, kDim);
    const int x = warp - 12;
    const uint32_t q = (uint32_t)i8_sdesc(smem_u32(sq)) + x * (kTile >> 4), k0 = (uint32_t)i8_sdesc(smem_u32(sk)), upper = (uint32_t)(i8_sdesc(0) >> 32);
    named_sync(1 + x, 160);
    const auto scores = [&](int j) {
      if (elect_one()) {
        const uint32_t k = k0 + j % kPromptStages * (kTile >> 4), d = tmem + 128 * x + 64 * (j & 1);
#pragma unroll
        for (int c = 0; c < kDim / 16; ++c)
          f16_mma(d, q + (c >> 2) * (128 * 128 >> 4) + 2 * (c & 3), k + (c >> 2) * (64 * 128 >> 4) + 2 * (c & 3), upper, to_s, c > 0);
        mma_commit(&s_full[x][j & 1]);
      }
      __syncwarp();
    };
    bool ok = true;
    for (int j = 0; ok && x < both && j < 2 && j < count; ++j) {
      ok = warp_wait_quick(&kv_full[j], 0);
      tc_fence_after();
      if (ok) scores(j);
    }
    for (int j = 0; ok && x < both && j < count; ++j) {
      const int st = j % kPromptStages;
      ok = warp_wait_quick(&p_full[x][j & 1], (j >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t v = k0 + st * (kTile >> 4) + (kTile / 2 >> 4), p = tmem + 128 * x + 64 * (j & 1), d = tmem + 256 + 128 * x;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          f16_mma_tmem(d, p + 32 * (c >> 1) + 8 * (c & 1), v + 2 * c, upper, to_o, (j & (aside_every - 1)) + c > 0);
          f16_mma_tmem(d, p + 32 * (c >> 1) + 8 * (c & 1) + 16, v + 2 * c, upper, to_o, true);
        }
        mma_commit(&kv_empty[st]);
        mma_commit(&o_full[x][j & 1]);  // the last word to arrive in this CTA is one that is waited for
      }
      __syncwarp();
      if (j + 2 < count) {
        ok = warp_wait_quick(&kv_full[(j + 2) % kPromptStages], ((j + 2) / kPromptStages) & 1);
        tc_fence_after();
        if (ok) scores(j + 2);
      }
    }
    if (!ok) s_bad = 1;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

}  // namespace qrb200
