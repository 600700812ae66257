// Matrices of 8-bit codes as the tensor-core products load them: by TMA into rows of 128 codes in the
// 128-byte swizzle, for one CTA or a pair, and operands whose rows TMA cannot load laid out anew.
#pragma once

#include <cuda.h>

#include "cluster.cuh"

namespace qrb200 {

constexpr int kI8Depth = 128;  // codes of one row per stage: one 128-byte swizzled row

// One box of a 2D tensor map into shared memory, completing on an mbarrier of this CTA.
__device__ __forceinline__ void i8_load(uint32_t dst, const CUtensorMap* map, uint32_t mbar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(mbar)
      : "memory");
}
__device__ __forceinline__ void i8_expect(uint32_t mbar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(mbar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// Descriptor of a K-major tile of 128-byte rows in the 128-byte swizzle (layout type 2): groups of
// 8 rows 1024 bytes apart; a step of 32 codes advances the start address by 32 bytes.
__device__ __forceinline__ uint64_t i8_sdesc(uint32_t saddr) { return make_sdesc(saddr, 16, 1024) | ((uint64_t)2 << 61); }

// ---- pairs of CTAs --------------------------------------------------------------------------

__device__ __forceinline__ uint32_t pair_leader(uint32_t addr) {  // the same address in the pair's first CTA
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(addr));
  return a;
}
__device__ __forceinline__ void i8_load_pair(uint32_t dst, const CUtensorMap* map, uint32_t leader_bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(leader_bar)
      : "memory");
}
__device__ __forceinline__ void commit_pair(uint64_t* mbar) {  // arrives on this barrier of both CTAs
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
      :
      : "r"(smem_u32(mbar)), "h"((uint16_t)3)
      : "memory");
}

// ---- rows off 16-byte boundaries -----------------------------------------------------------

struct I8Operand {
  const int8_t* base;
  long long rows, stride;  // bytes
  bool aligned;            // base and stride are multiples of 16
};

// Sixteen codes of a row from column k on, zeros past the row's end: one load from an aligned row;
// from any other address neighbouring aligned words, shifted, where those lie within the operand;
// else byte by byte.
template <bool kAligned>
__device__ __forceinline__ uint4 i8_codes16(const I8Operand& o, long long row, int k, int depth) {
  const int8_t* p = o.base + row * o.stride + k;
  const int n = depth - k;
  if (kAligned && n >= 16) return __ldg(reinterpret_cast<const uint4*>(p));
  uint32_t w[4] = {};
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  const uint32_t* word = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
  const int8_t* end = o.base + (o.rows - 1) * o.stride + depth;
  if (!kAligned && reinterpret_cast<const int8_t*>(word) >= o.base && reinterpret_cast<const int8_t*>(word + 5) <= end) {
    const int shift = 8 * (int)(at & 3);
    uint32_t v[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) v[i] = __ldg(word + i);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = __funnelshift_r(v[i], v[i + 1], shift);
      const int keep = n - 4 * i;  // bytes of this word inside the row
      if (keep < 4) w[i] = keep > 0 ? w[i] & (0xffffffffu >> (32 - 8 * keep)) : 0u;
    }
  } else {
    for (int i = 0; i < n && i < 16; ++i) w[i >> 2] |= (uint32_t)(uint8_t)__ldg(p + i) << (8 * (i & 3));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Lays an operand out for the tensor-core kernels, which load by TMA: rows of `packs` 16-byte packs.
static __global__ void __launch_bounds__(256) i8_pad_kernel(I8Operand a, uint4* to_a, I8Operand b, uint4* to_b, int depth, int packs) {
  griddep_launch_wait();
  long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long first = to_a ? a.rows * packs : 0;
  const bool second = at >= first;
  if (second) at -= first;
  const I8Operand o = second ? b : a;
  uint4* to = second ? to_b : to_a;
  if (!to || at >= o.rows * packs) return;
  to[at] = i8_codes16<false>(o, at / packs, (int)(at % packs) * 16, depth);
}

}  // namespace qrb200
