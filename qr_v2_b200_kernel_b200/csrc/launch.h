// What the operators' launchers share: the one-time check of a device, launch attributes, small sums.
// Included by one source file each that has device code, whose own failure words it registers.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <mutex>
#include <type_traits>

#include "internal.h"
#include "qrb200.h"
#include "tc.cuh"

namespace qrb200 {

// The device checked, and what an earlier kernel on it has reported. (Every source file's failure words are registered by the first
// call of any operator on a device: a symbol's copy could not be captured.)
static int quant_ready() {
  const int st = qrb200_internal_check_device();
  return st != QRB200_OK ? st : qrb200_last_status(nullptr);
}
static inline bool register_word(int* word) { return cudaMemcpyToSymbol(g_status_mapped, &word, sizeof(word)) == cudaSuccess; }

// Reads and clears this translation unit's device failure word; a site, 0, or -1 for a CUDA error.
static inline int take_site() {
  int v = 0;
  const int zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_device_status, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0 && cudaMemcpyToSymbol(g_device_status, &zero, sizeof(int)) != cudaSuccess) return -1;
  return v;
}

static int launched() {
  qrb200_internal_count_launch();
  return cudaGetLastError() == cudaSuccess ? QRB200_OK : QRB200_ERR_CUDA;
}

static inline bool type_ok(int t) { return t == QRB200_F32 || t == QRB200_BF16 || t == QRB200_F16; }
static inline bool type16_ok(int t) { return t == QRB200_BF16 || t == QRB200_F16; }

constexpr int kMaxCols = 32768;
constexpr int64_t kMaxRows = (1ll << 31) - 1;

static inline PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

struct LaunchShape {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  // A kernel that begins with griddep_launch_wait() may be set up while its predecessor ends.
  LaunchShape(dim3 grid, unsigned threads, size_t smem, cudaStream_t s) {
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    cfg.attrs = attr;
  }
  void cluster(unsigned x, unsigned y, unsigned z) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = x;
    attr[1].val.clusterDim.y = y;
    attr[1].val.clusterDim.z = z;
    cfg.numAttrs = 2;
  }
};

// Whether a one-time set-up of a kernel has been done on the current device; the caller marks it.
struct OncePerDevice {
  std::atomic<unsigned long long> bits{0};
  template <typename F>
  cudaError_t run(F&& set_up) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 64 && ((bits.load(std::memory_order_acquire) >> dev) & 1ull)) return cudaSuccess;
    const cudaError_t e = set_up();
    if (e == cudaSuccess && dev < 64) bits.fetch_or(1ull << dev, std::memory_order_acq_rel);
    return e;
  }
};

static int sm_count() {
  static std::atomic<int> sms[64];
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  if (dev < 64 && (n = sms[dev].load(std::memory_order_relaxed)) > 0) return n;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  if (dev < 64) sms[dev].store(n, std::memory_order_relaxed);
  return n;
}

static inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

static inline int page_shift(int page) {
  int s = 0;
  while (s < 10 && (1 << s) < page) ++s;
  return s;
}

template <int kValue>
using Int = std::integral_constant<int, kValue>;

}  // namespace qrb200
