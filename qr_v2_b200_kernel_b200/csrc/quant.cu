// C ABI of the operators on data in 8 and 4 bits: argument checks, choice of kernel, launches.
#include "codes.h"
#include "i8_linear.cuh"
#include "kv4_attention.cuh"
#include "quant_rows.cuh"

namespace qrb200 {

// Packs of a row to a thread, by the row's length: four (enough loads in flight, few threads at the
// two reductions), fewer where that would leave a warp idle. Short rows go several to a block, a
// warp each, where there are rows enough.
template <typename T, typename W, bool kNorm, bool kAligned>
static cudaError_t launch_rows_of(const RowsParams& p, cudaStream_t s) {
  const int packs = ceil_div(p.cols, 16 / sizeof(T));
  const int items = packs <= 32 ? 1 : packs <= 64 ? 2 : packs <= 4096 ? 4 : 8;
  const int threads = ceil_div(ceil_div(packs, items), 32) * 32;
  const int y = threads == 32 && p.rows > 4 * sm_count() ? 8 : 1;
  LaunchShape l(dim3(ceil_div(p.rows, y)), threads, 0, s);
  l.cfg.blockDim.y = y;
  switch (items) {
    case 1: return cudaLaunchKernelEx(&l.cfg, rows_int8_kernel<T, W, kNorm, kAligned, 1>, p);
    case 2: return cudaLaunchKernelEx(&l.cfg, rows_int8_kernel<T, W, kNorm, kAligned, 2>, p);
    case 4: return cudaLaunchKernelEx(&l.cfg, rows_int8_kernel<T, W, kNorm, kAligned, 4>, p);
  }
  if constexpr (sizeof(T) == 4) return cudaLaunchKernelEx(&l.cfg, rows_int8_kernel<T, W, kNorm, kAligned, 8>, p);
  return cudaErrorInvalidValue;  // 16-bit rows of up to 32768 have 4096 packs
}

template <typename T, bool kNorm>
static int launch_rows(RowsParams p, int weight_type, int dtype, cudaStream_t s) {
  constexpr int kVec = 16 / sizeof(T);
  const auto off = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) != 0; };
  const bool aligned = p.cols % kVec == 0 && !off(p.x) && !off(p.residual) && !off(p.weight) && !off(p.h_out) && !off(p.q) &&
                       p.x_stride % kVec == 0 && p.r_stride % kVec == 0 && p.q_stride % 16 == 0;
  p.q_aligned = !off(p.q) && p.q_stride % 16 == 0;
  cudaError_t e;
  if (p.weight && weight_type == QRB200_F32 && dtype != QRB200_F32)
    e = aligned ? launch_rows_of<T, float, kNorm, true>(p, s) : launch_rows_of<T, float, kNorm, false>(p, s);
  else
    e = aligned ? launch_rows_of<T, T, kNorm, true>(p, s) : launch_rows_of<T, T, kNorm, false>(p, s);
  if (e != cudaSuccess) return QRB200_ERR_CUDA;
  return launched();
}

template <typename T>
static int launch_dequant(const int8_t* q, int64_t q_stride, const float* scale, void* out, int64_t rows, int64_t cols,
                          cudaStream_t s) {
  // Sixteen codes to a thread where rows start on 16-byte boundaries on both sides, else eight, a
  // warp's side by side.
  const bool packed = (cols * sizeof(T)) % 16 == 0 && q_stride % 16 == 0 &&
                      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  const int64_t units = packed ? rows * ceil_div(cols, 16) : rows * ceil_div(cols, 256) * 32;
  if (units > ((int64_t)1 << 38)) return QRB200_ERR_ARG;
  LaunchShape l(dim3(ceil_div(units, 256)), 256, 0, s);
  const auto kernel = !packed     ? dequant_rows_kernel<T, false, true>
                      : cols % 16 ? dequant_rows_kernel<T, true, true>
                                  : dequant_rows_kernel<T, true, false>;
  const cudaError_t e = cudaLaunchKernelEx(
      &l.cfg, kernel, q, (long long)q_stride, scale, static_cast<T*>(out), (long long)rows, (int)cols);
  if (e != cudaSuccess) return QRB200_ERR_CUDA;
  return launched();
}

template <bool kNorm>
static int rows_int8(const RowsParams& p, int weight_type, int dtype, cudaStream_t s) {
  switch (dtype) {
    case QRB200_BF16: return launch_rows<__nv_bfloat16, kNorm>(p, weight_type, dtype, s);
    case QRB200_F16: return launch_rows<__half, kNorm>(p, weight_type, dtype, s);
    default: return launch_rows<float, kNorm>(p, weight_type, dtype, s);
  }
}


template <typename T, int kBN>
static cudaError_t launch_i8_few(const I8Params& p, const I8Operand& x, const I8Operand& w, unsigned split, cudaStream_t s) {
  using C = I8Few<kBN>;
  static OncePerDevice once;
  const cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(i8_few_kernel<T, kBN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::smem());
  });
  if (e != cudaSuccess) return e;
  CUtensorMap tw, tx;
  if (!encode_codes(&tw, w, p.depth, 128) || !encode_codes(&tx, x, p.depth, kBN)) return cudaErrorInvalidValue;
  const int tn = ceil_div(p.outs, 128), tm = ceil_div(p.rows, kBN);
  if (tm > 65535) return cudaErrorInvalidValue;
  LaunchShape l(dim3(tn, tm, split), 192, C::smem(), s);
  if (split > 1) l.cluster(1, 1, split);
  return cudaLaunchKernelEx(&l.cfg, i8_few_kernel<T, kBN>, p, tw, tx);
}

template <typename T>
static cudaError_t launch_i8_wide(I8Params p, const I8Operand& x, const I8Operand& w, cudaStream_t s) {
  static OncePerDevice once;
  const cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(i8_wide_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)i8_wide_smem());
  });
  if (e != cudaSuccess) return e;
  CUtensorMap tw, tx;
  if (!encode_codes(&tw, w, p.depth, 128) || !encode_codes(&tx, x, p.depth, 128)) return cudaErrorInvalidValue;
  p.tiles_n = ceil_div(p.outs, 256);
  const int64_t tiles = (int64_t)p.tiles_n * ceil_div(p.rows, 256);
  if (tiles > (1 << 30)) return cudaErrorInvalidValue;
  p.tiles = (int)tiles;
  const int pairs = std::min(p.tiles, sm_count() / 2);
  LaunchShape l(dim3(2 * pairs), 128 + 32 * kI8WideEpi, i8_wide_smem(), s);
  return cudaLaunchKernelEx(&l.cfg, i8_wide_kernel<T>, p, tx, tw);
}

// Which kernel, with how many rows a tile (`rows`) and over how many CTAs of the depth: the least
// of the estimated clocks. A CTA takes in its stages at about 40 bytes a clock; joining a split
// costs two cluster barriers (about 1500 clocks) and reading the sums at about 20 bytes a clock.
// Clusters of eight lose: a GPC holds two at best (64 x 1000 x 2048: 12 us against 9). The wide
// kernel's pair takes 512 clocks a stage and a tile's last epilogue is bare.
struct I8Plan {
  int rows;  // 16, 32, 64 or 128 (few), 256 (wide)
  unsigned split;
};
static I8Plan i8_plan(int64_t rows, int64_t outs, int64_t depth) {
  const int64_t sms = sm_count(), nk = (depth + kI8Depth - 1) / kI8Depth;
  const int64_t pairs = (rows + 255) / 256 * ((outs + 255) / 256);
  I8Plan best{256, 1};
  int64_t least = (pairs + sms / 2 - 1) / (sms / 2) * nk * 512 + 3000;
  for (int bn = 16; bn <= 128; bn *= 2) {
    const int64_t tiles = (rows + bn - 1) / bn * ((outs + 127) / 128);
    if ((rows + bn - 1) / bn > 65535) continue;
    for (unsigned split = 1; split <= kI8Split && split <= nk; split *= 2) {
      const int64_t clocks = (tiles * split + sms - 1) / sms *
                             ((nk + split - 1) / split * (128 + bn) * 128 / 40 + (split > 1 ? 1500 + bn * 24 : bn * 8));
      if (clocks < least) {
        least = clocks;
        best = I8Plan{bn, split};
      }
    }
    if (rows <= bn) break;
  }
  return best;
}

template <typename T>
static cudaError_t launch_i8_rows(const I8Params& p, const I8Operand& x, const I8Operand& w, cudaStream_t s) {
  const I8RowsParams r{p, x, w};
  LaunchShape l(dim3(ceil_div(p.outs, 8)), 128, 0, s);
  const bool aligned = x.aligned && w.aligned;
  if (p.rows == 1) return cudaLaunchKernelEx(&l.cfg, aligned ? i8_rows_kernel<T, 1, true> : i8_rows_kernel<T, 1, false>, r);
  if (p.rows == 2) return cudaLaunchKernelEx(&l.cfg, aligned ? i8_rows_kernel<T, 2, true> : i8_rows_kernel<T, 2, false>, r);
  return cudaLaunchKernelEx(&l.cfg, i8_rows_kernel<T, 4, true>, r);  // never unaligned
}

// Up to four rows by dot products (4096 x 4096: 3.2 us for one or two, 4.5 for four, against 5.7 in
// tiles); three or four off 16-byte boundaries are better laid out first (3 x 1641 x 1329: 6.6
// against 8.4). A warp walks its channels' whole depth, so a long one is left to the split of the
// tensor-core kernel.
static bool i8_by_rows(int64_t rows, int64_t depth, bool aligned) { return rows <= (aligned ? 4 : 2) && depth <= 8192; }

template <typename T>
static cudaError_t launch_i8(const I8Params& p, I8Operand x, I8Operand w, uint4* ws, cudaStream_t s) {
  if (i8_by_rows(p.rows, p.depth, x.aligned && w.aligned)) return launch_i8_rows<T>(p, x, w, s);
  const cudaError_t e = lay_out(x, w, p.depth, ws, s);
  if (e != cudaSuccess) return e;
  const I8Plan plan = i8_plan(p.rows, p.outs, p.depth);
  switch (plan.rows) {
    case 16: return launch_i8_few<T, 16>(p, x, w, plan.split, s);
    case 32: return launch_i8_few<T, 32>(p, x, w, plan.split, s);
    case 64: return launch_i8_few<T, 64>(p, x, w, plan.split, s);
    case 128: return launch_i8_few<T, 128>(p, x, w, plan.split, s);
    default: return launch_i8_wide<T>(p, x, w, s);
  }
}

static bool shape_ok(const Kv4Shape& h) {
  return h.pages >= 0 && h.pages <= (1ll << 31) - 1 && h.heads > 0 && h.heads <= 65535 && (h.dim == 64 || h.dim == 128) &&
         h.page >= 16 && h.page <= 1024 && (h.page & (h.page - 1)) == 0 && h.groups > 0 && h.dim % h.groups == 0 &&
         (h.dim / h.groups == 32 || h.dim / h.groups == 64 || h.dim / h.groups == 128);
}

// f(dim, groups) with both as types, for the layouts that shape_ok admits.
template <typename F>
static cudaError_t with_layout(const Kv4Shape& h, F&& f) {
  if (h.dim == 64) return h.groups == 1 ? f(Int<64>{}, Int<1>{}) : f(Int<64>{}, Int<2>{});
  if (h.groups == 1) return f(Int<128>{}, Int<1>{});
  return h.groups == 2 ? f(Int<128>{}, Int<2>{}) : f(Int<128>{}, Int<4>{});
}

// Heads to a CTA of the write and the read: as many as leave sixteen CTAs to an SM, so that a CTA's
// set-up is shared by more work without idling the GPU.
static int head_span(int64_t tokens, int heads) {
  const int64_t ctas = (tokens + 15) / 16 * heads;
  return (int)std::max<int64_t>(1, std::min<int64_t>(heads, ctas / (16 * sm_count())));
}

template <typename T>
static cudaError_t launch_write(Kv4IoParams p, bool vec, cudaStream_t s) {
  p.span = head_span(p.tokens, p.sh.heads);
  LaunchShape l(dim3(ceil_div(p.tokens, 16), ceil_div(p.sh.heads, p.span)), 2 * p.sh.dim, 0, s);
  return with_layout(p.sh, [&](auto dim, auto groups) {
    return cudaLaunchKernelEx(&l.cfg, vec ? kv4_write_kernel<T, dim(), groups(), true> : kv4_write_kernel<T, dim(), groups(), false>, p);
  });
}

template <typename T>
static cudaError_t launch_read(Kv4IoParams p, cudaStream_t s) {
  p.span = head_span(p.tokens, p.sh.heads);
  LaunchShape l(dim3(ceil_div(p.tokens, 16), ceil_div(p.sh.heads, p.span)), 2 * p.sh.dim, 0, s);
  return with_layout(p.sh, [&](auto dim, auto groups) { return cudaLaunchKernelEx(&l.cfg, kv4_read_kernel<T, dim(), groups()>, p); });
}

// How an attention call is cut: query rows per tile, and the token range over `splits` CTAs.
struct AttnPlan {
  int tile_rows, tiles, splits;
  bool brief;  // steps of half the size (kv_runs)
  size_t bytes;  // workspace: the parts and their (maximum, sum) pairs
};

// Eight rows a tile where a key head has no more than eight query rows, else sixteen. The token
// range is cut over the CTAs that make the least estimated time, in fifths of a step's share of a
// busy SM (0.63 us): a CTA alone takes 2.4 such shares for a step (1.8 with sixteen rows), so up to
// that many share an SM for nothing, and its set-up takes two steps; joining costs 1.5 in a cluster
// and 6 through memory. The length is the table's capacity or what a window leaves of it, all that
// the host knows.
static AttnPlan attn_plan(const Kv4Shape& h, int64_t batch, int64_t queries, int64_t q_heads, int64_t max_pages, int64_t span) {
  AttnPlan p{};
  const int64_t rows = queries * (q_heads / h.heads);
  p.tile_rows = rows <= 8 ? 8 : 16;
  p.tiles = ceil_div(rows, p.tile_rows);
  const int64_t ctas = batch * h.heads * p.tiles, tokens = std::min(max_pages * h.page, span), sms = sm_count();
  const auto plan = [&](bool brief) {  // steps of a warp
    const int64_t unit = 16 * kv_runs(h.dim, brief) * kKvWarps, steps = std::max<int64_t>(1, (tokens + unit - 1) / unit);
    int64_t best = -1, left = 0;
    for (int64_t n = 1; n <= std::min<int64_t>(steps, 128); ++n) {
      const int64_t share = std::max<int64_t>(p.tile_rows == 8 ? 12 : 9, 5 * ((ctas * n + sms - 1) / sms));
      const int64_t time = share * ((steps + n - 1) / n + 2) + (n > kKvCluster ? 30 : n > 1 ? 8 : 0);
      if (best < 0 || time < best) {
        best = time;
        left = (steps + n - 1) / n;
        p.splits = (int)n;
      }
    }
    return left;
  };
  p.brief = plan(false) <= 2 && h.dim == 64;
  if (p.brief) plan(true);
  if (p.splits > kKvCluster) p.bytes = (size_t)(ctas * p.splits * p.tile_rows) * (h.dim * sizeof(float) + sizeof(float2));
  return p;
}

template <typename T, int kDim, int kGroups, int kNT, bool kBrief>
static cudaError_t launch_attention_tile(const Kv4AttnParams& p, const AttnPlan& plan, cudaStream_t s) {
  constexpr int kSmem = kv_smem_bytes(kDim, kGroups, kNT, kBrief);
  static OncePerDevice once;
  const cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(kv4_attention_kernel<T, kDim, kGroups, kNT, kBrief>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  });
  if (e != cudaSuccess) return e;
  LaunchShape l(dim3(plan.splits * plan.tiles, p.sh.heads, p.batch), 32 * kKvWarps, kSmem, s);
  if (plan.splits > 1 && plan.splits <= kKvCluster) l.cluster(plan.splits, 1, 1);
  return cudaLaunchKernelEx(&l.cfg, kv4_attention_kernel<T, kDim, kGroups, kNT, kBrief>, p);
}

template <typename T, int kDim, int kGroups>
static cudaError_t launch_attention(Kv4AttnParams p, const AttnPlan& plan, cudaStream_t s) {
  const auto tile = [&](auto nt) {
    if constexpr (kDim == 64)
      if (plan.brief) return launch_attention_tile<T, kDim, kGroups, nt(), true>(p, plan, s);
    return launch_attention_tile<T, kDim, kGroups, nt(), false>(p, plan, s);
  };
  const cudaError_t e = plan.tile_rows == 8 ? tile(Int<1>{}) : tile(Int<2>{});
  if (e != cudaSuccess || plan.splits <= kKvCluster) return e;
  qrb200_internal_count_launch();
  LaunchShape j(dim3(p.batch * p.queries * p.q_heads), 32 * kKvJoinWarps, 0, s);
  return cudaLaunchKernelEx(&j.cfg, kv_join_kernel<T, kDim, Kv4AttnParams>, p, plan.tile_rows);
}

template <typename T>
static cudaError_t launch_attention_of(const Kv4AttnParams& p, const AttnPlan& plan, cudaStream_t s) {
  return with_layout(p.sh, [&](auto dim, auto groups) { return launch_attention<T, dim(), groups()>(p, plan, s); });
}

}  // namespace qrb200

using namespace qrb200;

int qrb200_internal_quant_site() { return take_site(); }
bool qrb200_internal_quant_register(int* word) { return register_word(word); }

extern "C" {

int qrb200_rms_norm_int8(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                         const void* weight, int weight_type, int8_t* q, int64_t q_stride, float* scale, void* h_out,
                         int64_t rows, int64_t cols, float eps, int dtype, void* stream) {
  if (rows < 0 || cols < 0 || rows > kMaxRows || cols > kMaxCols || !type_ok(dtype)) return QRB200_ERR_ARG;
  if (rows == 0 || cols == 0) return QRB200_OK;
  if (!x || !q || !scale || (residual != nullptr) != (h_out != nullptr) || !(eps >= 0.f)) return QRB200_ERR_ARG;
  if (weight && weight_type != dtype && weight_type != QRB200_F32) return QRB200_ERR_ARG;
  if (rows > 1 && (x_stride < cols || q_stride < cols || (residual && residual_stride < cols))) return QRB200_ERR_ARG;
  const int st = quant_ready();
  if (st != QRB200_OK) return st;
  RowsParams p{x, residual, weight, h_out, q, scale, rows, x_stride, residual_stride, q_stride, (int)cols, eps, 0};
  return rows_int8<true>(p, weight_type, dtype, static_cast<cudaStream_t>(stream));
}

int qrb200_quantize_int8(const void* x, int64_t x_stride, int8_t* q, int64_t q_stride, float* scale, int64_t rows,
                         int64_t cols, int dtype, void* stream) {
  if (rows < 0 || cols < 0 || rows > kMaxRows || cols > kMaxCols || !type_ok(dtype)) return QRB200_ERR_ARG;
  if (rows == 0 || cols == 0) return QRB200_OK;
  if (!x || !q || !scale || (rows > 1 && (x_stride < cols || q_stride < cols))) return QRB200_ERR_ARG;
  const int st = quant_ready();
  if (st != QRB200_OK) return st;
  RowsParams p{x, nullptr, nullptr, nullptr, q, scale, rows, x_stride, 0, q_stride, (int)cols, 0.f, 0};
  return rows_int8<false>(p, dtype, dtype, static_cast<cudaStream_t>(stream));
}

int qrb200_dequantize_int8(const int8_t* q, int64_t q_stride, const float* scale, void* out, int64_t rows,
                           int64_t cols, int dtype, void* stream) {
  if (rows < 0 || cols < 0 || rows > kMaxRows || cols > kMaxCols || !type_ok(dtype)) return QRB200_ERR_ARG;
  if (rows == 0 || cols == 0) return QRB200_OK;
  if (!q || !scale || !out || (rows > 1 && q_stride < cols)) return QRB200_ERR_ARG;
  const int st = quant_ready();
  if (st != QRB200_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == QRB200_BF16) return launch_dequant<__nv_bfloat16>(q, q_stride, scale, out, rows, cols, s);
  if (dtype == QRB200_F16) return launch_dequant<__half>(q, q_stride, scale, out, rows, cols, s);
  return launch_dequant<float>(q, q_stride, scale, out, rows, cols, s);
}

size_t qrb200_int8_linear_workspace_bytes(const int8_t* x, int64_t x_stride, const int8_t* w, int64_t w_stride,
                                          int64_t rows, int64_t outs, int64_t depth) {
  if (rows <= 0 || outs <= 0 || depth <= 0 || depth > QRB200_INT8_MAX_DEPTH) return 0;
  const I8Operand xo = i8_operand(x, rows, x_stride), wo = i8_operand(w, outs, w_stride);
  return i8_by_rows(rows, depth, xo.aligned && wo.aligned) ? 0 : layout_bytes(xo, wo, depth);
}

int qrb200_int8_linear(const int8_t* x, int64_t x_stride, const float* x_scale, const int8_t* w, int64_t w_stride,
                       const float* w_scale, const void* bias, void* y, int64_t rows, int64_t outs, int64_t depth,
                       int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (rows < 0 || outs < 0 || depth <= 0 || depth > QRB200_INT8_MAX_DEPTH || !type_ok(dtype)) return QRB200_ERR_ARG;
  if (rows > kMaxRows / 2 || outs > kMaxRows / 2) return QRB200_ERR_ARG;
  if (rows == 0 || outs == 0) return QRB200_OK;
  if (!x || !w || !x_scale || !w_scale || !y || (reinterpret_cast<uintptr_t>(y) & 15u)) return QRB200_ERR_ARG;
  if ((rows > 1 && x_stride < depth) || (outs > 1 && w_stride < depth)) return QRB200_ERR_ARG;
  const int st = quant_ready();
  if (st != QRB200_OK) return st;
  const size_t need = qrb200_int8_linear_workspace_bytes(x, x_stride, w, w_stride, rows, outs, depth);
  if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u)))
    return QRB200_ERR_WORKSPACE;
  const I8Params p{x_scale, w_scale, bias, y, (int)rows, (int)outs, (int)depth, 0, 0};
  const I8Operand xo = i8_operand(x, rows, x_stride), wo = i8_operand(w, outs, w_stride);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint4* ws = static_cast<uint4*>(workspace);
  cudaError_t e;
  if (dtype == QRB200_BF16) e = launch_i8<__nv_bfloat16>(p, xo, wo, ws, s);
  else if (dtype == QRB200_F16) e = launch_i8<__half>(p, xo, wo, ws, s);
  else e = launch_i8<float>(p, xo, wo, ws, s);
  if (e != cudaSuccess) return QRB200_ERR_CUDA;
  return launched();
}

int64_t qrb200_kv4_block_bytes(int64_t page_size, int64_t head_dim, int64_t group_size) {
  if (group_size <= 0 || page_size < 0 || page_size > 1024 || head_dim < 0 || head_dim > 128) return 0;
  const Kv4Shape h{1, (int)page_size, (int)head_dim, (int)(head_dim / std::min<int64_t>(group_size, 1024)), 0, 0};
  return shape_ok(h) && head_dim % group_size == 0 ? h.block_bytes() : 0;
}

int qrb200_kv4_write(void* cache, const qrb200_kv4_shape* shape, const void* k, int64_t k_token_stride,
                     int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
                     const int64_t* slots, int64_t tokens, void* stream) {
  if (!shape || tokens < 0 || !type16_ok(shape->dtype)) return QRB200_ERR_ARG;
  const Kv4Shape h{shape->kv_heads, shape->page_size, shape->head_dim, shape->groups, page_shift(shape->page_size), shape->pages};
  if (!shape_ok(h) || tokens > kMaxRows / h.heads) return QRB200_ERR_ARG;
  if (tokens == 0) return QRB200_OK;
  if (!cache || !k || !v || !slots || (reinterpret_cast<uintptr_t>(cache) & 15u)) return QRB200_ERR_ARG;
  const int st = quant_ready();
  if (st != QRB200_OK) return st;
  Kv4IoParams p{static_cast<unsigned char*>(cache), k, v, nullptr, nullptr, reinterpret_cast<const long long*>(slots),
                tokens, k_token_stride, k_head_stride, v_token_stride, v_head_stride, h};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = shape->dtype == QRB200_BF16;
  // 16-byte loads where every (token, head) starts on such a boundary.
  const bool vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0 &&
                   ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) == 0;
  const cudaError_t e = bf ? launch_write<__nv_bfloat16>(p, vec, s) : launch_write<__half>(p, vec, s);
  if (e != cudaSuccess) return QRB200_ERR_CUDA;
  return launched();
}

int qrb200_kv4_read(const void* cache, const qrb200_kv4_shape* shape, void* k, void* v, const int64_t* slots,
                    int64_t tokens, void* stream) {
  if (!shape || tokens < 0 || !type16_ok(shape->dtype)) return QRB200_ERR_ARG;
  const Kv4Shape h{shape->kv_heads, shape->page_size, shape->head_dim, shape->groups, page_shift(shape->page_size), shape->pages};
  if (!shape_ok(h) || tokens > kMaxRows / h.heads) return QRB200_ERR_ARG;
  if (tokens == 0) return QRB200_OK;
  if (!cache || !k || !v || !slots || (reinterpret_cast<uintptr_t>(cache) & 15u)) return QRB200_ERR_ARG;
  const int st = quant_ready();
  if (st != QRB200_OK) return st;
  Kv4IoParams p{static_cast<unsigned char*>(const_cast<void*>(cache)), nullptr, nullptr, k, v,
                reinterpret_cast<const long long*>(slots), tokens, 0, 0, 0, 0, h};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) return QRB200_ERR_ARG;
  const cudaError_t e = shape->dtype == QRB200_BF16 ? launch_read<__nv_bfloat16>(p, s) : launch_read<__half>(p, s);
  if (e != cudaSuccess) return QRB200_ERR_CUDA;
  return launched();
}

// The most tokens that a sequence's queries see between them.
static int64_t token_span(int64_t queries, int64_t window) { return window > 0 ? std::min(window, kMaxRows) + queries : kMaxRows; }

// The launch grid is (splits x row tiles) x key heads x batch, a large batch in several launches.
constexpr int64_t kGridZ = 65535;
static bool attention_args(const qrb200_kv4_shape* shape, int64_t batch, int64_t queries, int64_t q_heads,
                           int64_t max_pages, Kv4Shape* h) {
  if (!shape || batch < 0 || queries < 0 || q_heads < 0 || max_pages < 0 || !type16_ok(shape->dtype)) return false;
  *h = Kv4Shape{shape->kv_heads, shape->page_size, shape->head_dim, shape->groups, page_shift(shape->page_size), shape->pages};
  return shape_ok(*h) && q_heads % h->heads == 0 && batch <= kMaxRows && q_heads <= 65535 && queries <= (1 << 24) &&
         queries * (q_heads / h->heads) <= (1 << 24) && (queries * q_heads == 0 || batch <= kMaxRows / (queries * q_heads)) &&
         max_pages <= kMaxRows / h->page - 64 * (kKvWarps + 1);
}

size_t qrb200_kv4_attention_workspace_bytes(const qrb200_kv4_shape* shape, int64_t batch, int64_t queries,
                                            int64_t q_heads, int64_t max_pages, int64_t window) {
  Kv4Shape h;
  if (window < 0) return 0;
  if (!attention_args(shape, batch, queries, q_heads, max_pages, &h) || batch * queries * q_heads == 0) return 0;
  return attn_plan(h, batch, queries, q_heads, max_pages, token_span(queries, window)).bytes;
}

int qrb200_kv4_attention(const void* q, const int64_t* q_strides, const void* cache, const qrb200_kv4_shape* shape,
                         const int32_t* block_table, int64_t table_stride, const int32_t* lengths, void* out,
                         int64_t batch, int64_t queries, int64_t q_heads, int64_t max_pages, int64_t window,
                         int causal, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  Kv4Shape h;
  if (!q_strides || !(scale >= 0.f) || !(scale <= 3.0e38f) || window < 0 || !attention_args(shape, batch, queries, q_heads, max_pages, &h))
    return QRB200_ERR_ARG;
  if (batch == 0 || queries == 0 || q_heads == 0) return QRB200_OK;
  if (!q || !out || !lengths || (max_pages > 0 && !block_table) || (reinterpret_cast<uintptr_t>(cache) & 15u) ||
      (h.pages > 0 && !cache) || table_stride < 0)
    return QRB200_ERR_ARG;
  const int st = quant_ready();
  if (st != QRB200_OK) return st;
  const AttnPlan plan = attn_plan(h, batch, queries, q_heads, max_pages, token_span(queries, window));
  if (plan.bytes > 0 && (!workspace || workspace_bytes < plan.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255u)))
    return QRB200_ERR_WORKSPACE;
  Kv4AttnParams p{};
  p.cache = static_cast<const unsigned char*>(cache);
  p.q = q;
  p.out = out;
  p.part_o = static_cast<float*>(workspace);
  p.table = block_table;
  p.lengths = lengths;
  p.q_bs = q_strides[0], p.q_ts = q_strides[1], p.q_hs = q_strides[2], p.table_stride = table_stride;
  p.batch = (int)batch, p.queries = (int)queries, p.q_heads = (int)q_heads, p.share = (int)(q_heads / h.heads);
  // A window that reaches every token from every position is none (and cannot overflow a position).
  p.window = window >= max_pages * h.page + queries ? 0 : (int)window;
  p.max_pages = (int)max_pages, p.causal = causal, p.splits = plan.splits, p.tiles = plan.tiles;
  p.scale2 = scale * 1.4426950408889634f;
  p.sh = h;
  p.q_wide = (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && ((q_strides[0] | q_strides[1] | q_strides[2]) & 3) == 0;
  if (plan.splits > kKvCluster)
    p.part_ml = reinterpret_cast<float2*>(p.part_o + batch * h.heads * plan.tiles * plan.splits * plan.tile_rows * h.dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  for (int64_t b = 0; b < batch; b += kGridZ) {
    Kv4AttnParams part = p;
    const int64_t rows = b * queries * q_heads, parts = b * h.heads * plan.tiles * plan.splits * plan.tile_rows;
    part.batch = (int)std::min(kGridZ, batch - b);
    part.q = static_cast<const char*>(q) + 2 * b * p.q_bs;
    part.out = static_cast<char*>(out) + 2 * rows * h.dim;
    part.table += b * table_stride;
    part.lengths += b;
    if (p.part_ml) part.part_o += parts * h.dim, part.part_ml += parts;
    const cudaError_t e = shape->dtype == QRB200_BF16 ? launch_attention_of<__nv_bfloat16>(part, plan, s)
                                                      : launch_attention_of<__half>(part, plan, s);
    if (e != cudaSuccess) return QRB200_ERR_CUDA;
    const int ended = launched();
    if (ended != QRB200_OK) return ended;
  }
  return QRB200_OK;
}

}  // extern "C"
