// C ABI of the 8-bit key/value cache: argument checks, choice of kernel, launches.
#include <cmath>

#include "launch.h"
#include "kv8.cuh"
#include "kv8_attention.cuh"
#include "kv8_prompt.cuh"

namespace qrb200 {

static bool shape_of(const qrb200_kv8_shape* s, Kv8Shape* h) {
  if (!s || !type16_ok(s->dtype)) return false;
  *h = Kv8Shape{s->kv_heads, s->page_size, s->head_dim, page_shift(s->page_size), s->pages};
  return h->pages >= 0 && h->pages <= kMaxRows && h->heads > 0 && h->heads <= 65535 && (h->dim == 64 || h->dim == 128) &&
         h->page >= 16 && h->page <= 1024 && (h->page & (h->page - 1)) == 0;
}

// Codes by sixteen bytes, ranges by pairs.
static bool cache_ok(const Kv8Shape& h, const void* codes, const void* range) {
  return (h.pages == 0 || (codes && range)) && ((reinterpret_cast<uintptr_t>(codes) & 15u) | (reinterpret_cast<uintptr_t>(range) & 7u)) == 0;
}

// f(type, dim) with both as types.
template <typename F>
static cudaError_t with_shape(int dtype, int dim, F&& f) {
  if (dtype == QRB200_BF16) return dim == 64 ? f(__nv_bfloat16{}, Int<64>{}) : f(__nv_bfloat16{}, Int<128>{});
  return dim == 64 ? f(__half{}, Int<64>{}) : f(__half{}, Int<128>{});
}

// The pages' number and their list, before the slots' rows.
static size_t write_list_bytes(int64_t tokens) { return 256 + (size_t)(tokens + 63) / 64 * 256; }

// How an attention call is cut: query rows per tile, steps of 4 or 8 KB, and the token range over `splits` CTAs.
struct Kv8Plan {
  int tile_rows, tiles, splits;
  bool prompt;  // tiles of 256 rows on the tensor cores, not split; else
  bool brief;   // short steps
  bool memory;  // parts go through memory
  size_t bytes;  // workspace: the parts and their (maximum, sum) pairs, or a prompt's sums set aside
};

// Eight rows a tile where a key head has no more than eight query rows, else sixteen. Of both kinds of step and every number of
// splits the least estimated time, in ns: waves of CTAs, a wave's steps at what one takes with so many CTAs on an SM
// (measured with 128 channels), three steps for a CTA's set-up, 2 us for a join in a cluster and 4 through memory. Clusters of
// other than two or four CTAs place badly where they fill the GPU (24 x 8192 tokens, 8 heads in threes: 99 us, through memory 70; in
// pairs 64 x 8192 172, through memory 180), so those are left to thin waves. The length is the table's capacity or what a window leaves of it, all that the host knows.
static Kv8Plan attn_plan(const Kv8Shape& h, bool half, int64_t batch, int64_t queries, int64_t q_heads, int64_t max_pages, int64_t span) {
  static const int kShort[5] = {0, 750, 1000, 1300, 1400}, kLong[3] = {0, 1000, 1400}, kLong16[3] = {0, 1500, 2300};
  Kv8Plan p{};
  const int64_t rows = queries * (q_heads / h.heads);
  p.tile_rows = rows <= 8 ? 8 : 16;
  p.tiles = ceil_div(rows, p.tile_rows);
  const int64_t ctas = batch * h.heads * p.tiles, tokens = std::min(max_pages * h.page, span), sms = sm_count();
  int64_t best = -1;
  for (int brief = 0; brief <= (p.tile_rows == 8 ? 1 : 0); ++brief) {
    const int64_t unit = 16 * kv8_runs(h.dim, brief) * kKvWarps, steps = std::max<int64_t>(1, (tokens + unit - 1) / unit);
    const int* ns = brief ? kShort : p.tile_rows == 8 ? kLong : kLong16;
    const int per_sm = kv8_ctas(brief);
    for (int64_t n = 1; n <= std::min<int64_t>(steps, 128); ++n) {
      const int64_t all = ctas * n, waves = all / (per_sm * sms), rest = all - waves * per_sm * sms;
      const bool memory = n > kKvCluster || (n != 1 && n != 2 && n != 4 && all > 2 * sms);
      const int64_t time = ((steps + n - 1) / n + 3) * (waves * ns[per_sm] + ns[(rest + sms - 1) / sms]) + (memory ? 4000 : n > 1 ? 2000 : 0);
      if (best < 0 || time < best) {
        best = time;
        p.splits = (int)n, p.brief = brief, p.memory = memory;
      }
    }
  }
  // The prompt kernel does not split the tokens: 1.4 us for each 64 of them and 8 for the rest of a CTA, one an SM. (16 heads on 4 of 128
  // channels, over 4096 tokens: 1 x 512 queries 104 us for 122, 1 x 128 104 for 38; 32 on 8, 8 x 16 queries over 4096: 78 for
  // 65, 16 x 24 over 2048: 46 for 103.)
  const int64_t tiles = (rows + kPromptRows - 1) / kPromptRows, wide = (tiles * batch * h.heads + sms - 1) / sms * (tokens / kPromptTokens * 1400 + 8000);
  if (p.tile_rows == 16 && wide < best) {
    p.prompt = true;
    p.tile_rows = kPromptRows, p.tiles = (int)tiles, p.splits = 1, p.memory = false;
    if (tokens / kPromptTokens + 2 > prompt_aside(half))  // (the most steps, begun anywhere)
      p.bytes = (size_t)(tiles * batch * h.heads * kPromptRows) * (h.dim * sizeof(float));
    return p;
  }
  if (p.memory) p.bytes = (size_t)(ctas * p.splits * p.tile_rows) * (h.dim * sizeof(float) + sizeof(float2));
  return p;
}

template <typename T, int kDim, int kNT, bool kBrief>
static cudaError_t launch_attention(const Kv8AttnParams& p, const Kv8Plan& plan, cudaStream_t s) {
  constexpr int kSmem = kv8_smem_bytes(kDim, kNT, kBrief);
  static OncePerDevice once;
  cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(kv8_attention_kernel<T, kDim, kNT, kBrief>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  });
  if (e != cudaSuccess) return e;
  LaunchShape l(dim3(plan.splits * plan.tiles, p.sh.heads, p.batch), 32 * kKvWarps, kSmem, s);
  if (plan.splits > 1 && !plan.memory) l.cluster(plan.splits, 1, 1);
  e = cudaLaunchKernelEx(&l.cfg, kv8_attention_kernel<T, kDim, kNT, kBrief>, p);
  if (e != cudaSuccess || !plan.memory) return e;
  qrb200_internal_count_launch();
  LaunchShape j(dim3(p.batch * p.queries * p.q_heads), 32 * kKvJoinWarps, 0, s);
  return cudaLaunchKernelEx(&j.cfg, kv_join_kernel<T, kDim, Kv8AttnParams>, p, plan.tile_rows);
}

template <typename T, int kDim>
static cudaError_t launch_prompt(const Kv8AttnParams& p, cudaStream_t s) {
  constexpr int kSmem = prompt_smem_bytes(kDim);
  static OncePerDevice once;
  const cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(kv8_prompt_kernel<T, kDim>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  });
  if (e != cudaSuccess) return e;
  const int64_t ctas = (int64_t)p.tiles * p.sh.heads * p.batch;
  if (ctas > kMaxRows) return cudaErrorInvalidValue;
  LaunchShape l(dim3((unsigned)ctas), kPromptThreads, kSmem, s);
  return cudaLaunchKernelEx(&l.cfg, kv8_prompt_kernel<T, kDim>, p);
}

}  // namespace qrb200

using namespace qrb200;

int qrb200_internal_kv8_site() { return take_site(); }
bool qrb200_internal_kv8_register(int* word) { return register_word(word); }

extern "C" {

int64_t qrb200_kv8_block_bytes(int64_t page_size, int64_t head_dim) {
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0 || (head_dim != 64 && head_dim != 128)) return 0;
  return 2 * page_size * head_dim;
}

size_t qrb200_kv8_write_workspace_bytes(const qrb200_kv8_shape* shape, int64_t tokens) {
  Kv8Shape h;
  if (!shape_of(shape, &h) || tokens <= kKv8Few) return 0;
  return write_list_bytes(tokens) + (size_t)h.pages * h.page * sizeof(int);
}

int qrb200_kv8_write(void* codes, float* range, const qrb200_kv8_shape* shape, const void* k, int64_t k_token_stride,
                     int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride, const int64_t* slots,
                     int64_t tokens, void* workspace, size_t workspace_bytes, void* stream) {
  Kv8Shape h;
  if (tokens < 0 || !shape_of(shape, &h) || tokens > kMaxRows / h.heads) return QRB200_ERR_ARG;
  if (tokens == 0) return QRB200_OK;
  if (!k || !v || !slots || !cache_ok(h, codes, range)) return QRB200_ERR_ARG;
  const int st = quant_ready();
  if (st != QRB200_OK) return st;
  const size_t need = qrb200_kv8_write_workspace_bytes(shape, tokens);
  if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u)))
    return QRB200_ERR_WORKSPACE;
  Kv8IoParams p{static_cast<unsigned char*>(codes), range, k, v, nullptr, nullptr, reinterpret_cast<const long long*>(slots),
                nullptr, nullptr, nullptr, tokens, k_token_stride, k_head_stride, v_token_stride, v_head_stride, h};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (need > 0) {
    p.pages = static_cast<int*>(workspace);
    p.list = p.pages + 64;
    p.rows = p.pages + write_list_bytes(tokens) / sizeof(int);
    LaunchShape l(dim3(ceil_div(tokens, 256)), 256, 0, s);
    if (cudaLaunchKernelEx(&l.cfg, kv8_rows_kernel, p) != cudaSuccess) return QRB200_ERR_CUDA;
    LaunchShape m(dim3(ceil_div(tokens, 8 * kKv8Seek)), 256, 0, s);
    if (cudaLaunchKernelEx(&m.cfg, kv8_pages_kernel, p) != cudaSuccess) return QRB200_ERR_CUDA;
    qrb200_internal_count_launch();
    qrb200_internal_count_launch();
  }
  // 16-byte loads where every (token, head) starts on such a boundary.
  const bool vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0 &&
                   ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) == 0;
  const cudaError_t e = with_shape(shape->dtype, h.dim, [&](auto type, auto dim) {
    using E = decltype(type);
    if (!p.rows) {
      LaunchShape l(dim3((unsigned)tokens, ceil_div(h.heads, 8)), 256, 0, s);
      return cudaLaunchKernelEx(&l.cfg, vec ? kv8_write_few_kernel<E, dim(), true> : kv8_write_few_kernel<E, dim(), false>, p);
    }
    // Eight CTAs to an SM: a page's rows are looked up once for several heads then, and the next head's loads are under
    // way while one's bytes leave.
    const unsigned ctas = (unsigned)std::min<int64_t>(8 * sm_count(), tokens * h.heads);
    LaunchShape m(dim3(std::min<unsigned>(ctas, 4 * sm_count())), 32 * kKv8ThinWarps, 0, s);
    const cudaError_t thin = cudaLaunchKernelEx(&m.cfg, vec ? kv8_write_thin_kernel<E, dim(), true> : kv8_write_thin_kernel<E, dim(), false>, p);
    if (thin != cudaSuccess) return thin;
    qrb200_internal_count_launch();
    LaunchShape l(dim3(ctas), 2 * h.dim, 0, s);
    return cudaLaunchKernelEx(&l.cfg, vec ? kv8_write_kernel<E, dim(), true> : kv8_write_kernel<E, dim(), false>, p);
  });
  if (e != cudaSuccess) return QRB200_ERR_CUDA;
  return launched();
}

int qrb200_kv8_read(const void* codes, const float* range, const qrb200_kv8_shape* shape, void* k, void* v, const int64_t* slots,
                    int64_t tokens, void* stream) {
  Kv8Shape h;
  if (tokens < 0 || !shape_of(shape, &h) || tokens > kMaxRows / h.heads) return QRB200_ERR_ARG;
  if (tokens == 0) return QRB200_OK;
  if (!k || !v || !slots || !cache_ok(h, codes, range) || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u))
    return QRB200_ERR_ARG;
  const int st = quant_ready();
  if (st != QRB200_OK) return st;
  const Kv8IoParams p{static_cast<unsigned char*>(const_cast<void*>(codes)), const_cast<float*>(range), nullptr, nullptr, k, v,
                      reinterpret_cast<const long long*>(slots), nullptr, nullptr, nullptr, tokens, 0, 0, 0, 0, h};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = with_shape(shape->dtype, h.dim, [&](auto type, auto dim) {
    LaunchShape l(dim3(ceil_div((tokens + 15) / 16 * h.heads, 8)), 256, 0, s);
    return cudaLaunchKernelEx(&l.cfg, kv8_read_kernel<decltype(type), dim()>, p);
  });
  if (e != cudaSuccess) return QRB200_ERR_CUDA;
  return launched();
}

// The most tokens that a sequence's queries see between them.
static int64_t token_span(int64_t queries, int64_t window) { return window > 0 ? std::min(window, kMaxRows) + queries : kMaxRows; }

// The launch grid is (splits x row tiles) x key heads x batch, a large batch in several launches.
constexpr int64_t kGridZ = 65535;
static bool attention_args(const qrb200_kv8_shape* shape, int64_t batch, int64_t queries, int64_t q_heads, int64_t max_pages,
                           Kv8Shape* h) {
  if (batch < 0 || queries < 0 || q_heads < 0 || max_pages < 0 || !shape_of(shape, h)) return false;
  return q_heads % h->heads == 0 && batch <= kMaxRows && q_heads <= 65535 && queries <= (1 << 24) &&
         queries * (q_heads / h->heads) <= (1 << 24) && (queries * q_heads == 0 || batch <= kMaxRows / (queries * q_heads)) &&
         max_pages <= kMaxRows / h->page - 320;
}

size_t qrb200_kv8_attention_workspace_bytes(const qrb200_kv8_shape* shape, int64_t batch, int64_t queries, int64_t q_heads,
                                            int64_t max_pages, int64_t window) {
  Kv8Shape h;
  if (window < 0 || !attention_args(shape, batch, queries, q_heads, max_pages, &h)) return 0;
  return batch * queries * q_heads == 0 ? 0 : attn_plan(h, shape->dtype == QRB200_F16, batch, queries, q_heads, max_pages, token_span(queries, window)).bytes;
}

int qrb200_kv8_attention(const void* q, const int64_t* q_strides, const void* codes, const float* range,
                         const qrb200_kv8_shape* shape, const int32_t* block_table, int64_t table_stride, const int32_t* lengths,
                         void* out, int64_t batch, int64_t queries, int64_t q_heads, int64_t max_pages, int64_t window, int causal,
                         float scale, void* workspace, size_t workspace_bytes, void* stream) {
  Kv8Shape h;
  if (!q_strides || !(scale >= 0.f) || !(scale <= 3.0e38f) || window < 0 || !attention_args(shape, batch, queries, q_heads, max_pages, &h))
    return QRB200_ERR_ARG;
  if (batch == 0 || queries == 0 || q_heads == 0) return QRB200_OK;
  if (!q || !out || !lengths || (max_pages > 0 && !block_table) || !cache_ok(h, codes, range) || table_stride < 0)
    return QRB200_ERR_ARG;
  const int st = quant_ready();
  if (st != QRB200_OK) return st;
  const Kv8Plan plan = attn_plan(h, shape->dtype == QRB200_F16, batch, queries, q_heads, max_pages, token_span(queries, window));
  if (plan.bytes > 0 && (!workspace || workspace_bytes < plan.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255u)))
    return QRB200_ERR_WORKSPACE;
  Kv8AttnParams p{};
  p.codes = static_cast<const unsigned char*>(codes);
  p.range = range;
  p.q = q;
  p.out = out;
  p.table = block_table;
  p.lengths = lengths;
  p.q_bs = q_strides[0], p.q_ts = q_strides[1], p.q_hs = q_strides[2], p.table_stride = table_stride;
  p.batch = (int)batch, p.queries = (int)queries, p.q_heads = (int)q_heads, p.share = (int)(q_heads / h.heads);
  p.window = window >= max_pages * h.page ? 0 : (int)window;  // one that reaches every token from every position is none
  p.max_pages = (int)max_pages, p.causal = causal, p.splits = plan.splits, p.tiles = plan.tiles;
  p.scale_part = std::frexp(scale, &p.scale_power) * 2.f * 1.4426950408889634f;
  p.scale_power -= 1;
  p.sh = h;
  p.q_wide = (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && ((q_strides[0] | q_strides[1] | q_strides[2]) & 3) == 0;
  p.part_o = plan.bytes > 0 ? static_cast<float*>(workspace) : nullptr;
  if (plan.memory)
    p.part_ml = reinterpret_cast<float2*>(p.part_o + batch * h.heads * plan.tiles * plan.splits * plan.tile_rows * h.dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  for (int64_t b = 0; b < batch; b += kGridZ) {
    Kv8AttnParams part = p;
    const int64_t rows = b * queries * q_heads, parts = b * h.heads * plan.tiles * plan.splits * plan.tile_rows;
    part.batch = (int)std::min(kGridZ, batch - b);
    part.q = static_cast<const char*>(q) + 2 * b * p.q_bs;
    part.out = static_cast<char*>(out) + 2 * rows * h.dim;
    part.table += b * table_stride;
    part.lengths += b;
    if (p.part_o) part.part_o += parts * h.dim;
    if (p.part_ml) part.part_ml += parts;
    const cudaError_t e = with_shape(shape->dtype, h.dim, [&](auto type, auto dim) {
      using E = decltype(type);
      if (plan.prompt) return launch_prompt<E, dim()>(part, s);
      if (plan.tile_rows == 16) return launch_attention<E, dim(), 2, false>(part, plan, s);
      return plan.brief ? launch_attention<E, dim(), 1, true>(part, plan, s) : launch_attention<E, dim(), 1, false>(part, plan, s);
    });
    if (e != cudaSuccess) return QRB200_ERR_CUDA;
    const int ended = launched();
    if (ended != QRB200_OK) return ended;
  }
  return QRB200_OK;
}

}  // extern "C"
