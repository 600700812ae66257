// The operators on 8- and 4-bit data for Python: argument checks, outputs and workspaces from torch's
// allocator, and the C ABI call, in one native step. A small call costs the host more than the GPU;
// done through Python and ctypes its checks and allocations took 12-22 us, here 4-8 us.
//
// The functions are private (`_native`); quant.py documents the public ones that call them.
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <optional>

#include "qrb200.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

constexpr int64_t kMaxCols = 32768;

int type_code(at::ScalarType t) {
  return t == at::kFloat ? QRB200_F32 : t == at::kBFloat16 ? QRB200_BF16 : t == at::kHalf ? QRB200_F16 : -1;
}

std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

// Type, device and autograd checks that every tensor operand gets.
void operand(const Tensor& t, const char* name, std::initializer_list<at::ScalarType> types, const Tensor* like = nullptr) {
  if (std::find(types.begin(), types.end(), t.scalar_type()) == types.end()) {
    std::string want;
    for (at::ScalarType s : types) want += (want.empty() ? "" : " or ") + std::string(c10::toString(s));
    TORCH_CHECK_TYPE(false, name, " must be ", want, ", got ", c10::toString(t.scalar_type()));
  }
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor (qrb200 has no CPU path)");
  if (like) TORCH_CHECK_VALUE(t.device() == like->device(), name, " is on ", t.device(), ", expected ", like->device());
  TORCH_CHECK(!(t.requires_grad() && at::GradMode::is_enabled()), name,
              " requires grad, and quantised operators have no backward pass; use torch.no_grad()");
}

Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

// `t` as (rows, cols) with unit column stride, copied only where its strides need it.
Tensor as_rows(const Tensor& t) {
  const int64_t cols = t.size(-1);
  Tensor r = t;
  if (t.dim() != 2) {
    int64_t rows = 1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
    r = t.reshape({rows, cols});
  }
  if ((r.stride(1) != 1 && cols > 1) || (r.stride(0) < cols && r.size(0) > 1)) r = r.contiguous();
  return r;
}

// int8 rows that start on 16-byte boundaries, as the tensor-core product loads them.
Tensor empty_codes(int64_t rows, int64_t cols, const Tensor& like) {
  const int64_t padded = (cols + 15) / 16 * 16;
  Tensor q = empty({rows, padded}, at::kChar, like);
  return padded == cols ? q : q.slice(1, 0, cols);
}
Tensor shaped(const Tensor& q, const Tensor& x) {
  if (x.dim() == 2) return q;
  return x.dim() == 1 ? q.select(0, 0) : q.unflatten(0, x.sizes().slice(0, x.dim() - 1));
}

// Runs on the current stream of `like`'s device, which becomes the current device meanwhile.
struct OnDevice {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit OnDevice(const Tensor& like)
      : guard(like.device()), stream(c10::cuda::getCurrentCUDAStream(like.get_device()).stream()) {}
};

void check(int status, const char* what) {
  TORCH_CHECK_VALUE(status != QRB200_ERR_ARG, what, ": a size, stride or alignment is beyond what the library takes (include/qrb200.h)");
  if (status != QRB200_OK) py::module_::import("qr_v2_b200_kernel_b200._lib").attr("check")(status, what);
}

const void* ptr(const Tensor& t) { return t.const_data_ptr(); }
const void* ptr(const OptTensor& t) { return t ? t->const_data_ptr() : nullptr; }

void check_cols(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() > 0 && t.size(-1) <= kMaxCols, name, " must be (..., cols) with cols <= ", kMaxCols, ", got ",
                    shape_of(t));
}

py::tuple rms_norm_int8(const Tensor& x, OptTensor weight, const OptTensor& residual, double eps) {
  operand(x, "x", {at::kFloat, at::kBFloat16, at::kHalf});
  check_cols(x, "x");
  const int64_t cols = x.size(-1);
  if (residual) {
    operand(*residual, "residual", {x.scalar_type()}, &x);
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes(), "residual must be ", shape_of(x), ", got ", shape_of(*residual));
  }
  if (weight) {
    operand(*weight, "weight", {x.scalar_type(), at::kFloat}, &x);
    TORCH_CHECK_VALUE(weight->dim() == 1 && weight->size(0) == cols, "weight must be (", cols, ",), got ", shape_of(*weight));
    weight = weight->contiguous();
  }
  TORCH_CHECK_VALUE(eps >= 0, "eps must be >= 0, got ", eps);
  OnDevice on(x);
  const Tensor xr = as_rows(x);
  const int64_t rows = xr.size(0);
  OptTensor rr;
  if (residual) rr = as_rows(*residual);
  const Tensor q = empty_codes(rows, cols, x), scale = empty(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
  const Tensor h = residual ? empty(x.sizes(), x.scalar_type(), x) : x;
  if (rows == 0 || cols == 0) scale.zero_();
  else
    check(qrb200_rms_norm_int8(ptr(xr), xr.stride(0), ptr(rr), rr ? rr->stride(0) : 0, ptr(weight),
                               weight ? type_code(weight->scalar_type()) : 0, q.data_ptr<int8_t>(), q.stride(0),
                               scale.data_ptr<float>(), residual ? h.data_ptr() : nullptr, rows, cols, (float)eps,
                               type_code(x.scalar_type()), on.stream),
          "rms_norm_int8");
  return py::make_tuple(shaped(q, x), scale, h);
}

py::tuple quantize_int8(const Tensor& x) {
  operand(x, "x", {at::kFloat, at::kBFloat16, at::kHalf});
  check_cols(x, "x");
  OnDevice on(x);
  const Tensor xr = as_rows(x);
  const int64_t rows = xr.size(0), cols = xr.size(1);
  const Tensor q = empty_codes(rows, cols, x), scale = empty(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
  if (rows == 0 || cols == 0) scale.zero_();
  else
    check(qrb200_quantize_int8(ptr(xr), xr.stride(0), q.data_ptr<int8_t>(), q.stride(0), scale.data_ptr<float>(), rows, cols,
                               type_code(x.scalar_type()), on.stream),
          "quantize_int8");
  return py::make_tuple(shaped(q, x), scale);
}

Tensor dequantize_int8(const Tensor& codes, const Tensor& scale, at::ScalarType dtype) {
  operand(codes, "codes", {at::kChar});
  operand(scale, "scale", {at::kFloat}, &codes);
  TORCH_CHECK_TYPE(type_code(dtype) >= 0, "dtype must be float32, bfloat16 or float16, got ", c10::toString(dtype));
  check_cols(codes, "codes");
  TORCH_CHECK_VALUE(scale.sizes() == codes.sizes().slice(0, codes.dim() - 1), "scale must have the leading shape of codes ",
                    shape_of(codes), ", got ", shape_of(scale));
  OnDevice on(codes);
  const Tensor q = as_rows(codes), s = scale.contiguous(), out = empty(codes.sizes(), dtype, codes);
  if (q.numel() > 0)
    check(qrb200_dequantize_int8(q.const_data_ptr<int8_t>(), q.stride(0), s.const_data_ptr<float>(), out.data_ptr(), q.size(0),
                                 q.size(1), type_code(dtype), on.stream),
          "dequantize_int8");
  return out;
}

Tensor int8_linear(const Tensor& x, const Tensor& x_scale, const Tensor& weight, const Tensor& weight_scale, OptTensor bias,
                   at::ScalarType dtype) {
  operand(x, "x", {at::kChar});
  operand(weight, "weight", {at::kChar}, &x);
  operand(x_scale, "x_scale", {at::kFloat}, &x);
  operand(weight_scale, "weight_scale", {at::kFloat}, &x);
  TORCH_CHECK_TYPE(type_code(dtype) >= 0, "dtype must be float32, bfloat16 or float16, got ", c10::toString(dtype));
  TORCH_CHECK_VALUE(x.dim() > 0 && weight.dim() == 2 && x.size(-1) == weight.size(1),
                    "x must be (..., depth) and weight (outs, depth), got ", shape_of(x), " and ", shape_of(weight));
  const int64_t outs = weight.size(0), depth = weight.size(1);
  TORCH_CHECK_VALUE(depth >= 1 && depth <= QRB200_INT8_MAX_DEPTH, "depth must be from 1 to ", QRB200_INT8_MAX_DEPTH, ", got ",
                    depth);
  TORCH_CHECK_VALUE(x_scale.sizes() == x.sizes().slice(0, x.dim() - 1), "x_scale must have the leading shape of x ",
                    shape_of(x), ", got ", shape_of(x_scale));
  TORCH_CHECK_VALUE(weight_scale.dim() == 1 && weight_scale.size(0) == outs, "weight_scale must be (", outs, ",), got ",
                    shape_of(weight_scale));
  if (bias) {
    operand(*bias, "bias", {dtype}, &x);
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == outs, "bias must be (", outs, ",), got ", shape_of(*bias));
    bias = bias->contiguous();
  }
  OnDevice on(x);
  const Tensor xr = as_rows(x), wr = as_rows(weight);
  const int64_t rows = xr.size(0);
  c10::SmallVector<int64_t, 5> sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = outs;
  const Tensor y = empty(sizes, dtype, x);
  if (rows == 0 || outs == 0) return y;
  const int8_t *xp = xr.const_data_ptr<int8_t>(), *wp = wr.const_data_ptr<int8_t>();
  const size_t need = qrb200_int8_linear_workspace_bytes(xp, xr.stride(0), wp, wr.stride(0), rows, outs, depth);
  Tensor ws;
  if (need > 0) ws = empty({(int64_t)need}, at::kByte, x);
  const Tensor sx = x_scale.contiguous(), sw = weight_scale.contiguous();
  check(qrb200_int8_linear(xp, xr.stride(0), sx.const_data_ptr<float>(), wp, wr.stride(0), sw.const_data_ptr<float>(), ptr(bias),
                           y.data_ptr(), rows, outs, depth, type_code(dtype), need > 0 ? ws.data_ptr() : nullptr, need, on.stream),
        "int8_linear");
  return y;
}

// ---- the 4-bit cache: its bytes and what they mean ------------------------------------------

struct Cache {
  Tensor data;
  qrb200_kv4_shape shape;
  at::ScalarType type;
};

Cache make_cache(const Tensor& data, int32_t page_size, int32_t head_dim, int32_t groups, at::ScalarType type) {
  TORCH_CHECK_TYPE(type == at::kBFloat16 || type == at::kHalf, "a cache's dtype must be bfloat16 or float16, got ",
                   c10::toString(type));
  operand(data, "data", {at::kByte});
  const int64_t bytes = groups > 0 ? qrb200_kv4_block_bytes(page_size, head_dim, head_dim / groups) : 0;
  TORCH_CHECK_VALUE(bytes > 0 && head_dim % groups == 0 && data.dim() == 3 && data.size(2) == bytes && data.is_contiguous() &&
                        data.size(1) >= 1 && data.size(1) <= 65535 && (reinterpret_cast<uintptr_t>(data.const_data_ptr()) & 15u) == 0,
                    "data must be a contiguous, 16-byte aligned (pages, kv_heads, ", bytes,
                    ") tensor for this page_size, head_dim and group_size, got ", shape_of(data));
  return Cache{data, {data.size(0), (int32_t)data.size(1), page_size, head_dim, groups, type_code(type)}, type};
}

Tensor slots_operand(const Cache& c, const Tensor& slots) {
  operand(slots, "slots", {at::kLong}, &c.data);
  TORCH_CHECK_VALUE(slots.dim() == 1, "slots must be (tokens,), got ", shape_of(slots));
  return slots.contiguous();
}

void kv4_write(const Cache& c, Tensor k, Tensor v, const Tensor& slots) {
  operand(k, "k", {c.type}, &c.data);
  operand(v, "v", {c.type}, &c.data);
  const Tensor at = slots_operand(c, slots);
  const int64_t want[3] = {at.size(0), c.shape.kv_heads, c.shape.head_dim};
  TORCH_CHECK_VALUE(k.sizes() == at::IntArrayRef(want) && v.sizes() == at::IntArrayRef(want), "k and v must be (", want[0], ", ",
                    want[1], ", ", want[2], "), got ", shape_of(k), " and ", shape_of(v));
  if (want[0] == 0) return;
  OnDevice on(c.data);
  if (k.stride(2) != 1) k = k.contiguous();
  if (v.stride(2) != 1) v = v.contiguous();
  check(qrb200_kv4_write(c.data.data_ptr(), &c.shape, ptr(k), k.stride(0), k.stride(1), ptr(v), v.stride(0), v.stride(1),
                         at.const_data_ptr<int64_t>(), want[0], on.stream),
        "kv4_write");
}

py::tuple kv4_read(const Cache& c, const Tensor& slots) {
  const Tensor at = slots_operand(c, slots);
  OnDevice on(c.data);
  const int64_t sizes[3] = {at.size(0), c.shape.kv_heads, c.shape.head_dim};
  const Tensor k = empty(sizes, c.type, c.data), v = empty(sizes, c.type, c.data);
  if (sizes[0] > 0)
    check(qrb200_kv4_read(ptr(c.data), &c.shape, k.data_ptr(), v.data_ptr(), at.const_data_ptr<int64_t>(), sizes[0], on.stream),
          "kv4_read");
  return py::make_tuple(k, v);
}

Tensor kv4_attention(Tensor q, const Cache& c, Tensor table, Tensor lengths, std::optional<double> scale, bool causal,
                     std::optional<int64_t> window) {
  operand(q, "q", {c.type}, &c.data);
  operand(table, "block_table", {at::kInt}, &c.data);
  operand(lengths, "lengths", {at::kInt}, &c.data);
  const int64_t dim = c.shape.head_dim;
  TORCH_CHECK_VALUE(q.dim() == 4 && q.size(3) == dim && q.size(2) % c.shape.kv_heads == 0,
                    "q must be (batch, queries, heads, ", dim, ") with heads a multiple of ", c.shape.kv_heads, ", got ",
                    shape_of(q));
  const int64_t batch = q.size(0), queries = q.size(1), heads = q.size(2);
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) == batch, "block_table must be (", batch, ", max_pages), got ",
                    shape_of(table));
  TORCH_CHECK_VALUE(lengths.dim() == 1 && lengths.size(0) == batch, "lengths must be (", batch, ",), got ", shape_of(lengths));
  TORCH_CHECK_VALUE(!window || *window >= 1, "window must be at least 1, got ", *window);
  const double factor = scale ? *scale : 1 / std::sqrt((double)dim);
  TORCH_CHECK_VALUE(factor >= 0 && factor < 3e38, "scale must be finite and not negative, got ", factor);
  OnDevice on(c.data);
  if (q.stride(3) != 1) q = q.contiguous();
  if (table.size(1) > 1 && table.stride(1) != 1) table = table.contiguous();
  lengths = lengths.contiguous();
  const Tensor out = empty(q.sizes(), c.type, c.data);
  if (out.numel() == 0) return out;
  const int64_t pages = table.size(1);
  const size_t need = qrb200_kv4_attention_workspace_bytes(&c.shape, batch, queries, heads, pages, window.value_or(0));
  Tensor ws;
  if (need > 0) ws = empty({(int64_t)need}, at::kByte, c.data);
  const int64_t strides[3] = {q.stride(0), q.stride(1), q.stride(2)};
  check(qrb200_kv4_attention(ptr(q), strides, ptr(c.data), &c.shape, table.const_data_ptr<int32_t>(), table.stride(0),
                             lengths.const_data_ptr<int32_t>(), out.data_ptr(), batch, queries, heads, pages,
                             window.value_or(0), causal, (float)factor, need > 0 ? ws.data_ptr() : nullptr, need, on.stream),
        "kv4_attention");
  return out;
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.def("rms_norm_int8", &rms_norm_int8);
  m.def("quantize_int8", &quantize_int8);
  m.def("dequantize_int8", &dequantize_int8);
  m.def("int8_linear", &int8_linear);
  py::class_<Cache>(m, "Cache").def(py::init(&make_cache));
  m.def("kv4_write", &kv4_write);
  m.def("kv4_read", &kv4_read);
  m.def("kv4_attention", &kv4_attention);
}
