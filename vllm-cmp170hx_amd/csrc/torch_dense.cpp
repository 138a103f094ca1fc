// The dense linear layer (kernels/dense/ops.py) in host-only C++: tensor checks, outputs
// and scratch from torch's allocator (so of the current stream, and of a graph's pool
// under capture), the C-ABI calls on torch's current stream, and the gradient as an
// autograd node that calls operators of its own below autograd.
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/Tensor.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <optional>
#include <tuple>
#include <vector>

#include "../../include/vllm_mi355x.h"
#include "torch_common.h"

namespace {

using vq_torch::check_status;
using vq_torch::dtype_code;
using vq_torch::stream_of;

decltype(&dense_linear) native_linear = nullptr;
decltype(&dense_linear_workspace_size) native_workspace = nullptr;
decltype(&dense_linear_grad) native_grad = nullptr;
decltype(&dense_linear_grad_workspace_size) native_grad_workspace = nullptr;
decltype(&vllm_mi355x_last_error) native_error = nullptr;

constexpr const char* kWhat = "dense_linear";
constexpr int64_t kSwiglu = 5;

bool is_float(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat; }

template <typename Size>
std::vector<Size> with_last(c10::ArrayRef<Size> sizes, const Size& last) {
  std::vector<Size> v = sizes.vec();
  v.back() = last;
  return v;
}

// t as rows of its last axis at one row stride; stride -1: they do not lie so.
struct Rows {
  int64_t rows, k, stride;
};
Rows rows_of(const at::Tensor& t) {
  const int64_t k = t.size(-1);
  const int64_t rows = k ? t.numel() / k : 0;
  if (rows == 0) return {0, k, k};
  if (k > 1 && t.stride(-1) != 1) return {rows, k, -1};
  int64_t stride = k, count = 1;
  bool first = true;
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (first) stride = t.stride(d);
    else if (t.stride(d) != stride * count) return {rows, k, -1};
    first = false;
    count *= t.size(d);
  }
  return {rows, k, rows > 1 && stride < k ? -1 : stride};
}

// Shapes and types (not how tensors lie); sizes may be symbolic.
void check_kinds(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias, int64_t activation,
                 const std::optional<at::Tensor>& residual, at::ScalarType out_dtype, double limit) {
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, kWhat, ": x must be BF16 or FP16");
  TORCH_CHECK(w.scalar_type() == x.scalar_type(), kWhat, ": the weights must have x's type");
  TORCH_CHECK(x.dim() >= 1 && w.dim() == 2, kWhat, ": x must be [..., k], the weights [n, k]");
  TORCH_CHECK(is_float(out_dtype), kWhat, ": out_dtype must be BF16, FP16 or FP32");
  TORCH_CHECK(activation >= 0 && activation <= kSwiglu, kWhat, ": unknown activation");
  TORCH_CHECK(limit > 0, kWhat, ": clamp_limit must be positive");
  TORCH_CHECK(!bias || (bias->dim() == 1 && is_float(bias->scalar_type())), kWhat, ": bias must be BF16, FP16 or FP32, a value a weight row");
  TORCH_CHECK(!residual || (residual->dim() == x.dim() && is_float(residual->scalar_type())), kWhat,
              ": residual must be BF16, FP16 or FP32 of the output's shape");
  for (const at::Tensor* t : {&w, bias ? &*bias : nullptr, residual ? &*residual : nullptr}) {
    TORCH_CHECK(!t || t->device() == x.device(), kWhat, ": tensors must be on x's device");
  }
  const c10::SymInt k = x.sym_size(-1), lines = w.sym_size(0);
  TORCH_SYM_CHECK(k.sym_gt(0), kWhat, ": the weights must be [n, k] of x's k = ", k);
  TORCH_SYM_CHECK(w.sym_size(1).sym_eq(k), kWhat, ": the weights must be [n, k] of x's k = ", k);
  TORCH_SYM_CHECK(lines.sym_gt(0), kWhat, ": the weights must be [n, k], not without rows");
  if (activation == kSwiglu) {
    TORCH_SYM_CHECK((lines % 2).sym_eq(0), kWhat, ": a gated activation needs gate and up rows in equal number");
  }
  if (bias) TORCH_SYM_CHECK(bias->sym_size(0).sym_eq(lines), kWhat, ": bias must be a value a weight row");
  if (residual) {
    for (int64_t d = 0; d < x.dim(); ++d) {
      TORCH_SYM_CHECK(residual->sym_size(d).sym_eq(d + 1 < x.dim() ? x.sym_size(d) : activation == kSwiglu ? lines / 2 : lines), kWhat,
                      ": residual must have the output's shape");
    }
  }
}

int64_t columns_of(const at::Tensor& w, int64_t activation) { return activation == kSwiglu ? w.size(0) / 2 : w.size(0); }

void run(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias, int64_t activation,
         const std::optional<at::Tensor>& residual, double limit, const at::Tensor& out, const at::Tensor& z) {
  TORCH_CHECK(x.is_cuda(), kWhat, ": x must be on a GPU");
  const Rows r = rows_of(x);
  TORCH_CHECK(r.stride >= 0, kWhat, ": x needs unit stride along its last axis and leading axes that are one run of rows, not overlapping");
  TORCH_CHECK((r.k == 1 || w.stride(1) == 1) && (w.size(0) == 1 || w.stride(0) >= r.k), kWhat,
              ": the weights need unit inner stride and rows that do not overlap");
  const int64_t n = columns_of(w, activation);
  TORCH_CHECK(!bias || bias->is_contiguous(), kWhat, ": bias must be contiguous");
  Rows res{0, 0, 0};
  if (residual) {
    res = rows_of(*residual);
    TORCH_CHECK(res.stride >= 0, kWhat, ": residual needs unit stride along its last axis and leading axes that are one run of rows, not overlapping");
  }
  const c10::DeviceGuard guard(x.device());
  const int64_t w_stride = w.size(0) > 1 ? w.stride(0) : r.k;
  const int64_t bytes = native_workspace(x.const_data_ptr(), r.rows, r.k, r.stride, w.const_data_ptr(), n, w_stride, int(activation));
  if (bytes < 0) TORCH_CHECK(false, native_error());
  const at::Tensor ws = at::empty({bytes}, x.options().dtype(at::kByte));
  check_status(native_linear(x.const_data_ptr(), dtype_code(x.scalar_type()), r.rows, r.k, r.stride, w.const_data_ptr(), n, w_stride,
                             bias ? bias->const_data_ptr() : nullptr, bias ? dtype_code(bias->scalar_type()) : 0, int(activation),
                             static_cast<float>(limit), residual ? residual->const_data_ptr() : nullptr,
                             residual ? dtype_code(residual->scalar_type()) : 0, res.stride, out.mutable_data_ptr(),
                             dtype_code(out.scalar_type()), z.defined() ? z.mutable_data_ptr<float>() : nullptr, ws.mutable_data_ptr(), bytes,
                             stream_of(x)));
}

at::Tensor linear(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias, int64_t activation,
                  const std::optional<at::Tensor>& residual, at::ScalarType out_dtype, double limit) {
  check_kinds(x, w, bias, activation, residual, out_dtype, limit);
  const c10::DeviceGuard guard(x.device());
  at::Tensor out = at::empty(with_last(x.sizes(), columns_of(w, activation)), x.options().dtype(out_dtype).memory_format(at::MemoryFormat::Contiguous));
  run(x, w, bias, activation, residual, limit, out, at::Tensor());
  return out;
}

void check_out(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias, int64_t activation,
               const std::optional<at::Tensor>& residual, double limit, const at::Tensor& out) {
  check_kinds(x, w, bias, activation, residual, out.scalar_type(), limit);
  TORCH_CHECK(out.is_contiguous() && out.device() == x.device() && out.dim() == x.dim(), kWhat, ": out must be a contiguous [..., n] on x's GPU");
  for (int64_t d = 0; d < x.dim(); ++d) {
    const c10::SymInt lines = w.sym_size(0);
    TORCH_SYM_CHECK(out.sym_size(d).sym_eq(d + 1 < x.dim() ? x.sym_size(d) : activation == kSwiglu ? lines / 2 : lines), kWhat,
                    ": out must be a contiguous [..., n] on x's GPU");
  }
}

void linear_out(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias, int64_t activation,
                const std::optional<at::Tensor>& residual, double limit, const at::Tensor& out) {
  check_out(x, w, bias, activation, residual, limit, out);
  run(x, w, bias, activation, residual, limit, out, at::Tensor());
}

// Sizes that the gradient takes (so that it is not refused after the forward has run).
void check_trains(int64_t rows, int64_t k, int64_t n, int64_t activation) {
  if (rows > 0 && native_grad_workspace(rows, k, n, int(activation), 1, 1, 1) < 0) TORCH_CHECK(false, native_error());
}

// (y, z): z is what the gradient needs beside x and w, x w^T + bias in FP32 (nothing
// without an activation).
std::tuple<at::Tensor, at::Tensor> forward(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias, int64_t activation,
                                           const std::optional<at::Tensor>& residual, at::ScalarType out_dtype, double limit) {
  check_kinds(x, w, bias, activation, residual, out_dtype, limit);
  const c10::DeviceGuard guard(x.device());
  const int64_t n = columns_of(w, activation), k = x.size(-1);
  check_trains(x.numel() / k, k, n, activation);
  at::Tensor out = at::empty(with_last(x.sizes(), n), x.options().dtype(out_dtype).memory_format(at::MemoryFormat::Contiguous));
  at::Tensor z = at::empty({activation ? x.numel() / k : 0, w.size(0)}, x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
  run(x, w, bias, activation, residual, limit, out, activation ? z : at::Tensor());
  return {out, z};
}

// (dx, dw, dbias) from dy; those not asked for are empty.  x is read for dw alone, w for dx alone.
std::tuple<at::Tensor, at::Tensor, at::Tensor> gradient(const std::optional<at::Tensor>& x, const std::optional<at::Tensor>& w,
                                                        const at::Tensor& z, int64_t activation, double limit, const at::Tensor& given,
                                                        bool need_x, bool need_w, std::optional<at::ScalarType> bias_dtype) {
  TORCH_CHECK((x || !need_w) && (w || !need_x) && given.is_cuda() && z.device() == given.device() && given.dim() >= 1 && given.size(-1) > 0, kWhat,
              ": the gradient's tensors must be there, on a GPU");
  if (x && w) check_kinds(*x, *w, std::nullopt, activation, std::nullopt, given.scalar_type(), limit);
  const int64_t n = given.size(-1), rows = given.numel() / n, lines = activation == kSwiglu ? 2 * n : n;
  const Rows r = x ? rows_of(*x) : Rows{rows, w ? w->size(1) : 1, w ? w->size(1) : 1};
  TORCH_CHECK((!x || (x->device() == given.device() && x->dim() == given.dim() && r.stride >= 0 && r.rows == rows)) &&
                  (!w || (w->device() == given.device() && w->dim() == 2 && w->size(0) == lines && w->size(1) == r.k)) &&
                  (!activation || (z.is_contiguous() && z.numel() == rows * lines && z.scalar_type() == at::kFloat)),
              kWhat, ": the gradient's tensors must be the forward's");
  const at::ScalarType type = x ? x->scalar_type() : w ? w->scalar_type() : at::kBFloat16;
  const c10::DeviceGuard guard(given.device());
  const auto make = [&](at::IntArrayRef sizes, at::ScalarType t) {
    const auto options = given.options().dtype(t).memory_format(at::MemoryFormat::Contiguous);
    return rows ? at::empty(sizes, options) : at::zeros(sizes, given.options().dtype(t));
  };
  at::Tensor dx = need_x ? make(with_last(given.sizes(), r.k), type) : make({0}, type);
  at::Tensor dw = need_w ? make({lines, r.k}, type) : make({0}, type);
  at::Tensor db = bias_dtype ? make({lines}, *bias_dtype) : make({0}, type);
  if (rows == 0) return {dx, dw, db};
  // (autograd gives broadcast and transposed gradients too)
  const at::Tensor dy = rows_of(given).stride >= 0 ? given : given.contiguous();
  const int64_t bytes = native_grad_workspace(rows, r.k, n, int(activation), need_x, need_w, bias_dtype.has_value());
  if (bytes < 0) TORCH_CHECK(false, native_error());
  const at::Tensor ws = at::empty({bytes}, given.options().dtype(at::kByte));
  check_status(native_grad(x ? x->const_data_ptr() : nullptr, dtype_code(type), rows, r.k, r.stride, w ? w->const_data_ptr() : nullptr, n,
                           w && lines > 1 ? w->stride(0) : r.k, activation ? z.const_data_ptr<float>() : nullptr, int(activation),
                           static_cast<float>(limit), dy.const_data_ptr(), dtype_code(dy.scalar_type()), rows_of(dy).stride,
                           need_x ? dx.mutable_data_ptr() : nullptr, need_w ? dw.mutable_data_ptr() : nullptr,
                           bias_dtype ? db.mutable_data_ptr() : nullptr, bias_dtype ? dtype_code(*bias_dtype) : 0, ws.mutable_data_ptr(), bytes,
                           stream_of(given)));
  return {dx, dw, db};
}

template <typename F>
c10::TypedOperatorHandle<F> handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

struct DenseLinear : torch::autograd::Function<DenseLinear> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w,
                            const std::optional<at::Tensor>& bias, int64_t activation, const std::optional<at::Tensor>& residual,
                            at::ScalarType out_dtype, double limit) {
    const bool need_x = x.requires_grad(), need_w = w.requires_grad(), need_bias = bias && bias->requires_grad();
    const at::AutoDispatchBelowADInplaceOrView below;
    at::Tensor y, z;
    if (need_x || need_w || need_bias) {
      static const auto op = handle<decltype(::forward)>("_vllm_mi355x::dense_linear_forward");
      std::tie(y, z) = op.call(x, w, bias, activation, residual, out_dtype, limit);
    } else {  // (the residual's gradient is dy)
      static const auto op = handle<decltype(linear)>("_vllm_mi355x::dense_linear");
      y = op.call(x, w, bias, activation, residual, out_dtype, limit);
    }
    // (what no gradient is computed from is not kept, and may be written to)
    ctx->save_for_backward({need_w ? x : at::Tensor(), need_x ? w : at::Tensor(), z});
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["limit"] = limit;
    ctx->saved_data["x"] = need_x;
    ctx->saved_data["w"] = need_w;
    ctx->saved_data["has_bias"] = bias.has_value();
    ctx->saved_data["bias"] = need_bias ? int64_t(bias->scalar_type()) : int64_t(-1);
    ctx->saved_data["residual"] = residual && residual->requires_grad() ? int64_t(residual->scalar_type()) : int64_t(-1);
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(7);
    if (!grads[0].defined()) return out;
    TORCH_CHECK(!c10::GradMode::is_enabled(), kWhat, ": its gradient has no gradient (create_graph)");
    static const auto op = handle<decltype(::gradient)>("_vllm_mi355x::dense_linear_grad");
    const torch::autograd::variable_list saved = ctx->get_saved_variables();
    // what this pass asks for (an edge an input that is there: x, w, bias, residual)
    const bool has_bias = ctx->saved_data["has_bias"].toBool();
    const auto asked = [&](const char* name, size_t edge) {
      const int64_t type = ctx->saved_data[name].toInt();
      return type >= 0 && ctx->needs_input_grad(edge) ? type : int64_t(-1);
    };
    const int64_t bias = asked("bias", 2), residual = asked("residual", has_bias ? 3 : 2);
    const bool need_x = ctx->saved_data["x"].toBool() && ctx->needs_input_grad(0);
    const bool need_w = ctx->saved_data["w"].toBool() && ctx->needs_input_grad(1);
    if (residual >= 0) out[4] = grads[0].to(at::ScalarType(residual));
    if (need_x || need_w || bias >= 0) {
      const at::AutoDispatchBelowADInplaceOrView below;
      const auto kept = [&](size_t i) { return saved[i].defined() ? std::optional<at::Tensor>(saved[i]) : std::nullopt; };
      auto [dx, dw, db] = op.call(kept(0), kept(1), saved[2], ctx->saved_data["activation"].toInt(), ctx->saved_data["limit"].toDouble(),
                                  grads[0], need_x, need_w, bias >= 0 ? std::optional<at::ScalarType>(at::ScalarType(bias)) : std::nullopt);
      if (need_x) out[0] = dx;
      if (need_w) out[1] = dw;
      if (bias >= 0) out[2] = db;
    }
    return out;
  }
};

at::Tensor linear_autograd(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias, int64_t activation,
                           const std::optional<at::Tensor>& residual, at::ScalarType out_dtype, double limit) {
  bool needs = false;
  for (const at::Tensor* t : {&x, &w, bias ? &*bias : nullptr, residual ? &*residual : nullptr}) {
    if (!t) continue;
    TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), kWhat, ": no forward-mode derivative");
    needs = needs || t->requires_grad();
  }
  if (!needs || !c10::GradMode::is_enabled()) {
    static const auto op = handle<decltype(linear)>("_vllm_mi355x::dense_linear");
    const at::AutoDispatchBelowADInplaceOrView below;
    return op.call(x, w, bias, activation, residual, out_dtype, limit);
  }
  return DenseLinear::apply(x, w, bias, activation, residual, out_dtype, limit);
}

void linear_out_autograd(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias, int64_t activation,
                         const std::optional<at::Tensor>& residual, double limit, const at::Tensor& out) {
  for (const at::Tensor* t : {&x, &w, bias ? &*bias : nullptr, residual ? &*residual : nullptr, &out}) {
    if (!t) continue;
    TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), kWhat, ": no forward-mode derivative");
    TORCH_CHECK(!t->requires_grad() || !c10::GradMode::is_enabled(), kWhat, ": out carries no gradient");
  }
  static const auto op = handle<decltype(linear_out)>("_vllm_mi355x::dense_linear_out");
  const at::AutoDispatchBelowADInplaceOrView below;
  op.call(x, w, bias, activation, residual, limit, out);
  // (a gradient that was to use what out held finds it changed)
  if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}

// Shapes alone, for tracing.
at::Tensor linear_meta(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias, int64_t activation,
                       const std::optional<at::Tensor>& residual, at::ScalarType out_dtype, double limit) {
  check_kinds(x, w, bias, activation, residual, out_dtype, limit);
  const c10::SymInt lines = w.sym_size(0);
  return at::empty_symint(with_last(x.sym_sizes(), activation == kSwiglu ? lines / 2 : lines), x.options().dtype(out_dtype));
}
void linear_out_meta(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias, int64_t activation,
                     const std::optional<at::Tensor>& residual, double limit, const at::Tensor& out) {
  check_out(x, w, bias, activation, residual, limit, out);
}
std::tuple<at::Tensor, at::Tensor> forward_meta(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias,
                                                int64_t activation, const std::optional<at::Tensor>& residual, at::ScalarType out_dtype,
                                                double limit) {
  at::Tensor y = linear_meta(x, w, bias, activation, residual, out_dtype, limit);
  const c10::SymInt rows = activation ? x.sym_numel() / x.sym_size(-1) : c10::SymInt(0);
  const auto all = x.sym_numel().maybe_as_int(), k = x.sym_size(-1).maybe_as_int(), n = y.sym_size(-1).maybe_as_int();
  if (all && k && n) check_trains(*all / *k, *k, *n, activation);
  return {y, at::empty_symint({rows, w.sym_size(0)}, x.options().dtype(at::kFloat))};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> gradient_meta(const std::optional<at::Tensor>& x, const std::optional<at::Tensor>& w,
                                                             const at::Tensor&, int64_t activation, double, const at::Tensor& given,
                                                             bool need_x, bool need_w, std::optional<at::ScalarType> bias_dtype) {
  TORCH_CHECK((x || !need_w) && (w || !need_x), kWhat, ": the gradient's tensors must be there");
  const at::ScalarType type = x ? x->scalar_type() : w ? w->scalar_type() : at::kBFloat16;
  const auto make = [&](c10::SymIntArrayRef sizes, at::ScalarType t) { return at::empty_symint(sizes, given.options().dtype(t)); };
  const c10::SymInt n = given.sym_size(-1), lines = activation == kSwiglu ? n * 2 : n;
  return {need_x ? make(with_last(given.sym_sizes(), w->sym_size(1)), type) : make({c10::SymInt(0)}, type),
          need_w ? make({lines, x->sym_size(-1)}, type) : make({c10::SymInt(0)}, type),
          bias_dtype ? make({lines}, *bias_dtype) : make({c10::SymInt(0)}, type)};
}

template <typename F>
bool find(void* library, const char* name, F& f) {
  f = reinterpret_cast<F>(dlsym(library, name));
  return f != nullptr;
}

}  // namespace

bool vq_torch::bind_dense(void* library) {
  return find(library, "dense_linear", native_linear) && find(library, "dense_linear_workspace_size", native_workspace) &&
         find(library, "dense_linear_grad", native_grad) && find(library, "dense_linear_grad_workspace_size", native_grad_workspace) &&
         find(library, "vllm_mi355x_last_error", native_error);
}

TORCH_LIBRARY_FRAGMENT(_vllm_mi355x, m) {
  m.def("dense_linear(Tensor x, Tensor w, Tensor? bias, int activation, Tensor? residual, ScalarType out_dtype, float limit) -> Tensor");
  m.def("dense_linear_out(Tensor x, Tensor w, Tensor? bias, int activation, Tensor? residual, float limit, Tensor(a!) out) -> ()");
  m.def(
      "dense_linear_forward(Tensor x, Tensor w, Tensor? bias, int activation, Tensor? residual, ScalarType out_dtype, float limit) "
      "-> (Tensor, Tensor)");
  m.def(
      "dense_linear_grad(Tensor? x, Tensor? w, Tensor z, int activation, float limit, Tensor dy, bool need_x, bool need_w, "
      "ScalarType? bias_dtype) -> (Tensor, Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(_vllm_mi355x, CUDA, m) {
  m.impl("dense_linear", &linear);
  m.impl("dense_linear_out", &linear_out);
  m.impl("dense_linear_forward", &forward);
  m.impl("dense_linear_grad", &gradient);
}
TORCH_LIBRARY_IMPL(_vllm_mi355x, Meta, m) {
  m.impl("dense_linear", &linear_meta);
  m.impl("dense_linear_out", &linear_out_meta);
  m.impl("dense_linear_forward", &forward_meta);
  m.impl("dense_linear_grad", &gradient_meta);
}
TORCH_LIBRARY_IMPL(_vllm_mi355x, Autograd, m) {
  m.impl("dense_linear", &linear_autograd);
  m.impl("dense_linear_out", &linear_out_autograd);
}
