// Routing from logits (kernels/moe/route.py: moe_route_logits) in host-only C++: the
// choice and its weights, and the weights' gradient as an autograd node that calls an
// operator of its own below autograd.
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/Tensor.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <cmath>
#include <optional>
#include <tuple>

#include "../../include/vllm_mi355x.h"
#include "torch_common.h"

namespace {

using vq_torch::check_status;
using vq_torch::dtype_code;
using vq_torch::stream_of;

decltype(&moe_route_logits) native_route = nullptr;
decltype(&moe_route_grad) native_grad = nullptr;

constexpr const char* kWhat = "moe_route_logits";

// Shapes, types and options; sizes may be symbolic.
void check_call(const at::Tensor& logits, const std::optional<at::Tensor>& bias, int64_t topk, int64_t groups, int64_t topk_groups,
                int64_t scoring, double scale, const std::optional<at::Tensor>& padding) {
  TORCH_CHECK(logits.dim() == 2, kWhat, ": logits must be [rows, experts]");
  TORCH_CHECK(logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kHalf || logits.scalar_type() == at::kFloat, kWhat,
              ": logits must be BF16, FP16 or FP32");
  const c10::SymInt rows = logits.sym_size(0), experts = logits.sym_size(1);
  TORCH_SYM_CHECK(experts.sym_gt(0), kWhat, ": between 1 and 1024 experts");
  TORCH_SYM_CHECK(experts.sym_le(1024), kWhat, ": between 1 and 1024 experts");
  TORCH_CHECK(topk > 0 && topk <= 64, kWhat, ": topk must be between 1 and 64, and at most the experts");
  TORCH_SYM_CHECK(experts.sym_ge(topk), kWhat, ": topk must be between 1 and 64, and at most the experts");
  TORCH_CHECK(groups > 0 && groups <= 64, kWhat, ": up to 64 groups of equal size");
  TORCH_SYM_CHECK((experts % groups).sym_eq(0), kWhat, ": up to 64 groups of equal size");
  TORCH_CHECK(topk_groups > 0 && topk_groups <= groups, kWhat, ": topk_groups must be between 1 and the groups");
  TORCH_SYM_CHECK((experts / groups * topk_groups).sym_ge(topk), kWhat, ": topk experts do not fit topk_groups groups");
  TORCH_CHECK(scoring == 0 || scoring == 1, kWhat, ": scoring must be softmax (0) or sigmoid (1)");
  TORCH_CHECK(std::isfinite(static_cast<float>(scale)), kWhat, ": the scale must be finite");
  if (bias) {
    TORCH_CHECK(bias->dim() == 1 && bias->device() == logits.device() && bias->scalar_type() == at::kFloat, kWhat,
                ": bias must be FP32 [experts] on the logits' GPU");
    TORCH_SYM_CHECK(bias->sym_size(0).sym_eq(experts), kWhat, ": bias must be FP32 [experts] on the logits' GPU");
  }
  if (padding) {
    TORCH_CHECK(padding->dim() == 1 && padding->device() == logits.device() &&
                    (padding->scalar_type() == at::kBool || padding->scalar_type() == at::kByte),
                kWhat, ": is_padding must be a contiguous bool or uint8 [rows] on the logits' GPU");
    TORCH_SYM_CHECK(padding->sym_size(0).sym_eq(rows), kWhat, ": is_padding must be a contiguous bool or uint8 [rows] on the logits' GPU");
  }
}

void check_logits(const at::Tensor& logits) {
  TORCH_CHECK(logits.is_cuda(), kWhat, ": logits must be on a GPU");
  TORCH_CHECK(logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kHalf || logits.scalar_type() == at::kFloat, kWhat,
              ": logits must be BF16, FP16 or FP32");
  TORCH_CHECK(logits.dim() == 2 && logits.size(1) > 0 && (logits.numel() == 0 || logits.size(1) == 1 || logits.stride(1) == 1), kWhat,
              ": logits must be [rows, experts] with unit inner stride");
}

// A row of one expert may have any inner stride: rows are one element then.
int64_t stride_of(const at::Tensor& logits) { return logits.size(0) > 1 ? logits.stride(0) : logits.size(1); }

std::tuple<at::Tensor, at::Tensor> route(const at::Tensor& logits, const std::optional<at::Tensor>& bias, int64_t topk, int64_t groups,
                                         int64_t topk_groups, int64_t scoring, bool renormalize, double scale,
                                         const std::optional<at::Tensor>& padding) {
  check_call(logits, bias, topk, groups, topk_groups, scoring, scale, padding);
  check_logits(logits);
  const int64_t rows = logits.size(0), experts = logits.size(1);
  TORCH_CHECK(!padding || padding->is_contiguous(), kWhat, ": is_padding must be a contiguous bool or uint8 [rows] on the logits' GPU");
  const c10::DeviceGuard guard(logits.device());
  const at::Tensor close = bias ? bias->contiguous() : at::Tensor();
  at::Tensor weights = at::empty({rows, topk}, logits.options().dtype(at::kFloat));
  at::Tensor ids = at::empty({rows, topk}, logits.options().dtype(at::kInt));
  check_status(native_route(logits.const_data_ptr(), dtype_code(logits.scalar_type()), rows, experts, stride_of(logits),
                            bias ? close.const_data_ptr<float>() : nullptr, topk, groups, topk_groups, int(scoring), renormalize,
                            static_cast<float>(scale), padding ? static_cast<const uint8_t*>(padding->const_data_ptr()) : nullptr,
                            weights.mutable_data_ptr<float>(), ids.mutable_data_ptr<int32_t>(), stream_of(logits)));
  return {weights, ids};
}

at::Tensor gradient(const at::Tensor& logits, const at::Tensor& weights, const at::Tensor& ids, const at::Tensor& upstream,
                    int64_t scoring, bool renormalize) {
  check_logits(logits);
  TORCH_CHECK(weights.dim() == 2 && weights.size(0) == logits.size(0) && ids.sizes() == weights.sizes() && upstream.sizes() == weights.sizes(),
              kWhat, ": the gradient's weights, ids and upstream must be [rows, topk]");
  TORCH_CHECK(weights.scalar_type() == at::kFloat && ids.scalar_type() == at::kInt && upstream.scalar_type() == at::kFloat &&
                  weights.is_contiguous() && ids.is_contiguous() && upstream.is_contiguous() && weights.device() == logits.device() &&
                  ids.device() == logits.device() && upstream.device() == logits.device(),
              kWhat, ": the gradient's weights, ids and upstream must be contiguous FP32, int32 and FP32 on the logits' GPU");
  const int64_t rows = logits.size(0), experts = logits.size(1);
  const c10::DeviceGuard guard(logits.device());
  at::Tensor grad = at::empty({rows, experts}, logits.options());
  check_status(native_grad(logits.const_data_ptr(), dtype_code(logits.scalar_type()), rows, experts, stride_of(logits),
                           weights.const_data_ptr<float>(), ids.const_data_ptr<int32_t>(), weights.size(1), int(scoring), renormalize,
                           upstream.const_data_ptr<float>(), grad.mutable_data_ptr(), stream_of(logits)));
  return grad;
}

template <typename F>
c10::TypedOperatorHandle<F> handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

std::tuple<at::Tensor, at::Tensor> route_below(const at::Tensor& logits, const std::optional<at::Tensor>& bias, int64_t topk, int64_t groups,
                                               int64_t topk_groups, int64_t scoring, bool renormalize, double scale,
                                               const std::optional<at::Tensor>& padding) {
  static const auto op = handle<decltype(route)>("_vllm_mi355x::moe_route_logits");
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(logits, bias, topk, groups, topk_groups, scoring, renormalize, scale, padding);
}

struct RouteWeights : torch::autograd::Function<RouteWeights> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits,
                                                const std::optional<at::Tensor>& bias, int64_t topk, int64_t groups, int64_t topk_groups,
                                                int64_t scoring, bool renormalize, double scale, const std::optional<at::Tensor>& padding) {
    auto [weights, ids] = route_below(logits, bias, topk, groups, topk_groups, scoring, renormalize, scale, padding);
    ctx->save_for_backward({logits, weights, ids});
    ctx->saved_data["scoring"] = scoring;
    ctx->saved_data["renormalize"] = renormalize;
    ctx->mark_non_differentiable({ids});
    return {weights, ids};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    torch::autograd::variable_list none(9);
    if (!grads[0].defined()) return none;
    TORCH_CHECK(!c10::GradMode::is_enabled(), kWhat, ": its gradient has no gradient (create_graph)");
    static const auto op = handle<decltype(::gradient)>("_vllm_mi355x::moe_route_grad");
    const torch::autograd::variable_list saved = ctx->get_saved_variables();
    const at::Tensor upstream = grads[0].to(at::kFloat).contiguous();
    const at::AutoDispatchBelowADInplaceOrView below;
    none[0] = op.call(saved[0], saved[1], saved[2], upstream, ctx->saved_data["scoring"].toInt(), ctx->saved_data["renormalize"].toBool());
    return none;
  }
};

std::tuple<at::Tensor, at::Tensor> route_autograd(const at::Tensor& logits, const std::optional<at::Tensor>& bias, int64_t topk,
                                                  int64_t groups, int64_t topk_groups, int64_t scoring, bool renormalize, double scale,
                                                  const std::optional<at::Tensor>& padding) {
  TORCH_CHECK(!logits._fw_grad(/*level=*/0).defined(), kWhat, ": no forward-mode derivative");
  if (!c10::GradMode::is_enabled() || !logits.requires_grad()) {
    return route_below(logits, bias, topk, groups, topk_groups, scoring, renormalize, scale, padding);
  }
  const torch::autograd::variable_list out = RouteWeights::apply(logits, bias, topk, groups, topk_groups, scoring, renormalize, scale, padding);
  return {out[0], out[1]};
}

// Shapes alone, for tracing.
std::tuple<at::Tensor, at::Tensor> route_meta(const at::Tensor& logits, const std::optional<at::Tensor>& bias, int64_t topk, int64_t groups,
                                              int64_t topk_groups, int64_t scoring, bool, double scale,
                                              const std::optional<at::Tensor>& padding) {
  check_call(logits, bias, topk, groups, topk_groups, scoring, scale, padding);
  const c10::SymInt rows = logits.sym_size(0);
  return {at::empty_symint({rows, topk}, logits.options().dtype(at::kFloat)), at::empty_symint({rows, topk}, logits.options().dtype(at::kInt))};
}
at::Tensor gradient_meta(const at::Tensor& logits, const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t, bool) {
  return at::empty_symint(logits.sym_sizes(), logits.options());
}

template <typename F>
bool find(void* library, const char* name, F& f) {
  f = reinterpret_cast<F>(dlsym(library, name));
  return f != nullptr;
}

}  // namespace

bool vq_torch::bind_route(void* library) {
  return find(library, "moe_route_logits", native_route) && find(library, "moe_route_grad", native_grad);
}

TORCH_LIBRARY_FRAGMENT(_vllm_mi355x, m) {
  m.def(
      "moe_route_logits(Tensor logits, Tensor? bias, int topk, int num_groups, int topk_groups, int scoring, bool renormalize, "
      "float scale, Tensor? is_padding) -> (Tensor, Tensor)");
  m.def(
      "moe_route_grad(Tensor logits, Tensor topk_weights, Tensor topk_ids, Tensor upstream, int scoring, bool renormalize) "
      "-> Tensor");
}
TORCH_LIBRARY_IMPL(_vllm_mi355x, CUDA, m) {
  m.impl("moe_route_logits", &route);
  m.impl("moe_route_grad", &gradient);
}
TORCH_LIBRARY_IMPL(_vllm_mi355x, Meta, m) {
  m.impl("moe_route_logits", &route_meta);
  m.impl("moe_route_grad", &gradient_meta);
}
TORCH_LIBRARY_IMPL(_vllm_mi355x, Autograd, m) { m.impl("moe_route_logits", &route_autograd); }
