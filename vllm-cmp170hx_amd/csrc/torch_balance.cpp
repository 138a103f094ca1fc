// The router's load operators (kernels/moe/balance.py), in host-only C++: the
// expert counts, and the balance loss with its gradient as an autograd node.
// The node and the call without gradients reach the kernels through operators of
// their own (moe_balance_forward, moe_balance_grad), below autograd: tracers, fake
// tensors and dispatch modes see these as any other operator.
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/Tensor.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "../../include/vllm_mi355x.h"
#include "torch_common.h"

namespace {

using vq_torch::check_status;
using vq_torch::dtype_code;
using vq_torch::stream_of;

decltype(&moe_expert_counts) native_counts = nullptr;
decltype(&moe_balance_loss) native_loss = nullptr;
decltype(&moe_balance_grad) native_grad = nullptr;
decltype(&moe_balance_workspace_size) native_workspace = nullptr;
decltype(&vllm_mi355x_last_error) native_error = nullptr;

at::Tensor scratch(int64_t rows, int64_t experts, const at::Tensor& on) {
  const int64_t bytes = native_workspace(rows, experts);
  if (bytes < 0) TORCH_CHECK(false, native_error());
  return at::empty({bytes}, on.options().dtype(at::kByte));
}

void check_padding(const std::optional<at::Tensor>& padding, int64_t rows, const at::Tensor& on, const char* what) {
  TORCH_CHECK(!padding || (padding->device() == on.device() && (padding->scalar_type() == at::kBool || padding->scalar_type() == at::kByte) &&
                           padding->dim() == 1 && padding->size(0) == rows && padding->is_contiguous()),
              what, ": is_padding must be a contiguous bool or uint8 [rows] on the same GPU");
}

void check_routing(const at::Tensor& ids, const std::optional<at::Tensor>& padding, const at::Tensor& on, const char* what) {
  TORCH_CHECK(ids.is_cuda() && ids.device() == on.device(), what, ": topk_ids must be on the logits' GPU");
  TORCH_CHECK(ids.scalar_type() == at::kInt && ids.dim() == 2 && ids.is_contiguous() && ids.size(1) > 0, what,
              ": topk_ids must be a contiguous int32 [rows, topk]");
  check_padding(padding, ids.size(0), on, what);
}

void check_logits(const at::Tensor& logits, const char* what) {
  TORCH_CHECK(logits.is_cuda(), what, ": logits must be on a GPU");
  TORCH_CHECK(logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kHalf || logits.scalar_type() == at::kFloat, what,
              ": logits must be BF16, FP16 or FP32");
  TORCH_CHECK(logits.dim() == 2 && logits.size(1) > 0 && (logits.numel() == 0 || logits.size(1) == 1 || logits.stride(1) == 1), what,
              ": logits must be [rows, experts] with unit inner stride");
}

const uint8_t* bytes_of(const std::optional<at::Tensor>& t) { return t ? static_cast<const uint8_t*>(t->const_data_ptr()) : nullptr; }

void expert_counts(const at::Tensor& ids, const std::optional<at::Tensor>& padding, const at::Tensor& out, bool add) {
  constexpr const char* what = "moe_expert_counts";
  TORCH_CHECK(ids.is_cuda(), what, ": topk_ids must be on a GPU");
  check_routing(ids, padding, ids, what);
  TORCH_CHECK(out.device() == ids.device() && out.scalar_type() == at::kLong && out.dim() == 1 && out.is_contiguous(), what,
              ": out must be a contiguous int64 [num_experts] on the ids' GPU");
  const c10::DeviceGuard guard(ids.device());
  at::Tensor ws = scratch(ids.size(0), out.size(0), ids);
  check_status(native_counts(static_cast<const int32_t*>(ids.const_data_ptr()), bytes_of(padding), ids.size(0), ids.size(1),
                             out.size(0), add, static_cast<int64_t*>(out.mutable_data_ptr()), ws.mutable_data_ptr(), ws.numel(),
                             stream_of(ids)));
}

// (loss, counts, stats): stats is what the gradient needs beside the logits.
std::tuple<at::Tensor, at::Tensor, at::Tensor> forward(const at::Tensor& logits, const at::Tensor& ids,
                                                       const std::optional<at::Tensor>& padding, int64_t scoring) {
  constexpr const char* what = "moe_balance_loss";
  check_logits(logits, what);
  check_routing(ids, padding, logits, what);
  const int64_t rows = logits.size(0), experts = logits.size(1);
  TORCH_CHECK(ids.size(0) == rows, what, ": topk_ids must have a row for each row of the logits");
  const c10::DeviceGuard guard(logits.device());
  at::Tensor ws = scratch(rows, experts, logits);
  at::Tensor loss = at::empty({}, logits.options().dtype(at::kFloat));
  at::Tensor counts = at::empty({experts}, logits.options().dtype(at::kLong));
  at::Tensor stats = at::empty({experts + 1}, logits.options().dtype(at::kFloat));
  check_status(native_loss(logits.const_data_ptr(), dtype_code(logits.scalar_type()), rows, experts, rows > 1 ? logits.stride(0) : experts,
                           static_cast<const int32_t*>(ids.const_data_ptr()), ids.size(1), bytes_of(padding), int(scoring),
                           static_cast<float*>(loss.mutable_data_ptr()), static_cast<int64_t*>(counts.mutable_data_ptr()),
                           static_cast<float*>(stats.mutable_data_ptr()), ws.mutable_data_ptr(), ws.numel(), stream_of(logits)));
  return {loss, counts, stats};
}

// The loss's gradient in the logits from upstream, one FP32 value on their GPU.
at::Tensor gradient(const at::Tensor& logits, const std::optional<at::Tensor>& padding, const at::Tensor& stats,
                    const at::Tensor& upstream, int64_t scoring) {
  constexpr const char* what = "moe_balance_grad";
  check_logits(logits, what);
  check_padding(padding, logits.size(0), logits, what);
  TORCH_CHECK(stats.dim() == 1 && stats.size(0) == logits.size(1) + 1 && stats.is_contiguous() &&
                  stats.scalar_type() == at::kFloat && stats.device() == logits.device(),
              what, ": stats must be the forward's");
  TORCH_CHECK(upstream.scalar_type() == at::kFloat && upstream.numel() == 1 && upstream.device() == logits.device(), what,
              ": upstream must be one FP32 value on the logits' GPU");
  const int64_t rows = logits.size(0), experts = logits.size(1);
  const c10::DeviceGuard guard(logits.device());
  at::Tensor grad = at::empty({rows, experts}, logits.options());
  check_status(native_grad(logits.const_data_ptr(), dtype_code(logits.scalar_type()), rows, experts, rows > 1 ? logits.stride(0) : experts,
                           bytes_of(padding), int(scoring), static_cast<const float*>(stats.const_data_ptr()),
                           static_cast<const float*>(upstream.const_data_ptr()), grad.mutable_data_ptr(), stream_of(logits)));
  return grad;
}

std::tuple<at::Tensor, at::Tensor> loss_only(const at::Tensor& logits, const at::Tensor& ids, const std::optional<at::Tensor>& padding,
                                             int64_t scoring) {
  auto [loss, counts, stats] = forward(logits, ids, padding, scoring);
  return {loss, counts};
}

// The operators by their names in the dispatcher.
template <typename F>
c10::TypedOperatorHandle<F> handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

struct BalanceLoss : torch::autograd::Function<BalanceLoss> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& ids,
                                                const std::optional<at::Tensor>& padding, int64_t scoring) {
    static const auto op = handle<decltype(::forward)>("_vllm_mi355x::moe_balance_forward");
    const at::AutoDispatchBelowADInplaceOrView below;
    auto [loss, counts, stats] = op.call(logits, ids, padding, scoring);
    ctx->save_for_backward({logits, stats, padding.value_or(at::Tensor())});
    ctx->saved_data["scoring"] = scoring;
    ctx->mark_non_differentiable({counts});
    return {loss, counts};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    TORCH_CHECK(!c10::GradMode::is_enabled(), "moe_balance_loss: its gradient has no gradient (create_graph)");
    static const auto op = handle<decltype(::gradient)>("_vllm_mi355x::moe_balance_grad");
    const torch::autograd::variable_list saved = ctx->get_saved_variables();
    const at::Tensor &logits = saved[0], &stats = saved[1], &padding = saved[2];
    // (one FP32 value on the device, as a rule)
    const at::Tensor& given = grads[0];
    const at::Tensor upstream = given.scalar_type() == at::kFloat && given.device() == logits.device()
                                    ? given : given.to(logits.device(), at::kFloat);
    const at::AutoDispatchBelowADInplaceOrView below;
    return {op.call(logits, padding.defined() ? std::optional<at::Tensor>(padding) : std::nullopt, stats, upstream,
                    ctx->saved_data["scoring"].toInt()),
            at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

std::tuple<at::Tensor, at::Tensor> loss_autograd(const at::Tensor& logits, const at::Tensor& ids, const std::optional<at::Tensor>& padding,
                                                 int64_t scoring) {
  TORCH_CHECK(!logits._fw_grad(/*level=*/0).defined(), "moe_balance_loss: no forward-mode derivative");
  if (!c10::GradMode::is_enabled() || !logits.requires_grad()) {
    static const auto op = handle<decltype(loss_only)>("_vllm_mi355x::moe_balance_loss");
    const at::AutoDispatchBelowADInplaceOrView below;
    return op.call(logits, ids, padding, scoring);
  }
  const torch::autograd::variable_list out = BalanceLoss::apply(logits, ids, padding, scoring);
  return {out[0], out[1]};
}

// Shapes alone, for tracing.
std::tuple<at::Tensor, at::Tensor, at::Tensor> forward_meta(const at::Tensor& logits, const at::Tensor& ids,
                                                            const std::optional<at::Tensor>&, int64_t) {
  TORCH_CHECK(logits.dim() == 2 && ids.dim() == 2, "moe_balance_loss: logits must be [rows, experts], topk_ids [rows, topk]");
  const c10::SymInt experts = logits.sym_size(1);
  return {at::empty({}, logits.options().dtype(at::kFloat)), at::empty_symint({experts}, logits.options().dtype(at::kLong)),
          at::empty_symint({experts + 1}, logits.options().dtype(at::kFloat))};
}
std::tuple<at::Tensor, at::Tensor> loss_meta(const at::Tensor& logits, const at::Tensor& ids, const std::optional<at::Tensor>& padding,
                                             int64_t scoring) {
  auto [loss, counts, stats] = forward_meta(logits, ids, padding, scoring);
  return {loss, counts};
}
at::Tensor gradient_meta(const at::Tensor& logits, const std::optional<at::Tensor>&, const at::Tensor&, const at::Tensor&, int64_t) {
  return at::empty_symint(logits.sym_sizes(), logits.options());
}

template <typename F>
bool find(void* library, const char* name, F& f) {
  f = reinterpret_cast<F>(dlsym(library, name));
  return f != nullptr;
}

}  // namespace

bool vq_torch::bind_balance(void* library) {
  return find(library, "moe_expert_counts", native_counts) && find(library, "moe_balance_loss", native_loss) &&
         find(library, "moe_balance_grad", native_grad) && find(library, "moe_balance_workspace_size", native_workspace) &&
         find(library, "vllm_mi355x_last_error", native_error);
}

TORCH_LIBRARY_FRAGMENT(_vllm_mi355x, m) {
  m.def("moe_expert_counts(Tensor topk_ids, Tensor? is_padding, Tensor(a!) out, bool add) -> ()");
  m.def("moe_balance_loss(Tensor logits, Tensor topk_ids, Tensor? is_padding, int scoring) -> (Tensor, Tensor)");
  m.def("moe_balance_forward(Tensor logits, Tensor topk_ids, Tensor? is_padding, int scoring) -> (Tensor, Tensor, Tensor)");
  m.def("moe_balance_grad(Tensor logits, Tensor? is_padding, Tensor stats, Tensor upstream, int scoring) -> Tensor");
}
TORCH_LIBRARY_IMPL(_vllm_mi355x, CUDA, m) {
  m.impl("moe_expert_counts", &expert_counts);
  m.impl("moe_balance_loss", &loss_only);
  m.impl("moe_balance_forward", &forward);
  m.impl("moe_balance_grad", &gradient);
}
TORCH_LIBRARY_IMPL(_vllm_mi355x, Meta, m) {
  m.impl("moe_balance_loss", &loss_meta);
  m.impl("moe_balance_forward", &forward_meta);
  m.impl("moe_balance_grad", &gradient_meta);
}
TORCH_LIBRARY_IMPL(_vllm_mi355x, Autograd, m) {
  m.impl("moe_expert_counts", torch::CppFunction::makeFallthrough());
  m.impl("moe_balance_loss", &loss_autograd);
}
