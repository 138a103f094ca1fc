// The MXFP4 operators (kernels/mxfp4/ops.py), in host-only C++: tensor checks,
// outputs and scratch from torch's allocator (so of the current stream, and of a
// graph's pool under capture), and the C-ABI call on torch's current stream.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <dlfcn.h>
#include <torch/library.h>

#include <cmath>
#include <limits>
#include <optional>
#include <tuple>
#include <vector>

#include "../../include/vllm_mi355x.h"
#include "torch_common.h"

namespace {

using vq_torch::check_status;
using vq_torch::dtype_code;
using vq_torch::stream_of;

decltype(&mxfp4_quantize) native_quantize = nullptr;
decltype(&mxfp4_dequantize) native_dequantize = nullptr;
decltype(&mxfp4_matmul) native_matmul = nullptr;
decltype(&mxfp4_matmul_workspace_size) native_matmul_workspace = nullptr;
decltype(&mxfp4_linear) native_linear = nullptr;
decltype(&mxfp4_linear_workspace_size) native_linear_workspace = nullptr;
decltype(&mxfp4_moe) native_moe = nullptr;
decltype(&mxfp4_moe_workspace_size) native_moe_workspace = nullptr;
decltype(&vllm_mi355x_last_error) native_error = nullptr;

constexpr int64_t kBlock = 32;

bool is_float(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat; }

std::vector<int64_t> with_last(const at::Tensor& t, int64_t last) {
  std::vector<int64_t> sizes = t.sizes().vec();
  sizes.back() = last;
  return sizes;
}

// x as rows of its last axis at one row stride.
struct Rows {
  int64_t rows, k, stride;
};

Rows rows_of(const at::Tensor& x, const char* what) {
  TORCH_CHECK(x.dim() >= 1, what, ": x needs at least one axis");
  const int64_t k = x.size(-1);
  TORCH_CHECK(k > 0 && k % kBlock == 0, what, ": the last axis must be a positive multiple of 32, got ", k);
  const int64_t rows = x.numel() / k;
  if (rows == 0) return {0, k, k};
  TORCH_CHECK(x.stride(-1) == 1, what, ": x needs unit stride along its last axis");
  int64_t stride = k, count = 1;
  bool first = true;
  for (int64_t d = x.dim() - 2; d >= 0; --d) {
    if (x.size(d) == 1) continue;
    if (first) stride = x.stride(d);
    else TORCH_CHECK(x.stride(d) == stride * count, what, ": the leading axes of x must be one run of rows (a view as [-1, k])");
    first = false;
    count *= x.size(d);
  }
  TORCH_CHECK(rows == 1 || stride >= k, what, ": rows of x must not overlap");
  return {rows, k, stride};
}

void check_float(const at::Tensor& x, const char* what) {
  TORCH_CHECK(x.is_cuda(), what, ": x must be on a GPU");
  TORCH_CHECK(is_float(x.scalar_type()), what, ": x must be BF16, FP16 or FP32");
}

// codes [..., k / 2] and scales [..., k / 32], contiguous bytes on `on`'s device.
void check_packed(const at::Tensor& codes, const at::Tensor& scales, const at::Tensor& on, const char* what) {
  TORCH_CHECK(codes.is_cuda() && codes.device() == on.device() && scales.device() == on.device(), what,
              ": codes and scales must be on the input's GPU");
  TORCH_CHECK(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte, what, ": codes and scales must be uint8");
  TORCH_CHECK(codes.is_contiguous() && scales.is_contiguous(), what, ": codes and scales must be contiguous");
  TORCH_CHECK(codes.dim() >= 1 && codes.dim() == scales.dim() && codes.size(-1) > 0 && codes.size(-1) == 16 * scales.size(-1) &&
                  codes.sizes().slice(0, codes.dim() - 1) == scales.sizes().slice(0, codes.dim() - 1),
              what, ": codes [..., k / 2] and scales [..., k / 32] do not fit each other");
}

at::Tensor scratch(int64_t bytes, const at::Tensor& on) {
  if (bytes < 0) TORCH_CHECK(false, native_error());
  return at::empty({bytes}, on.options().dtype(at::kByte));
}

std::tuple<at::Tensor, at::Tensor> quantize(const at::Tensor& x) {
  check_float(x, "mxfp4_quantize");
  const Rows r = rows_of(x, "mxfp4_quantize");
  const c10::DeviceGuard guard(x.device());
  at::Tensor codes = at::empty(with_last(x, r.k / 2), x.options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous));
  at::Tensor scales = at::empty(with_last(x, r.k / kBlock), x.options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous));
  check_status(native_quantize(x.const_data_ptr(), dtype_code(x.scalar_type()), r.rows, r.k, r.stride,
                               codes.mutable_data_ptr<uint8_t>(), scales.mutable_data_ptr<uint8_t>(), stream_of(x)));
  return {codes, scales};
}

at::Tensor dequantize(const at::Tensor& codes, const at::Tensor& scales, at::ScalarType out_dtype) {
  TORCH_CHECK(is_float(out_dtype), "mxfp4_dequantize: out_dtype must be BF16, FP16 or FP32");
  check_packed(codes, scales, codes, "mxfp4_dequantize");
  const int64_t k = codes.size(-1) * 2;
  const c10::DeviceGuard guard(codes.device());
  at::Tensor out = at::empty(with_last(codes, k), codes.options().dtype(out_dtype));
  check_status(native_dequantize(codes.const_data_ptr<uint8_t>(), scales.const_data_ptr<uint8_t>(), out.numel() / k, k,
                                 out.mutable_data_ptr(), dtype_code(out_dtype), stream_of(codes)));
  return out;
}

void check_weight(const at::Tensor& w, const at::Tensor& w_scale, int64_t k, const at::Tensor& on, const char* what) {
  check_packed(w, w_scale, on, what);
  TORCH_CHECK(w.dim() == 2 && 2 * w.size(1) == k, what, ": the weights must be [n, k / 2] codes of the input's k = ", k);
}

at::Tensor matmul(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& w, const at::Tensor& w_scale,
                  at::ScalarType out_dtype) {
  TORCH_CHECK(is_float(out_dtype), "mxfp4_matmul: out_dtype must be BF16, FP16 or FP32");
  check_packed(a, a_scale, a, "mxfp4_matmul");
  const int64_t k = 2 * a.size(-1), rows = a.numel() / a.size(-1);
  check_weight(w, w_scale, k, a, "mxfp4_matmul");
  const int64_t n = w.size(0);
  const c10::DeviceGuard guard(a.device());
  at::Tensor out = at::empty(with_last(a, n), a.options().dtype(out_dtype));
  at::Tensor ws = scratch(native_matmul_workspace(rows, k, n), a);
  check_status(native_matmul(a.const_data_ptr<uint8_t>(), a_scale.const_data_ptr<uint8_t>(), rows, k,
                             w.const_data_ptr<uint8_t>(), w_scale.const_data_ptr<uint8_t>(), n, out.mutable_data_ptr(),
                             dtype_code(out_dtype), ws.mutable_data_ptr(), ws.numel(), stream_of(a)));
  return out;
}

at::Tensor linear(const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_scale, std::optional<at::ScalarType> out_dtype) {
  check_float(x, "mxfp4_linear");
  const at::ScalarType type = out_dtype.value_or(x.scalar_type());
  TORCH_CHECK(is_float(type), "mxfp4_linear: out_dtype must be BF16, FP16 or FP32");
  const Rows r = rows_of(x, "mxfp4_linear");
  check_weight(w, w_scale, r.k, x, "mxfp4_linear");
  const int64_t n = w.size(0);
  const c10::DeviceGuard guard(x.device());
  at::Tensor out = at::empty(with_last(x, n), x.options().dtype(type).memory_format(at::MemoryFormat::Contiguous));
  at::Tensor ws = scratch(native_linear_workspace(r.rows, r.k, n), x);
  check_status(native_linear(x.const_data_ptr(), dtype_code(x.scalar_type()), r.rows, r.k, r.stride, w.const_data_ptr<uint8_t>(),
                             w_scale.const_data_ptr<uint8_t>(), n, out.mutable_data_ptr(), dtype_code(type),
                             ws.mutable_data_ptr(), ws.numel(), stream_of(x)));
  return out;
}

int64_t moe_workspace(const at::Tensor& x, const at::Tensor& w1, const at::Tensor& w2, const at::Tensor& topk_ids) {
  TORCH_CHECK(x.dim() == 2 && w1.dim() == 3 && w2.dim() == 3 && topk_ids.dim() == 2, "fused_mxfp4_moe: tensor ranks mismatch");
  const int64_t bytes = native_moe_workspace(x.size(0), topk_ids.size(1), x.size(1), 2 * w2.size(2), w1.size(0));
  if (bytes < 0) TORCH_CHECK(false, native_error());
  return bytes;
}

void moe(const at::Tensor& x, const at::Tensor& w1, const at::Tensor& w2, const at::Tensor& s1, const at::Tensor& s2,
         const at::Tensor& topk_w, const at::Tensor& topk_ids, const std::optional<at::Tensor>& expert_map, double limit,
         const at::Tensor& workspace, const at::Tensor& out) {
  constexpr const char* what = "fused_mxfp4_moe";
  const at::ScalarType type = x.scalar_type();
  TORCH_CHECK(x.is_cuda(), what, ": hidden_states must be on a GPU");
  TORCH_CHECK((type == at::kBFloat16 || type == at::kHalf) && x.dim() == 2 && (x.numel() == 0 || x.stride(1) == 1), what,
              ": hidden_states must be BF16 or FP16 [tokens, hidden], unit inner stride");
  check_packed(w1, s1, x, what);
  check_packed(w2, s2, x, what);
  const int64_t tokens = x.size(0), hidden = x.size(1);
  TORCH_CHECK(w1.dim() == 3 && w2.dim() == 3, what, ": weights must be [experts, rows, k / 2] codes");
  const int64_t experts = w1.size(0), inter = 2 * w2.size(2);
  TORCH_CHECK(2 * w1.size(2) == hidden && w1.size(1) == 2 * inter && w2.size(0) == experts && w2.size(1) == hidden, what,
              ": weights must be [E, 2 I, hidden / 2] and [E, hidden, I / 2] codes");
  TORCH_CHECK(topk_ids.dim() == 2 && topk_ids.size(0) == tokens && topk_w.sizes() == topk_ids.sizes(), what, ": routing shape mismatch");
  TORCH_CHECK(topk_ids.scalar_type() == at::kInt && topk_ids.is_contiguous() && topk_w.scalar_type() == at::kFloat &&
                  topk_w.is_contiguous(),
              what, ": routing must be contiguous, ids int32, weights FP32");
  TORCH_CHECK(out.scalar_type() == type && out.is_contiguous() && out.sizes() == x.sizes(), what,
              ": output must be a contiguous tensor like hidden_states");
  TORCH_CHECK(workspace.scalar_type() == at::kByte && workspace.is_contiguous(), what, ": the workspace must be contiguous bytes");
  for (const at::Tensor* t : {&topk_w, &topk_ids, &out, &workspace}) {
    TORCH_CHECK(t->is_cuda() && t->device() == x.device(), what, ": tensors must be on the activation device");
  }
  TORCH_CHECK(!expert_map || (expert_map->scalar_type() == at::kInt && expert_map->is_contiguous() && expert_map->dim() == 1 &&
                              expert_map->numel() > 0 && expert_map->is_cuda() && expert_map->device() == x.device()),
              what, ": expert_map must be a contiguous int32 vector on the activation device");
  const c10::DeviceGuard guard(x.device());
  check_status(native_moe(x.const_data_ptr(), dtype_code(type), tokens, tokens > 1 ? x.stride(0) : hidden,
                          w1.const_data_ptr<uint8_t>(), s1.const_data_ptr<uint8_t>(), w2.const_data_ptr<uint8_t>(),
                          s2.const_data_ptr<uint8_t>(), experts, topk_ids.const_data_ptr<int32_t>(),
                          topk_w.const_data_ptr<float>(), topk_ids.size(1),
                          expert_map ? expert_map->const_data_ptr<int32_t>() : nullptr, expert_map ? expert_map->numel() : 0, hidden,
                          inter, static_cast<float>(limit), out.mutable_data_ptr(), workspace.mutable_data_ptr(),
                          workspace.numel(), stream_of(x)));
}

// Shapes alone, for tracing.
std::tuple<at::Tensor, at::Tensor> quantize_meta(const at::Tensor& x) {
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) % kBlock == 0, "mxfp4_quantize: the last axis must be a positive multiple of 32");
  return {at::empty(with_last(x, x.size(-1) / 2), x.options().dtype(at::kByte)),
          at::empty(with_last(x, x.size(-1) / kBlock), x.options().dtype(at::kByte))};
}
at::Tensor dequantize_meta(const at::Tensor& codes, const at::Tensor& scales, at::ScalarType out_dtype) {
  (void)scales;
  return at::empty(with_last(codes, codes.size(-1) * 2), codes.options().dtype(out_dtype));
}
at::Tensor matmul_meta(const at::Tensor& a, const at::Tensor&, const at::Tensor& w, const at::Tensor&, at::ScalarType out_dtype) {
  return at::empty(with_last(a, w.size(0)), a.options().dtype(out_dtype));
}
at::Tensor linear_meta(const at::Tensor& x, const at::Tensor& w, const at::Tensor&, std::optional<at::ScalarType> out_dtype) {
  return at::empty(with_last(x, w.size(0)), x.options().dtype(out_dtype.value_or(x.scalar_type())));
}

template <typename F>
bool find(void* library, const char* name, F& f) {
  f = reinterpret_cast<F>(dlsym(library, name));
  return f != nullptr;
}

}  // namespace

bool vq_torch::bind_mxfp4(void* library) {
  return find(library, "mxfp4_quantize", native_quantize) && find(library, "mxfp4_dequantize", native_dequantize) &&
         find(library, "mxfp4_matmul", native_matmul) && find(library, "mxfp4_matmul_workspace_size", native_matmul_workspace) &&
         find(library, "mxfp4_linear", native_linear) && find(library, "mxfp4_linear_workspace_size", native_linear_workspace) &&
         find(library, "mxfp4_moe", native_moe) && find(library, "mxfp4_moe_workspace_size", native_moe_workspace) &&
         find(library, "vllm_mi355x_last_error", native_error);
}

TORCH_LIBRARY_FRAGMENT(_vllm_mi355x, m) {
  m.def("mxfp4_quantize(Tensor x) -> (Tensor, Tensor)");
  m.def("mxfp4_dequantize(Tensor codes, Tensor scales, ScalarType out_dtype) -> Tensor");
  m.def("mxfp4_matmul(Tensor a, Tensor a_scale, Tensor w, Tensor w_scale, ScalarType out_dtype) -> Tensor");
  m.def("mxfp4_linear(Tensor x, Tensor w, Tensor w_scale, ScalarType? out_dtype=None) -> Tensor");
  m.def("mxfp4_moe_workspace(Tensor x, Tensor w1, Tensor w2, Tensor topk_ids) -> int", &moe_workspace);
  m.def(
      "mxfp4_moe(Tensor x, Tensor w1, Tensor w2, Tensor s1, Tensor s2, Tensor topk_w, Tensor topk_ids, Tensor? expert_map, "
      "float limit, Tensor(a!) workspace, Tensor(b!) out) -> ()");
}

TORCH_LIBRARY_IMPL(_vllm_mi355x, CUDA, m) {
  m.impl("mxfp4_quantize", &quantize);
  m.impl("mxfp4_dequantize", &dequantize);
  m.impl("mxfp4_matmul", &matmul);
  m.impl("mxfp4_linear", &linear);
  m.impl("mxfp4_moe", &moe);
}
TORCH_LIBRARY_IMPL(_vllm_mi355x, Meta, m) {
  m.impl("mxfp4_quantize", &quantize_meta);
  m.impl("mxfp4_dequantize", &dequantize_meta);
  m.impl("mxfp4_matmul", &matmul_meta);
  m.impl("mxfp4_linear", &linear_meta);
}
// inference calls: inputs that require gradients are read as they are
TORCH_LIBRARY_IMPL(_vllm_mi355x, Autograd, m) {
  for (const char* name : {"mxfp4_quantize", "mxfp4_dequantize", "mxfp4_matmul", "mxfp4_linear", "mxfp4_moe"}) {
    m.impl(name, torch::CppFunction::makeFallthrough());
  }
}
