// What the operators' host files share: dtype codes, the current stream, and the
// library's error text (torch_ops.cpp defines them).
#pragma once

#include <ATen/core/Tensor.h>

#include <cstdint>

namespace vq_torch {

int dtype_code(at::ScalarType t);
void* stream_of(const at::Tensor& x);
// Throws the library's last error for a nonzero status.
void check_status(int status);

// The entry points that each host file takes from the loaded library (its
// dlopen handle); false when one is missing.
bool bind_mxfp4(void* library);
bool bind_balance(void* library);
bool bind_route(void* library);
bool bind_dense(void* library);

}  // namespace vq_torch
