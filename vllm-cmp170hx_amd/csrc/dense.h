// The dense linear layer: what its kernels share.
//
//   y = act(x W^T + b) + residual
//
// x [rows][k] and W [lines][k] are BF16 or FP16 (one type), sums and all that follows
// FP32, rounded once to y's type.  A gated activation has lines = 2 n (n gate rows,
// then n up rows), else lines = n.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

namespace dense {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

enum Activation : int { kNone = 0, kRelu = 1, kGelu = 2, kGeluTanh = 3, kSilu = 4, kSwiglu = 5 };

constexpr int kChunk = 8;  // elements of 16 bytes

// Rows of k 16-bit elements that lie together.
struct Operand {
  const uint16_t* p;
  int64_t rows, stride;
};

struct Epilogue {
  const void* bias;  // [lines] or null
  int bias_dtype;
  int activation;
  float limit;  // of a gated activation, infinity: none
  const void* residual;  // [rows][n], stride residual_stride, or null
  int residual_dtype;
  int64_t residual_stride;
  void* out;  // [rows][n]
  int out_dtype;
  int64_t n;
  // x W^T + b for the gradient, [rows][lines], or null.  (In 16 bits its rounding would add as
  // much to gradients as that of dz: of 4096 rows through 4096 x 28672 gated, in BF16, 1.7
  // times the result's own rounding for 1.4.)
  float* z;
  const uint32_t* top;  // the sums are over scale_of(*top), or null
};

inline bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Two values rounded to nearest even, the first one in the low half.
__device__ __forceinline__ uint32_t pack16(int dtype, float a, float b) {
  if (dtype == vq::kBF16) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, bf16x2_t{__bf16(a), __bf16(b)});  // v_cvt_pk_bf16_f32
  }
  return uint32_t(__builtin_bit_cast(uint16_t, _Float16(a))) | (uint32_t(__builtin_bit_cast(uint16_t, _Float16(b))) << 16);
}

// Elements at .. at + kC - 1 of an array of dtype, of which the first `valid` exist, in
// loads and stores of 16 bytes whatever their alignment.
template <int kC>
__device__ __forceinline__ void load_columns(const void* p, int dtype, int64_t at, int64_t valid, float (&v)[kC]) {
  if (kC == 1 || valid < kC) {
#pragma unroll
    for (int q = 0; q < kC; ++q) v[q] = q < valid ? vq::load_act(p, dtype, at + q) : 0.0f;
  } else if (dtype == vq::kFP32) {
    __builtin_memcpy(v, static_cast<const float*>(p) + at, 4 * kC);
  } else {
    uint32_t w[(kC + 1) / 2];
    __builtin_memcpy(w, static_cast<const uint16_t*>(p) + at, 2 * kC);
#pragma unroll
    for (int q = 0; q < kC; ++q) {
      const uint16_t h = uint16_t(w[q / 2] >> (16 * (q & 1)));
      v[q] = dtype == vq::kBF16 ? vq::bf16_to_f32(h) : vq::f16_to_f32(h);
    }
  }
}
template <int kC>
__device__ __forceinline__ void store_columns(void* p, int dtype, int64_t at, int64_t valid, const float (&v)[kC]) {
  if (kC == 1 || valid < kC) {
#pragma unroll
    for (int q = 0; q < kC; ++q) {
      if (q < valid) vq::store_act(p, dtype, at + q, v[q]);
    }
  } else if (dtype == vq::kFP32) {
    __builtin_memcpy(static_cast<float*>(p) + at, v, 4 * kC);
  } else {
    uint32_t w[(kC + 1) / 2];
#pragma unroll
    for (int q = 0; q < kC / 2; ++q) w[q] = pack16(dtype, v[2 * q], v[2 * q + 1]);
    __builtin_memcpy(static_cast<uint16_t*>(p) + at, w, 2 * kC);
  }
}

// 1 / (1 + e^-v).
__device__ __forceinline__ float sigmoid(float v) { return 1 / (1 + __expf(-v)); }

constexpr float kTanhA = 0.797884561f, kTanhB = 0.044715f;  // sqrt(2 / pi)

__device__ __forceinline__ float relu(float z) { return z > 0 || z != z ? z : 0.0f; }
__device__ __forceinline__ float gelu(float z) { return 0.5f * z * erfcf(z * -0.707106781f); }
// (1 + tanh u) / 2 is the sigmoid of 2 u
__device__ __forceinline__ float gelu_tanh(float z) { return z * sigmoid(2 * kTanhA * (z + kTanhB * z * z * z)); }
__device__ __forceinline__ float silu(float z) { return z * sigmoid(z); }

// (a NaN passes gradients as it passes relu)
__device__ __forceinline__ float relu_slope(float z) { return z > 0 || z != z ? 1.0f : 0.0f; }
__device__ __forceinline__ float gelu_slope(float z) { return 0.5f * erfcf(z * -0.707106781f) + z * 0.398942280f * __expf(-0.5f * z * z); }
__device__ __forceinline__ float gelu_tanh_slope(float z) {
  const float s = sigmoid(2 * kTanhA * (z + kTanhB * z * z * z));
  return s + z * s * (1 - s) * 2 * kTanhA * (1 + 3 * kTanhB * z * z);
}
__device__ __forceinline__ float silu_slope(float z) {
  const float s = sigmoid(z);
  return s * (1 + z * (1 - s));
}

// min(v, limit) and clamp(v, -limit, limit); a NaN stays one.
__device__ __forceinline__ float clamp_above(float v, float limit) { return v > limit ? limit : v; }
__device__ __forceinline__ float clamp_both(float v, float limit) { return v > limit ? limit : (v < -limit ? -limit : v); }

// FP16 holds gradients over a power of two that brings the largest magnitude to 2^13 .. 2^14:
// those of a mean are often below what FP16 holds, and products with up lines may be above.
// top: the FP32 bits of that (finite) magnitude.
__device__ __forceinline__ float scale_of(uint32_t top) {
  const int e = int(top >> 23);
  if (e == 0) return 1.0f;  // nothing
  return __builtin_amdgcn_ldexpf(1.0f, min(13 - (e - 127), 126));
}

// What all rows have at columns c .. c + kC - 1.
template <int kC, bool kGated>
struct Columns {
  float bias[kC], up_bias[kC], factor;
  __device__ __forceinline__ Columns(const Epilogue& e, int64_t c) {
    factor = e.top ? 1 / scale_of(*e.top) : 1.0f;
#pragma unroll
    for (int q = 0; q < kC; ++q) bias[q] = up_bias[q] = 0;
    if (!e.bias || c >= e.n) return;
    load_columns<kC>(e.bias, e.bias_dtype, c, e.n - c, bias);
    if constexpr (kGated) load_columns<kC>(e.bias, e.bias_dtype, e.n + c, e.n - c, up_bias);
  }
};

// A row's residual there.
template <int kC>
__device__ __forceinline__ void load_residual(const Epilogue& e, int64_t row, int64_t c, float (&r)[kC]) {
  if (e.residual && c < e.n) load_columns<kC>(e.residual, e.residual_dtype, row * e.residual_stride + c, e.n - c, r);
}

// Columns c .. c + kC - 1 of a row from its sums (u: of a gated activation's up lines).
template <int kC, bool kGated>
__device__ __forceinline__ void finish_columns(const Epilogue& e, int64_t row, int64_t c, float (&v)[kC], float (&u)[kC],
                                               const Columns<kC, kGated>& columns, const float (&residual)[kC]) {
  const int64_t valid = e.n - c;
  if (valid <= 0) return;
#pragma unroll
  for (int q = 0; q < kC; ++q) v[q] = v[q] * columns.factor + columns.bias[q];
  if constexpr (kGated) {
#pragma unroll
    for (int q = 0; q < kC; ++q) u[q] += columns.up_bias[q];
    if (e.z) {
      store_columns<kC>(e.z, vq::kFP32, row * 2 * e.n + c, valid, v);
      store_columns<kC>(e.z, vq::kFP32, row * 2 * e.n + e.n + c, valid, u);
    }
#pragma unroll
    for (int q = 0; q < kC; ++q) {
      const float g = clamp_above(v[q], e.limit);
      v[q] = g * sigmoid(g) * clamp_both(u[q], e.limit);
    }
  } else {
    if (e.z) store_columns<kC>(e.z, vq::kFP32, row * e.n + c, valid, v);
    const auto each = [&](float (*f)(float)) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < kC; ++q) v[q] = f(v[q]);
    };
    switch (e.activation) {
      case kRelu: each(relu); break;
      case kGelu: each(gelu); break;
      case kGeluTanh: each(gelu_tanh); break;
      case kSilu: each(silu); break;
    }
  }
  if (e.residual) {
#pragma unroll
    for (int q = 0; q < kC; ++q) v[q] += residual[q];
  }
  store_columns<kC>(e.out, e.out_dtype, row * e.n + c, valid, v);
}
template <int kC, bool kGated>
__device__ __forceinline__ void finish_columns(const Epilogue& e, int64_t row, int64_t c, float (&v)[kC], float (&u)[kC]) {
  float r[kC];
  load_residual<kC>(e, row, c, r);
  finish_columns<kC, kGated>(e, row, c, v, u, Columns<kC, kGated>(e, c), r);
}

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));

// acc += A B, A and B of 32 (16) lines and 16 (32) k: a lane holds eight k of line lane &
// 31 (15); its sums are of B's line lane & 31 (15).
template <bool kBf16>
__device__ __forceinline__ void mfma32(f32x16_t& acc, const u32x4_t& a, const u32x4_t& b) {
  if constexpr (kBf16) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), acc, 0, 0, 0);
  } else {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), acc, 0, 0, 0);
  }
}
template <bool kBf16>
__device__ __forceinline__ void mfma16(f32x4_t& acc, const u32x4_t& a, const u32x4_t& b) {
  if constexpr (kBf16) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), acc, 0, 0, 0);
  } else {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), acc, 0, 0, 0);
  }
}

}  // namespace dense
