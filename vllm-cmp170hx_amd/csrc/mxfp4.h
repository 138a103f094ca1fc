// The MXFP4 format on gfx950, and the quantization that the MXFP4 kernels share.
//
// A block is 32 consecutive elements of a row: 32 E2M1 codes (0, 0.5, 1, 1.5,
// 2, 3, 4, 6 and their negatives; two a byte, the even element in the low
// nibble, so 16 bytes) under one E8M0 scale byte b, the power of two 2^(b -
// 127).  Rows of k elements are k / 2 code bytes and k / 32 scale bytes.
//
// Quantization of a block with the largest magnitude m: b = max(0,
// exponent(m) - 2) with exponent() the biased FP32 exponent, so that m * 2^(127
// - b) lies in [4, 8) (below it where b is 0); each element's code is the
// nearest of the grid to x * 2^(127 - b), ties to the even code, 6 for what
// lies above 6; the sign is kept, of zeros too.  A block that holds a NaN or an
// infinity becomes b = 255 (the format's NaN) over zero codes, so that products
// with it are NaN.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

namespace mx {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));

constexpr int kBlock = 32;       // elements under one scale
constexpr int kBlockBytes = 16;  // their codes

inline bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// The scale byte of a block whose largest magnitude has the FP32 bits `top`
// (sign clear; NaNs are the largest patterns).
__device__ __forceinline__ uint32_t block_scale(uint32_t top) {
  const int e = int(top >> 23);
  return top >= 0x7f800000u ? 255u : uint32_t(max(e - 2, 0));
}

// Eight codes of v under the scale byte b (not 255): v_cvt_scalef32_pk_fp4_f32
// divides by the power of two whose exponent field b is (2^-127 for 0), rounds
// to nearest even, saturates at 6 and keeps the sign.
__device__ __forceinline__ uint32_t codes8(const float* v, uint32_t b) {
  const float scale = __builtin_bit_cast(float, b << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
  return w;
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// Eight consecutive elements as they lie in memory.
template <int kDtype>
struct Eight {
  static constexpr int kWords = kDtype == vq::kFP32 ? 8 : 4;
  uint32_t w[kWords];
};

// Elements i .. i + 7 of p; `wide`: their address is 16-byte aligned.
template <int kDtype>
__device__ __forceinline__ Eight<kDtype> load8(const void* p, int64_t i, bool wide) {
  constexpr int kWords = Eight<kDtype>::kWords;
  Eight<kDtype> v;
  if (wide) {
    const u32x4_t* q = reinterpret_cast<const u32x4_t*>(static_cast<const uint8_t*>(p) + i * (kWords / 2));
#pragma unroll
    for (int k = 0; k < kWords / 4; ++k) {
      const u32x4_t a = q[k];
#pragma unroll
      for (int j = 0; j < 4; ++j) v.w[4 * k + j] = a[j];
    }
  } else if constexpr (kDtype == vq::kFP32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v.w[j] = static_cast<const uint32_t*>(p)[i + j];
  } else {
    const uint16_t* h = static_cast<const uint16_t*>(p) + i;
#pragma unroll
    for (int j = 0; j < 4; ++j) v.w[j] = uint32_t(h[2 * j]) | (uint32_t(h[2 * j + 1]) << 16);
  }
  return v;
}

// The FP32 bits of the largest magnitude of eight elements.  (16-bit magnitudes
// order as whole numbers do, two at a time.)
template <int kDtype>
__device__ __forceinline__ uint32_t top8(const Eight<kDtype>& v) {
  if constexpr (kDtype == vq::kFP32) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, v.w[j] & 0x7fffffffu);
    return top;
  } else {
    typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
    u16x2_t m = __builtin_bit_cast(u16x2_t, v.w[0] & 0x7fff7fffu);
#pragma unroll
    for (int j = 1; j < 4; ++j) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, v.w[j] & 0x7fff7fffu));
    const uint16_t top = m[0] > m[1] ? m[0] : m[1];
    return kDtype == vq::kBF16 ? uint32_t(top) << 16 : __builtin_bit_cast(uint32_t, vq::f16_to_f32(top));
  }
}

// Their codes under the scale byte b, as codes8.
template <int kDtype>
__device__ __forceinline__ uint32_t codes_of(const Eight<kDtype>& v, uint32_t b) {
  const float scale = __builtin_bit_cast(float, b << 23);
  uint32_t w = 0;
  if constexpr (kDtype == vq::kFP32) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = __builtin_bit_cast(float, v.w[j]);
    w = codes8(f, b);
  } else if constexpr (kDtype == vq::kBF16) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    const auto pair = [&](int j) { return __builtin_bit_cast(bf16x2_t, v.w[j]); };
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, pair(0), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, pair(1), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, pair(2), scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, pair(3), scale, 3);
  } else {
    typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
    const auto pair = [&](int j) { return __builtin_bit_cast(half2_t, v.w[j]); };
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, pair(0), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, pair(1), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, pair(2), scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, pair(3), scale, 3);
  }
  return w;
}

// A quarter of a block held by lane j of a quad (elements 8 j .. 8 j + 7): its
// four code bytes, and the block's scale byte in every lane of the quad.
template <int kDtype>
__device__ __forceinline__ uint32_t quantize_quarter(const Eight<kDtype>& v, uint32_t& scale) {
  uint32_t top = top8(v);
  top = max(top, uint32_t(__builtin_amdgcn_mov_dpp(int(top), 0xB1, 0xF, 0xF, false)));
  top = max(top, uint32_t(__builtin_amdgcn_mov_dpp(int(top), 0x4E, 0xF, 0xF, false)));
  scale = block_scale(top);
  const uint32_t w = codes_of(v, scale);
  return scale == 255u ? 0u : w;
}

// The FP32 value of the low nibble of c: the doubled magnitudes, a nibble each.
__device__ __forceinline__ float code_value(uint32_t c) {
  const float v = float((0xC8643210u >> (4 * (c & 7))) & 15u) * 0.5f;
  return (c & 8) ? -v : v;
}

// 2^(b - 127) (NaN for 255).
__device__ __forceinline__ float scale_value(uint32_t b) {
  return b == 255u ? __builtin_nanf("") : b == 0 ? __builtin_bit_cast(float, 0x00400000u) : __builtin_bit_cast(float, b << 23);
}

}  // namespace mx
