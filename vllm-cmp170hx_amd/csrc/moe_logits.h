// Rows of a router's logits in the lanes of wavefronts: what the balance loss and
// the routing from logits share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

namespace logits {

// How experts lie in lanes: kLanes lanes a row (64 / kLanes rows a wavefront), four
// consecutive experts a lane and step, kSteps steps.
template <int kLanes_, int kSteps_>
struct Shape {
  static constexpr int kLanes = kLanes_, kSteps = kSteps_, kRows = 64 / kLanes_;
};

template <int kLanes>
__device__ __forceinline__ float lanes_sum(float v, int lane) {
  if constexpr (kLanes > 32) v += vq::xor_lanes<32>(v, lane);
  if constexpr (kLanes > 16) v += vq::xor_lanes<16>(v, lane);
  v += vq::xor_lanes<8>(v, lane);
  v += vq::xor_lanes<4>(v, lane);
  v += vq::xor_lanes<2>(v, lane);
  v += vq::xor_lanes<1>(v, lane);
  return v;
}
template <int kLanes>
__device__ __forceinline__ float lanes_max(float v, int lane) {
  if constexpr (kLanes > 32) v = fmaxf(v, vq::xor_lanes<32>(v, lane));
  if constexpr (kLanes > 16) v = fmaxf(v, vq::xor_lanes<16>(v, lane));
  v = fmaxf(v, vq::xor_lanes<8>(v, lane));
  v = fmaxf(v, vq::xor_lanes<4>(v, lane));
  v = fmaxf(v, vq::xor_lanes<2>(v, lane));
  v = fmaxf(v, vq::xor_lanes<1>(v, lane));
  return v;
}

constexpr float kLog2e = 1.44269504f;

// Sigmoids of logits below it are below 2^-1022, the smallest that 64 bits hold in full.
constexpr float kNothing = -708.396f;

// e^x / 2^k for x <= 0 and a whole k, 0 or at least x log2(e): 2^(y - k) of y = x
// log2(e) as rounded (its difference to k is exact), corrected by what the rounding
// took.  Off by 2^-22 of it whatever x (by y alone |x| 2^-24); 0 where it is below
// 2^-126.
__device__ __forceinline__ float exp_nonpositive(float x, float k = 0) {
#pragma clang fp contract(off)  // (y - k is of the rounded y)
  constexpr float kLow = 1.925963033e-8f, kLn2 = 0.693147181f;
  const float y = x * kLog2e;
  float low = __builtin_fmaf(x, kLow, __builtin_fmaf(x, kLog2e, -y));
  low = x > -2048.0f ? low : 0.0f;  // (infinities have no difference)
  const float p = __builtin_amdgcn_exp2f(y - k);
  return __builtin_fmaf(p, low * kLn2, p);
}

// a b rounded by itself, whatever is added to it (r: the same in loss and gradient).
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

struct Rows {
  const void* logits;
  int64_t stride;
  const uint8_t* padding;
  int64_t rows;
  int experts;
  bool wide;  // four experts at a time: whole fours, rows on whole fours
};

template <typename S>
struct Values {
  float v[S::kSteps][4];
};

// Row t's logits (experts past the last are -inf).
template <typename S, int kDtype>
__device__ __forceinline__ Values<S> load_row(const Rows& g, int64_t t, int l) {
  Values<S> o;
#pragma unroll
  for (int i = 0; i < S::kSteps; ++i) {
    const int e = 4 * (S::kLanes * i + l);
    if (g.wide && e < g.experts) {
      const int64_t at = t * g.stride + e;
      if constexpr (kDtype == vq::kFP32) {
        typedef float f4_t __attribute__((ext_vector_type(4)));
        const f4_t w = *reinterpret_cast<const f4_t*>(static_cast<const float*>(g.logits) + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) o.v[i][j] = w[j];
      } else {
        typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
        const u2_t w = *reinterpret_cast<const u2_t*>(static_cast<const uint16_t*>(g.logits) + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint16_t u = uint16_t(w[j >> 1] >> (16 * (j & 1)));
          o.v[i][j] = kDtype == vq::kBF16 ? vq::bf16_to_f32(u) : vq::f16_to_f32(u);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o.v[i][j] = e + j < g.experts ? vq::load_act(g.logits, kDtype, t * g.stride + e + j) : -__builtin_inff();
      }
    }
  }
  return o;
}

template <typename S>
__device__ __forceinline__ float row_max(const Values<S>& x, int lane) {
  float m = x.v[0][0];
#pragma unroll
  for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) m = fmaxf(m, x.v[i][j]);
  return lanes_max<S::kLanes>(m, lane);
}

}  // namespace logits
