// The dense linear layer: few rows, many rows (dense_tile.h), the sum of K splits, and
// the gradient.
//
// With dy the gradient of y and z = x W^T + b,
//
//   dz = dy act'(z)   (gated: dg = dy clamp(u) silu'(g) where g <= L, du = dy silu(min(g, L))
//                      where |u| <= L)
//   dx = dz W,   dW = dz^T x,   db = sum over rows of dz,
//
// so two more products, whose sums run over the lines and over the rows.  Both run on
// the tiles of dense_tile.h, which want what is summed over to lie together: W and x
// are transposed into the workspace, dz is written both ways.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <initializer_list>

#include "../../include/vllm_mi355x.h"
#include "common.h"
#include "dense.h"
#include "dense_tile.h"

namespace dense {
namespace {

constexpr int64_t kMaxK = 1 << 21;  // 256 rows of a tile stay below 2^31 bytes
constexpr int64_t kMaxRows = 1 << 26, kMaxLines = 1 << 24;
constexpr int64_t kMaxGroups = 1 << 22;  // tiles, of up to 512 threads: below 2^32

// ---- eight rows at most -------------------------------------------------------------
//
// A wavefront takes kLines lines of W (a gated activation: a gate line and its up line), its
// lanes 512 k of each at a time, 16 bytes a lane and load: a line streams from memory
// as it lies.  x comes from the caches, its chunks held for all the wavefront's lines; products are
// v_dot2 with FP32 sums, a lane's own until the end.  Where lines are few, `parts` wavefronts
// of a workgroup share them, every parts-th 512 k each, and add up in LDS.  Bound by memory:
// one row of 4096 x 2 x 14336, gated, takes 41 us, 5.7 TB/s (a large copy: 5.1); on matrix
// instructions, whose 16 columns one row leaves empty, it took 54.

constexpr int kGemvRows = 8, kGemvWaves = 8, kGemvStep = 64 * kChunk;

template <bool kBf16>
__device__ __forceinline__ float dot8(const u32x4_t& a, const u32x4_t& b, float sum) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kBf16) {
      typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
      const uint32_t ai = a[i], bi = b[i];
      sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, ai), __builtin_bit_cast(bf16x2_t, bi), sum, false);
    } else {
      typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
      const uint32_t ai = a[i], bi = b[i];
      sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, ai), __builtin_bit_cast(half2_t, bi), sum, false);
    }
  }
  return sum;
}

template <bool kBf16>
__device__ __forceinline__ u32x4_t load_chunk(const uint16_t* row, int64_t b, int64_t k) {
  u32x4_t v{0, 0, 0, 0};
  if (kChunk * b + kChunk <= k) {
    __builtin_memcpy(&v, row + kChunk * b, 16);  // (of any alignment)
  } else if (kChunk * b < k) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      if (kChunk * b + i < k) w[i / 2] |= uint32_t(row[kChunk * b + i]) << (16 * (i & 1));
    }
    v = u32x4_t{w[0], w[1], w[2], w[3]};
  }
  return v;
}

__device__ __forceinline__ float wave_sum(float v, int lane) {
  v += vq::xor_lanes<32>(v, lane);
  v += vq::xor_lanes<16>(v, lane);
  v += vq::xor_lanes<8>(v, lane);
  v += vq::xor_lanes<4>(v, lane);
  v += vq::xor_lanes<2>(v, lane);
  return v + vq::xor_lanes<1>(v, lane);
}

template <int kRows, int kLines, bool kGated, bool kBf16>
__global__ __launch_bounds__(64 * kGemvWaves) void gemv_kernel(Operand x, Operand w, int64_t k, int parts, Epilogue e) {
  static_assert(!kGated || kLines == 2, "a gate and an up line");
  constexpr int kCols = kGated ? 1 : kLines;
  constexpr int kAhead = kRows * kLines > 8 ? 2 : 4;  // steps whose loads are on their way together
  __shared__ float sums[kGemvWaves][kLines][kRows];
  const int tid = threadIdx.x, lane = tid & 63, wave = vq::uniform(tid >> 6);
  const int part = wave % parts, set = wave / parts;
  const int64_t c = (int64_t(blockIdx.x) * (kGemvWaves / parts) + set) * kCols;
  const uint16_t* wrow[kLines];
#pragma unroll
  for (int l = 0; l < kLines; ++l) wrow[l] = w.p + (min(c + (kGated ? 0 : l), e.n - 1) + (kGated && l ? e.n : 0)) * w.stride;
  const uint16_t* xrow[kRows];
#pragma unroll
  for (int m = 0; m < kRows; ++m) xrow[m] = x.p + min(int64_t(m), x.rows - 1) * x.stride;
  float acc[kLines][kRows];
#pragma unroll
  for (int l = 0; l < kLines; ++l)
#pragma unroll
    for (int m = 0; m < kRows; ++m) acc[l][m] = 0;
  const int64_t chunks = (k + kChunk - 1) / kChunk;
  if (c < e.n) {
    for (int64_t b = 64 * part + lane; b < chunks; b += 64 * kAhead * parts) {
      u32x4_t a[kAhead][kLines], v[kAhead][kRows];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
#pragma unroll
        for (int l = 0; l < kLines; ++l) a[i][l] = load_chunk<kBf16>(wrow[l], b + 64 * i * parts, k);
#pragma unroll
        for (int m = 0; m < kRows; ++m) v[i][m] = load_chunk<kBf16>(xrow[m], b + 64 * i * parts, k);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int l = 0; l < kLines; ++l)
#pragma unroll
          for (int m = 0; m < kRows; ++m) acc[l][m] = dot8<kBf16>(a[i][l], v[i][m], acc[l][m]);
    }
  }
  // lane m keeps row m's
  float mine[kLines];
#pragma unroll
  for (int l = 0; l < kLines; ++l) {
    mine[l] = 0;
#pragma unroll
    for (int m = 0; m < kRows; ++m) {
      const float all = wave_sum(acc[l][m], lane);
      if (lane == m) mine[l] = all;
    }
  }
  if (parts > 1) {
    if (lane < kRows) {
#pragma unroll
      for (int l = 0; l < kLines; ++l) sums[wave][l][lane] = mine[l];
    }
    __syncthreads();
    if (part || lane >= kRows) return;
#pragma unroll
    for (int l = 0; l < kLines; ++l) {
      mine[l] = 0;
      for (int p = 0; p < parts; ++p) mine[l] += sums[wave + p][l][lane];
    }
  }
  if (lane >= kRows || lane >= x.rows || c >= e.n) return;
  float v[kCols], u[kCols];
#pragma unroll
  for (int q = 0; q < kCols; ++q) {
    v[q] = mine[q];
    u[q] = kGated ? mine[1] : 0.0f;
  }
  finish_columns<kCols, kGated>(e, lane, c, v, u);
}

// ---- 16 rows at most ------------------------------------------------------------------
//
// W is read once, from memory to the registers of the wavefront that multiplies it: a
// wavefront holds 16 lines (a gated activation: 16 gate and the 16 up lines of the same
// columns), per step 128 k, in which lane (r = lane & 15, q = lane >> 4) loads the
// chunks 4 j + q (j < 4) of line r and of x's row r and multiplies them in four
// v_mfma_16x16x32.  K is split over the wavefronts of a workgroup, whose sums meet in
// LDS and are added in order.  Bound by the loads' latency: 8 rows of 4096 x 4096 take 9.2 us
// (3.6 TB/s; tiles with K splits and their sum 12.3).  From 17 rows on tiles are the faster ones
// (20 rows of 2592 x 5003: 15 us for 20 with two of these products a lane).

constexpr int kSmallRows = 16;  // of one B operand
constexpr int kStepChunks = 16;

template <bool kGated, bool kBf16>
__global__ __launch_bounds__(1024) void small_kernel(Operand x, Operand w, int64_t k, Epilogue e) {
  constexpr int kOps = kGated ? 2 : 1;
  __shared__ __attribute__((aligned(16))) float sums[16][kOps][64 * 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = vq::uniform(tid >> 6), waves = int(blockDim.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int64_t c0 = int64_t(blockIdx.x) * 16;
  const int64_t line = min(c0 + r, e.n - 1);
  const uint16_t* wrow[kOps];
#pragma unroll
  for (int o = 0; o < kOps; ++o) wrow[o] = w.p + (line + o * e.n) * w.stride;
  const uint16_t* xrow = x.p + min(int64_t(r), x.rows - 1) * x.stride;
  f32x4_t acc[kOps];
#pragma unroll
  for (int o = 0; o < kOps; ++o) acc[o] = f32x4_t{0, 0, 0, 0};
  const int64_t steps = (k + kChunk * kStepChunks - 1) / (kChunk * kStepChunks);
  for (int64_t s = wave; s < steps; s += waves) {
    u32x4_t a[kOps][4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t at = s * kStepChunks + 4 * j + q;
#pragma unroll
      for (int o = 0; o < kOps; ++o) a[o][j] = load_chunk<kBf16>(wrow[o], at, k);
      b[j] = load_chunk<kBf16>(xrow, at, k);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int o = 0; o < kOps; ++o) mfma16<kBf16>(acc[o], a[o][j], b[j]);
  }
#pragma unroll
  for (int o = 0; o < kOps; ++o) *reinterpret_cast<f32x4_t*>(&sums[wave][o][4 * lane]) = acc[o];
  __syncthreads();
  if (wave) return;
  float v[4], u[4] = {0, 0, 0, 0};
#pragma unroll
  for (int o = 0; o < kOps; ++o) {
    f32x4_t all{0, 0, 0, 0};
    for (int from = 0; from < waves; ++from) all += *reinterpret_cast<const f32x4_t*>(&sums[from][o][4 * lane]);
#pragma unroll
    for (int i = 0; i < 4; ++i) (o ? u : v)[i] = all[i];
  }
  if (r < x.rows) finish_columns<4, kGated>(e, r, c0 + 4 * q, v, u);
}

// ---- the sum of K splits --------------------------------------------------------------

// Four columns a thread, the splits' sums of four splits on their way at a time: 6.4 us for 20
// rows of 5003 in six splits (the launch and two waits for memory), 7.5 for 400 of 4096 in four.
template <bool kGated>
__global__ __launch_bounds__(256) void finish_kernel(const float* sums, int splits, int64_t rows, Epilogue e) {
  const int64_t lines = kGated ? 2 * e.n : e.n, quarters = (e.n + 3) / 4;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < rows * quarters; i += int64_t(gridDim.x) * 256) {
    const int64_t m = i / quarters, c = i % quarters * 4;
    float v[4] = {0, 0, 0, 0}, u[4] = {0, 0, 0, 0}, residual[4];
    const Columns<4, kGated> columns(e, c);
    load_residual<4>(e, m, c, residual);
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      float a[4];
      const float* from = sums + (s * rows + m) * lines + c;
      load_columns<4>(from, vq::kFP32, 0, e.n - c, a);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] += a[q];
      if constexpr (kGated) {
        load_columns<4>(from + e.n, vq::kFP32, 0, e.n - c, a);
#pragma unroll
        for (int q = 0; q < 4; ++q) u[q] += a[q];
      }
    }
    finish_columns<4, kGated>(e, m, c, v, u, columns, residual);
  }
}

// ---- operands that do not lie as the tiles want them -----------------------------------

// out [rows][stride] = in's rows of k, zeros up to whole chunks.
__global__ __launch_bounds__(256) void pack_kernel(Operand in, int64_t k, uint16_t* out, int64_t stride) {
  const int64_t chunks = stride / kChunk;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < in.rows * chunks; i += int64_t(gridDim.x) * 256) {
    const int64_t m = i / chunks, b = i % chunks;
    *reinterpret_cast<u32x4_t*>(out + m * stride + kChunk * b) = load_chunk<true>(in.p + m * in.stride, b, k);
  }
}

// A 64 x 64 part of a transposition through LDS: rows of 64 elements and one dword more.
constexpr int kPart = 64, kPartStride = kPart + 2;
constexpr int64_t kMaxParts = 1 << 23;  // workgroups of 256 threads: below 2^32

// out [k][out_stride] = the transpose of in [rows][k], zeros up to whole chunks of rows.
__global__ __launch_bounds__(256) void transpose_kernel(Operand in, int64_t k, uint16_t* out, int64_t out_stride) {
  __shared__ uint16_t part[kPart * kPartStride];
  const int64_t across = (k + kPart - 1) / kPart, m0 = blockIdx.x / across * kPart, k0 = blockIdx.x % across * kPart;
  const int ch = threadIdx.x & 7, row = threadIdx.x >> 3;
#pragma unroll
  for (int i = 0; i < kPart; i += 32) {
    const int64_t m = m0 + row + i;
    u32x4_t v{0, 0, 0, 0};
    if (m < in.rows) v = load_chunk<true>(in.p + m * in.stride, k0 / kChunk + ch, k);
    uint32_t* to = reinterpret_cast<uint32_t*>(part + (row + i) * kPartStride + kChunk * ch);
#pragma unroll
    for (int j = 0; j < 4; ++j) to[j] = v[j];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPart; i += 32) {
    const int64_t line = k0 + row + i, m = m0 + kChunk * ch;
    u32x4_t v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint16_t* from = part + (kChunk * ch + 2 * j) * kPartStride + row + i;
      v[j] = uint32_t(from[0]) | (uint32_t(from[kPartStride]) << 16);
    }
    if (line < k && m < out_stride) *reinterpret_cast<u32x4_t*>(out + line * out_stride + m) = v;
  }
}

// ---- the gradient of z ------------------------------------------------------------------

struct Slopes {
  const void* dy;  // [rows][n], stride dy_stride
  int dy_dtype;
  int64_t dy_stride;
  const float* z;  // [rows][lines], or null without an activation
  int dtype, activation;
  float limit;
  int64_t rows, n, lines;
};

// Slopes are 0 or 1 from here on.
constexpr float kFar = 104.0f;

// dz at row m of columns c .. c + 7 (zeros past the last): of z's lines there, with a gated
// activation v of the gate lines and u of the up lines.
template <bool kGated>
__device__ __forceinline__ void slopes8(const Slopes& g, int64_t m, int64_t c, float (&v)[8], float (&u)[8]) {
  const int64_t valid = m < g.rows ? g.n - c : 0;
#pragma unroll
  for (int q = 0; q < 8; ++q) v[q] = u[q] = 0;
  if (valid <= 0) return;
  float dy[8];
  load_columns<8>(g.dy, g.dy_dtype, m * g.dy_stride + c, valid, dy);
  if constexpr (kGated) {
    float a[8], b[8];
    load_columns<8>(g.z, vq::kFP32, m * g.lines + c, valid, a);
    load_columns<8>(g.z, vq::kFP32, m * g.lines + g.n + c, valid, b);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      // (an infinite gate has slope 0 or 1, and nothing or all of it passes)
      const float gate = clamp_above(a[q], g.limit);
      v[q] = a[q] > g.limit ? 0.0f : dy[q] * clamp_both(b[q], g.limit) * silu_slope(clamp_both(gate, kFar));
      u[q] = fabsf(b[q]) > g.limit ? 0.0f : dy[q] * silu(gate < -kFar ? -kFar : gate);
    }
  } else if (g.z) {
    float z[8];
    load_columns<8>(g.z, vq::kFP32, m * g.lines + c, valid, z);
    const auto each = [&](float (*f)(float)) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = dy[q] * f(clamp_both(z[q], kFar));
    };
    switch (g.activation) {
      case kRelu: each(relu_slope); break;
      case kGelu: each(gelu_slope); break;
      case kGeluTanh: each(gelu_tanh_slope); break;
      default: each(silu_slope); break;
    }
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = dy[q];
  }
}

// The largest finite magnitude of dz: each workgroup's, and of these all's (in whole numbers,
// as FP32's magnitudes order; a row without numbers leaves the others' scale).
constexpr int kTops = 256;

__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
  return bits < 0x7f800000u ? bits : 0;
}

__device__ __forceinline__ uint32_t block_top(uint32_t mine, uint32_t (&lds)[4]) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2) mine = max(mine, uint32_t(__shfl_xor(int(mine), d)));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = mine;
  __syncthreads();
  return max(max(lds[0], lds[1]), max(lds[2], lds[3]));
}

template <bool kGated>
__global__ __launch_bounds__(256) void top_kernel(Slopes g, uint32_t* tops) {
  __shared__ uint32_t lds[4];
  const int64_t eighths = (g.n + 7) / 8;
  uint32_t most = 0;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < g.rows * eighths; i += int64_t(gridDim.x) * 256) {
    float v[8], u[8];
    slopes8<kGated>(g, i / eighths, i % eighths * 8, v, u);
#pragma unroll
    for (int q = 0; q < 8; ++q) most = max(most, finite_bits(v[q]));
    if constexpr (kGated) {
#pragma unroll
      for (int q = 0; q < 8; ++q) most = max(most, finite_bits(u[q]));
    }
  }
  most = block_top(most, lds);
  if (threadIdx.x == 0) tops[blockIdx.x] = most;
}

// Bound by memory: 4096 rows of a gated 14336 take 207 us (FP32 z read, dz written twice in 16
// bits, dy read: 1.06 GB at 5.1 TB/s).
//
// dz of 64 rows and 64 columns (gated: of the gate and of the up lines; FP16 over scale_of
// the largest of `tops`): by rows (stride `ld`, zeros up to whole chunks of lines), by lines
// (stride `ldt`, zeros up to whole chunks of rows), and the lines' sums over these rows.
//
// dz is rounded to x's type: the matrix cores multiply 16-bit operands of one type, and a second
// product for what the rounding takes off would double the time of both gradients.  It is all that dx
// and dW lose beside their own rounding: against 64 bits they are off by 0.00235 in BF16 and 0.00029
// in FP16 (norms; rounded once 0.00166 and 0.00021), against 64 bits from the rounded dz by
// 0.00166 and 0.00021 (4096 x 4096 x 288, 1000 x 2048 x 768, 4096 x 4096 x 28672).
template <bool kGated>
__global__ __launch_bounds__(256) void slopes_kernel(Slopes g, const uint32_t* tops, int parts, uint32_t* top, uint16_t* dz, int64_t ld,
                                                     uint16_t* dzt, int64_t ldt, float* partial) {
  constexpr int kHalves = kGated ? 2 : 1;
  __shared__ uint16_t part[kHalves][kPart * kPartStride];
  __shared__ float sum[kHalves][32][kPart + 1];
  const int64_t across = (g.n + kPart - 1) / kPart, down = blockIdx.x / across, m0 = down * kPart, c0 = blockIdx.x % across * kPart;
  const int ch = threadIdx.x & 7, row = threadIdx.x >> 3;
  const int64_t c = c0 + kChunk * ch;
  float scale = 1.0f;
  if (tops) {
    __shared__ uint32_t lds[4];
    const uint32_t all = block_top(int(threadIdx.x) < parts ? tops[threadIdx.x] : 0, lds);
    scale = scale_of(all);
    if (blockIdx.x == 0 && threadIdx.x == 0) *top = all;  // for the products
  }
  float mine[kHalves][8];
#pragma unroll
  for (int o = 0; o < kHalves; ++o)
#pragma unroll
    for (int q = 0; q < 8; ++q) mine[o][q] = 0;
#pragma unroll
  for (int i = 0; i < kPart; i += 32) {
    const int64_t m = m0 + row + i;
    float v[2][8];
    slopes8<kGated>(g, m, c, v[0], v[1]);
#pragma unroll
    for (int o = 0; o < kHalves; ++o) {
      uint32_t w[4];
#pragma unroll
      for (int q = 0; q < 8; ++q) mine[o][q] += v[o][q];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = pack16(g.dtype, v[o][2 * j] * scale, v[o][2 * j + 1] * scale);
      if (dz && m < g.rows && c < g.n) {
        const int64_t at = o * g.n + c;
        uint16_t* to = dz + m * ld + at;
        if (c + kChunk <= g.n) {
          __builtin_memcpy(to, w, 16);
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            if (c + q < g.n) to[q] = uint16_t(w[q / 2] >> (16 * (q & 1)));
          }
        }
        if (o == kHalves - 1 && c + kChunk >= g.n) {
          for (int64_t past = g.lines; past < ld; ++past) dz[m * ld + past] = 0;
        }
      }
      uint32_t* to = reinterpret_cast<uint32_t*>(part[o] + (row + i) * kPartStride + kChunk * ch);
#pragma unroll
      for (int j = 0; j < 4; ++j) to[j] = w[j];
    }
  }
#pragma unroll
  for (int o = 0; o < kHalves; ++o)
#pragma unroll
    for (int q = 0; q < 8; ++q) sum[o][row][kChunk * ch + q] = mine[o][q];
  __syncthreads();
  if (dzt) {
#pragma unroll
    for (int o = 0; o < kHalves; ++o)
#pragma unroll
      for (int i = 0; i < kPart; i += 32) {
        const int64_t col = c0 + row + i, m = m0 + kChunk * ch;
        u32x4_t v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint16_t* from = part[o] + (kChunk * ch + 2 * j) * kPartStride + row + i;
          v[j] = uint32_t(from[0]) | (uint32_t(from[kPartStride]) << 16);
        }
        if (col < g.n && m < ldt) *reinterpret_cast<u32x4_t*>(dzt + (o * g.n + col) * ldt + m) = v;
      }
  }
  if (partial && threadIdx.x < kHalves * kPart) {
    const int o = threadIdx.x / kPart, col = threadIdx.x % kPart;
    if (c0 + col < g.n) {
      float all = 0;
      for (int i = 0; i < 32; ++i) all += sum[o][i][col];
      partial[down * g.lines + o * g.n + c0 + col] = all;
    }
  }
}

// db = the parts' sums, in 64 bits: 2^21 rows have 32768 of them, whose sum in FP32 one after
// another was off by 2^-12.6 of itself where gradients have one sign.  32 threads a line take every
// 32nd part, and one adds theirs up in order.  Bound by the loads' latency: 65536 rows of 256 take
// 3.9 us (a thread a line 37), 2^21 of 24 51 (1080), 1000 of 768 2.6 (2.1).
constexpr int kSumLines = 32, kSumRuns = 32;

__global__ __launch_bounds__(kSumLines * kSumRuns) void bias_kernel(const float* partial, int64_t parts, int64_t lines, void* out,
                                                                    int dtype) {
  __shared__ double sums[kSumRuns][kSumLines];
  const int col = threadIdx.x % kSumLines, run = threadIdx.x / kSumLines;
  const int64_t c = int64_t(blockIdx.x) * kSumLines + col;
  double all = 0;
  if (c < lines) {
#pragma unroll 8
    for (int64_t p = run; p < parts; p += kSumRuns) all += partial[p * lines + c];
  }
  sums[run][col] = all;
  __syncthreads();
  if (run || c >= lines) return;
  for (int r = 1; r < kSumRuns; ++r) all += sums[r][col];
  vq::store_act(out, dtype, c, float(all));
}

// ---- how a product runs -----------------------------------------------------------------

int64_t up_to(int64_t v, int64_t step) { return (v + step - 1) / step * step; }
int64_t parts_of(int64_t v, int64_t step) { return (v + step - 1) / step; }

// The tiles, and for the choice between them what they take in us: a round of workgroups
// `start` (and `residual` with one), a stage `alone` on a card hardly filled or `full` on a
// full one.  The last two have four parts in their ring in the place of six and eight: of
// few stages more workgroups a CU, which store while others load, are worth more than loads
// far ahead (8179 rows of 192 x 1152: 16 us for 20; of 4096 x 1152, on 64 x 64: 129 for 111).
struct Shape {
  int lines, rows, parts, places;  // places: workgroups that the card holds
  double start, alone, full, residual;
};
constexpr int kCus = 256, kShapes = 6;
constexpr Shape kShape[kShapes] = {{256, 256, 5, kCus, 17.1, 0.32, 1.70, 13.6}, {256, 128, 6, kCus, 9.1, 0.31, 0.90, 2.4},
                                   {64, 128, 6, 2 * kCus, 5.5, 0.17, 0.55, 1.8},  {64, 64, 8, 2 * kCus, 4.0, 0.11, 0.33, 0.9},
                                   {64, 128, 4, 3 * kCus, 4.6, 0.38, 0.88, 1.7},  {64, 64, 4, 5 * kCus, 3.5, 0.28, 1.02, 1.2}};

enum Kind : int { kTiles = 0, kSmall = 1, kGemv = 2 };

struct Plan {
  Kind kind;
  int shape, splits;  // of the tiles
  int waves;          // of the small kernel: a workgroup's; of the gemv: those that share a line
  int lines;          // of the gemv: a wavefront's
};

// The figures above are fitted to 245 sizes (17 to 8179 rows, k 64 to 14336, n 128 to 20434; of
// small k with an FP32 residual and without), each on all tiles and up to 16 splits; the choice
// by them is 1% slower than the best of each on average, 30% at worst (300 rows of 360 x
// 20434 with a residual: 28 us for 22).
//
// Up to 16 rows (us, a wavefront a line / the small kernel / tiles; k x lines): 4096 x 28672
// 4 rows 48 / 59 / 46, 8 rows 73 / 60 / 45, 16 rows - / 70 / 45; 14336 x 4096 2 rows 25 / 26 /
// 26, 4 rows 35 / 28 / 26; 4096 x 4096 4 rows 9.4 / 9.0 / 12, 8 rows 15 / 9.2 / 12, 16 rows
// - / 10.4 / 12.3; 7168 x 256 8 rows 5.9 / 12 / 8.7, 16 rows - / 14.6 / 9.0.  So W of more than
// 2^25 elements goes to the tiles from three rows on (if it lies as they want it: a packed copy
// costs more than it gains), few and long lines from nine.
constexpr int64_t kLargeW = int64_t(1) << 25, kFewLines = 512;

// direct: x and W lie as the tiles want them.
Plan plan_of(int64_t rows, int64_t k, int64_t n, bool gated, bool residual, bool direct) {
  const int64_t lines = gated ? 2 * n : n;
  const bool large = direct && lines * k > kLargeW;
  if (rows <= kGemvRows && !(large && rows > 2) && !(rows > 4 && lines > kFewLines)) {
    // a line a wavefront, and as many wavefronts a line as fill the card with four each SIMD
    const int64_t steps = parts_of(k, kGemvStep);
    Plan p{kGemv, 0, 1, 1, lines >= 8192 || gated ? 2 : 1};
    while (p.waves < kGemvWaves && p.waves < steps && parts_of(lines, p.lines) * p.waves < 16 * kCus) p.waves *= 2;
    return p;
  }
  const int64_t steps = parts_of(k, kChunk * kStepChunks);
  if (rows <= kSmallRows && !large && !(direct && rows > kGemvRows && lines <= kFewLines && steps > 32)) {
    return {kSmall, 0, 1, steps >= 16 ? 16 : steps >= 8 ? 8 : 4, 0};
  }
  const int64_t stages = parts_of(k, kChunk * kStageChunks);
  Plan best{kTiles, 0, 1, 0, 0};
  double least = 0;
  for (int i = 0; i < kShapes; ++i) {
    const Shape& t = kShape[i];
    const int64_t tiles = parts_of(rows, t.rows) * parts_of(n, gated ? t.lines / 2 : t.lines);
    if (i && tiles > kMaxGroups) continue;  // (a result that fits a card has no more of the largest)
    for (int64_t splits = 1; splits <= 16 && splits <= std::max<int64_t>(1, stages / 4); ++splits) {
      if (splits > 1 && tiles * splits > 8 * kCus) break;
      const int64_t each = parts_of(stages, splits), all = tiles * parts_of(stages, each);
      const int64_t rest = all % t.places;
      const double start = t.start + (residual && splits == 1 ? t.residual : 0);
      double cost = double(all / t.places) * (start + double(each) * t.full);
      if (rest) cost += start + double(each) * (t.alone + (t.full - t.alone) * double(rest) / t.places);
      if (splits > 1) cost += 4 + double(splits) * (0.25 + double(rows) * double(lines) * 4 / 8e6);  // written and added up
      if (least == 0 || cost < least) {
        least = cost;
        best = {kTiles, i, int(splits), 0, 0};
      }
    }
  }
  return best;
}

bool direct(const Operand& o, int64_t k) { return aligned(o.p, 16) && o.stride % kChunk == 0 && k % kChunk == 0 && o.stride <= kMaxK; }

int64_t sums_bytes(const Plan& p, int64_t rows, int64_t lines) { return p.splits > 1 ? p.splits * rows * lines * 4 : 0; }

template <bool kBf16>
void launch_small(const Operand& x, const Operand& w, int64_t k, const Epilogue& e, int waves, hipStream_t s) {
  const dim3 grid(unsigned(parts_of(e.n, 16))), block(unsigned(64 * waves));
  if (e.activation == kSwiglu) hipLaunchKernelGGL((small_kernel<true, kBf16>), grid, block, 0, s, x, w, k, e);
  else hipLaunchKernelGGL((small_kernel<false, kBf16>), grid, block, 0, s, x, w, k, e);
}

template <int kRows, bool kBf16>
void launch_gemv(const Operand& x, const Operand& w, int64_t k, const Epilogue& e, const Plan& p, hipStream_t s) {
  const bool gated = e.activation == kSwiglu;
  const int64_t each = kGemvWaves / p.waves * (gated ? 1 : p.lines);
  const dim3 grid(unsigned(parts_of(e.n, each))), block(64 * kGemvWaves);
  if (gated) hipLaunchKernelGGL((gemv_kernel<kRows, 2, true, kBf16>), grid, block, 0, s, x, w, k, p.waves, e);
  else if (p.lines == 2) hipLaunchKernelGGL((gemv_kernel<kRows, 2, false, kBf16>), grid, block, 0, s, x, w, k, p.waves, e);
  else hipLaunchKernelGGL((gemv_kernel<kRows, 1, false, kBf16>), grid, block, 0, s, x, w, k, p.waves, e);
}

// Plain: without a gated activation.
template <typename Plain, typename Gated, bool kBf16>
void launch_tile(const TileArgs& t, int64_t splits, hipStream_t s) {
  const dim3 grid(unsigned(up_to(int64_t(t.tiles_n) * t.tiles_m, 8)), unsigned(splits));
  if (t.e.activation == kSwiglu) hipLaunchKernelGGL((tile_kernel<Gated, true, kBf16>), grid, dim3(Gated::kThreads), 0, s, t);
  else hipLaunchKernelGGL((tile_kernel<Plain, false, kBf16>), grid, dim3(Plain::kThreads), 0, s, t);
}

// x [rows][k] times W's transpose, finished by e; sums: the plan's K splits' room.
template <bool kBf16>
int product(const Operand& x, const Operand& w, int64_t k, const Epilogue& e, float* sums, const Plan& p, hipStream_t s) {
  if (p.kind == kGemv) {
    if (x.rows == 1) launch_gemv<1, kBf16>(x, w, k, e, p, s);
    else if (x.rows == 2) launch_gemv<2, kBf16>(x, w, k, e, p, s);
    else if (x.rows <= 4) launch_gemv<4, kBf16>(x, w, k, e, p, s);
    else launch_gemv<8, kBf16>(x, w, k, e, p, s);
    return vq::check_launch("dense_linear");
  }
  if (p.kind == kSmall) {
    launch_small<kBf16>(x, w, k, e, p.waves, s);
    return vq::check_launch("dense_linear");
  }
  const bool gated = e.activation == kSwiglu;
  const Shape& shape = kShape[p.shape];
  const int64_t stages = parts_of(k, kChunk * kStageChunks);
  const int64_t tiles_n = parts_of(e.n, gated ? shape.lines / 2 : shape.lines), tiles_m = parts_of(x.rows, shape.rows);
  if (tiles_n * tiles_m > kMaxGroups) return vq::fail("dense_linear: too many rows and columns");
  const int64_t split = parts_of(stages, p.splits);
  const int64_t splits = parts_of(stages, split);  // (none without a stage)
  const double at_work = std::min(double(tiles_n * tiles_m), double(shape.places)) / 8;  // on an XCD
  const int64_t band = std::max<int64_t>(1, std::min<int64_t>(tiles_m, int64_t(std::sqrt(at_work * shape.lines / shape.rows) + 0.5)));
  const TileArgs t{x, w, int(parts_of(k, kChunk)), int(tiles_n), int(tiles_m), int(band), int(split), sums, e};
  switch (p.shape) {
    case 0: launch_tile<Tile<4, 2, 2, 4, 5>, Tile<4, 2, 2, 4, 5>, kBf16>(t, splits, s); break;
    case 1: launch_tile<Tile<4, 2, 2, 2, 6>, Tile<4, 2, 2, 2, 6>, kBf16>(t, splits, s); break;
    case 2: launch_tile<Tile<2, 2, 1, 2, 6>, Tile<1, 4, 2, 1, 6>, kBf16>(t, splits, s); break;
    case 3: launch_tile<Tile<2, 2, 1, 1, 8>, Tile<1, 2, 2, 1, 8>, kBf16>(t, splits, s); break;
    case 4: launch_tile<Tile<2, 2, 1, 2, 4>, Tile<1, 4, 2, 1, 4>, kBf16>(t, splits, s); break;
    default: launch_tile<Tile<2, 2, 1, 1, 4>, Tile<1, 2, 2, 1, 4>, kBf16>(t, splits, s); break;
  }
  if (int rc = vq::check_launch("dense_linear")) return rc;
  if (splits == 1) return vq::kOk;
  const dim3 groups(unsigned(std::min<int64_t>(parts_of(x.rows * parts_of(e.n, 4), 256), 8192)));
  if (gated) hipLaunchKernelGGL(finish_kernel<true>, groups, dim3(256), 0, s, sums, int(splits), x.rows, e);
  else hipLaunchKernelGGL(finish_kernel<false>, groups, dim3(256), 0, s, sums, int(splits), x.rows, e);
  return vq::check_launch("dense_linear");
}
int product(const Operand& x, const Operand& w, int64_t k, const Epilogue& e, bool bf16, float* sums, const Plan& p, hipStream_t s) {
  return bf16 ? product<true>(x, w, k, e, sums, p, s) : product<false>(x, w, k, e, sums, p, s);
}

int pack(Operand& o, int64_t k, uint16_t* to, hipStream_t s) {
  const int64_t stride = up_to(k, kChunk), groups = parts_of(o.rows * (stride / kChunk), 256);
  hipLaunchKernelGGL(pack_kernel, dim3(unsigned(std::min<int64_t>(groups, 16384))), dim3(256), 0, s, o, k, to, stride);
  o.p = to;
  o.stride = stride;
  return vq::check_launch("dense_linear");
}

int transpose(const Operand& o, int64_t k, uint16_t* to, int64_t stride, hipStream_t s) {
  const int64_t groups = parts_of(k, kPart) * parts_of(o.rows, kPart);  // (check_grad_sizes)
  hipLaunchKernelGGL(transpose_kernel, dim3(unsigned(groups)), dim3(256), 0, s, o, k, to, stride);
  return vq::check_launch("dense_linear");
}

int check_sizes(int64_t rows, int64_t k, int64_t n, int activation) {
  if (rows < 0 || rows > kMaxRows) return vq::fail("dense_linear: rows out of range");
  if (k <= 0 || k > kMaxK) return vq::fail("dense_linear: k must be between 1 and 2^21");
  if (n <= 0 || (activation == kSwiglu ? 2 * n : n) > kMaxLines) return vq::fail("dense_linear: columns out of range");
  if (activation < kNone || activation > kSwiglu) return vq::fail("dense_linear: unknown activation");
  return vq::kOk;
}

int check_grad_sizes(int64_t rows, int64_t k, int64_t n, int activation) {
  if (int rc = check_sizes(rows, k, n, activation)) return rc;
  const int64_t lines = activation == kSwiglu ? 2 * n : n;
  // (the products' sums run over the lines and the rows)
  if (rows > kMaxK || lines > kMaxK) return vq::fail("dense_linear: a gradient takes up to 2^21 rows and weight rows");
  const int64_t across = parts_of(std::max(lines, k), kPart);
  if (across * parts_of(rows, kPart) > kMaxParts || parts_of(k, kPart) * parts_of(lines, kPart) > kMaxParts) {
    return vq::fail("dense_linear: too many rows and columns");
  }
  return vq::kOk;
}

bool is_half(int dtype) { return dtype == vq::kBF16 || dtype == vq::kFP16; }
bool is_float(int dtype) { return is_half(dtype) || dtype == vq::kFP32; }

int check_inputs(const void* x, int dtype, int64_t rows, int64_t k, int64_t x_stride, const void* w, int64_t w_stride, float limit,
                 bool read_x = true, bool read_w = true) {
  if (!is_half(dtype)) return vq::fail("dense_linear: x and the weights must be BF16 or FP16");
  if ((read_x && !x) || (read_w && !w)) return vq::fail("dense_linear: null pointer");
  if (x_stride < 0 || (rows > 1 && x_stride < k) || x_stride > (int64_t(1) << 40) || w_stride < k || w_stride > (int64_t(1) << 40)) {
    return vq::fail("dense_linear: row stride out of range");
  }
  if (!(limit > 0)) return vq::fail("dense_linear: the clamp limit must be positive");
  return vq::kOk;
}

struct Span {
  const void* p;
  int64_t bytes, element;
};
int check_spans(std::initializer_list<Span> outputs, std::initializer_list<Span> inputs) {
  for (const Span* a = outputs.begin(); a != outputs.end(); ++a) {
    for (const Span* b = outputs.begin(); b != a; ++b) {
      if (vq::overlaps(a->p, a->bytes, b->p, b->bytes)) return vq::fail("dense_linear: arguments must not overlap");
    }
    for (const Span& b : inputs) {
      if (vq::overlaps(a->p, a->bytes, b.p, b.bytes)) return vq::fail("dense_linear: arguments must not overlap");
    }
  }
  for (const auto* list : {&outputs, &inputs}) {
    for (const Span& a : *list) {
      if (reinterpret_cast<uintptr_t>(a.p) % uintptr_t(a.element)) return vq::fail("dense_linear: misaligned pointer");
    }
  }
  return vq::kOk;
}
int64_t span_bytes(int64_t rows, int64_t cols, int64_t stride, int dtype) {
  return rows > 0 ? ((rows - 1) * stride + cols) * vq::dtype_bytes(dtype) : 0;
}

// The forward's workspace: the K splits' sums, then packed operands.
struct Room {
  int64_t sums, x, w, bytes;
  Room(int64_t rows, int64_t k, int64_t lines, const Plan& p, bool pack_x, bool pack_w) {
    const int64_t row = up_to(k, kChunk) * 2;
    sums = up_to(sums_bytes(p, rows, lines), 256);
    x = pack_x ? up_to(rows * row, 256) : 0;
    w = pack_w ? up_to(lines * row, 256) : 0;
    bytes = sums + x + w;
  }
};

// The gradient's: the sums (of either product), then the operands by what they are summed over.
struct GradRoom {
  Plan px, pw;
  int64_t sums, wt, xt, dz, dzt, partial, top, bytes;
  GradRoom(int64_t rows, int64_t k, int64_t lines, bool need_x, bool need_w, bool need_bias) {
    px = plan_of(rows, lines, k, false, false, true);
    pw = plan_of(lines, rows, k, false, false, true);
    const int64_t ld = up_to(lines, kChunk) * 2, ldt = up_to(rows, kChunk) * 2;
    sums = up_to(std::max(need_x ? sums_bytes(px, rows, k) : 0, need_w ? sums_bytes(pw, lines, k) : 0), 256);
    wt = need_x ? up_to(k * ld, 256) : 0;
    xt = need_w ? up_to(k * ldt, 256) : 0;
    dz = need_x ? up_to(rows * ld, 256) : 0;
    dzt = need_w ? up_to(lines * ldt, 256) : 0;
    partial = need_bias ? up_to(parts_of(rows, kPart) * lines * 4, 256) : 0;
    top = up_to((1 + kTops) * 4, 256);  // all's, then the workgroups'
    bytes = sums + wt + xt + dz + dzt + partial + top;
  }
};

}  // namespace
}  // namespace dense

extern "C" int64_t dense_linear_workspace_size(const void* x, int64_t rows, int64_t k, int64_t x_stride, const void* w, int64_t n,
                                               int64_t w_stride, int activation) {
  using namespace dense;
  if (check_sizes(rows, k, n, activation)) return -1;
  if (rows == 0) return 0;
  const bool gated = activation == kSwiglu;
  const int64_t lines = gated ? 2 * n : n;
  const Operand xo{static_cast<const uint16_t*>(x), rows, rows > 1 ? x_stride : k}, wo{static_cast<const uint16_t*>(w), lines, w_stride};
  int64_t most = 0;
  for (const bool residual : {false, true}) {
    const Plan p = plan_of(rows, k, n, gated, residual, direct(xo, k) && direct(wo, k));
    const bool tiles = p.kind == kTiles;
    most = std::max(most, Room(rows, k, lines, p, tiles && !direct(xo, k), tiles && !direct(wo, k)).bytes);
  }
  return most;
}

extern "C" int dense_linear_plan(int64_t rows, int64_t k, int64_t n, int activation, int has_residual, int32_t* plan) {
  using namespace dense;
  if (int rc = check_sizes(rows, k, n, activation)) return rc;
  if (!plan) return vq::fail("dense_linear: null pointer");
  const Plan p = plan_of(rows, k, n, activation == kSwiglu, has_residual, k % kChunk == 0);
  plan[0] = p.kind;
  plan[1] = p.kind == kTiles ? kShape[p.shape].rows : 0;
  plan[2] = p.kind == kTiles ? kShape[p.shape].lines : p.lines;
  plan[3] = p.kind == kTiles ? p.splits : p.waves;
  plan[4] = p.kind == kTiles ? kShape[p.shape].parts : 0;
  return vq::kOk;
}

extern "C" int dense_linear(const void* x, int dtype, int64_t rows, int64_t k, int64_t x_stride, const void* w, int64_t n, int64_t w_stride,
                            const void* bias, int bias_dtype, int activation, float limit, const void* residual, int residual_dtype,
                            int64_t residual_stride, void* out, int out_dtype, float* z, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  using namespace dense;
  if (int rc = check_sizes(rows, k, n, activation)) return rc;
  if (!is_float(out_dtype) || (bias && !is_float(bias_dtype)) || (residual && !is_float(residual_dtype))) {
    return vq::fail("dense_linear: bias, residual and output must be BF16, FP16 or FP32");
  }
  if (rows == 0) return vq::kOk;
  if (int rc = check_inputs(x, dtype, rows, k, x_stride, w, w_stride, limit)) return rc;
  if (!out) return vq::fail("dense_linear: null pointer");
  if (residual && (residual_stride < 0 || (rows > 1 && residual_stride < n))) return vq::fail("dense_linear: residual stride out of range");
  const bool gated = activation == kSwiglu;
  const int64_t lines = gated ? 2 * n : n;
  Operand xo{static_cast<const uint16_t*>(x), rows, rows > 1 ? x_stride : k}, wo{static_cast<const uint16_t*>(w), lines, w_stride};
  const Plan p = plan_of(rows, k, n, gated, residual, direct(xo, k) && direct(wo, k));
  const bool pack_x = p.kind == kTiles && !direct(xo, k), pack_w = p.kind == kTiles && !direct(wo, k);
  const Room room(rows, k, lines, p, pack_x, pack_w);
  if (room.bytes && (!workspace || workspace_bytes < room.bytes || !aligned(workspace, 16))) {
    return vq::fail("dense_linear: workspace too small or misaligned");
  }
  // (the output may be the residual: an element is read before it is written, by the same lane)
  const bool in_place = residual == out && residual_dtype == out_dtype && (rows == 1 || residual_stride == n);
  if (int rc = check_spans({{out, rows * n * vq::dtype_bytes(out_dtype), vq::dtype_bytes(out_dtype)},
                            {z, z ? rows * lines * 4 : 0, 4},
                            {workspace, room.bytes, 1}},
                           {{x, span_bytes(rows, k, xo.stride, dtype), 2},
                            {w, span_bytes(lines, k, w_stride, dtype), 2},
                            {bias, bias ? lines * vq::dtype_bytes(bias_dtype) : 0, bias ? vq::dtype_bytes(bias_dtype) : 1},
                            {in_place ? nullptr : residual, residual ? span_bytes(rows, n, residual_stride, residual_dtype) : 0,
                             residual ? vq::dtype_bytes(residual_dtype) : 1}})) {
    return rc;
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  uint8_t* at = static_cast<uint8_t*>(workspace);
  float* sums = reinterpret_cast<float*>(at);
  at += room.sums;
  if (pack_x) {
    if (int rc = pack(xo, k, reinterpret_cast<uint16_t*>(at), s)) return rc;
  }
  at += room.x;
  if (pack_w) {
    if (int rc = pack(wo, k, reinterpret_cast<uint16_t*>(at), s)) return rc;
  }
  const Epilogue e{bias, bias_dtype, activation, limit, residual, residual_dtype, residual_stride, out, out_dtype, n, z, nullptr};
  return product(xo, wo, k, e, dtype == vq::kBF16, sums, p, s);
}

extern "C" int64_t dense_linear_grad_workspace_size(int64_t rows, int64_t k, int64_t n, int activation, int need_x, int need_w, int need_bias) {
  using namespace dense;
  if (check_grad_sizes(rows, k, n, activation)) return -1;
  if (rows == 0) return 0;
  return GradRoom(rows, k, activation == kSwiglu ? 2 * n : n, need_x, need_w, need_bias).bytes;
}

extern "C" int dense_linear_grad(const void* x, int dtype, int64_t rows, int64_t k, int64_t x_stride, const void* w, int64_t n,
                                 int64_t w_stride, const float* z, int activation, float limit, const void* dy, int dy_dtype,
                                 int64_t dy_stride, void* dx, void* dw, void* dbias, int bias_dtype, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  using namespace dense;
  if (int rc = check_grad_sizes(rows, k, n, activation)) return rc;
  if (!is_float(dy_dtype) || (dbias && !is_float(bias_dtype))) return vq::fail("dense_linear: bias and output must be BF16, FP16 or FP32");
  if (rows == 0) return vq::fail("dense_linear: no rows have no gradient to compute");
  if (int rc = check_inputs(x, dtype, rows, k, x_stride, w, w_stride, limit, dw, dx)) return rc;
  if (!dy || (activation != kNone && !z)) return vq::fail("dense_linear: null pointer");
  if (dy_stride < 0 || (rows > 1 && dy_stride < n)) return vq::fail("dense_linear: gradient stride out of range");
  const bool gated = activation == kSwiglu;
  const int64_t lines = gated ? 2 * n : n;
  const GradRoom room(rows, k, lines, dx, dw, dbias);
  if (!workspace || workspace_bytes < room.bytes || !aligned(workspace, 16)) return vq::fail("dense_linear: workspace too small or misaligned");
  const Operand xo{static_cast<const uint16_t*>(x), rows, rows > 1 ? x_stride : k}, wo{static_cast<const uint16_t*>(w), lines, w_stride};
  if (int rc = check_spans({{dx, dx ? rows * k * 2 : 0, 2},
                            {dw, dw ? lines * k * 2 : 0, 2},
                            {dbias, dbias ? lines * vq::dtype_bytes(bias_dtype) : 0, dbias ? vq::dtype_bytes(bias_dtype) : 1},
                            {workspace, room.bytes, 1}},
                           {{x, span_bytes(rows, k, xo.stride, dtype), 2},
                            {w, span_bytes(lines, k, w_stride, dtype), 2},
                            {z, activation != kNone ? rows * lines * 4 : 0, 4},
                            {dy, span_bytes(rows, n, dy_stride, dy_dtype), vq::dtype_bytes(dy_dtype)}})) {
    return rc;
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  uint8_t* at = static_cast<uint8_t*>(workspace);
  const auto take = [&](int64_t bytes) {
    uint8_t* p = bytes ? at : nullptr;
    at += bytes;
    return p;
  };
  float* sums = reinterpret_cast<float*>(take(room.sums));
  uint16_t* wt = reinterpret_cast<uint16_t*>(take(room.wt));
  uint16_t* xt = reinterpret_cast<uint16_t*>(take(room.xt));
  uint16_t* dz = reinterpret_cast<uint16_t*>(take(room.dz));
  uint16_t* dzt = reinterpret_cast<uint16_t*>(take(room.dzt));
  float* partial = reinterpret_cast<float*>(take(room.partial));
  uint32_t* top = reinterpret_cast<uint32_t*>(take(room.top));
  const int64_t ld = up_to(lines, kChunk), ldt = up_to(rows, kChunk);
  const Slopes g{dy, dy_dtype, rows > 1 ? dy_stride : n, activation == kNone ? nullptr : z, dtype, activation, limit,
                 rows, n, lines};
  const bool scaled = dtype == vq::kFP16 && (dx || dw);
  int tops = 0;
  if (scaled) {
    tops = int(std::min<int64_t>(parts_of(rows * parts_of(n, 8), 256), kTops));
    if (gated) hipLaunchKernelGGL(top_kernel<true>, dim3(unsigned(tops)), dim3(256), 0, s, g, top + 1);
    else hipLaunchKernelGGL(top_kernel<false>, dim3(unsigned(tops)), dim3(256), 0, s, g, top + 1);
    if (int rc = vq::check_launch("dense_linear gradient")) return rc;
  }
  const dim3 parts(unsigned(parts_of(n, kPart) * parts_of(rows, kPart)));
  if (gated) hipLaunchKernelGGL(slopes_kernel<true>, parts, dim3(256), 0, s, g, scaled ? top + 1 : nullptr, tops, top, dz, ld, dzt, ldt, partial);
  else hipLaunchKernelGGL(slopes_kernel<false>, parts, dim3(256), 0, s, g, scaled ? top + 1 : nullptr, tops, top, dz, ld, dzt, ldt, partial);
  if (int rc = vq::check_launch("dense_linear gradient")) return rc;
  if (dbias) {
    hipLaunchKernelGGL(bias_kernel, dim3(unsigned(parts_of(lines, kSumLines))), dim3(kSumLines * kSumRuns), 0, s, partial, parts_of(rows, kPart),
                       lines, dbias, bias_dtype);
    if (int rc = vq::check_launch("dense_linear gradient")) return rc;
  }
  const bool bf16 = dtype == vq::kBF16;
  const auto plain = [&](void* out) {
    return Epilogue{nullptr, 0, kNone, __builtin_inff(), nullptr, 0, 0, out, dtype, k, nullptr, scaled ? top : nullptr};
  };
  if (dx) {
    if (int rc = transpose(wo, k, wt, ld, s)) return rc;
    if (int rc = product({dz, rows, ld}, {wt, k, ld}, lines, plain(dx), bf16, sums, room.px, s)) return rc;
  }
  if (dw) {
    if (int rc = transpose(xo, k, xt, ldt, s)) return rc;
    if (int rc = product({dzt, lines, ldt}, {xt, k, ldt}, rows, plain(dw), bf16, sums, room.pw, s)) return rc;
  }
  return vq::kOk;
}
