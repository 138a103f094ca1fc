// MXFP4 (mxfp4.h): quantization, dequantization, and the product of MXFP4
// activations with MXFP4 weights.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "../../include/vllm_mi355x.h"
#include "mxfp4.h"
#include "mxfp4_tile.h"

namespace mx {
namespace {

constexpr int kThreads = 256;

// ---- quantization ------------------------------------------------------------

// Four lanes a block, eight elements each.
template <int kDtype>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const void* x, int64_t rows, int blocks, int64_t stride,
                                                            bool wide, uint32_t* codes, uint8_t* scales) {
  const int64_t quarter = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t b = quarter >> 2;
  const int j = int(quarter & 3);
  if (b >= rows * blocks) return;
  const int64_t r = b / blocks;
  const int c = int(b - r * blocks);
  float v[8];
  load8<kDtype>(x, r * stride + int64_t(c) * kBlock + 8 * j, wide, v);
  uint32_t s;
  codes[quarter] = quantize_quarter(v, s);
  if (j == 0) scales[b] = uint8_t(s);
}

__global__ __launch_bounds__(kThreads) void dequantize_kernel(const uint32_t* codes, const uint8_t* scales,
                                                              int64_t quarters, void* out, int dtype) {
  const int64_t quarter = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (quarter >= quarters) return;
  const uint32_t w = codes[quarter];
  const float s = scale_value(scales[quarter >> 2]);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = code_value(w >> (4 * i)) * s;
  vq::store8_act(out, dtype, 8 * quarter, v, 8);
}

// ---- product -------------------------------------------------------------------

struct MatmulArgs {
  const uint8_t *a, *as, *w, *ws;
  int64_t rows, n;
  int blocks;  // k / 32
  void* out;
  int out_dtype;
};

// One wavefront: 16 rows x 16 columns, every operand from global memory.
__global__ __launch_bounds__(64) void matmul_kernel(MatmulArgs g) {
  const int lane = threadIdx.x;
  const int r = lane & 15, q = lane >> 4;
  const int64_t n0 = int64_t(blockIdx.x) * 16, m0 = int64_t(blockIdx.y) * 16;
  const int64_t wrow = min(n0 + r, g.n - 1), arow = min(m0 + r, g.rows - 1);
  const uint8_t* a = g.a + arow * g.blocks * kBlockBytes;
  const uint8_t* w = g.w + wrow * g.blocks * kBlockBytes;
  const uint8_t* as = g.as + arow * g.blocks;
  const uint8_t* ws = g.ws + wrow * g.blocks;
  f32x4_t acc{0, 0, 0, 0};
  for (int b0 = 0; b0 < g.blocks; b0 += 4) {
    // blocks past the last multiply zeros by zeros
    const int b = b0 + q;
    u32x4_t av{0, 0, 0, 0}, wv{0, 0, 0, 0};
    uint32_t sa = 127, sw = 127;
    if (b < g.blocks) {
      av = *reinterpret_cast<const u32x4_t*>(a + int64_t(b) * kBlockBytes);
      wv = *reinterpret_cast<const u32x4_t*>(w + int64_t(b) * kBlockBytes);
      sa = as[b];
      sw = ws[b];
    }
    acc = mfma16(wv, sw, av, sa, acc);
  }
  if (m0 + r >= g.rows) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t n = n0 + 4 * q + i;
    if (n < g.n) vq::store_act(g.out, g.out_dtype, (m0 + r) * g.n + n, acc[i]);
  }
}

#ifdef MX_TUNE
int g_force = 0;
#endif

template <int kN, int kM>
int launch_tile(const MatmulArgs& g, hipStream_t s) {
  TileArgs t{};
  t.a = g.a;
  t.as = g.as;
  t.w = g.w;
  t.ws = g.ws;
  t.rows = g.rows;
  t.n = g.n;
  t.blocks = g.blocks;
  t.out = g.out;
  t.out_dtype = g.out_dtype;
  t.wide = g.n % 8 == 0 && aligned(g.out, 16);
  t.tiles_n = int((g.n + 64 * kN - 1) / (64 * kN));
  t.tiles_m = int((g.rows + 64 * kM - 1) / (64 * kM));
  const int64_t total = int64_t(t.tiles_n) * t.tiles_m;
  hipLaunchKernelGGL((tile_kernel<kN, kM, kDense>), dim3(unsigned((total + 7) / 8 * 8)), dim3(kTileThreads), 0, s, t);
  return vq::check_launch("mxfp4 tile");
}

int64_t tiles_of(const MatmulArgs& g, int cols, int rows) { return ((g.n + cols - 1) / cols) * ((g.rows + rows - 1) / rows); }

int launch_matmul(const MatmulArgs& g, hipStream_t s) {
  // the tile kernel: whole stages of blocks, tiles below 2 GiB, a grid in 32 bits
  if (g.rows > 32 && g.blocks >= kStageBlocks && int64_t(g.blocks) * kBlockBytes * 256 <= INT_MAX && tiles_of(g, 64, 64) <= INT_MAX / 8) {
    int force = 0;
#ifdef MX_TUNE
    force = g_force;
#endif
    if (force == 44 || (!force && tiles_of(g, 256, 256) >= 200)) return launch_tile<4, 4>(g, s);
    if (force == 22 || (!force && tiles_of(g, 128, 128) >= 200)) return launch_tile<2, 2>(g, s);
    if (force == 11 || !force) return launch_tile<1, 1>(g, s);
  }
  const int64_t tiles_n = (g.n + 15) / 16, tiles_m = (g.rows + 15) / 16;
  if (tiles_n > INT_MAX || tiles_m > 65535) return vq::fail("mxfp4: too many rows or columns");
  hipLaunchKernelGGL(matmul_kernel, dim3(unsigned(tiles_n), unsigned(tiles_m)), dim3(64), 0, s, g);
  return vq::check_launch("mxfp4 matmul");
}

int launch_quantize(const void* x, int dtype, int64_t rows, int64_t k, int64_t stride, uint8_t* codes, uint8_t* scales,
                    hipStream_t s) {
  const int64_t blocks = k / kBlock;
  const int64_t groups = (rows * blocks * 4 + kThreads - 1) / kThreads;
  if (groups > INT_MAX || blocks > INT_MAX) return vq::fail("mxfp4: too many elements");
  // 16-byte loads where every eight elements begin on a 16-byte line
  const bool wide = aligned(x, 16) && stride * vq::dtype_bytes(dtype) % 16 == 0;
  const dim3 grid{unsigned(groups)};
  uint32_t* words = reinterpret_cast<uint32_t*>(codes);
  if (dtype == vq::kBF16) {
    hipLaunchKernelGGL(quantize_kernel<vq::kBF16>, grid, dim3(kThreads), 0, s, x, rows, int(blocks), stride, wide, words, scales);
  } else if (dtype == vq::kFP16) {
    hipLaunchKernelGGL(quantize_kernel<vq::kFP16>, grid, dim3(kThreads), 0, s, x, rows, int(blocks), stride, wide, words, scales);
  } else {
    hipLaunchKernelGGL(quantize_kernel<vq::kFP32>, grid, dim3(kThreads), 0, s, x, rows, int(blocks), stride, wide, words, scales);
  }
  return vq::check_launch("mxfp4 quantize");
}

// Sizes below which every offset of a matrix fits 62 bits, whatever the strides.
bool sane(int64_t rows, int64_t cols) {
  return rows >= 0 && cols >= 0 && (rows == 0 || cols <= (int64_t(1) << 60) / std::max<int64_t>(rows, 1));
}

bool known_dtype(int dtype) { return dtype == vq::kBF16 || dtype == vq::kFP16 || dtype == vq::kFP32; }

int check_product(int64_t rows, int64_t k, int64_t n, const uint8_t* w, const uint8_t* w_scales, int out_dtype, const void* out) {
  if (!known_dtype(out_dtype)) return vq::fail("mxfp4: out must be BF16, FP16 or FP32");
  if (rows < 0 || n < 0 || k <= 0 || k % kBlock != 0) return vq::fail("mxfp4: k must be a positive multiple of 32");
  if (!sane(rows, k) || !sane(n, k) || !sane(rows, n)) return vq::fail("mxfp4: sizes out of range");
  if (rows == 0 || n == 0) return vq::kOk;
  if (!w || !w_scales || !out) return vq::fail("mxfp4: null pointer");
  if (!aligned(w, 16)) return vq::fail("mxfp4: codes must be 16-byte aligned");
  if (!aligned(out, vq::dtype_bytes(out_dtype))) return vq::fail("mxfp4: out must be aligned to its elements");
  if (vq::overlaps(out, rows * n * vq::dtype_bytes(out_dtype), w, n * k / 2) ||
      vq::overlaps(out, rows * n * vq::dtype_bytes(out_dtype), w_scales, n * k / kBlock)) {
    return vq::fail("mxfp4: out must not overlap the weights");
  }
  return vq::kOk;
}

int check_rows(const void* x, int x_dtype, int64_t rows, int64_t k, int64_t x_stride) {
  if (!known_dtype(x_dtype)) return vq::fail("mxfp4: x must be BF16, FP16 or FP32");
  if (rows < 0 || k <= 0 || k % kBlock != 0) return vq::fail("mxfp4: the last axis must be a positive multiple of 32");
  if (x_stride < 0 || (rows > 1 && x_stride < k) || !sane(rows, std::max(x_stride, k))) return vq::fail("mxfp4: row stride out of range");
  if (rows == 0) return vq::kOk;
  if (!x) return vq::fail("mxfp4: null pointer");
  if (!aligned(x, vq::dtype_bytes(x_dtype))) return vq::fail("mxfp4: x must be aligned to its elements");
  return vq::kOk;
}

}  // namespace
}  // namespace mx

extern "C" int mxfp4_quantize(const void* x, int x_dtype, int64_t rows, int64_t k, int64_t x_stride, uint8_t* codes,
                              uint8_t* scales, void* stream) {
  using namespace mx;
  if (int rc = check_rows(x, x_dtype, rows, k, x_stride)) return rc;
  if (rows == 0) return vq::kOk;
  if (!codes || !scales) return vq::fail("mxfp4: null pointer");
  if (!aligned(codes, 16)) return vq::fail("mxfp4: codes must be 16-byte aligned");
  const int64_t x_bytes = ((rows - 1) * x_stride + k) * vq::dtype_bytes(x_dtype);
  if (vq::overlaps(codes, rows * k / 2, x, x_bytes) || vq::overlaps(scales, rows * k / kBlock, x, x_bytes) ||
      vq::overlaps(codes, rows * k / 2, scales, rows * k / kBlock)) {
    return vq::fail("mxfp4: codes and scales must not overlap x or each other");
  }
  return launch_quantize(x, x_dtype, rows, k, x_stride, codes, scales, static_cast<hipStream_t>(stream));
}

extern "C" int mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t k, void* out, int out_dtype,
                                void* stream) {
  using namespace mx;
  if (!known_dtype(out_dtype)) return vq::fail("mxfp4: out must be BF16, FP16 or FP32");
  if (rows < 0 || k <= 0 || k % kBlock != 0 || !sane(rows, k)) return vq::fail("mxfp4: the last axis must be a positive multiple of 32");
  if (rows == 0) return vq::kOk;
  if (!codes || !scales || !out) return vq::fail("mxfp4: null pointer");
  if (!aligned(codes, 16)) return vq::fail("mxfp4: codes must be 16-byte aligned");
  if (!aligned(out, vq::dtype_bytes(out_dtype))) return vq::fail("mxfp4: out must be aligned to its elements");
  const int64_t out_bytes = rows * k * vq::dtype_bytes(out_dtype);
  if (vq::overlaps(out, out_bytes, codes, rows * k / 2) || vq::overlaps(out, out_bytes, scales, rows * k / kBlock)) {
    return vq::fail("mxfp4: out must not overlap codes or scales");
  }
  const int64_t quarters = rows * k / 8;
  const int64_t groups = (quarters + kThreads - 1) / kThreads;
  if (groups > INT_MAX) return vq::fail("mxfp4: too many elements");
  hipLaunchKernelGGL(dequantize_kernel, dim3(unsigned(groups)), dim3(kThreads), 0, static_cast<hipStream_t>(stream),
                     reinterpret_cast<const uint32_t*>(codes), scales, quarters, out, out_dtype);
  return vq::check_launch("mxfp4 dequantize");
}

extern "C" int mxfp4_matmul(const uint8_t* a, const uint8_t* a_scales, int64_t rows, int64_t k, const uint8_t* w,
                            const uint8_t* w_scales, int64_t n, void* out, int out_dtype, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  using namespace mx;
  if (int rc = check_product(rows, k, n, w, w_scales, out_dtype, out)) return rc;
  if (rows == 0 || n == 0) return vq::kOk;
  if (!a || !a_scales) return vq::fail("mxfp4: null pointer");
  if (!aligned(a, 16)) return vq::fail("mxfp4: codes must be 16-byte aligned");
  const int64_t out_bytes = rows * n * vq::dtype_bytes(out_dtype);
  if (vq::overlaps(out, out_bytes, a, rows * k / 2) || vq::overlaps(out, out_bytes, a_scales, rows * k / kBlock)) {
    return vq::fail("mxfp4: out must not overlap the activations");
  }
  (void)workspace;
  (void)workspace_bytes;
  return launch_matmul({a, a_scales, w, w_scales, rows, n, int(k / kBlock), out, out_dtype}, static_cast<hipStream_t>(stream));
}

extern "C" int64_t mxfp4_matmul_workspace_size(int64_t rows, int64_t k, int64_t n) {
  using namespace mx;
  if (rows < 0 || n < 0 || k <= 0 || k % kBlock != 0 || !sane(rows, k) || !sane(rows, n)) {
    vq::fail("mxfp4: k must be a positive multiple of 32, sizes not negative");
    return -1;
  }
  return 0;
}

extern "C" int64_t mxfp4_linear_workspace_size(int64_t rows, int64_t k, int64_t n) {
  using namespace mx;
  if (rows < 0 || n < 0 || k <= 0 || k % kBlock != 0 || !sane(rows, k) || !sane(rows, n)) {
    vq::fail("mxfp4: k must be a positive multiple of 32, sizes not negative");
    return -1;
  }
  return rows * (k / 2) + (rows * (k / kBlock) + 15) / 16 * 16;
}

extern "C" int mxfp4_linear(const void* x, int x_dtype, int64_t rows, int64_t k, int64_t x_stride, const uint8_t* w,
                            const uint8_t* w_scales, int64_t n, void* out, int out_dtype, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  using namespace mx;
  if (int rc = check_rows(x, x_dtype, rows, k, x_stride)) return rc;
  if (int rc = check_product(rows, k, n, w, w_scales, out_dtype, out)) return rc;
  if (rows == 0 || n == 0) return vq::kOk;
  const int64_t x_bytes = ((rows - 1) * x_stride + k) * vq::dtype_bytes(x_dtype);
  const int64_t out_bytes = rows * n * vq::dtype_bytes(out_dtype);
  if (vq::overlaps(out, out_bytes, x, x_bytes)) return vq::fail("mxfp4: out must not overlap x");
  const int64_t need = mxfp4_linear_workspace_size(rows, k, n);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16)) {
    return vq::fail("mxfp4: workspace too small or not 16-byte aligned");
  }
  if (vq::overlaps(workspace, need, x, x_bytes) || vq::overlaps(workspace, need, out, out_bytes) ||
      vq::overlaps(workspace, need, w, n * k / 2) || vq::overlaps(workspace, need, w_scales, n * k / kBlock)) {
    return vq::fail("mxfp4: the workspace must not overlap another argument");
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  uint8_t* scales = codes + rows * (k / 2);
  if (int rc = launch_quantize(x, x_dtype, rows, k, x_stride, codes, scales, s)) return rc;
  return launch_matmul({codes, scales, w, w_scales, rows, n, int(k / kBlock), out, out_dtype}, s);
}

#ifdef MX_TUNE
extern "C" void mx_force(int f) { mx::g_force = f; }
#endif
