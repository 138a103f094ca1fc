// MXFP4 (mxfp4.h): quantization, dequantization, and the product of MXFP4
// activations with MXFP4 weights.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "../../include/vllm_mi355x.h"
#include "mxfp4.h"
#include "mxfp4_small.h"
#include "mxfp4_tile.h"

namespace mx {
namespace {

constexpr int kThreads = 256;

// ---- quantization ------------------------------------------------------------

// Four lanes a block, eight elements each: one pass, bound by its bytes (14336 x 4096 in
// FP32, 266 MB: 61-64 us).
template <int kDtype>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const void* x, int64_t rows, int blocks, int64_t stride,
                                                            bool wide, uint32_t* codes, uint8_t* scales) {
  const int64_t quarter = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t b = quarter >> 2;
  const int j = int(quarter & 3);
  if (b >= rows * blocks) return;
  const int64_t r = b / blocks;
  const int c = int(b - r * blocks);
  uint32_t s;
  codes[quarter] = quantize_quarter(load8<kDtype>(x, r * stride + int64_t(c) * kBlock + 8 * j, wide), s);
  if (j == 0) scales[b] = uint8_t(s);
}

// Eight elements a thread, bound by its bytes (the same matrix to FP32, 266 MB: 46 us).
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

struct SmallArgs {
  const void* x;            // unquantized rows, or
  int64_t stride;
  bool wide;
  const uint8_t *a, *as;    // their codes and scales
  const uint8_t *w, *ws;
  int64_t rows, n;
  int blocks;  // k / 32
  void* out;
  int out_dtype;
  int64_t groups_n;  // column groups
  int groups_m;      // row groups
};

struct MatmulArgs {
  const uint8_t *a, *as, *w, *ws;
  int64_t rows, n;
  int blocks;  // k / 32
  void* out;
  int out_dtype;
};

// Few rows: a workgroup of kCols x `parts` wavefronts has 16 kCols columns and 16
// rows, chunk c of K multiplied by part c % parts; the parts' sums are added
// through LDS in order.  kQuantize: x comes unquantized and is quantized into
// LDS, while the first weights are on their way; else its codes come from memory
// (L2, after the first workgroup).  Bound by the weight stream or, of small matrices,
// by one chain of loads: 4096 x 14336, one row, 9.0 us (31 MB); 2592 x 5003, 20 rows,
// 6.7 us (7 MB).
template <int kCols, bool kQuantize, int kDtype>
__global__ __launch_bounds__(1024, 4) void small_kernel(SmallArgs g) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63;
  const int wave = vq::uniform(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int col = wave % kCols, part = wave / kCols, parts = threads / 64 / kCols;
  const int chunks = (g.blocks + kChunk - 1) / kChunk;
  // workgroups b, b + 8, ... run on one XCD: the row groups of a column group
  // follow each other there, so that its L2 fetches the weights once
  const int local = int(blockIdx.x >> 3);
  const int64_t group = int64_t(local / g.groups_m) * 8 + (blockIdx.x & 7);
  if (group >= g.groups_n) return;
  const int64_t n0 = (group * kCols + col) * 16;
  const int64_t m0 = int64_t(local % g.groups_m) * 16;
  const int rows = int(min(int64_t(16), g.rows - m0));
  const int64_t wrow = min(n0 + r, g.n - 1);
  const uint8_t* w = g.w + wrow * g.blocks * kBlockBytes;
  const uint8_t* ws = g.ws + wrow * g.blocks;
  const auto weights = [&](int c) {
    ChunkOperand o{};
    if (c < chunks) o = load_chunk(w, ws, c, g.blocks, q);
    return o;
  };
  f32x4_t acc{0, 0, 0, 0};
  if constexpr (kQuantize) {
    ChunkOperand a = weights(part), b = weights(part + parts);
    quantize_to_lds<kDtype>(g.x, [&](int m) { return (m0 + m) * g.stride; }, rows, g.blocks, chunks, g.wide, lds, tid, threads);
    __syncthreads();
    for (int c = part; c < chunks; c += parts) {
      const ChunkOperand next = weights(c + 2 * parts);
      multiply_lds(a, lds, c, rows, chunks, r, q, acc);
      a = b;
      b = next;
    }
  } else {
    const int64_t row = m0 + min(r, rows - 1);
    const uint8_t* x = g.a + row * g.blocks * kBlockBytes;
    const uint8_t* xs = g.as + row * g.blocks;
    const auto activations = [&](int c) {
      ChunkOperand o{};
      if (c < chunks) o = load_chunk(x, xs, c, g.blocks, q);
      return o;
    };
    ChunkOperand a = weights(part), ax = activations(part);
    for (int c = part; c < chunks; c += parts) {
      const ChunkOperand next = weights(c + parts), nx = activations(c + parts);
      multiply_loaded(a, ax, acc);
      a = next;
      ax = nx;
    }
  }
  // the sums of parts 1, 2, ... through LDS, [part - 1][col][lane]
  f32x4_t* sums = reinterpret_cast<f32x4_t*>(lds);
  __syncthreads();
  if (part > 0) sums[((part - 1) * kCols + col) * 64 + lane] = acc;
  __syncthreads();
  if (part > 0) return;
  for (int p = 1; p < parts; ++p) acc += sums[((p - 1) * kCols + col) * 64 + lane];
  if (r >= rows) return;
  const int64_t at = (m0 + r) * g.n;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t n = n0 + 4 * q + i;
    if (n < g.n) vq::store_act(g.out, g.out_dtype, at + n, acc[i]);
  }
}

// out[i] = RN(part 0's i + part 1's i + ...), eight elements a thread (two parts of
// 400 x 4096: 5 us, most of it the launch).
__global__ __launch_bounds__(kThreads) void combine_kernel(const float* part, int splits, int64_t numel, void* out, int dtype) {
  const int64_t i = (int64_t(blockIdx.x) * kThreads + threadIdx.x) * 8;
  if (i >= numel) return;
  float v[8];
  if (i + 8 <= numel && (numel & 3) == 0) {
    f32x4_t a{0, 0, 0, 0}, b{0, 0, 0, 0};
    for (int p = 0; p < splits; ++p) {
      a += *reinterpret_cast<const f32x4_t*>(part + p * numel + i);
      b += *reinterpret_cast<const f32x4_t*>(part + p * numel + i + 4);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = a[j];
      v[4 + j] = b[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = 0;
      for (int p = 0; p < splits && i + j < numel; ++p) v[j] += part[p * numel + i + j];
    }
  }
  vq::store8_act(out, dtype, i, v, numel - i);
}

template <int kSize, int kBufs>
int launch_tile(const MatmulArgs& g, int splits, float* part, hipStream_t s) {
  TileArgs t{};
  t.a = g.a;
  t.as = g.as;
  t.w = g.w;
  t.ws = g.ws;
  t.rows = g.rows;
  t.n = g.n;
  t.blocks = g.blocks;
  t.out = splits > 1 ? part : g.out;
  t.out_dtype = splits > 1 ? int(vq::kFP32) : g.out_dtype;
  t.tiles_n = int((g.n + 64 * kSize - 1) / (64 * kSize));
  t.tiles_m = int((g.rows + 64 * kSize - 1) / (64 * kSize));
  const int stages = (g.blocks + kStageBlocks - 1) / kStageBlocks;
  t.split_stages = (stages + splits - 1) / splits;
  const int64_t total = int64_t(t.tiles_n) * t.tiles_m;
  hipLaunchKernelGGL((tile_kernel<kSize, kSize, kDense, kBufs>), dim3(unsigned((total + 7) / 8 * 8), unsigned(splits)), dim3(kTileThreads), 0, s, t);
  if (int rc = vq::check_launch("mxfp4 tile")) return rc;
  if (splits == 1) return vq::kOk;
  const int64_t numel = g.rows * g.n;
  hipLaunchKernelGGL(combine_kernel, dim3(unsigned((numel + 8 * kThreads - 1) / (8 * kThreads))), dim3(kThreads), 0, s, part, splits,
                     numel, g.out, g.out_dtype);
  return vq::check_launch("mxfp4 combine");
}

// ---- which kernel ------------------------------------------------------------

// How a product runs.  tile 0: the few-rows kernel, `cols` column tiles and
// `parts` parts of K a workgroup, `fused`: it quantizes x itself; else the tile
// kernel with 64 `tile` columns and rows, K in `splits`, `deep`: four stage
// buffers instead of two.
struct Plan {
  int tile, splits, cols, parts;
  bool fused, deep;
};

constexpr int kCUs = 256;

// The tile kernel's time in us as its workgroups fill the chip: a stage costs
// `alone` where a workgroup has a CU's loads and matrix cores for itself, and
// `shared` per workgroup of a CU that is full; K splits write and read FP32 sums
// at about 3 TB/s, in one more launch.  Fitted to the tile sizes and splits
// measured at 24 to 4096 rows of 4096 x 14336, 14336 x 4096, 4096 x 4096 and
// 2592 x 5003: at 52 sizes the fastest, or one within 12% of it, is picked.  `lines`: rows of codes
// begin on 128-byte lines; the others' stages take longer, most of all the largest
// tiles' (1500 rows of 2592 x 5003: 38 us, 26 on 128 x 128).
double tile_cost(int size, bool deep, bool lines, int64_t rows, int64_t n, int64_t stages, int64_t splits) {
  const double alone = size == 4 ? (lines ? 1.48 : 2.4) : size == 2 ? (deep ? 0.52 : 0.72) * (lines ? 1 : 1.12) : lines ? 0.30 : 0.33;
  const double shared = (size == 4 ? 2.2 : size == 2 ? (deep ? 0.60 : 0.80) : 0.385) * (lines ? 1 : 1.25);
  const int64_t groups = ((n + 64 * size - 1) / (64 * size)) * ((rows + 64 * size - 1) / (64 * size)) * splits;
  // whole rounds where a CU holds one workgroup
  const bool one = size == 4 || deep;
  const double load = one ? double((groups + kCUs - 1) / kCUs) : double(groups) / kCUs;
  // (four buffers' workgroups gain nothing from each other over rounds)
  const double each = one && groups < kCUs / 2 ? alone : std::max(alone, (deep && load > 1 ? (lines ? 0.95 : 1.19) : shared) * load);
  const double sums = splits > 1 ? 3.0 + double(rows) * double(n) * 8.0 * double(splits) / 3e6 : 0.0;
  return double((stages + splits - 1) / splits) * each + sums;
}

Plan plan_of(int64_t rows, int64_t k, int64_t n) {
  Plan p{0, 1, 1, 1, false, false};
  const int64_t blocks = k / kBlock, stages = (blocks + kStageBlocks - 1) / kStageBlocks;
  // the tile kernel wants whole stages, buffers below 2 GiB and a 32-bit grid
  const bool tiles = rows > 16 && blocks >= kStageBlocks && k <= (int64_t(1) << 22) &&
                     ((n + 63) / 64) * ((rows + 63) / 64) <= INT_MAX / 8;
  // A group of 16 rows reads the weights once more, from L2: 20 rows of 2592 x
  // 5003 10.6 us (tiles 13.0), 64 rows 11.4 (13.9), but 20 rows of 4096 x 14336
  // 20.9 (15.3).  Near the border the product alone may lose a fifth by it (40 rows
  // of 4096 x 4096 10.2, on tiles 8.4).
  if (tiles && (rows > 64 || (rows + 15) / 16 * double(n) * double(k) > 64e6)) {
    double best = 0;
    for (const int kind : {1, 2, 3, 4}) {  // 3: size 2 with four buffers
      const int size = kind == 3 ? 2 : kind;
      for (const int splits : {1, 2, 4, 8}) {
        if (splits > 1 && stages < 4 * splits) continue;
        const double cost = tile_cost(size, kind == 3, k % (2 * 128) == 0, rows, n, stages, splits);
        if (!p.tile || cost < best) {
          best = cost;
          p.tile = size;
          p.splits = splits;
          p.deep = kind == 3;
        }
      }
    }
  }
  if (!p.tile) {
    // wide enough workgroups to share the activations, wavefronts enough to have
    // all of a small matrix in flight: one row of 4096 x 14336 9.1 us with 4 column
    // tiles and 4 parts (1 and 4: 9.8, 1 and 16: 13.6), of 14336 x 4096 9.2 with 1
    // and 16 (4 and 4: 18.5)
    const int64_t groups = (n + 15) / 16, chunks = (blocks + kChunk - 1) / kChunk;
    p.cols = groups >= 800 ? 4 : groups >= 400 ? 2 : 1;
    while (2 * p.parts * p.cols <= 16 && 2 * p.parts <= chunks && groups * p.parts < 3500) p.parts *= 2;
    // every workgroup quantizes its rows itself, as long as that is less than a
    // launch (per CU 28k elements 11.7 against 13.2 us, 57k 15.6 against 14.7 and
    // 11.8 against 11.4)
    const int64_t groups_cu = ((groups + p.cols - 1) / p.cols + kCUs - 1) / kCUs;
    p.fused = rows <= 16 && groups_cu * rows * k <= 40960;
  }
  if (p.splits > 1) p.splits = int((stages + (stages + p.splits - 1) / p.splits - 1) / ((stages + p.splits - 1) / p.splits));
  return p;
}

// Bytes of rows' codes and scales, in whole sixteens.
int64_t packed_bytes(int64_t rows, int64_t k) { return rows * (k / 2) + (rows * (k / kBlock) + 15) / 16 * 16; }

// Bytes of a plan's K splits.
int64_t split_bytes(const Plan& p, int64_t rows, int64_t n) { return p.tile && p.splits > 1 ? p.splits * rows * n * 4 : 0; }

template <int kCols, bool kQuantize, int kDtype>
int launch_small_as(SmallArgs g, int parts, hipStream_t s) {
  g.groups_n = (g.n + 16 * kCols - 1) / (16 * kCols);
  g.groups_m = int((g.rows + 15) / 16);
  const int64_t chunks = (g.blocks + kChunk - 1) / kChunk, rows = std::min<int64_t>(g.rows, 16);
  const int64_t lds = std::max<int64_t>(kQuantize ? small_bytes(rows, chunks) : 0, int64_t(parts - 1) * kCols * 1024);
  const int64_t grid = (g.groups_n + 7) / 8 * 8 * ((g.rows + 15) / 16);
  if (grid > INT_MAX) return vq::fail("mxfp4: too many rows or columns");
  hipLaunchKernelGGL((small_kernel<kCols, kQuantize, kDtype>), dim3(unsigned(grid)), dim3(64 * kCols * parts), size_t(lds), s, g);
  return vq::check_launch("mxfp4 few rows");
}

template <bool kQuantize, int kDtype>
int launch_small(const SmallArgs& g, const Plan& p, hipStream_t s) {
  if (p.cols == 4) return launch_small_as<4, kQuantize, kDtype>(g, p.parts, s);
  if (p.cols == 2) return launch_small_as<2, kQuantize, kDtype>(g, p.parts, s);
  return launch_small_as<1, kQuantize, kDtype>(g, p.parts, s);
}

SmallArgs small_args(const MatmulArgs& g) {
  SmallArgs m{};
  m.a = g.a;
  m.as = g.as;
  m.w = g.w;
  m.ws = g.ws;
  m.rows = g.rows;
  m.n = g.n;
  m.blocks = g.blocks;
  m.out = g.out;
  m.out_dtype = g.out_dtype;
  return m;
}

int launch_matmul(const MatmulArgs& g, const Plan& p, float* part, hipStream_t s) {
  if (p.tile == 4) return launch_tile<4, 2>(g, p.splits, part, s);
  if (p.tile == 2) return p.deep ? launch_tile<2, 4>(g, p.splits, part, s) : launch_tile<2, 2>(g, p.splits, part, s);
  if (p.tile == 1) return launch_tile<1, 4>(g, p.splits, part, s);
  return launch_small<false, vq::kBF16>(small_args(g), p, s);
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

// The longest sum of a product: a row's blocks, and what the kernels count in them, fit
// 32 bits.
constexpr int64_t kMaxK = int64_t(1) << 32;

bool known_dtype(int dtype) { return dtype == vq::kBF16 || dtype == vq::kFP16 || dtype == vq::kFP32; }

int check_product(int64_t rows, int64_t k, int64_t n, const uint8_t* w, const uint8_t* w_scales, int out_dtype, const void* out) {
  if (!known_dtype(out_dtype)) return vq::fail("mxfp4: out must be BF16, FP16 or FP32");
  if (rows < 0 || n < 0 || k <= 0 || k % kBlock != 0) return vq::fail("mxfp4: k must be a positive multiple of 32");
  if (k > kMaxK || !sane(rows, k) || !sane(n, k) || !sane(rows, n)) return vq::fail("mxfp4: sizes out of range");
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
  const Plan p = plan_of(rows, k, n);
  const int64_t need = split_bytes(p, rows, n);
  if (need > 0) {
    if (!workspace || workspace_bytes < need || !aligned(workspace, 16)) {
      return vq::fail("mxfp4: workspace too small or not 16-byte aligned");
    }
    if (vq::overlaps(workspace, need, a, rows * k / 2) || vq::overlaps(workspace, need, a_scales, rows * k / kBlock) ||
        vq::overlaps(workspace, need, out, out_bytes) || vq::overlaps(workspace, need, w, n * k / 2) ||
        vq::overlaps(workspace, need, w_scales, n * k / kBlock)) {
      return vq::fail("mxfp4: the workspace must not overlap another argument");
    }
  }
  return launch_matmul({a, a_scales, w, w_scales, rows, n, int(k / kBlock), out, out_dtype}, p, static_cast<float*>(workspace),
                       static_cast<hipStream_t>(stream));
}

extern "C" int64_t mxfp4_matmul_workspace_size(int64_t rows, int64_t k, int64_t n) {
  using namespace mx;
  if (rows < 0 || n < 0 || k <= 0 || k % kBlock != 0 || k > kMaxK || !sane(rows, k) || !sane(rows, n)) {
    vq::fail("mxfp4: k must be a positive multiple of 32 up to 2^32, sizes not negative");
    return -1;
  }
  return split_bytes(plan_of(rows, k, n), rows, n);
}

extern "C" int mxfp4_matmul_plan(int64_t rows, int64_t k, int64_t n, int32_t* plan) {
  using namespace mx;
  if (!plan) return vq::fail("mxfp4: null pointer");
  if (mxfp4_matmul_workspace_size(rows, k, n) < 0) return vq::kInvalidArgument;
  const Plan p = plan_of(rows, k, n);
  plan[0] = 64 * p.tile;
  plan[1] = p.tile == 1 || p.deep ? 4 : p.tile ? 2 : 0;
  plan[2] = p.splits;
  plan[3] = p.cols;
  plan[4] = p.parts;
  plan[5] = p.fused;
  return vq::kOk;
}

extern "C" int64_t mxfp4_linear_workspace_size(int64_t rows, int64_t k, int64_t n) {
  using namespace mx;
  if (rows < 0 || n < 0 || k <= 0 || k % kBlock != 0 || k > kMaxK || !sane(rows, k) || !sane(rows, n)) {
    vq::fail("mxfp4: k must be a positive multiple of 32 up to 2^32, sizes not negative");
    return -1;
  }
  const Plan p = plan_of(rows, k, n);
  return (p.fused ? 0 : packed_bytes(rows, k)) + split_bytes(p, rows, n);
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
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const Plan p = plan_of(rows, k, n);
  const MatmulArgs g{nullptr, nullptr, w, w_scales, rows, n, int(k / kBlock), out, out_dtype};
  if (p.fused) {
    SmallArgs m = small_args(g);
    m.x = x;
    m.stride = x_stride;
    m.wide = aligned(x, 16) && x_stride * vq::dtype_bytes(x_dtype) % 16 == 0;
    if (x_dtype == vq::kBF16) return launch_small<true, vq::kBF16>(m, p, s);
    if (x_dtype == vq::kFP16) return launch_small<true, vq::kFP16>(m, p, s);
    return launch_small<true, vq::kFP32>(m, p, s);
  }
  const int64_t need = mxfp4_linear_workspace_size(rows, k, n);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16)) {
    return vq::fail("mxfp4: workspace too small or not 16-byte aligned");
  }
  if (vq::overlaps(workspace, need, x, x_bytes) || vq::overlaps(workspace, need, out, out_bytes) ||
      vq::overlaps(workspace, need, w, n * k / 2) || vq::overlaps(workspace, need, w_scales, n * k / kBlock)) {
    return vq::fail("mxfp4: the workspace must not overlap another argument");
  }
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  uint8_t* scales = codes + rows * (k / 2);
  if (int rc = launch_quantize(x, x_dtype, rows, k, x_stride, codes, scales, s)) return rc;
  MatmulArgs packed = g;
  packed.a = codes;
  packed.as = scales;
  return launch_matmul(packed, p, reinterpret_cast<float*>(codes + packed_bytes(rows, k)), s);
}
