// The fused MoE with MXFP4 weights (mxfp4.h): the routed slots grouped by
// expert (moe_rows.h), gate | up with the SwiGLU, down with the router weight,
// the slot sum.  Activations are quantized to MXFP4 on the way in, and the
// SwiGLU's output on its way to the down projection.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "../../include/vllm_mi355x.h"
#include "moe_rows.h"
#include "mxfp4.h"
#include "mxfp4_tile.h"

namespace mx {
namespace {

constexpr int kThreads = 256;
constexpr int kTaskRows = 16;
constexpr int kTileRows = 128;  // rows of a task on the tile kernel
#ifdef MX_TUNE
int g_moe_force = 0;
#endif

// The local expert of a slot: through the map where the call brings one, -1
// outside [0, experts).
struct ExpertOf {
  const int32_t *ids, *map;
  int64_t map_size;
  int experts;
  __device__ __forceinline__ int operator()(int64_t slot) const {
    int id = ids[slot];
    if (map) id = id >= 0 && id < map_size ? map[id] : -1;
    return id >= 0 && id < experts ? id : -1;
  }
};

// Workgroups 0 .. parts - 1 count the slots; the others quantize the rows of x,
// four lanes a block.
template <int kDtype>
__global__ __launch_bounds__(moe::kRowsPartThreads) void count_quantize_kernel(ExpertOf of, moe::RowsLayout lay, int32_t* table,
                                                                               const void* x, int64_t tokens, int blocks,
                                                                               int64_t stride, bool wide, uint32_t* codes,
                                                                               uint8_t* scales) {
  extern __shared__ int part_count[];
  const int64_t parts = lay.parts();
  if (blockIdx.x < parts) {
    moe::rows_count_part(of, lay, table, int(blockIdx.x), part_count);
    return;
  }
  const int64_t quarter = int64_t(blockIdx.x - parts) * moe::kRowsPartThreads + threadIdx.x;
  const int64_t b = quarter >> 2;
  const int j = int(quarter & 3);
  if (b >= tokens * blocks) return;
  const int64_t r = b / blocks;
  const int c = int(b - r * blocks);
  uint32_t s;
  codes[quarter] = quantize_quarter(load8<kDtype>(x, r * stride + int64_t(c) * kBlock + 8 * j, wide), s);
  if (j == 0) scales[b] = uint8_t(s);
}

__global__ __launch_bounds__(moe::kRowsPartThreads) void fill_kernel(moe::RowsLayout lay, int32_t* table, int task_rows) {
  extern __shared__ int first[];
  moe::rows_fill_part(lay, table, task_rows, int(blockIdx.x), first);
}

struct GemmArgs {
  const uint8_t *a, *as;  // rows of k: tokens (gate | up), sorted rows (down)
  const uint8_t *w, *ws;  // [experts][n][k]
  const int32_t* table;
  int64_t tasks, sorted;  // offsets in the table
  const float* topk_w;
  int top_k, n, blocks;   // k / 32
  float limit;
  uint8_t *h, *hs;        // gate | up: rows of n / 2
  float* out;             // down: [slots][n]
};

// 16 x 16 sums of rows `arow` (one per lane & 15) with weight rows `wrow`.
__device__ __forceinline__ f32x4_t row_tile(const GemmArgs& g, int64_t arow, int64_t wrow, int q) {
  const uint8_t* a = g.a + arow * g.blocks * kBlockBytes;
  const uint8_t* w = g.w + wrow * g.blocks * kBlockBytes;
  const uint8_t* as = g.as + arow * g.blocks;
  const uint8_t* ws = g.ws + wrow * g.blocks;
  f32x4_t acc{0, 0, 0, 0};
  for (int b0 = 0; b0 < g.blocks; b0 += 4) {
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
  return acc;
}

// One wavefront: a task's rows (at most 16) by 32 columns of h.
__global__ __launch_bounds__(64) void gate_up_kernel(GemmArgs g) {
  const int task = blockIdx.y;
  if (task >= g.table[0]) return;
  const int4 tk = reinterpret_cast<const int4*>(g.table + g.tasks)[task];
  const int lane = threadIdx.x, r = lane & 15, q = lane >> 4;
  const int inter = g.n / 2;
  const int c0 = blockIdx.x * kBlock;
  const int t = min(r, tk.z - 1);
  const int64_t row = tk.y + t;
  const int64_t token = g.table[g.sorted + row] / g.top_k;
  const int64_t w0 = int64_t(tk.x) * g.n + c0 + r;
  float v[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x4_t gate = row_tile(g, token, w0 + 16 * i, q);
    const f32x4_t up = row_tile(g, token, w0 + inter + 16 * i, q);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[4 * i + j] = swiglu(gate[j], up[j], g.limit);
  }
  // the row's 32 columns lie in its four lanes (q): elements 4 q + j and 16 + 4 q + j
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, magnitude(v[j]));
  top = max(top, uint32_t(__shfl_xor(int(top), 16)));
  top = max(top, uint32_t(__shfl_xor(int(top), 32)));
  const uint32_t s = block_scale(top);
  const uint32_t w = s == 255u ? 0u : codes8(v, s);
  if (r >= tk.z) return;
  uint16_t* out = reinterpret_cast<uint16_t*>(g.h + row * (inter / 2) + c0 / 2);
  out[q] = uint16_t(w);
  out[4 + q] = uint16_t(w >> 16);
  if (q == 0) g.hs[row * (inter / kBlock) + blockIdx.x] = uint8_t(s);
}

// One wavefront: a task's rows by 16 columns of the slot rows.
__global__ __launch_bounds__(64) void down_kernel(GemmArgs g) {
  const int task = blockIdx.y;
  if (task >= g.table[0]) return;
  const int4 tk = reinterpret_cast<const int4*>(g.table + g.tasks)[task];
  const int lane = threadIdx.x, r = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int64_t row = tk.y + min(r, tk.z - 1);
  const int slot = g.table[g.sorted + row];
  const f32x4_t acc = row_tile(g, row, int64_t(tk.x) * g.n + min(n0 + r, g.n - 1), q);
  if (r >= tk.z) return;
  const float weight = g.topk_w[slot];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = n0 + 4 * q + i;
    if (n < g.n) g.out[int64_t(slot) * g.n + n] = weight * acc[i];
  }
}

// out[t][c] = RN(sum over t's slots with a local expert, in slot order).
__global__ __launch_bounds__(kThreads) void slot_sum_kernel(const float* in, ExpertOf of, int64_t tokens, int top_k, int hidden,
                                                            void* out, int dtype) {
  const int64_t i = (int64_t(blockIdx.x) * kThreads + threadIdx.x) * 4;
  if (i >= tokens * hidden) return;
  const int64_t t = i / hidden;
  const int64_t c = i - t * hidden;
  f32x4_t sum{0, 0, 0, 0};
  for (int k = 0; k < top_k; ++k) {
    if (of(t * top_k + k) < 0) continue;
    const f32x4_t v = *reinterpret_cast<const f32x4_t*>(in + (t * top_k + k) * hidden + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] += v[j];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) vq::store_act(out, dtype, i + j, sum[j]);
}

// Byte offsets of a call's workspace, each part 16-byte aligned.
struct Workspace {
  int64_t xq, xs, hq, hs, c3, table, total;
};

moe::RowsLayout layout_of(int64_t slots, int64_t experts) { return {slots, experts, slots / 16 + std::min(experts, slots)}; }

Workspace workspace_of(int64_t tokens, int64_t top_k, int64_t hidden, int64_t inter, int64_t experts) {
  const int64_t slots = tokens * top_k;
  Workspace w{};
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t start = at;
    at += (bytes + 15) / 16 * 16;
    return start;
  };
  w.xq = take(tokens * hidden / 2);
  w.xs = take(tokens * hidden / kBlock);
  w.hq = take(slots * inter / 2);
  w.hs = take(slots * inter / kBlock);
  w.c3 = take(slots * hidden * 4);
  w.table = take(layout_of(slots, experts).total() * 4);
  w.total = at;
  return w;
}

}  // namespace
}  // namespace mx

extern "C" int64_t mxfp4_moe_workspace_size(int64_t tokens, int64_t top_k, int64_t hidden, int64_t inter, int64_t experts) {
  using namespace mx;
  if (tokens < 0 || top_k <= 0 || tokens > INT_MAX / top_k || hidden <= 0 || inter <= 0 || hidden % kBlock != 0 ||
      inter % kBlock != 0 || hidden > (1 << 24) || inter > (1 << 24) || experts <= 0 || experts > moe::kRowsMaxExperts) {
    vq::fail("mxfp4 moe: sizes out of range (hidden and intermediate multiples of 32, at most 1024 experts)");
    return -1;
  }
  return workspace_of(tokens, top_k, hidden, inter, experts).total;
}

extern "C" int mxfp4_moe(const void* x, int act_dtype, int64_t tokens, int64_t x_stride, const uint8_t* w13, const uint8_t* s13,
                         const uint8_t* w2, const uint8_t* s2, int64_t experts, const int32_t* topk_ids, const float* topk_w,
                         int64_t top_k, const int32_t* expert_map, int64_t map_size, int64_t hidden, int64_t inter, float limit,
                         void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace mx;
  if (act_dtype != vq::kBF16 && act_dtype != vq::kFP16) return vq::fail("mxfp4 moe: bf16 or fp16 activations");
  const int64_t need = mxfp4_moe_workspace_size(tokens, top_k, hidden, inter, experts);
  if (need < 0) return vq::kInvalidArgument;
  if (x_stride < hidden || x_stride > (int64_t(1) << 40)) return vq::fail("mxfp4 moe: row stride out of range");
  if (std::isnan(limit) || limit <= 0) return vq::fail("mxfp4 moe: limit must be positive");
  if (tokens == 0) return vq::kOk;
  if (!x || !w13 || !s13 || !w2 || !s2 || !topk_ids || !topk_w || !out || map_size < 0 || (map_size > 0 && !expert_map)) {
    return vq::fail("mxfp4 moe: null pointer");
  }
  if (!aligned(w13, 16) || !aligned(w2, 16)) return vq::fail("mxfp4 moe: codes must be 16-byte aligned");
  if (!aligned(x, 2) || !aligned(out, 2) || !aligned(topk_ids, 4) || !aligned(topk_w, 4)) return vq::fail("mxfp4 moe: misaligned pointer");
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16)) return vq::fail("mxfp4 moe: workspace too small or not 16-byte aligned");
  const int64_t slots = tokens * top_k;
  const Workspace ws = workspace_of(tokens, top_k, hidden, inter, experts);
  const moe::RowsLayout lay = layout_of(slots, experts);
  uint8_t* base = static_cast<uint8_t*>(workspace);
  int32_t* table = reinterpret_cast<int32_t*>(base + ws.table);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const ExpertOf of{topk_ids, map_size > 0 ? expert_map : nullptr, map_size, int(experts)};
  const int64_t hb = hidden / kBlock, ib = inter / kBlock;
  const int64_t groups = lay.parts() + (tokens * hb * 4 + moe::kRowsPartThreads - 1) / moe::kRowsPartThreads;
  const int64_t sums = (tokens * hidden / 4 + kThreads - 1) / kThreads;
  if (groups > INT_MAX || sums > INT_MAX || lay.max_tasks > 65535) return vq::fail("mxfp4 moe: too many rows");
  const bool wide = aligned(x, 16) && x_stride % 8 == 0;
  const size_t lds = size_t(experts) * sizeof(int);
  bool tiles = slots >= 24 * std::min(experts, slots) && hb >= kStageBlocks && ib >= kStageBlocks && hidden * inter < (int64_t(1) << 31) &&
               tokens * hidden / 2 < (int64_t(1) << 31);
#ifdef MX_TUNE
  if (g_moe_force) tiles = g_moe_force == 2;
#endif
  uint32_t* xq = reinterpret_cast<uint32_t*>(base + ws.xq);
  if (act_dtype == vq::kBF16) {
    hipLaunchKernelGGL(count_quantize_kernel<vq::kBF16>, dim3(unsigned(groups)), dim3(moe::kRowsPartThreads), lds, st, of, lay, table,
                       x, tokens, int(hb), x_stride, wide, xq, base + ws.xs);
  } else {
    hipLaunchKernelGGL(count_quantize_kernel<vq::kFP16>, dim3(unsigned(groups)), dim3(moe::kRowsPartThreads), lds, st, of, lay, table,
                       x, tokens, int(hb), x_stride, wide, xq, base + ws.xs);
  }
  if (int rc = vq::check_launch("mxfp4 moe count")) return rc;
  hipLaunchKernelGGL(fill_kernel, dim3(unsigned(lay.parts())), dim3(moe::kRowsPartThreads), lds, st, lay, table, tiles ? kTileRows : kTaskRows);
  if (int rc = vq::check_launch("mxfp4 moe fill")) return rc;
  if (tiles) {
    TileArgs t{};
    t.a = base + ws.xq;
    t.as = base + ws.xs;
    t.a_rows = tokens;
    t.w = w13;
    t.ws = s13;
    t.n = 2 * inter;
    t.blocks = int(hb);
    t.tiles_n = int((inter + 63) / 64);
    t.table = table;
    t.tasks = lay.tasks();
    t.sorted = lay.sorted();
    t.topk_w = topk_w;
    t.top_k = int(top_k);
    t.limit = limit;
    t.h = base + ws.hq;
    t.hs = base + ws.hs;
    const int64_t bound = (slots / kTileRows + std::min(experts, slots) + 7) / 8 * 8;
    hipLaunchKernelGGL((tile_kernel<2, 2, kGateUp>), dim3(unsigned(bound * t.tiles_n)), dim3(kTileThreads), 0, st, t);
    if (int rc = vq::check_launch("mxfp4 moe gate_up")) return rc;
    t.a = base + ws.hq;
    t.as = base + ws.hs;
    t.w = w2;
    t.ws = s2;
    t.n = hidden;
    t.blocks = int(ib);
    t.tiles_n = int((hidden + 127) / 128);
    t.out = base + ws.c3;
    hipLaunchKernelGGL((tile_kernel<2, 2, kDown>), dim3(unsigned(bound * t.tiles_n)), dim3(kTileThreads), 0, st, t);
    if (int rc = vq::check_launch("mxfp4 moe down")) return rc;
    hipLaunchKernelGGL(slot_sum_kernel, dim3(unsigned(sums)), dim3(kThreads), 0, st, static_cast<const float*>(t.out), of, tokens, int(top_k), int(hidden), out, act_dtype);
    return vq::check_launch("mxfp4 moe sum");
  }
  GemmArgs g{};
  g.a = base + ws.xq;
  g.as = base + ws.xs;
  g.w = w13;
  g.ws = s13;
  g.table = table;
  g.tasks = lay.tasks();
  g.sorted = lay.sorted();
  g.topk_w = topk_w;
  g.top_k = int(top_k);
  g.n = int(2 * inter);
  g.blocks = int(hb);
  g.limit = limit;
  g.h = base + ws.hq;
  g.hs = base + ws.hs;
  hipLaunchKernelGGL(gate_up_kernel, dim3(unsigned(ib), unsigned(lay.max_tasks)), dim3(64), 0, st, g);
  if (int rc = vq::check_launch("mxfp4 moe gate_up")) return rc;
  g.a = base + ws.hq;
  g.as = base + ws.hs;
  g.w = w2;
  g.ws = s2;
  g.n = int(hidden);
  g.blocks = int(ib);
  g.out = reinterpret_cast<float*>(base + ws.c3);
  hipLaunchKernelGGL(down_kernel, dim3(unsigned((hidden + 15) / 16), unsigned(lay.max_tasks)), dim3(64), 0, st, g);
  if (int rc = vq::check_launch("mxfp4 moe down")) return rc;
  hipLaunchKernelGGL(slot_sum_kernel, dim3(unsigned(sums)), dim3(kThreads), 0, st, g.out, of, tokens, int(top_k), int(hidden), out, act_dtype);
  return vq::check_launch("mxfp4 moe sum");
}

#ifdef MX_TUNE
extern "C" void mx_moe_force(int f) { mx::g_moe_force = f; }
#endif
