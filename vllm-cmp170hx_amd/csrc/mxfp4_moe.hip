// The fused MoE with MXFP4 weights (mxfp4.h): the routed slots grouped by
// expert (moe_rows.h), gate | up with the SwiGLU, down with the router weight,
// the slot sum.  Activations are quantized to MXFP4 on the way in, and the
// SwiGLU's output on its way to the down projection.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <utility>

#include "../../include/vllm_mi355x.h"
#include "moe_rows.h"
#include "mxfp4.h"
#include "mxfp4_small.h"
#include "mxfp4_tile.h"

namespace mx {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxSize = 65536;  // hidden and intermediate: a row fits LDS
constexpr int kTaskRows = 16;
constexpr int kTileRows = 128;  // rows of a task on the tile kernel

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

// Workgroups 0 .. parts - 1 count the slots (one alone also lists them: no launch
// for that); the others quantize the rows of x, four lanes a block.
// 2048 tokens of 2048 and 16384 slots 6 us, 300 tokens of 2592 with their list 5 us (in
// two launches 4.9 + 4.8).
template <int kDtype>
__global__ __launch_bounds__(moe::kRowsPartThreads) void count_quantize_kernel(ExpertOf of, moe::RowsLayout lay, int32_t* table,
                                                                               int task_rows, const void* x, int64_t tokens, int blocks,
                                                                               int64_t stride, bool wide, uint32_t* codes,
                                                                               uint8_t* scales) {
  extern __shared__ int part_count[];
  const int64_t parts = lay.parts();
  if (blockIdx.x < parts) {
    moe::rows_count_part(of, lay, table, int(blockIdx.x), part_count);
    if (parts == 1) {
      __syncthreads();
      moe::rows_fill_part(lay, table, task_rows, 0, part_count);
    }
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

// ---- few rows an expert ---------------------------------------------------------

constexpr int kScanSlots = 1024;  // slots that a workgroup looks through itself

struct SmallMoeArgs {
  ExpertOf of;
  const void* x;            // kScan: unquantized rows, else
  int64_t stride;
  bool wide;
  const uint8_t *a, *as;    // their codes and scales
  const uint8_t *w, *ws;    // [experts][n][k]
  int slots, top_k;
  int pass;                 // rows that a workgroup takes at a time, 16 or what LDS holds
  int by_slot;              // kScan: workgroups go by slot, the first of an expert's does the work
  const int32_t* table;
  int64_t tasks, sorted;    // offsets in the table
  const float* topk_w;
  int n, blocks;            // k / 32
  float limit;
  uint8_t *h, *hs;          // [slots][inter]
  float* c3;                // [slots][n]
  void* out;
};

// Rows of `chunks` chunks that the kernels below take at a time.  A task of more rows
// goes over its weights again: with LDS for 16 rows of 7168, 2048 tokens on 32 experts
// of 7168 x 192, four a token, take 436 us; with 56 KB, for 15 rows, 575.
int rows_at_once(int64_t slots, int64_t chunks) {
  constexpr int64_t kLds = small_bytes(kTaskRows, 7168 / kBlock / kChunk);
  static_assert(kLds + (kScanSlots + 1) * 4 <= 64 * 1024, "beside the list of slots");
  static_assert(small_bytes(1, kMaxSize / kBlock / kChunk) <= kLds, "one row fits");
  return int(std::min({slots, int64_t(16), kLds / small_bytes(1, chunks)}));
}

// The expert and the slots of workgroup `index`, in slot order; count 0: no work.
// kScan: from the ids themselves (list: LDS of kScanSlots entries); else a task of
// the table.
struct RowsOf {
  int expert, count;
  const int32_t* slots;
};

template <bool kScan>
__device__ __forceinline__ RowsOf rows_of(const SmallMoeArgs& g, int index, int32_t* list, int* count) {
  if constexpr (!kScan) {
    (void)list;
    (void)count;
    if (index >= g.table[0]) return {0, 0, nullptr};
    const int4 tk = reinterpret_cast<const int4*>(g.table + g.tasks)[index];
    return {vq::uniform(tk.x), vq::uniform(tk.z), g.table + g.sorted + vq::uniform(tk.y)};
  } else {
    const int e = g.by_slot ? vq::uniform(g.of(index)) : index;
    if (e < 0) return {0, 0, nullptr};
    if (threadIdx.x < 64) {
      const int lane = threadIdx.x;
      int n = 0;
      constexpr int kEach = 4;
      for (int s0 = 0; s0 < g.slots; s0 += 64 * kEach) {
        int id[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
          const int s = s0 + 64 * u + lane;
          id[u] = s < g.slots ? g.of(s) : -1;
        }
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
          const bool mine = id[u] == e;
          const uint64_t all = __ballot(mine);
          if (mine) list[n + __popcll(all & ((uint64_t(1) << lane) - 1))] = s0 + 64 * u + lane;
          n += __popcll(all);
        }
      }
      // (by slot: an expert's first one has the work)
      if (lane == 0) *count = g.by_slot && list[0] != index ? 0 : n;
    }
    __syncthreads();
    return {e, vq::uniform(*count), list};
  }
}

// gate | up and the SwiGLU for the rows of one expert, 16 at a time, by one block
// of 32 columns of h: wavefront (tile = wave % 4: gate 0, gate 1, up 0, up 1; part
// = wave / 4 of K).  Its sums meet in LDS; one wavefront forms h, four lanes a row.
// For calls of few blocks, whose time is one block's: in us of the call, these and
// whole blocks a wavefront (gate_up_kernel), 1152 blocks of 2048 33 and 38, 1792 blocks
// of 4096 91 and 78.  One token, eight of 128 experts of 2048 x 768: 6.6 us for 13 MB, the
// list, one chain of loads and the sums.
template <int kDtype>
__global__ __launch_bounds__(1024, 4) void gate_up_split_kernel(SmallMoeArgs g) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ int32_t list[kScanSlots];
  __shared__ int count;
  constexpr int kRow = 20;  // floats of a row's 16 sums in LDS
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63;
  const int wave = vq::uniform(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int tile = wave & 3, part = wave >> 2, parts = threads >> 8;
  const int inter = g.n / 2, groups = inter / kBlock;
  const int c0 = int(blockIdx.x) % groups * kBlock;
  const RowsOf rows = rows_of<true>(g, int(blockIdx.x) / groups, list, &count);
  if (rows.count == 0) return;
  const int chunks = (g.blocks + kChunk - 1) / kChunk;
  const int64_t wrow = int64_t(rows.expert) * g.n + (tile & 2 ? inter : 0) + c0 + 16 * (tile & 1) + r;
  const uint8_t* w = g.w + wrow * g.blocks * kBlockBytes;
  const uint8_t* ws = g.ws + wrow * g.blocks;
  const auto weights = [&](int c) {
    ChunkOperand o{};
    if (c < chunks) o = load_chunk(w, ws, c, g.blocks, q);
    return o;
  };
  float* sums = reinterpret_cast<float*>(lds);
  for (int m0 = 0; m0 < rows.count; m0 += g.pass) {
    const int here = min(rows.count - m0, g.pass);
    f32x4_t acc{0, 0, 0, 0};
    ChunkOperand a = weights(part), b = weights(part + parts);
    quantize_to_lds<kDtype>(g.x, [&](int m) { return int64_t(rows.slots[m0 + m] / g.top_k) * g.stride; }, here, g.blocks, chunks,
                            g.wide, lds, tid, threads);
    __syncthreads();
    for (int c = part; c < chunks; c += parts) {
      const ChunkOperand next = weights(c + 2 * parts);
      multiply_lds(a, lds, c, here, chunks, r, q, acc);
      a = b;
      b = next;
    }
    __syncthreads();
    *reinterpret_cast<f32x4_t*>(sums + ((part * 4 + tile) * 16 + r) * kRow + 4 * q) = acc;
    __syncthreads();
    if (wave == 0) {
      const int m = lane >> 2, j = lane & 3;
      // columns 8 j .. 8 j + 7 of the block: tile j / 2, 8 (j & 1) on
      float gate[8], up[8];
      const auto eight = [&](int t, float (&v)[8]) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 0;
        for (int p = 0; p < parts; ++p) {
          const float* at = sums + ((p * 4 + t) * 16 + m) * kRow + 8 * (j & 1);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] += at[k];
        }
      };
      eight(j >> 1, gate);
      eight(2 + (j >> 1), up);
      Eight<vq::kFP32> v;
#pragma unroll
      for (int k = 0; k < 8; ++k) v.w[k] = __builtin_bit_cast(uint32_t, swiglu(gate[k], up[k], g.limit));
      uint32_t s;
      const uint32_t code = quantize_quarter(v, s);
      if (m < here) {
        const int64_t slot = rows.slots[m0 + m];
        *reinterpret_cast<uint32_t*>(g.h + slot * (inter / 2) + c0 / 2 + 4 * j) = code;
        if (j == 0) g.hs[slot * groups + c0 / kBlock] = uint8_t(s);
      }
    }
    __syncthreads();
  }
}

// A wavefront's way through weight tiles of 16 rows, chunk by chunk, its loads
// kAhead chunks in front of what it multiplies: tile i of the run lies at
// base(i), its chunks follow each other.
constexpr int kAhead = 2;
template <typename Base>
struct WeightStream {
  const Base& base;
  int tiles, chunks, blocks, q;
  int tile, chunk;  // the next chunk to load
  ChunkOperand ring[kAhead];

  __device__ __forceinline__ ChunkOperand load() {
    ChunkOperand o{};
    if (tile < tiles) {
      const uint8_t *w, *ws;
      base(tile, w, ws);
      o = load_chunk(w, ws, chunk, blocks, q);
      if (++chunk == chunks) {
        chunk = 0;
        ++tile;
      }
    }
    return o;
  }
  __device__ __forceinline__ void start() {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ring[i] = load();
  }
  __device__ __forceinline__ ChunkOperand next() {
    const ChunkOperand o = ring[0];
#pragma unroll
    for (int i = 0; i + 1 < kAhead; ++i) ring[i] = ring[i + 1];
    ring[kAhead - 1] = load();
    return o;
  }
};

// gate | up and the SwiGLU for the rows of one expert, 16 (or g.pass) at a time: the rows
// in LDS, a wavefront whole blocks of 32 columns of h (four weight tiles each), one after
// another with no barrier between.  `wgs` workgroups an expert.  Bound by the weight
// stream: 8 tokens, eight of 128 experts of 2048 x 768 each, 25 us for the 87 MB of 52
// experts.
template <bool kScan, int kDtype>
__global__ __launch_bounds__(256, 4) void gate_up_kernel(SmallMoeArgs g, int wgs) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ int32_t list[kScan ? kScanSlots : 1];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = vq::uniform(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int inter = g.n / 2, groups = inter / kBlock;
  const RowsOf rows = rows_of<kScan>(g, int(blockIdx.x) / wgs, list, &count);
  if (rows.count == 0) return;
  const int chunks = (g.blocks + kChunk - 1) / kChunk;
  const int first = int(blockIdx.x) % wgs * 4 + wave, stride = 4 * wgs;
  const int mine = first < groups ? (groups - first + stride - 1) / stride : 0;  // blocks of h
  const int64_t line = int64_t(g.blocks) * kBlockBytes;
  const uint8_t* w = g.w + (int64_t(rows.expert) * g.n + r) * line;
  const uint8_t* ws = g.ws + (int64_t(rows.expert) * g.n + r) * g.blocks;
  const auto base = [&](int i, const uint8_t*& wt, const uint8_t*& wst) {  // gate 0, gate 1, up 0, up 1
    const int64_t row = int64_t(first + (i >> 2) * stride) * kBlock + 16 * (i & 1) + (i & 2 ? inter : 0);
    wt = w + row * line;
    wst = ws + row * g.blocks;
  };
  for (int m0 = 0; m0 < rows.count; m0 += g.pass) {
    const int here = min(rows.count - m0, g.pass);
    WeightStream<decltype(base)> stream{base, 4 * mine, chunks, g.blocks, q, 0, 0, {}};
    stream.start();
    if (m0) __syncthreads();
    if constexpr (kScan) {
      quantize_to_lds<kDtype>(g.x, [&](int m) { return int64_t(rows.slots[m0 + m] / g.top_k) * g.stride; }, here, g.blocks, chunks,
                              g.wide, lds, tid, 256);
    } else {
      copy_to_lds(g.a, g.as, [&](int m) { return int64_t(rows.slots[m0 + m] / g.top_k); }, here, g.blocks, chunks, lds, tid, 256);
    }
    __syncthreads();
    const int64_t slot = rows.slots[m0 + min(r, here - 1)];
    for (int i = 0; i < mine; ++i) {
      f32x4_t acc[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        acc[t] = f32x4_t{0, 0, 0, 0};
        for (int c = 0; c < chunks; ++c) {
          const ChunkOperand a = stream.next();
          multiply_lds(a, lds, c, here, chunks, r, q, acc[t]);
        }
      }
      // row r's block of h lies in its four lanes (q): elements 4 q + j and 16 + 4 q + j
      float v[8];
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = swiglu(acc[0][j], acc[2][j], g.limit);
        v[4 + j] = swiglu(acc[1][j], acc[3][j], g.limit);
        top = max(top, max(magnitude(v[j]), magnitude(v[4 + j])));
      }
      top = max(top, uint32_t(__shfl_xor(int(top), 16)));
      top = max(top, uint32_t(__shfl_xor(int(top), 32)));
      const uint32_t s = block_scale(top);
      const uint32_t code = s == 255u ? 0u : codes8(v, s);
      if (r < here) {
        const int block = first + i * stride;
        uint16_t* out = reinterpret_cast<uint16_t*>(g.h + slot * (inter / 2) + block * kBlockBytes);
        out[q] = uint16_t(code);
        out[4 + q] = uint16_t(code >> 16);
        if (q == 0) g.hs[slot * groups + block] = uint8_t(s);
      }
    }
  }
}

// down for the rows of one expert: the rows of h in LDS, a wavefront 16 columns
// after another; the weighted slot rows.  16 tokens of the layer above 22 us (69 MB).
template <bool kScan>
__global__ __launch_bounds__(256, 4) void down_kernel(SmallMoeArgs g, int wgs) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ int32_t list[kScan ? kScanSlots : 1];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = vq::uniform(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const RowsOf rows = rows_of<kScan>(g, int(blockIdx.x) / wgs, list, &count);
  if (rows.count == 0) return;
  const int groups = g.n / 16, chunks = (g.blocks + kChunk - 1) / kChunk;  // n: whole sixteens
  const int first = int(blockIdx.x) % wgs * 4 + wave, stride = 4 * wgs;
  const int mine = first < groups ? (groups - first + stride - 1) / stride : 0;
  const int64_t line = int64_t(g.blocks) * kBlockBytes;
  const uint8_t* w = g.w + (int64_t(rows.expert) * g.n + r) * line;
  const uint8_t* ws = g.ws + (int64_t(rows.expert) * g.n + r) * g.blocks;
  const auto base = [&](int i, const uint8_t*& wt, const uint8_t*& wst) {
    const int64_t row = int64_t(first + i * stride) * 16;
    wt = w + row * line;
    wst = ws + row * g.blocks;
  };
  for (int m0 = 0; m0 < rows.count; m0 += g.pass) {
    const int here = min(rows.count - m0, g.pass);
    WeightStream<decltype(base)> stream{base, mine, chunks, g.blocks, q, 0, 0, {}};
    stream.start();
    if (m0) __syncthreads();
    copy_to_lds(g.h, g.hs, [&](int m) { return int64_t(rows.slots[m0 + m]); }, here, g.blocks, chunks, lds, tid, 256);
    __syncthreads();
    const int64_t slot = rows.slots[m0 + min(r, here - 1)];
    const float weight = g.topk_w[slot];
    float* out = g.c3 + slot * g.n + 4 * q;
    for (int i = 0; i < mine; ++i) {
      f32x4_t acc{0, 0, 0, 0};
      for (int c = 0; c < chunks; ++c) {
        const ChunkOperand a = stream.next();
        multiply_lds(a, lds, c, here, chunks, r, q, acc);
      }
      if (r < here) *reinterpret_cast<f32x4_t*>(out + (first + i * stride) * 16) = acc * weight;
    }
  }
}

// down and the slot sum for one token by 16 columns, 2^log_parts wavefronts a slot (chunk
// c of K multiplied by part c % parts, of at least as many chunks): where tokens are few, their experts' weights are
// read a token at a time (those two share come from L2) and the slot rows never leave
// the workgroup.  One token, eight experts of 2048 x 768: 5 us (6.7 MB), two of 4096 x
// 14336: 15 us (62 MB; 29 without parts).
template <int kDtype>
__global__ __launch_bounds__(1024, 4) void down_sum_kernel(SmallMoeArgs g, int log_parts) {
  extern __shared__ float sums[];  // [top_k][parts][16]
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = vq::uniform(int(threadIdx.x) >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int groups = g.n / 16, parts = 1 << log_parts;
  const int n0 = int(blockIdx.x) % groups * 16;
  const int token = int(blockIdx.x) / groups;
  const int chunks = (g.blocks + kChunk - 1) / kChunk;
  for (int i = wave; i < g.top_k << log_parts; i += waves) {
    const int64_t slot = int64_t(token) * g.top_k + (i >> log_parts);
    const int part = i & (parts - 1);
    const int e = vq::uniform(g.of(slot));
    f32x4_t acc{0, 0, 0, 0};
    if (e >= 0) {
      const int64_t wrow = int64_t(e) * g.n + n0 + r;
      const uint8_t* w = g.w + wrow * g.blocks * kBlockBytes;
      const uint8_t* ws = g.ws + wrow * g.blocks;
      const uint8_t* x = g.h + slot * g.blocks * kBlockBytes;
      const uint8_t* xs = g.hs + slot * g.blocks;
      ChunkOperand a = load_chunk(w, ws, part, g.blocks, q), ax = load_chunk(x, xs, part, g.blocks, q);
      for (int c = part; c < chunks; c += parts) {
        ChunkOperand next{}, nx{};
        if (c + parts < chunks) {
          next = load_chunk(w, ws, c + parts, g.blocks, q);
          nx = load_chunk(x, xs, c + parts, g.blocks, q);
        }
        multiply_loaded(a, ax, acc);
        a = next;
        ax = nx;
      }
      acc = acc * g.topk_w[slot];
    }
    if (r == 0) *reinterpret_cast<f32x4_t*>(sums + i * 16 + 4 * q) = acc;
  }
  __syncthreads();
  if (threadIdx.x >= 16) return;
  float sum = 0;  // (masked slots: zeros)
#pragma unroll 4
  for (int i = 0; i < g.top_k << log_parts; ++i) sum += sums[i * 16 + threadIdx.x];
  vq::store_act(g.out, kDtype, int64_t(token) * g.n + n0 + threadIdx.x, sum);
}

// out[t][c] = RN(sum over t's slots with a local expert, in slot order).  2048 tokens of
// eight slots of 2048: 22 us, 142 MB at 6.4 TB/s (the slot rows were just written); 64
// tokens 4.6 us (5.8 with a slot's load behind the one before).
__global__ __launch_bounds__(kThreads) void slot_sum_kernel(const float* in, ExpertOf of, int64_t tokens, int top_k, int hidden,
                                                            void* out, int dtype) {
  const int64_t i = (int64_t(blockIdx.x) * kThreads + threadIdx.x) * 4;
  if (i >= tokens * hidden) return;
  const int64_t t = i / hidden;
  const int64_t c = i - t * hidden;
  f32x4_t sum{0, 0, 0, 0};
  constexpr int kEach = 4;  // slots whose loads are on their way together
  for (int k0 = 0; k0 < top_k; k0 += kEach) {
    f32x4_t v[kEach];
    bool local[kEach];
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int64_t slot = t * top_k + min(k0 + u, top_k - 1);
      v[u] = *reinterpret_cast<const f32x4_t*>(in + slot * hidden + c);  // (of a masked slot whatever lies there)
      local[u] = k0 + u < top_k && of(slot) >= 0;
    }
#pragma unroll
    for (int u = 0; u < kEach; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] = local[u] ? sum[j] + v[u][j] : sum[j];
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
      inter % kBlock != 0 || hidden > kMaxSize || inter > kMaxSize || experts <= 0 || experts > moe::kRowsMaxExperts) {
    vq::fail("mxfp4 moe: sizes out of range (hidden and intermediate multiples of 32 up to 65536, at most 1024 experts)");
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
  if (!aligned(x, 2) || !aligned(out, 2) || !aligned(topk_ids, 4) || !aligned(topk_w, 4) || !aligned(expert_map, 4)) return vq::fail("mxfp4 moe: misaligned pointer");
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16)) return vq::fail("mxfp4 moe: workspace too small or not 16-byte aligned");
  const int64_t slots = tokens * top_k, codes = experts * inter * hidden;  // of w13, bytes
  for (const auto& other : {std::pair<const void*, int64_t>{x, ((tokens - 1) * x_stride + hidden) * 2}, {w13, codes}, {s13, codes / 16},
                            {w2, codes / 2}, {s2, codes / 32}, {topk_ids, slots * 4}, {topk_w, slots * 4}, {expert_map, map_size * 4}}) {
    if (vq::overlaps(workspace, need, other.first, other.second)) return vq::fail("mxfp4 moe: the workspace must not overlap another argument");
    if (other.first != x && vq::overlaps(out, tokens * hidden * 2, other.first, other.second)) {
      return vq::fail("mxfp4 moe: out must not overlap the weights or the routing");
    }
  }
  if (vq::overlaps(workspace, need, out, tokens * hidden * 2)) return vq::fail("mxfp4 moe: the workspace must not overlap another argument");
  const Workspace ws = workspace_of(tokens, top_k, hidden, inter, experts);
  const moe::RowsLayout lay = layout_of(slots, experts);
  uint8_t* base = static_cast<uint8_t*>(workspace);
  int32_t* table = reinterpret_cast<int32_t*>(base + ws.table);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const ExpertOf of{topk_ids, map_size > 0 ? expert_map : nullptr, map_size, int(experts)};
  const int64_t hb = hidden / kBlock, ib = inter / kBlock;
  const int64_t groups = lay.parts() + (tokens * hb * 4 + moe::kRowsPartThreads - 1) / moe::kRowsPartThreads;
  const int64_t sums = (tokens * hidden / 4 + kThreads - 1) / kThreads;
  if (groups > INT_MAX || sums > INT_MAX) return vq::fail("mxfp4 moe: too many rows");
  const bool wide = aligned(x, 16) && x_stride % 8 == 0;
  const size_t lds = size_t(experts) * sizeof(int);
  const int64_t chunks = (hb + kChunk - 1) / kChunk, chunks2 = (ib + kChunk - 1) / kChunk;
  // Tiles where more than 16 rows may meet at an expert, which the few rows' kernels
  // would take one pass over its weights after another, or where it may expect ten (a
  // map says how many share the slots); whole stages and buffers below 2 GiB.  In us,
  // few rows' kernels and tiles, 128 experts of 2048 x 768, eight a token: 8 tokens
  // 44 and 53, 16 evenly routed 64 and 74, routed by a power law 66 and 55, 64 evenly
  // 82 and 91, by the power law 152 and 84; 8 experts of 4096 x 14336, two a token: 16
  // tokens 162 and 179, 32 198 and 180.
  const bool can_tile = hb >= kStageBlocks && ib >= kStageBlocks && hidden * inter < (int64_t(1) << 31) && tokens * hidden / 2 < (int64_t(1) << 31);
  const bool tile = can_tile && (tokens > 16 || slots >= 10 * std::max(experts, map_size));
  SmallMoeArgs m{};
  m.of = of;
  m.x = x;
  m.stride = x_stride;
  m.wide = wide;
  m.a = base + ws.xq;
  m.as = base + ws.xs;
  m.w = w13;
  m.ws = s13;
  m.slots = int(slots);
  m.top_k = int(top_k);
  m.pass = rows_at_once(slots, chunks);
  m.table = table;
  m.tasks = lay.tasks();
  m.sorted = lay.sorted();
  m.topk_w = topk_w;
  m.n = int(2 * inter);
  m.blocks = int(hb);
  m.limit = limit;
  m.h = base + ws.hq;
  m.hs = base + ws.hs;
  m.c3 = reinterpret_cast<float*>(base + ws.c3);
  m.out = out;
  const size_t rows13 = size_t(small_bytes(m.pass, chunks)), rows2 = size_t(small_bytes(rows_at_once(slots, chunks2), chunks2));
  // workgroups an expert: about four a CU in all
  const auto wgs_of = [&](int64_t units, int64_t most) { return int(std::max<int64_t>(1, std::min(most, 1024 / units))); };
  const int parts = chunks >= 8 ? 4 : chunks >= 2 ? 2 : 1;
  const size_t sums_lds = size_t(parts) * 4 * 16 * 20 * sizeof(float);
  const auto second = [&](SmallMoeArgs& a) {
    a.w = w2;
    a.ws = s2;
    a.n = int(hidden);
    a.blocks = int(ib);
    a.pass = rows_at_once(slots, chunks2);
  };
  const auto sum = [&] {
    hipLaunchKernelGGL(slot_sum_kernel, dim3(unsigned(sums)), dim3(kThreads), 0, st, m.c3, of, tokens, int(top_k), int(hidden), out, act_dtype);
    return vq::check_launch("mxfp4 moe sum");
  };
  if (!tile && slots <= kScanSlots) {
    m.by_slot = slots < experts;
    const int64_t units = m.by_slot ? slots : experts;
    if (units * ib < 1024) {
      const size_t need13 = std::max<size_t>(sums_lds, rows13);
      const dim3 grid13(unsigned(units * ib)), block13(256 * parts);
      if (act_dtype == vq::kBF16) hipLaunchKernelGGL(gate_up_split_kernel<vq::kBF16>, grid13, block13, need13, st, m);
      else hipLaunchKernelGGL(gate_up_split_kernel<vq::kFP16>, grid13, block13, need13, st, m);
    } else {
      const int wgs = wgs_of(units, (ib + 3) / 4);
      const dim3 grid13(unsigned(units * wgs)), block13(256);
      if (act_dtype == vq::kBF16) hipLaunchKernelGGL((gate_up_kernel<true, vq::kBF16>), grid13, block13, rows13, st, m, wgs);
      else hipLaunchKernelGGL((gate_up_kernel<true, vq::kFP16>), grid13, block13, rows13, st, m, wgs);
    }
    if (int rc = vq::check_launch("mxfp4 moe gate_up")) return rc;
    second(m);
    // A token at a time while experts are hardly shared: in us, a token at a time and
    // an expert at a time, 128 experts of 2048 x 768, eight a token: 4 tokens 25 and 30,
    // 12 58 and 61, 16 67 and 65; 8 experts of 4096 x 14336, two a token: 2 tokens 78 and
    // 86, 4 126 and 119.  K split where slots are few (the same 8 experts, one token: 51
    // for 65).
    if ((m.by_slot || tokens == 1) && top_k <= 64) {
      int split = 0;  // log2
      while ((2 << split) * std::min<int64_t>(top_k, 8) <= 16 && 4 << split <= chunks2) ++split;
      const dim3 grid(unsigned(tokens * (hidden / 16))), block(unsigned((64 << split) * std::min<int64_t>(top_k, 8)));
      const size_t bytes = (size_t(top_k) << split) * 16 * sizeof(float);
      if (act_dtype == vq::kBF16) hipLaunchKernelGGL(down_sum_kernel<vq::kBF16>, grid, block, bytes, st, m, split);
      else hipLaunchKernelGGL(down_sum_kernel<vq::kFP16>, grid, block, bytes, st, m, split);
      return vq::check_launch("mxfp4 moe down");
    }
    const int wgs = wgs_of(units, (hidden + 63) / 64);
    hipLaunchKernelGGL(down_kernel<true>, dim3(unsigned(units * wgs)), dim3(256), rows2, st, m, wgs);
    if (int rc = vq::check_launch("mxfp4 moe down")) return rc;
    return sum();
  }
  const int task_rows = tile ? kTileRows : kTaskRows;
  uint32_t* xq = reinterpret_cast<uint32_t*>(base + ws.xq);
  if (act_dtype == vq::kBF16) {
    hipLaunchKernelGGL(count_quantize_kernel<vq::kBF16>, dim3(unsigned(groups)), dim3(moe::kRowsPartThreads), lds, st, of, lay, table,
                       task_rows, x, tokens, int(hb), x_stride, wide, xq, base + ws.xs);
  } else {
    hipLaunchKernelGGL(count_quantize_kernel<vq::kFP16>, dim3(unsigned(groups)), dim3(moe::kRowsPartThreads), lds, st, of, lay, table,
                       task_rows, x, tokens, int(hb), x_stride, wide, xq, base + ws.xs);
  }
  if (int rc = vq::check_launch("mxfp4 moe count")) return rc;
  if (lay.parts() > 1) {
    hipLaunchKernelGGL(fill_kernel, dim3(unsigned(lay.parts())), dim3(moe::kRowsPartThreads), lds, st, lay, table, task_rows);
    if (int rc = vq::check_launch("mxfp4 moe fill")) return rc;
  }
  if (!tile) {
    const int wgs13 = wgs_of(lay.max_tasks, (ib + 3) / 4), wgs2 = wgs_of(lay.max_tasks, (hidden + 63) / 64);
    if (lay.max_tasks * std::max(wgs13, wgs2) > INT_MAX) return vq::fail("mxfp4 moe: too many rows");
    hipLaunchKernelGGL((gate_up_kernel<false, vq::kBF16>), dim3(unsigned(lay.max_tasks * wgs13)), dim3(256),
                       rows13, st, m, wgs13);
    if (int rc = vq::check_launch("mxfp4 moe gate_up")) return rc;
    second(m);
    hipLaunchKernelGGL(down_kernel<false>, dim3(unsigned(lay.max_tasks * wgs2)), dim3(256), rows2, st, m, wgs2);
    if (int rc = vq::check_launch("mxfp4 moe down")) return rc;
    return sum();
  }
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
  if (bound * std::max((inter + 63) / 64, (hidden + 127) / 128) > INT_MAX) return vq::fail("mxfp4 moe: too many rows");
  hipLaunchKernelGGL((tile_kernel<2, 2, kGateUp, 2>), dim3(unsigned(bound * t.tiles_n)), dim3(kTileThreads), 0, st, t);
  if (int rc = vq::check_launch("mxfp4 moe gate_up")) return rc;
  t.a = base + ws.hq;
  t.as = base + ws.hs;
  t.w = w2;
  t.ws = s2;
  t.n = hidden;
  t.blocks = int(ib);
  t.tiles_n = int((hidden + 127) / 128);
  t.out = base + ws.c3;
  hipLaunchKernelGGL((tile_kernel<2, 2, kDown, 2>), dim3(unsigned(bound * t.tiles_n)), dim3(kTileThreads), 0, st, t);
  if (int rc = vq::check_launch("mxfp4 moe down")) return rc;
  return sum();
}
