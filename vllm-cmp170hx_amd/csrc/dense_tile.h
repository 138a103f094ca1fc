// Many rows of the dense linear layer: tiles of the product through LDS.
//
// A workgroup of four or eight wavefronts computes kCols lines of W by kRows rows of x, each
// wavefront 32 kN x 32 kM of v_mfma_f32_32x32x16 tiles.  A stage is 64 k: 128
// bytes of every row and line, in one of kBufs buffers, one barrier a stage.
//  * Rows come to LDS by DMA, one 128-byte line in eight lanes, up to kBufs - 1 stages
//    ahead.  A line's eight 16-byte chunks lie in LDS in the order chunk ^ (line / 2 &
//    7), so that the 16 lines that a ds_read_b128 reads at once, all at one chunk, lie
//    on 16 different 16-byte columns of the 64 banks.
//  * A lane of the MFMA holds one chunk: line lane & 31, chunk 2 sub + (lane >> 5) of
//    the stage's 16-k sub-step `sub`.  W is the A operand, x the B operand, so that a
//    lane's sums are of one row.
//  * A gated activation's tile has the gate and the up lines of the same columns in one
//    wavefront.
#pragma once

#include <type_traits>

#include "dense.h"

namespace dense {

typedef __attribute__((address_space(3))) void* lds_ptr_t;

constexpr int kStageChunks = 8;  // 64 k
constexpr int kChunkBytes = 16;
constexpr int kStageBytes = kStageChunks * kChunkBytes;  // a line

// f(std::integral_constant<int, i>) for i = first .. last - 1.
template <int first, int last, typename F>
__device__ __forceinline__ void for_range(F&& f) {
  if constexpr (first < last) {
    f(std::integral_constant<int, first>{});
    for_range<first + 1, last>(f);
  }
}

struct TileArgs {
  Operand x, w;      // rows on 16 bytes, k whole chunks
  int chunks;        // of a row
  int tiles_n, tiles_m;
  int split_stages;  // stages of one split of K (gridDim.y splits)
  float* sums;       // more than one split: FP32 [split][rows][lines] for finish_kernel
  Epilogue e;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, int(bytes), 0x00020000);
}

// An offset past any buffer: such loads give zeros.
constexpr uint32_t kPastEnd = 0x80000000u;

// A workgroup's kWn x kWm wavefronts, each of 32 kN lines by 32 kM rows, and its stage buffers.
template <int kWn_, int kWm_, int kN_, int kM_, int kBufs_>
struct Tile {
  static constexpr int kWn = kWn_, kWm = kWm_, kN = kN_, kM = kM_, kBufs = kBufs_;
  static constexpr int kWaves = kWn * kWm, kThreads = 64 * kWaves;
  static constexpr int kCols = 32 * kN * kWn, kRows = 32 * kM * kWm, kLines = kCols + kRows;
  // workgroups that a CU's LDS holds, two at most
  static constexpr int kGroups = kLines * kStageBytes * kBufs > 80 * 1024 ? 1 : 2;
};

template <typename T, bool kGated, bool kBf16>
__global__ __launch_bounds__(T::kThreads, T::kGroups * T::kWaves / 4) void tile_kernel(TileArgs g) {
  constexpr int kN = T::kN, kM = T::kM, kBufs = T::kBufs, kWaves = T::kWaves;
  constexpr int kCols = T::kCols, kRows = T::kRows, kLines = T::kLines;
  constexpr int kLoadRows = 8;  // lines of a 1 KB DMA load
  constexpr int kLoadsW = kCols / (kWaves * kLoadRows), kLoadsX = kRows / (kWaves * kLoadRows);  // loads a wavefront and stage
  constexpr int kLoads = kLoadsW + kLoadsX;
  static_assert(kBufs >= 2 && kBufs <= 4, "stage buffers");
  static_assert(kLoadsW * kWaves * kLoadRows == kCols && kLoadsX * kWaves * kLoadRows == kRows, "whole loads");
  static_assert(!kGated || (kN >= 2 && kLoadRows * kLoadsW <= 16 * kN), "a wavefront loads gate or up lines alone");
  // (buffers by name: the compiler then sees that a stage's reads are not of the
  // buffer that the DMA is filling, and does not wait for it)
  constexpr int kBufBytes = kLines * kStageBytes;
  __shared__ __attribute__((aligned(1024))) uint8_t buf0[kBufBytes], buf1[kBufBytes], buf2[kBufs > 2 ? kBufBytes : 16],
      buf3[kBufs > 3 ? kBufBytes : 16];
  const auto buf = [&](auto i_c) -> uint8_t* {
    constexpr int i = decltype(i_c)::value % kBufs;
    if constexpr (i == 0) return buf0;
    else if constexpr (i == 1) return buf1;
    else if constexpr (i == 2) return buf2;
    else return buf3;
  };

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = vq::uniform(tid >> 6);
  const int r = lane & 31, h = lane >> 5;
  const int wn = wave % T::kWn, wm = wave / T::kWn;

  // XCD x (workgroups x, x + 8, ...) takes a run of tiles, rows first: it fetches few
  // lines of W and its L2 keeps them for all the rows
  const int total = g.tiles_n * g.tiles_m, per = (total + 7) / 8;
  const int t = int(blockIdx.x & 7) * per + int(blockIdx.x >> 3);
  if (int(blockIdx.x >> 3) >= per || t >= total) return;
  constexpr int kOut = kGated ? kCols / 2 : kCols;  // output columns
  const int64_t c0 = int64_t(t / g.tiles_m) * kOut;
  const int64_t m0 = int64_t(t % g.tiles_m) * kRows;
  const int nrows = int(min(int64_t(kRows), g.x.rows - m0));
  const int ncols = int(min(int64_t(kOut), g.e.n - c0));
  const uint32_t wline = uint32_t(g.w.stride) * 2, xline = uint32_t(g.x.stride) * 2;
  // Loads: 1 KB each, 8 lines, of which the first one's offset is scalar and the lane's part
  // has two values, by the parity of the load's place.  A wavefront's first kLoadsW
  // bring lines of W: with a gated activation all gate or all up lines.
  const int w_first = kLoadRows * kLoadsW * wave;
  const bool up = kGated && w_first % (32 * kN) >= 16 * kN;
  const uint32_t line_bytes = uint32_t(g.chunks) * kChunkBytes;
  const __amdgpu_buffer_rsrc_t wbuf = buffer(g.w.p + (c0 + (up ? g.e.n : 0)) * g.w.stride, uint32_t(ncols - 1) * wline + line_bytes);
  const __amdgpu_buffer_rsrc_t xbuf = buffer(g.x.p + m0 * g.x.stride, uint32_t(nrows - 1) * xline + line_bytes);
  const int sub_row = lane >> 3;
  const auto first_line = [&](int i) {
    return i < kLoadsW ? w_first + kLoadRows * i : kCols + kLoadRows * (kLoadsX * wave + i - kLoadsW);
  };
  const auto swizzle_of = [](int l) { return (l >> 1) & 7; };
  const int kb[2] = {(lane & 7) ^ swizzle_of(sub_row), (lane & 7) ^ swizzle_of(kLoadRows + sub_row)};
  // the scalar first row of load i (a row of the buffer also where the load's lie past
  // its end: their sums are not stored; the rest of a load that begins inside it is zeros)
  const auto first_row = [&](int i) -> int {
    int l;
    if (i >= kLoadsW) {
      l = first_line(i) - kCols;
      return l < nrows ? l : 0;
    }
    l = first_line(i);
    if constexpr (kGated) l = l / (32 * kN) * (16 * kN) + l % (16 * kN);
    return l < ncols ? l : 0;
  };
  const uint32_t wlane[2] = {sub_row * wline + kb[0] * kChunkBytes, sub_row * wline + kb[1] * kChunkBytes};
  const uint32_t xlane[2] = {sub_row * xline + kb[0] * kChunkBytes, sub_row * xline + kb[1] * kChunkBytes};
  const int all_stages = (g.chunks + kStageChunks - 1) / kStageChunks;
  const int first = int(blockIdx.y) * g.split_stages;
  const int stages = min(first + g.split_stages, all_stages);
  // DMA load i of stage s (zeros past the last stage)
  const auto fetch = [&](auto i_c, int s, uint8_t* into) __attribute__((always_inline)) {
    constexpr int i = decltype(i_c)::value;
    const int left = s < stages ? g.chunks - s * kStageChunks : 0;
    const int parity = (i < kLoadsW ? kLoadsW * wave + i : kLoadsX * wave + i - kLoadsW) & 1;
    const uint32_t lane_part = i < kLoadsW ? wlane[parity] : xlane[parity];
    const uint32_t o = left >= kStageChunks || kb[parity] < left ? lane_part : kPastEnd;
    const int row_part = first_row(i) * int(i < kLoadsW ? wline : xline);
    // (the scalar offset stays below the buffer's size, or its bounds check would wrap)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(i < kLoadsW ? wbuf : xbuf, (lds_ptr_t)(into + first_line(i) * kStageBytes), 16, int(o),
                                             row_part + (left > 0 ? s * kStageBytes : 0), 0, 0);
  };
  // a stage has landed (its loads of this wavefront, behind which kBufs - 2 stages'
  // stay on their way, then everyone's), and no wavefront reads the one before any more
  const auto land = [&]() __attribute__((always_inline)) {
    vq::wait_vmcnt<(kBufs - 2) * kLoads>();
    // (a barrier that leaves the loads on their way: __syncthreads() waits for them)
    vq::wait_lgkmcnt0();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  f32x16_t acc[kN][kM];
#pragma unroll
  for (int i = 0; i < kN; ++i)
#pragma unroll
    for (int j = 0; j < kM; ++j)
#pragma unroll
      for (int k = 0; k < 16; ++k) acc[i][j][k] = 0;

  const int wl = 32 * kN * wn + r, xl = kCols + 32 * kM * wm + r;
  const int swizzle = swizzle_of(r);
  u32x4_t fw[2][kN], fx[2][kM];  // this sub-step's operands and the next one's
  // operand i of a sub-step: kN of W, then kM of x
  const auto read = [&](auto i_c, const uint8_t* from, int sub, int set) __attribute__((always_inline)) {
    constexpr int i = decltype(i_c)::value;
    const int at = ((2 * sub + h) ^ swizzle) * kChunkBytes;
    if constexpr (i < kN) fw[set][i] = *reinterpret_cast<const u32x4_t*>(from + (wl + 32 * i) * kStageBytes + at);
    else fx[set][i - kN] = *reinterpret_cast<const u32x4_t*>(from + (xl + 32 * (i - kN)) * kStageBytes + at);
  };
  // Sub-step `sub` of a stage: between its kN kM MFMAs, one or two at a time, the
  // next sub-step's operands are read (of `next`, at sub-step next_sub) and loads
  // kFirst .. kLast - 1 of stage s issued into `into`.
  const auto step = [&](auto sub_c, auto first_c, auto last_c, const uint8_t* next, int next_sub, int s,
                        uint8_t* into) __attribute__((always_inline)) {
    constexpr int sub = decltype(sub_c)::value, kFirst = decltype(first_c)::value, kLast = decltype(last_c)::value;
    constexpr int kReads = kN + kM, kSlots = kN * kM;
    for_range<0, kSlots>([&](auto slot_c) __attribute__((always_inline)) {
      constexpr int slot = decltype(slot_c)::value, i = slot / kM, j = slot % kM;
      for_range<slot * kReads / kSlots, (slot + 1) * kReads / kSlots>([&](auto k) __attribute__((always_inline)) {
        read(k, next, next_sub, (sub + 1) & 1);
      });
      constexpr int kFetch = kLast - kFirst, kTurn = (slot + kSlots / 2) % kSlots;  // in other slots than the reads
      for_range<kFirst + kTurn * kFetch / kSlots, kFirst + (kTurn + 1) * kFetch / kSlots>(
          [&](auto k) __attribute__((always_inline)) { fetch(k, s, into); });
      __builtin_amdgcn_sched_barrier(0);
      mfma32<kBf16>(acc[i][j], fw[sub & 1][i], fx[sub & 1][j]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // Stage s, the i-th of a round of kBufs.  The barrier comes before the last sub-step,
  // whose operands are in registers by then: its MFMAs run while the next stage's first
  // operands are read, and its buffer takes stage s + kBufs: half of those loads here,
  // the others in the next stage's first sub-steps.
  constexpr int kHalf = kLoads / 2, kMore = kHalf + kLoads / 4;
  const auto stage = [&](auto i_c, int s) __attribute__((always_inline)) {
    constexpr int i = decltype(i_c)::value;
    using std::integral_constant;
    constexpr integral_constant<int, 0> none{};
    uint8_t* const cur = buf(i_c);
    uint8_t* const next = buf(integral_constant<int, i + 1>{});
    uint8_t* const prev = buf(integral_constant<int, i + kBufs - 1>{});
    step(none, integral_constant<int, kHalf>{}, integral_constant<int, kMore>{}, cur, 1, s + kBufs - 1, prev);
    step(integral_constant<int, 1>{}, integral_constant<int, kMore>{}, integral_constant<int, kLoads>{}, cur, 2, s + kBufs - 1, prev);
    step(integral_constant<int, 2>{}, none, none, cur, 3, 0, cur);
    land();
    step(integral_constant<int, 3>{}, none, integral_constant<int, kHalf>{}, next, 0, s + kBufs, cur);
  };
  for_range<0, kBufs - 1>([&](auto b_c) {
    for_range<0, kLoads>([&](auto k) { fetch(k, first + decltype(b_c)::value, buf(b_c)); });
  });
  land();
  for_range<0, kHalf>([&](auto k) { fetch(k, first + kBufs - 1, buf(std::integral_constant<int, kBufs - 1>{})); });
  for_range<0, kN + kM>([&](auto k) { read(k, buf0, 0, 0); });
  int s = first;
  for (; s + kBufs <= stages; s += kBufs) {
    for_range<0, kBufs>([&](auto i) __attribute__((always_inline)) { stage(i, s + decltype(i)::value); });
  }
  for_range<0, kBufs - 1>([&](auto i) __attribute__((always_inline)) {
    if (s + decltype(i)::value < stages) stage(i, s + decltype(i)::value);
  });
  vq::wait_vmcnt<0>();  // the last loads (zeros) are in before their buffers are used again

  // Results: each row tile through LDS (a wavefront's own part, four columns a chunk, the
  // chunks in an order by the row), then four columns of a row a lane.
  constexpr int kStride = 32 * kN;
  const auto exchange_at = [](int row, int chunk) { return row * kStride + 4 * (chunk ^ (kN > 1 ? row & 15 : (row >> 1) & 7)); };
  constexpr int kEach = (kWaves + kBufs - 1) / kBufs;  // exchanges in one buffer
  static_assert(kEach * 32 * kStride * 4 <= kBufBytes, "the wavefronts' exchanges fit the stage buffers");
  const int in = wave / kEach;
  float* part = reinterpret_cast<float*>(in == 0 ? buf0 : in == 1 ? buf1 : in == 2 ? buf2 : buf3) + wave % kEach * 32 * kStride;
  __syncthreads();
  const bool split = gridDim.y > 1;
  constexpr int kWave = kGated ? 16 * kN : 32 * kN;  // a wavefront's output columns
  // (a loop, so that there is one copy of what follows the sums)
#pragma unroll 1
  for (int i = 0; i < kM; ++i) {
    for_range<0, kM>([&](auto i_c) __attribute__((always_inline)) {
      constexpr int row_tile = decltype(i_c)::value;
      if (i != row_tile) return;
#pragma unroll
      for (int j = 0; j < kN; ++j) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          f32x4_t v;
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q] = acc[j][row_tile][4 * p + q];
          *reinterpret_cast<f32x4_t*>(part + exchange_at(r, 8 * j + 2 * p + h)) = v;
        }
      }
    });
    const int mt = 32 * (kM * wm + i);
    const int64_t ct = c0 + kWave * wn;
    constexpr int kChunksRow = kWave / 4;  // of four columns
    const int chunk = lane % kChunksRow, r0 = lane / kChunksRow;
#pragma unroll 1
    for (int k = 0; k < kChunksRow / 2; ++k) {
      const int mr = r0 + k * (64 / kChunksRow), m = mt + mr;
      const f32x4_t a = *reinterpret_cast<const f32x4_t*>(part + exchange_at(mr, chunk));
      const f32x4_t b = *reinterpret_cast<const f32x4_t*>(part + exchange_at(mr, chunk + (kGated ? 4 * kN : 0)));
      const int64_t c = ct + 4 * chunk;
      if (m >= nrows || c >= g.e.n) continue;
      float v[4] = {a[0], a[1], a[2], a[3]}, u[4] = {b[0], b[1], b[2], b[3]};
      if (split) {
        const int64_t lines = kGated ? 2 * g.e.n : g.e.n;
        float* to = g.sums + (int64_t(blockIdx.y) * g.x.rows + m0 + m) * lines + c;
        store_columns<4>(to, vq::kFP32, 0, g.e.n - c, v);
        if constexpr (kGated) store_columns<4>(to + g.e.n, vq::kFP32, 0, g.e.n - c, u);
      } else {
        finish_columns<4, kGated>(g.e, m0 + m, c, v, u);
      }
    }
  }
}

}  // namespace dense
