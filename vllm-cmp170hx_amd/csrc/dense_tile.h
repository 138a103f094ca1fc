// Many rows of the dense linear layer: tiles of the product through LDS.
//
// A workgroup of four or eight wavefronts computes kCols lines of W by kRows rows of x, each
// wavefront 32 kN x 32 kM of v_mfma_f32_32x32x16 tiles.  A stage is 64 k: 128
// bytes of every row and line, one barrier a stage.
//  * Rows come to LDS by DMA, one 128-byte line in eight lanes, into a ring of kParts
//    buffers, each a stage's lines of W or its rows of x: odd numbers of them keep LDS
//    full, and some loads are on their way whenever a stage is waited for.  A line's eight
//    16-byte chunks lie in LDS in the order chunk ^ (line / 2 & 7), so that the 16 lines that
//    a ds_read_b128 reads at once, all at one chunk, lie on 16 different 16-byte columns
//    of the 64 banks.
//  * A lane of the MFMA holds one chunk: line lane & 31, chunk 2 sub + (lane >> 5) of
//    the stage's 16-k sub-step `sub`.  W is the A operand, x the B operand, so that a
//    lane's sums are of one row.
//  * A gated activation's tile has the gate and the up lines of the same columns in one
//    wavefront.
//
// What bounds it: 2048 rows of 8192 x 28672 in BF16 take 803-833 us, 1.16-1.2 PFLOP/s (the
// library's product of these sizes 765): the card then clocks at about 1.8 of its 2.4 GHz,
// the last of 3.5 rounds of 256 workgroups is half full, and each round has a start and an end
// (stores) in which the matrix cores rest, about 17 us of 235.  Workgroups that go on to the
// next tile, its first loads on their way while they store, were slower (845 us for 774 in a
// loop of launches): their stores from registers are of 32 bytes.
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
  int band;          // rows of tiles that are gone through together, column by column
  int split_stages;  // stages of one split of K (gridDim.y splits)
  float* sums;       // more than one split: FP32 [split][rows][lines] for finish_kernel
  Epilogue e;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, int(bytes), 0x00020000);
}

// An offset past any buffer: such loads give zeros.
constexpr uint32_t kPastEnd = 0x80000000u;

// A workgroup's kWn x kWm wavefronts, each of 32 kN lines by 32 kM rows, and its ring's parts.
template <int kWn_, int kWm_, int kN_, int kM_, int kParts_>
struct Tile {
  static constexpr int kWn = kWn_, kWm = kWm_, kN = kN_, kM = kM_, kParts = kParts_;
  static constexpr int kWaves = kWn * kWm, kThreads = 64 * kWaves;
  static constexpr int kCols = 32 * kN * kWn, kRows = 32 * kM * kWm;
  // part i's bytes: even ones hold lines of W and odd ones rows of x, where there is an odd
  // number of them each both in turn
  static constexpr int part_bytes(int i) {
    return kStageBytes * (kParts % 2 ? (kCols > kRows ? kCols : kRows) : i % 2 ? kRows : kCols);
  }
  static constexpr int kBytes = part_bytes(0) * ((kParts + 1) / 2) + part_bytes(1) * (kParts / 2);
  // workgroups that a CU's LDS holds, and whose registers (128 a lane) it does
  static constexpr int kGroups = 160 * 1024 / kBytes < 4 ? 160 * 1024 / kBytes : 4;
};

// Part i of the ring.  (Buffers by name: the compiler then sees that a stage's reads are
// not of the buffer that the DMA is filling, and does not wait for it.)
template <typename T, int i>
__device__ __forceinline__ uint8_t* ring_part() {
  static __shared__ __attribute__((aligned(1024))) uint8_t part[T::part_bytes(i)];
  return part;
}

template <typename T, bool kGated, bool kBf16>
__global__ __launch_bounds__(T::kThreads, T::kGroups * T::kWaves / 4) void tile_kernel(TileArgs g) {
  constexpr int kN = T::kN, kM = T::kM, kParts = T::kParts, kWaves = T::kWaves;
  constexpr int kCols = T::kCols, kRows = T::kRows;
  constexpr int kLoadRows = 8;  // lines of a 1 KB DMA load
  constexpr int kLoadsW = kCols / (kWaves * kLoadRows), kLoadsX = kRows / (kWaves * kLoadRows);  // loads a wavefront and stage
  constexpr int kLoads = kLoadsW + kLoadsX;
  static_assert(kParts >= 4, "two stages");
  static_assert(kLoadsW * kWaves * kLoadRows == kCols && kLoadsX * kWaves * kLoadRows == kRows, "whole loads");
  static_assert(!kGated || (kN >= 2 && kLoadRows * kLoadsW <= 16 * kN), "a wavefront loads gate or up lines alone");
  const auto part_of = [](auto i_c) { return ring_part<T, decltype(i_c)::value % kParts>(); };

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = vq::uniform(tid >> 6);
  const int r = lane & 31, h = lane >> 5;
  const int wn = wave % T::kWn, wm = wave / T::kWn;

  // XCD x (workgroups x, x + 8, ...) takes a run of tiles, in bands of rows about as high as
  // the tiles at work at a time are wide, so that its L2 fetches few rows and lines for them
  const int total = g.tiles_n * g.tiles_m, per = (total + 7) / 8;
  const int t = int(blockIdx.x & 7) * per + int(blockIdx.x >> 3);
  if (int(blockIdx.x >> 3) >= per || t >= total) return;
  constexpr int kOut = kGated ? kCols / 2 : kCols;  // output columns
  const int top = t / (g.band * g.tiles_n) * g.band, height = min(g.band, g.tiles_m - top), in_band = t - top * g.tiles_n;
  const int64_t c0 = int64_t(in_band / height) * kOut;
  const int64_t m0 = int64_t(top + in_band % height) * kRows;
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
  const int x_first = kLoadRows * kLoadsX * wave;
  const auto swizzle_of = [](int l) { return (l >> 1) & 7; };
  const int kb[2] = {(lane & 7) ^ swizzle_of(sub_row), (lane & 7) ^ swizzle_of(kLoadRows + sub_row)};
  // the scalar first row of load i of W (x) (a row of the buffer also where the load's lie past
  // its end: their sums are not stored; the rest of a load that begins inside it is zeros)
  const auto w_row = [&](int i) -> int {
    int l = w_first + kLoadRows * i;
    if constexpr (kGated) l = l / (32 * kN) * (16 * kN) + l % (16 * kN);
    return l < ncols ? l : 0;
  };
  const auto x_row = [&](int i) -> int {
    const int l = x_first + kLoadRows * i;
    return l < nrows ? l : 0;
  };
  const uint32_t wlane[2] = {sub_row * wline + kb[0] * kChunkBytes, sub_row * wline + kb[1] * kChunkBytes};
  const uint32_t xlane[2] = {sub_row * xline + kb[0] * kChunkBytes, sub_row * xline + kb[1] * kChunkBytes};
  const int all_stages = (g.chunks + kStageChunks - 1) / kStageChunks;
  const int first = int(blockIdx.y) * g.split_stages;
  const int stages = min(first + g.split_stages, all_stages);
  // DMA load i of stage s's lines of W or rows of x (zeros past the last stage)
  const auto fetch = [&](auto x_c, int i, int s, uint8_t* into) __attribute__((always_inline)) {
    constexpr bool kX = decltype(x_c)::value;
    const int left = s < stages ? g.chunks - s * kStageChunks : 0;
    const int parity = ((kX ? kLoadsX : kLoadsW) * wave + i) & 1;
    const uint32_t o = left >= kStageChunks || kb[parity] < left ? (kX ? xlane[parity] : wlane[parity]) : kPastEnd;
    const int row_part = kX ? x_row(i) * int(xline) : w_row(i) * int(wline);
    // (the scalar offset stays below the buffer's size, or its bounds check would wrap)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(kX ? xbuf : wbuf, (lds_ptr_t)(into + ((kX ? x_first : w_first) + kLoadRows * i) * kStageBytes),
                                             16, int(o), row_part + (left > 0 ? s * kStageBytes : 0), 0, 0);
  };
  // Part kFrom + 2 s (an odd one is of x) and the next one are loaded together, load i of
  // kLoads; both take the places of stage s - kParts / 2's.
  const auto fetch_pair = [&](auto from_c, auto place_c, int i, int s) __attribute__((always_inline)) {
    constexpr int kFrom = decltype(from_c)::value, kPlace = decltype(place_c)::value;
    constexpr int kFirst = kFrom % 2 ? kLoadsX : kLoadsW;
    using std::integral_constant;
    if (i < kFirst) {
      fetch(integral_constant<bool, kFrom % 2 != 0>{}, i, s + kFrom / 2, part_of(integral_constant<int, kPlace>{}));
    } else {
      fetch(integral_constant<bool, kFrom % 2 == 0>{}, i - kFirst, s + (kFrom + 1) / 2, part_of(integral_constant<int, kPlace + 1>{}));
    }
  };
  // a stage has landed (this wavefront's loads of it, behind which those of kBehind more parts
  // stay on their way, then everyone's), and no wavefront reads the one before any more
  const auto land = [&](auto behind_c) __attribute__((always_inline)) {
    constexpr int kBehind = decltype(behind_c)::value;  // (the first of them a part of W)
    vq::wait_vmcnt<(kBehind + 1) / 2 * kLoadsW + kBehind / 2 * kLoadsX>();
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

  const int wl = 32 * kN * wn + r, xl = 32 * kM * wm + r;
  const int swizzle = swizzle_of(r);
  u32x4_t fw[2][kN], fx[2][kM];  // this sub-step's operands and the next one's
  // operand i of a sub-step: kN of W, then kM of x
  const auto read = [&](auto i_c, const uint8_t* w, const uint8_t* x, int sub, int set) __attribute__((always_inline)) {
    constexpr int i = decltype(i_c)::value;
    const int at = ((2 * sub + h) ^ swizzle) * kChunkBytes;
    if constexpr (i < kN) fw[set][i] = *reinterpret_cast<const u32x4_t*>(w + (wl + 32 * i) * kStageBytes + at);
    else fx[set][i - kN] = *reinterpret_cast<const u32x4_t*>(x + (xl + 32 * (i - kN)) * kStageBytes + at);
  };
  // Sub-step `sub` of stage s, in place `i` of the ring's turn: between its kN kM MFMAs, one or
  // two at a time, the next sub-step's operands are read and a quarter of the loads issued
  // that take the places of the stage before (after the barrier: of this one).
  const auto step = [&](auto i_c, auto sub_c, int s) __attribute__((always_inline)) {
    constexpr int i = decltype(i_c)::value, sub = decltype(sub_c)::value;
    using std::integral_constant;
    constexpr int kReads = kN + kM, kSlots = kN * kM;
    constexpr int kAt = sub == 3 ? 2 * i : 2 * i + 2 * kParts - 2;  // the freed places
    constexpr int kNext = 2 * i + (sub == 3 ? 2 : 0);
    const uint8_t* const w = part_of(integral_constant<int, kNext>{});
    const uint8_t* const x = part_of(integral_constant<int, kNext + 1>{});
    for_range<0, kSlots>([&](auto slot_c) __attribute__((always_inline)) {
      constexpr int slot = decltype(slot_c)::value, a = slot / kM, b = slot % kM;
      for_range<slot * kReads / kSlots, (slot + 1) * kReads / kSlots>([&](auto k) __attribute__((always_inline)) {
        read(k, w, x, (sub + 1) & 3, (sub + 1) & 1);
      });
      constexpr int kTurn = (slot + kSlots / 2) % kSlots;  // in other slots than the reads
      constexpr int kQuarter = (sub + 1) & 3;  // of the loads
      constexpr int kFirst = kQuarter * kLoads / 4, kFetch = (kQuarter + 1) * kLoads / 4 - kFirst;
      for_range<kFirst + kTurn * kFetch / kSlots, kFirst + (kTurn + 1) * kFetch / kSlots>([&](auto k) __attribute__((always_inline)) {
        fetch_pair(integral_constant<int, kParts>{}, integral_constant<int, kAt>{}, decltype(k)::value, sub == 3 ? s : s - 1);
      });
      __builtin_amdgcn_sched_barrier(0);
      mfma32<kBf16>(acc[a][b], fw[sub & 1][a], fx[sub & 1][b]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // Stage s, in place i.  The barrier comes before the last sub-step, whose operands are in
  // registers by then: its MFMAs run while the next stage's first operands are read.
  const auto stage = [&](auto i_c, int s) __attribute__((always_inline)) {
    using std::integral_constant;
    step(i_c, integral_constant<int, 0>{}, s);
    step(i_c, integral_constant<int, 1>{}, s);
    step(i_c, integral_constant<int, 2>{}, s);
    land(integral_constant<int, kParts - 4>{});
    step(i_c, integral_constant<int, 3>{}, s);
  };
  // The ring's first turn of loads: its last two parts come in the place of a stage before
  // the first one's, so that the first sub-steps load most of them.
  for_range<0, kParts - 2>([&](auto p_c) {
    constexpr int p = decltype(p_c)::value;
    for_range<0, p % 2 ? kLoadsX : kLoadsW>([&](auto k) {
      fetch(std::integral_constant<bool, p % 2 != 0>{}, decltype(k)::value, first + p / 2, part_of(p_c));
    });
  });
  land(std::integral_constant<int, kParts - 4>{});
  for_range<0, kLoads / 4>([&](auto k) {
    fetch_pair(std::integral_constant<int, kParts>{}, std::integral_constant<int, 2 * kParts - 2>{}, decltype(k)::value, first - 1);
  });
  for_range<0, kN + kM>([&](auto k) {
    read(k, part_of(std::integral_constant<int, 0>{}), part_of(std::integral_constant<int, 1>{}), 0, 0);
  });
  constexpr int kTurn = kParts % 2 ? kParts : kParts / 2;  // stages
  int s = first;
  for (; s + kTurn <= stages; s += kTurn) {
    for_range<0, kTurn>([&](auto i) __attribute__((always_inline)) { stage(i, s + decltype(i)::value); });
  }
  for_range<0, kTurn - 1>([&](auto i) __attribute__((always_inline)) {
    if (s + decltype(i)::value < stages) stage(i, s + decltype(i)::value);
  });
  vq::wait_vmcnt<0>();  // the last loads (zeros) are in before their buffers are used again

  // Results: each row tile through LDS (a wavefront's own part, four columns a chunk, the
  // chunks in an order by the row), then four columns of a row a lane.
  constexpr int kStride = 32 * kN;
  const auto exchange_at = [](int row, int chunk) { return row * kStride + 4 * (chunk ^ (kN > 1 ? row & 15 : (row >> 1) & 7)); };
  // exchanges in one part of the ring (the smaller ones' share)
  constexpr int kEach = (T::part_bytes(0) < T::part_bytes(1) ? T::part_bytes(0) : T::part_bytes(1)) / (32 * kStride * 4);
  static_assert(kEach * kParts >= kWaves, "the wavefronts' exchanges fit the ring");
  float* part = nullptr;
  for_range<0, (kWaves + kEach - 1) / kEach>([&](auto p_c) {
    if (wave / kEach == decltype(p_c)::value) part = reinterpret_cast<float*>(part_of(p_c)) + wave % kEach * 32 * kStride;
  });
  __syncthreads();
  const bool split = gridDim.y > 1;
  constexpr int kWave = kGated ? 16 * kN : 32 * kN;  // a wavefront's output columns
  // (Loops, so that there are few copies of what follows the sums.)  A lane's columns are the same
  // in all its rows; the residuals of two or four rows are on their way while those before are
  // finished (asked for before their stores, which a wait would count otherwise).
  constexpr int kChunksRow = kWave / 4;  // of four columns
  static_assert(kChunksRow % 8 == 0, "whole groups of rows");
  const int chunk = lane % kChunksRow, r0 = lane / kChunksRow;
  const int64_t c = c0 + kWave * wn + 4 * chunk;
  const Columns<4, kGated> columns(g.e, split ? g.e.n : c);
  const auto row_at = [&](int i, int k) { return 32 * (kM * wm + i) + r0 + k * (64 / kChunksRow); };
  constexpr int kTogether = kM == 4 ? 2 : 4;  // (registers)
  float next[kTogether][4];
  const auto ask = [&](int i, int k) __attribute__((always_inline)) {
#pragma unroll
    for (int y = 0; y < kTogether; ++y) {
      const int m = row_at(i, k + y);
      if (!split && m < nrows) load_residual<4>(g.e, m0 + m, c, next[y]);
    }
  };
  ask(0, 0);
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
#pragma unroll 1
    for (int k = 0; k < kChunksRow / 2; k += kTogether) {
      float residual[kTogether][4];
#pragma unroll
      for (int y = 0; y < kTogether; ++y)
#pragma unroll
        for (int q = 0; q < 4; ++q) residual[y][q] = next[y][q];
      if (k + kTogether < kChunksRow / 2) ask(i, k + kTogether);
      else if (i + 1 < kM) ask(i + 1, 0);
#pragma unroll
      for (int y = 0; y < kTogether; ++y) {
        const int m = row_at(i, k + y), mr = m & 31;
        const f32x4_t a = *reinterpret_cast<const f32x4_t*>(part + exchange_at(mr, chunk));
        const f32x4_t b = *reinterpret_cast<const f32x4_t*>(part + exchange_at(mr, chunk + (kGated ? 4 * kN : 0)));
        if (m >= nrows || c >= g.e.n) continue;
        float v[4] = {a[0], a[1], a[2], a[3]}, u[4] = {b[0], b[1], b[2], b[3]};
        if (split) {
          const int64_t lines = kGated ? 2 * g.e.n : g.e.n;
          float* to = g.sums + (int64_t(blockIdx.y) * g.x.rows + m0 + m) * lines + c;
          store_columns<4>(to, vq::kFP32, 0, g.e.n - c, v);
          if constexpr (kGated) store_columns<4>(to + g.e.n, vq::kFP32, 0, g.e.n - c, u);
        } else {
          finish_columns<4, kGated>(g.e, m0 + m, c, v, u, columns, residual[y]);
        }
      }
    }
  }
}

}  // namespace dense
