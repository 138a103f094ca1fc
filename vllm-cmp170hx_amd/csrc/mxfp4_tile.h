// The many-row product of MXFP4 activations with MXFP4 weights, dense and for
// the routed experts' tasks.
//
// One workgroup of four wavefronts (2 x 2) computes 64 kN columns by 64 kM
// rows, each wavefront 32 kN x 32 kM of v_mfma_scale_f32_32x32x64 tiles (its
// rate is twice the 16x16x128 form's: 8.9 against 4.6 PFLOP/s in a loop of
// nothing else).  A stage is 256 k: the 128 code bytes and 8 scale bytes of every
// row and column, in one of kBufs buffers; one barrier a stage.
//  * Codes come to LDS by DMA, one 128-byte line of a row in eight lanes, up to
//    kBufs - 1 stages ahead.  A row's eight 16-byte blocks lie in LDS in the order
//    kb ^ (row / 2 & 7), so that the 16 rows that a ds_read_b128 reads at once, all
//    at one kb, lie on 16 different 16-byte columns of the 64 banks.
//  * A lane of the 32x32x64 form holds one block: row lane & 31, block 2 sub +
//    (lane >> 5) of the stage's 64-k sub-step `sub`.  Scales come through
//    registers, a row's even blocks' bytes in one half of its LDS entry and the
//    odd blocks' in the other: a lane reads one half a row and stage, and the
//    MFMA's byte selector is `sub`.
//  * Weights are the A operand, rows the B operand, so that a lane's sums are
//    of one row: 16 of a 32-column block, the other 16 in lane ^ 32.
// What bounds it: where a CU holds one workgroup and all comes from caches, a stage of
// the 128 x 128 tile takes 0.53 us with four buffers and 0.74 with two, its MFMAs
// 0.21; the LDS moves 96 KB a stage (0.32 us), 256 x 256 half as much an MFMA.  2048 rows
// of 8192 x 28672 take 248 us (3.9 PFLOP/s; 3.5 rounds of workgroups), 400 rows of
// 14336 x 4096 in two K splits 23.5.  Routed, 16384 slots over 128 experts of 2048 x 768:
// gate | up 79 us (234 MB), down 65 (117 MB and 134 MB of slot rows).  Tried without gain:
// stages of 128 k in four buffers (half lines cost the loads more than the depth gains:
// 266 us for 250), a wavefront that asks for weights ahead.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "mxfp4.h"

namespace mx {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;

constexpr int kTileThreads = 256;
constexpr int kStageBlocks = 8;                          // 256 k; the fewest that the kernel takes
constexpr int kStageBytes = kStageBlocks * kBlockBytes;  // of codes, a row

// f(std::integral_constant<int, i>) for i = first .. last - 1.
template <int first, int last, typename F>
__device__ __forceinline__ void for_range(F&& f) {
  if constexpr (first < last) {
    f(std::integral_constant<int, first>{});
    for_range<first + 1, last>(f);
  }
}
template <int n, typename F>
__device__ __forceinline__ void for_each(F&& f) {
  for_range<0, n>(f);
}

enum TileMode : int { kDense = 0, kGateUp = 1, kDown = 2 };

struct TileArgs {
  const uint8_t *a, *as;  // activations: rows of `blocks` blocks
  int64_t a_rows;         // kGateUp: tokens
  const uint8_t *w, *ws;  // kDense [n], kGateUp [experts][n = 2 inter], kDown [experts][n]
  int64_t rows, n;
  int blocks;
  void* out;              // kDense: [rows][n] of out_dtype; kDown: FP32 [slots][n]
  int out_dtype;
  int tiles_n, tiles_m;   // kDense: workgroups; else tiles_n alone
  int split_stages;       // kDense: stages of one split of K (gridDim.y splits, whose
                          // sums go to FP32 [split][rows][n] at out)
  // the routed forms
  const int32_t* table;
  int64_t tasks, sorted;  // offsets in the table
  const float* topk_w;
  int top_k;
  float limit;
  uint8_t *h, *hs;        // kGateUp: rows of n / 2
};

// SiLU(min(g, L)) clamp(u, -L, L); a NaN stays one (comparisons, not fminf).
__device__ __forceinline__ float swiglu(float g, float u, float limit) {
  g = g > limit ? limit : g;
  u = u > limit ? limit : (u < -limit ? -limit : u);
  return g / (1.0f + __expf(-g)) * u;
}

// Two values rounded to nearest even, the first one in the low half.
template <int kDtype>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (kDtype == vq::kBF16) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, bf16x2_t{__bf16(a), __bf16(b)});  // v_cvt_pk_bf16_f32
  } else {
    return uint32_t(__builtin_bit_cast(uint16_t, _Float16(a))) | (uint32_t(__builtin_bit_cast(uint16_t, _Float16(b))) << 16);
  }
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, int(bytes), 0x00020000);
}

// An offset past any buffer: such loads give zeros.
constexpr uint32_t kPastEnd = 0x80000000u;

// A stage's scale bytes of a row of at least eight blocks, from block b0 on (the
// last eight, where fewer are left), as they come from memory,
__device__ __forceinline__ uint64_t load_scales(const uint8_t* row, int b0, int blocks) {
  uint64_t v;
  __builtin_memcpy(&v, row + min(b0, blocks - kStageBlocks), 8);
  return v;
}
// and block b0's first, 127 past the row, as the even blocks' dword and the odd
// blocks'.
__device__ __forceinline__ uint2 order_scales(uint64_t v, int b0, int blocks) {
  const int past = max(b0 - (blocks - kStageBlocks), 0) * 8;  // bits, less than 64
  if (past) v = (v >> past) | (0x7f7f7f7f7f7f7f7full << (64 - past));
  const uint32_t lo = uint32_t(v), hi = uint32_t(v >> 32);
  return make_uint2(__builtin_amdgcn_perm(hi, lo, 0x06040200u), __builtin_amdgcn_perm(hi, lo, 0x07050301u));
}

template <int kSub>
__device__ __forceinline__ void mfma32(f32x16_t& acc, const u32x4_t& a, uint32_t sa, const u32x4_t& b, uint32_t sb) {
  const i32x8_t av{int(a[0]), int(a[1]), int(a[2]), int(a[3]), 0, 0, 0, 0};
  const i32x8_t bv{int(b[0]), int(b[1]), int(b[2]), int(b[3]), 0, 0, 0, 0};
  acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, acc, 4, 4, kSub, int(sa), kSub, int(sb));
}

// 32 rows of 32 kN columns from LDS to the output, eight columns a lane, in 16-byte
// stores whatever the rows' alignment (1500 x 2592 x 5003 on 128 x 128 tiles: 26 us,
// with an element a store 33).  slots (LDS): the rows' slots and their
// router weights, which multiply them.
template <int kN, int kDtype>
__device__ __forceinline__ void store_rows(const float* part, int stride, int lane, int mt, int nrows, int ct, const TileArgs& g,
                                           int64_t m0, const int2* slots) {
  constexpr int kChunks = 4 * kN;  // of eight columns, a row
  const int ch = lane % kChunks, r0 = lane / kChunks;
  const int c = ct + 8 * ch;
#pragma unroll
  for (int k = 0; k < kChunks / 2; ++k) {
    const int mr = r0 + k * (64 / kChunks);
    const int m = mt + mr;
    const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(part + mr * stride + 8 * ch);
    const f32x4_t hi = *reinterpret_cast<const f32x4_t*>(part + mr * stride + 8 * ch + 4);
    if (m >= nrows || c >= g.n) continue;
    int64_t row = m0 + m;
    float weight = 1;
    if (slots) {
      row = slots[m].x;
      weight = __builtin_bit_cast(float, slots[m].y);
    }
    const int64_t at = row * g.n + c;
    if (c + 8 > g.n) {  // the last columns
      for (int q = 0; q < g.n - c; ++q) vq::store_act(g.out, kDtype, at + q, part[mr * stride + 8 * ch + q] * weight);
    } else if constexpr (kDtype == vq::kFP32) {
      const f32x4_t v[2] = {lo * weight, hi * weight};
      __builtin_memcpy(static_cast<float*>(g.out) + at, v, 32);
    } else {
      u32x4_t w;
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = pack16<kDtype>((q < 2 ? lo : hi)[2 * (q & 1)], (q < 2 ? lo : hi)[2 * (q & 1) + 1]);
      __builtin_memcpy(static_cast<uint16_t*>(g.out) + at, &w, 16);
    }
  }
}

// Workgroups of a size that a CU's LDS (and registers) hold, two at most.
constexpr int tile_groups(int n, int m, int bufs) { return n * m > 8 || 64 * (n + m) * (kStageBytes * bufs + 16) > 80 * 1024 ? 1 : 2; }

template <int kN, int kM, int kMode, int kBufs>
__global__ __launch_bounds__(kTileThreads, tile_groups(kN, kM, kBufs)) void tile_kernel(TileArgs g) {
  constexpr int kCols = 64 * kN, kRows = 64 * kM, kLines = kCols + kRows;
  constexpr int kLoadRows = 8;  // lines of a 1 KB DMA load
  constexpr int kLoadsW = kCols / (4 * kLoadRows), kLoadsA = kRows / (4 * kLoadRows);  // loads a wavefront and stage
  constexpr int kLoads = kLoadsW + kLoadsA;
  static_assert(kBufs == 2 || kBufs == 4, "stage buffers");
  constexpr int kScaleRows = (kLines + kTileThreads - 1) / kTileThreads;
  // (buffers by name: the compiler then sees that a stage's reads are not of the
  // buffer that the DMA is filling, and does not wait for it)
  constexpr int kBufBytes = kLines * kStageBytes;
  __shared__ __attribute__((aligned(1024))) uint8_t buf0[kBufBytes], buf1[kBufBytes], buf2[kBufs > 2 ? kBufBytes : 16],
      buf3[kBufs > 2 ? kBufBytes : 16];
  __shared__ __attribute__((aligned(16))) uint2 scale0[kLines], scale1[kLines];
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
  const int wn = wave & 1, wm = wave >> 1;

  // ---- which columns and rows
  int64_t wbase = 0;   // first weight row of the matrix
  int c0, nrows;       // first column (kGateUp: of h); rows of this tile
  int64_t m0 = 0;      // kDense: first row; else the task's first sorted row
  const int32_t* sorted = nullptr;
  const int inter = int(g.n / 2);
  if constexpr (kMode == kDense) {
    // XCD x (workgroups x, x + 8, ...) takes a run of tiles, rows first: it
    // fetches few weight columns and its L2 keeps them for all the rows
    const int total = g.tiles_n * g.tiles_m, per = (total + 7) / 8;
    const int t = int(blockIdx.x & 7) * per + int(blockIdx.x >> 3);
    if (int(blockIdx.x >> 3) >= per || t >= total) return;
    c0 = t / g.tiles_m * kCols;
    m0 = int64_t(t % g.tiles_m) * kRows;
    nrows = int(min(int64_t(kRows), g.rows - m0));
  } else {
    // XCD x takes a run of tasks, a task's columns one after another: the tasks of
    // one expert share its weights in L2
    const int local = int(blockIdx.x >> 3), all = g.table[0], per = (all + 7) / 8;
    const int task = int(blockIdx.x & 7) * per + local / g.tiles_n;
    if (local / g.tiles_n >= per) return;
    if (task >= all) return;
    const int4 tk = reinterpret_cast<const int4*>(g.table + g.tasks)[task];
    wbase = int64_t(vq::uniform(tk.x)) * g.n;
    m0 = vq::uniform(tk.y);
    nrows = vq::uniform(tk.z);
    sorted = g.table + g.sorted + m0;
    c0 = local % g.tiles_n * (kMode == kGateUp ? kCols / 2 : kCols);
  }
  // the weight row of the tile's line i (< kCols): kGateUp has, per wavefront
  // column, kN / 2 gate blocks and then their up blocks
  const auto weight_row = [&](int i) -> int64_t {
    if constexpr (kMode == kGateUp) {
      const int half = i / (32 * kN), j = i % (32 * kN) / 32;
      const bool up = j >= kN / 2;
      const int c = c0 + 16 * kN * half + 32 * (up ? j - kN / 2 : j) + (i & 31);
      return min(c, inter - 1) + (up ? inter : 0);
    } else {
      return min(int64_t(c0 + i), g.n - 1);
    }
  };
  const auto act_row = [&](int i) -> int64_t {  // relative to the activations' base
    const int t = min(i, nrows - 1);
    if constexpr (kMode == kGateUp) return sorted[t] / g.top_k;
    return t;
  };
  static_assert(kMode != kDown || kRows <= kTileThreads, "a thread a row");
  const int64_t act0 = kMode == kGateUp ? 0 : m0;
  const int64_t line = int64_t(g.blocks) * kBlockBytes;
  // this tile's weight rows from the first one's address on
  const int64_t w0 = kMode == kGateUp ? 0 : c0;
  const int w_rows = kMode == kGateUp ? int(g.n) : int(min(int64_t(kCols), g.n - c0));
  const __amdgpu_buffer_rsrc_t wbuf = buffer(g.w + (wbase + w0) * line, uint32_t(w_rows) * uint32_t(line));
  const __amdgpu_buffer_rsrc_t abuf =
      buffer(g.a + act0 * line, uint32_t(kMode == kGateUp ? g.a_rows : int64_t(nrows)) * uint32_t(line));

  // ---- loads: 1 KB each, kLoadRows lines; a wavefront's first kLoadsW bring
  // weights.  Rows that follow each other: the first one's offset is scalar (a row
  // of the buffer also where the load's lie past its end: their sums are not
  // stored; the rest of a load that begins inside it is zeros), and the lane's part
  // has two values, by the parity of the load's place.  Scattered rows (kGateUp's
  // tokens): an offset a lane and load.
  const uint32_t rline = uint32_t(line);
  const int sub_row = lane >> 3;
  const auto first_line = [&](int i) {
    return i < kLoadsW ? kLoadRows * (kLoadsW * wave + i) : kCols + kLoadRows * (kLoadsA * wave + i - kLoadsW);
  };
  const auto swizzle_of = [](int l) { return (l >> 1) & 7; };
  const int kb[2] = {(lane & 7) ^ swizzle_of(sub_row), (lane & 7) ^ swizzle_of(kLoadRows + sub_row)};
  const uint32_t lane_off[2] = {sub_row * rline + kb[0] * kBlockBytes, sub_row * rline + kb[1] * kBlockBytes};
  uint32_t token_off[kMode == kGateUp ? kLoadsA : 1];
  if constexpr (kMode == kGateUp) {
#pragma unroll
    for (int i = 0; i < kLoadsA; ++i) {
      token_off[i] = uint32_t(act_row(first_line(kLoadsW + i) - kCols + sub_row)) * rline + kb[(kLoadsA * wave + i) & 1] * kBlockBytes;
    }
  }
  // the scalar first row of load i
  const auto first_row = [&](int i) -> int {
    if (i >= kLoadsW) return first_line(i) - kCols < nrows ? first_line(i) - kCols : 0;
    if constexpr (kMode == kGateUp) {
      const int l = first_line(i), half = l / (32 * kN), j = l % (32 * kN) / 32;
      const bool up = j >= kN / 2;
      const int c = c0 + 16 * kN * half + 32 * (up ? j - kN / 2 : j) + (l & 31);
      return (c < inter ? c : 0) + (up ? inter : 0);  // inter: whole 32s
    }
    return first_line(i) < w_rows ? first_line(i) : 0;
  };
  const uint8_t* srow[kScaleRows];
#pragma unroll
  for (int i = 0; i < kScaleRows; ++i) {
    const int l = min(tid + i * kTileThreads, kLines - 1);
    srow[i] = l < kCols ? g.ws + (wbase + weight_row(l)) * g.blocks : g.as + (act0 + act_row(l - kCols)) * g.blocks;
  }
  const int all_stages = (g.blocks + kStageBlocks - 1) / kStageBlocks;
  int first = 0, stages = all_stages;  // this split's, up to `stages`
  if constexpr (kMode == kDense) {
    first = int(blockIdx.y) * g.split_stages;
    stages = min(first + g.split_stages, all_stages);
  }
  // kDown: the rows' slots, and (below, behind the first loads) their weights, for the end
  __shared__ int2 slots[kMode == kDown ? kRows : 1];
  int slot = 0;
  float slot_weight = 0;
  if constexpr (kMode == kDown) slot = sorted[min(tid, nrows - 1)];
  // DMA load i of stage s (zeros past the last stage)
  const auto fetch = [&](auto i_c, int s, uint8_t* buf) __attribute__((always_inline)) {
    constexpr int i = decltype(i_c)::value;
    const int left = s < stages ? g.blocks - s * kStageBlocks : 0;
    const int parity = (i < kLoadsW ? kLoadsW * wave + i : kLoadsA * wave + i - kLoadsW) & 1;
    constexpr bool scattered = kMode == kGateUp && i >= kLoadsW;
    const uint32_t lane_part = scattered ? token_off[scattered ? i - kLoadsW : 0] : lane_off[parity];
    const uint32_t o = left >= kStageBlocks || kb[parity] < left ? lane_part : kPastEnd;
    const int row_part = scattered ? 0 : first_row(i) * int(rline);
    // (the scalar offset stays below the buffer's size, or its bounds check would wrap)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(i < kLoadsW ? wbuf : abuf, (lds_ptr_t)(buf + first_line(i) * kStageBytes), 16,
                                             int(o), row_part + (left > 0 ? s * kStageBytes : 0), 0, 0);
  };
  // Scale bytes come for four stages at a time: a stage's eight bytes of a row by
  // themselves would ask L2 for as many lines as the codes do.
  uint64_t scales_now[4][kScaleRows], scales_next[4][kScaleRows];
  const auto fetch_scales = [&](uint64_t (&to)[4][kScaleRows], int s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kScaleRows; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) to[k][i] = load_scales(srow[i], (s + k) * kStageBlocks, g.blocks);
  };
  // stage s has landed (its loads of this wavefront, behind which kBufs - 2 stages'
  // stay on their way, then everyone's), and no wavefront reads the stage before it
  // any more
  const auto land = [&](const uint64_t (&from)[kScaleRows], int s, uint2* scales) __attribute__((always_inline)) {
    vq::wait_vmcnt<(kBufs - 2) * kLoads>();
    const int b0 = min(s, all_stages - 1) * kStageBlocks;
#pragma unroll
    for (int i = 0; i < kScaleRows; ++i) {
      if (kLines % kTileThreads == 0 || tid + i * kTileThreads < kLines) {
        scales[tid + i * kTileThreads] = order_scales(from[i], b0, g.blocks);
      }
    }
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

  const int wline = 32 * kN * wn + r, aline = kCols + 32 * kM * wm + r;
  const int swizzle = swizzle_of(r);
  uint32_t sw[2][kN], sa[2][kM];          // this stage's scales and the next one's
  u32x4_t fw[2][kN], fa[2][kM];           // this sub-step's operands and the next one's
  const auto read_scales = [&](const uint2* scales, uint32_t (&w)[kN], uint32_t (&a)[kM]) {
    const uint32_t* words = reinterpret_cast<const uint32_t*>(scales);
#pragma unroll
    for (int i = 0; i < kN; ++i) w[i] = words[2 * (wline + 32 * i) + h];
#pragma unroll
    for (int j = 0; j < kM; ++j) a[j] = words[2 * (aline + 32 * j) + h];
  };
  // operand i of a sub-step: kN of weights, then kM of rows
  const auto read = [&](auto i_c, const uint8_t* buf, int sub, int set) __attribute__((always_inline)) {
    constexpr int i = decltype(i_c)::value;
    const int at = ((2 * sub + h) ^ swizzle) * kBlockBytes;
    if constexpr (i < kN) fw[set][i] = *reinterpret_cast<const u32x4_t*>(buf + (wline + 32 * i) * kStageBytes + at);
    else fa[set][i - kN] = *reinterpret_cast<const u32x4_t*>(buf + (aline + 32 * (i - kN)) * kStageBytes + at);
  };
  // Sub-step `sub` of a stage: between its kN kM MFMAs, one or two at a time, the
  // next sub-step's operands are read (of `next`, at sub-step next_sub) and loads
  // kFirst .. kLast - 1 of stage s issued into `into`.  A wavefront issues in order
  // and alone on its SIMD: what stands between two MFMAs hides behind the first
  // one's 32 cycles (six or seven instructions), and loads in one burst would hold
  // up the MFMAs behind them (16 cycles a load and CU).
  const auto step = [&](auto sub_c, auto first_c, auto last_c, int set, const uint8_t* next, int next_sub, int s,
                        uint8_t* into) __attribute__((always_inline)) {
    constexpr int sub = decltype(sub_c)::value, kFirst = decltype(first_c)::value, kLast = decltype(last_c)::value;
    constexpr int kReads = kN + kM, kSlots = kN * kM;
    for_each<kSlots>([&](auto slot_c) __attribute__((always_inline)) {
      constexpr int slot = decltype(slot_c)::value, i = slot / kM, j = slot % kM;
      for_range<slot * kReads / kSlots, (slot + 1) * kReads / kSlots>([&](auto k) __attribute__((always_inline)) {
        read(k, next, next_sub, (sub + 1) & 1);
      });
      constexpr int kFetch = kLast - kFirst, kTurn = (slot + kSlots / 2) % kSlots;  // in other slots than the reads
      for_range<kFirst + kTurn * kFetch / kSlots, kFirst + (kTurn + 1) * kFetch / kSlots>(
          [&](auto k) __attribute__((always_inline)) { fetch(k, s, into); });
      __builtin_amdgcn_sched_barrier(0);
      mfma32<sub>(acc[i][j], fw[sub & 1][i], sw[set][i], fa[sub & 1][j], sa[set][j]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // Stage s, the i-th of a round of four.  The barrier comes before the last
  // sub-step, whose operands are in registers by then: its MFMAs run while the next
  // stage's first operands are read, and its buffer takes stage s + kBufs: half of
  // those loads here, the others in the next stage's first sub-steps.
  constexpr int kHalf = kLoads / 2, kMore = kHalf + kLoads / 4;
  const auto stage = [&](auto i_c, auto whole_c, int s) __attribute__((always_inline)) {
    constexpr int i = decltype(i_c)::value;
    using std::integral_constant;
    constexpr integral_constant<int, 0> c0{};
    constexpr integral_constant<int, i + 1> c1{};
    uint8_t* const cur = buf(i_c);
    uint8_t* const next = buf(c1);
    uint8_t* const prev = buf(integral_constant<int, i + kBufs - 1>{});
    uint2* const next_scales = i & 1 ? scale0 : scale1;
    constexpr int set = i & 1;
    step(c0, integral_constant<int, kHalf>{}, integral_constant<int, kMore>{}, set, cur, 1, s + kBufs - 1, prev);
    step(integral_constant<int, 1>{}, integral_constant<int, kMore>{}, integral_constant<int, kLoads>{}, set, cur, 2, s + kBufs - 1, prev);
    step(integral_constant<int, 2>{}, c0, c0, set, cur, 3, 0, cur);
    land(i < 3 ? scales_now[(i + 1) & 3] : scales_next[0], s + 1, next_scales);
    if constexpr (i == 0 && decltype(whole_c)::value) fetch_scales(scales_next, s + 4);
    read_scales(next_scales, sw[set ^ 1], sa[set ^ 1]);
    step(integral_constant<int, 3>{}, c0, integral_constant<int, kHalf>{}, set, next, 0, s + kBufs, cur);
  };
  fetch_scales(scales_now, first);
  for_range<0, kBufs - 1>([&](auto b_c) {
    for_range<0, kLoads>([&](auto k) { fetch(k, first + decltype(b_c)::value, buf(b_c)); });
  });
  if constexpr (kMode == kDown) slot_weight = g.topk_w[slot];
  land(scales_now[0], first, scale0);
  for_range<0, kHalf>([&](auto k) { fetch(k, first + kBufs - 1, buf(std::integral_constant<int, kBufs - 1>{})); });
  read_scales(scale0, sw[0], sa[0]);
  for_range<0, kN + kM>([&](auto k) { read(k, buf0, 0, 0); });
  int s = first;
  for (; s + 4 <= stages; s += 4) {
    for_range<0, 4>([&](auto i) __attribute__((always_inline)) { stage(i, std::true_type{}, s + decltype(i)::value); });
#pragma unroll
    for (int i = 0; i < kScaleRows; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) scales_now[k][i] = scales_next[k][i];
  }
  if (s < stages) {
    stage(std::integral_constant<int, 0>{}, std::false_type{}, s);
    if (s + 1 < stages) {
      stage(std::integral_constant<int, 1>{}, std::false_type{}, s + 1);
      if (s + 2 < stages) stage(std::integral_constant<int, 2>{}, std::false_type{}, s + 2);
    }
  }
  vq::wait_vmcnt<0>();  // the last loads (zeros) are in before their buffers are used again

  // ---- results
  if constexpr (kMode == kGateUp) {
    // block j of this wavefront: column cb .. cb + 31 of h, row m = lane & 31 of
    // row tile i; this lane holds elements 8 p + 4 h + q (p, q < 4)
#pragma unroll
    for (int j = 0; j < kN / 2; ++j) {
      const int cb = c0 + 16 * kN * wn + 32 * j;
      if (cb >= inter) continue;
#pragma unroll
      for (int i = 0; i < kM; ++i) {
        float v[16];
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          v[k] = swiglu(acc[j][i][k], acc[j + kN / 2][i][k], g.limit);
          top = max(top, magnitude(v[k]));
        }
        top = max(top, uint32_t(__shfl_xor(int(top), 32)));
        const uint32_t s = block_scale(top);
        const uint32_t w0v = s == 255u ? 0u : codes8(v, s), w1v = s == 255u ? 0u : codes8(v + 8, s);
        // halves 8 p + 4 h: even h low, odd h high in dword p
        const uint32_t o0 = uint32_t(__shfl_xor(int(w0v), 32)), o1 = uint32_t(__shfl_xor(int(w1v), 32));
        const int m = 32 * (kM * wm + i) + r;
        if (h == 0 && m < nrows) {
          u32x4_t block;
          block[0] = (w0v & 0xffffu) | (o0 << 16);
          block[1] = (w0v >> 16) | (o0 & 0xffff0000u);
          block[2] = (w1v & 0xffffu) | (o1 << 16);
          block[3] = (w1v >> 16) | (o1 & 0xffff0000u);
          const int64_t row = m0 + m;
          *reinterpret_cast<u32x4_t*>(g.h + row * (inter / 2) + cb / 2) = block;
          g.hs[row * (inter / kBlock) + cb / kBlock] = uint8_t(s);
        }
      }
    }
  } else {
    // each row tile through LDS (a wavefront's own part, rows 16 bytes apart
    // from a bank's multiple), then whole rows of 32 kN columns
    constexpr int kStride = 32 * kN + 4;
    static_assert((4 / kBufs) * 32 * kStride * 4 <= kBufBytes, "the wavefronts' exchanges fit the stage buffers");
    float* part = kBufs == 2 ? reinterpret_cast<float*>(wave < 2 ? buf0 : buf1) + (wave & 1) * 32 * kStride
                             : reinterpret_cast<float*>(wave < 2 ? (wave ? buf1 : buf0) : (wave == 2 ? buf2 : buf3));
    if constexpr (kMode == kDown) {
      if (tid < kRows) slots[tid] = make_int2(slot, __builtin_bit_cast(int, slot_weight));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kM; ++i) {
#pragma unroll
      for (int j = 0; j < kN; ++j) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          f32x4_t v;
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q] = acc[j][i][4 * p + q];
          *reinterpret_cast<f32x4_t*>(part + r * kStride + 32 * j + 8 * p + 4 * h) = v;
        }
      }
      const int mt = 32 * (kM * wm + i), ct = c0 + 32 * kN * wn;
      const int64_t o0 = kMode == kDense ? m0 + int64_t(blockIdx.y) * g.rows : m0;  // first output row
      if constexpr (kMode == kDense) {
        if (g.out_dtype == vq::kBF16) store_rows<kN, vq::kBF16>(part, kStride, lane, mt, nrows, ct, g, o0, nullptr);
        else if (g.out_dtype == vq::kFP16) store_rows<kN, vq::kFP16>(part, kStride, lane, mt, nrows, ct, g, o0, nullptr);
        else store_rows<kN, vq::kFP32>(part, kStride, lane, mt, nrows, ct, g, o0, nullptr);
      } else {
        store_rows<kN, vq::kFP32>(part, kStride, lane, mt, nrows, ct, g, o0, slots);
      }
    }
  }
}

}  // namespace mx
