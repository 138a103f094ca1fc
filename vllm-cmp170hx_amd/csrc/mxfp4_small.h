// Few rows times MXFP4 weights, dense and for the routed experts: the weights
// are read once, straight from memory to the registers of the wavefront that
// multiplies them, K split over the wavefronts of a workgroup.
//
// A wavefront holds 16 columns (weight rows): per chunk of 512 k a lane (r =
// lane & 15, q = lane >> 4) loads column r's blocks 4 j + q (j < 4; 16 rows of 64
// bytes a load) and the column's 16 scale bytes, and multiplies them in four
// v_mfma_scale_f32_16x16x128 with the activations' blocks 4 j + q of row r.
// Activations lie in LDS as [block][row] (16-byte blocks: a lane's operand in one
// conflict-free read) with the four j's scale bytes of a (chunk, q, row) in one
// dword, whose byte j the MFMA selects.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mxfp4.h"

namespace mx {

constexpr int kChunk = 16;  // blocks, 512 k

// acc += A B over 128 k: A 16 rows, B 16 columns, lane (r = lane & 15, q = lane
// >> 4) holding the block of k 32 q .. 32 q + 31 of row / column r, its scale in
// byte 0 of sa and byte kByte of sb; lane's acc[i] is row 4 q + i, column r.
template <int kByte>
__device__ __forceinline__ f32x4_t mfma16_byte(const u32x4_t& a, uint32_t sa, const u32x4_t& b, uint32_t sb, const f32x4_t& acc) {
  const i32x8_t av{int(a[0]), int(a[1]), int(a[2]), int(a[3]), 0, 0, 0, 0};
  const i32x8_t bv{int(b[0]), int(b[1]), int(b[2]), int(b[3]), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc, 4, 4, 0, int(sa), kByte, int(sb));
}

// One chunk of one row's operand: blocks 4 j + q and their scale bytes.
struct ChunkOperand {
  u32x4_t code[4];
  uint32_t scale[4];
};

// Chunk c of a row of `blocks` blocks; past the row zeros under scale 1.
__device__ __forceinline__ ChunkOperand load_chunk(const uint8_t* codes, const uint8_t* scales, int c, int blocks, int q) {
  ChunkOperand o;
  const int b0 = c * kChunk;
  if (b0 + kChunk <= blocks) {
#pragma unroll
    for (int j = 0; j < 4; ++j) o.code[j] = *reinterpret_cast<const u32x4_t*>(codes + int64_t(b0 + 4 * j + q) * kBlockBytes);
    uint32_t s[4];
    __builtin_memcpy(s, scales + b0, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) o.scale[j] = s[j] >> (8 * q);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int b = b0 + 4 * j + q;
      o.code[j] = u32x4_t{0, 0, 0, 0};
      o.scale[j] = 127;
      if (b < blocks) {
        o.code[j] = *reinterpret_cast<const u32x4_t*>(codes + int64_t(b) * kBlockBytes);
        o.scale[j] = scales[b];
      }
    }
  }
  return o;
}

// LDS of `rows` activation rows of `chunks` chunks: codes, then scale dwords.
__host__ __device__ constexpr int64_t small_codes_bytes(int64_t rows, int64_t chunks) { return rows * chunks * kChunk * kBlockBytes; }
__host__ __device__ constexpr int64_t small_bytes(int64_t rows, int64_t chunks) {
  return small_codes_bytes(rows, chunks) + rows * chunks * kChunk;
}

// Rows row_at(0 .. rows - 1) of x (element offsets) quantized into LDS by
// `threads` threads, a quarter block each at a time; blocks past the row are
// zeros under scale 1.
template <int kDtype, typename RowAt>
__device__ __forceinline__ void quantize_to_lds(const void* x, const RowAt& row_at, int rows, int blocks, int chunks, bool wide,
                                                uint8_t* lds, int tid, int threads) {
  uint8_t* scale = lds + small_codes_bytes(rows, chunks);
  const int per_row = chunks * kChunk * 4;
  for (int m = 0; m < rows; ++m) {
    const int64_t at = row_at(m);
    for (int i = tid; i < per_row; i += threads) {
      const int b = i >> 2, j = i & 3;
      uint32_t s = 127, w = 0;
      // (all four lanes of the quad alike)
      if (b < blocks) w = quantize_quarter(load8<kDtype>(x, at + int64_t(b) * kBlock + 8 * j, wide), s);
      *reinterpret_cast<uint32_t*>(lds + (b * rows + m) * kBlockBytes + 4 * j) = w;
      if (j == 0) scale[(((b >> 4) * 4 + (b & 3)) * rows + m) * 4 + ((b >> 2) & 3)] = uint8_t(s);
    }
  }
}

// The same of rows that are codes and scales already (row_at: their numbers).
template <typename RowAt>
__device__ __forceinline__ void copy_to_lds(const uint8_t* codes, const uint8_t* scales, const RowAt& row_at, int rows, int blocks,
                                            int chunks, uint8_t* lds, int tid, int threads) {
  uint8_t* scale = lds + small_codes_bytes(rows, chunks);
  for (int m = 0; m < rows; ++m) {
    const int64_t row = row_at(m) * blocks;
    for (int b = tid; b < chunks * kChunk; b += threads) {
      u32x4_t w{0, 0, 0, 0};
      uint8_t s = 127;
      if (b < blocks) {
        w = *reinterpret_cast<const u32x4_t*>(codes + (row + b) * kBlockBytes);
        s = scales[row + b];
      }
      *reinterpret_cast<u32x4_t*>(lds + (b * rows + m) * kBlockBytes) = w;
      scale[(((b >> 4) * 4 + (b & 3)) * rows + m) * 4 + ((b >> 2) & 3)] = s;
    }
  }
}

// acc += chunk c of the weights times row r of the LDS activations (lanes past
// the rows repeat the last one).
__device__ __forceinline__ void multiply_lds(const ChunkOperand& w, const uint8_t* lds, int c, int rows, int chunks, int r, int q,
                                             f32x4_t& acc) {
  const uint8_t* scale = lds + small_codes_bytes(rows, chunks);
  const int m = min(r, rows - 1);
  const uint32_t s = *reinterpret_cast<const uint32_t*>(scale + ((c * 4 + q) * rows + m) * 4);
  const uint8_t* at = lds + ((c * kChunk + q) * rows + m) * kBlockBytes;
  const int step = 4 * rows * kBlockBytes;
  const auto code = [&](int j) { return *reinterpret_cast<const u32x4_t*>(at + j * step); };
  acc = mfma16_byte<0>(w.code[0], w.scale[0], code(0), s, acc);
  acc = mfma16_byte<1>(w.code[1], w.scale[1], code(1), s, acc);
  acc = mfma16_byte<2>(w.code[2], w.scale[2], code(2), s, acc);
  acc = mfma16_byte<3>(w.code[3], w.scale[3], code(3), s, acc);
}

// The same with both operands loaded from memory.
__device__ __forceinline__ void multiply_loaded(const ChunkOperand& w, const ChunkOperand& x, f32x4_t& acc) {
#pragma unroll
  for (int j = 0; j < 4; ++j) acc = mfma16_byte<0>(w.code[j], w.scale[j], x.code[j], x.scale[j], acc);
}

}  // namespace mx
