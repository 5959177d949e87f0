// fp32 contractions on the matrix cores and the fp32 tiles that feed them.
//
// MFMA 32x32x2 f32, lane l = 32 h + c: A[m = c][k = h], B[k = h][n = c], C as
// in mfma_common.h.  A contraction over K elements runs K / 2 MFMAs; lane half
// h supplies element k = perm(s, h) of step s, any bijection shared by both
// operands.  Over a head dimension the kernels take d = h D / 2 + s, so each
// lane walks a contiguous half of every row (16-byte LDS reads serve four
// steps); over a 32-row tile of an accumulator layout they take the row
// crow(i, h) of register i, so a C tile feeds the next contraction as it is.
//
// LDS tiles hold 32 rows x D floats, row-major, 16-byte chunk q of row r at
// q ^ fsw(r): 16 lanes reading one chunk each of 16 consecutive rows hit 16
// different bank groups (the operands whose rows are lanes), and 64 lanes
// reading a 32-float segment of rows r and r + 4 (the operands whose rows are
// accumulator rows) hit the two halves of the banks (D >= 64; at D = 32 a row
// is half the banks and the segment reads take two passes).  Tiles reach LDS
// by direct buffer loads (DMA), each lane fetching the global chunk its
// swizzled position holds; rows past the buffer range arrive as zeros.
#pragma once

#include "mfma_common.h"

namespace tsattn {

__device__ __forceinline__ f32x16 mfma32f(float a, float b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

template <int D>
__host__ __device__ __forceinline__ constexpr int fsw(int r) {
  return D >= 64 ? ((r & 3) | ((r & 4) << 1) | ((r & 8) >> 1)) : ((r >> 1) & 7);
}

// A [32 x D] fp32 tile in LDS (the layout above).
template <int D>
struct FTile {
  static constexpr int CPR = D / 4;                  // 16-byte chunks per row
  static constexpr int BYTES = 32 * D * 4;           // per tile
  static constexpr int BLOCKS = BYTES / 1024;        // 1 KiB DMA blocks per tile
  static constexpr int RPB = 1024 / (D * 4);         // rows per DMA block

  // Byte offset (within the block's rows) of the global chunk lane l of a
  // DMA of block n fetches: its LDS slot is 16 l of the block.
  __device__ __forceinline__ static uint32_t dma_off(int n, int lane, uint32_t stride_b) {
    const int rr = lane / CPR, p = lane % CPR, row = n * RPB + rr;
    return static_cast<uint32_t>(rr) * stride_b + static_cast<uint32_t>((p ^ fsw<D>(row)) * 16);
  }
  // 16 bytes of row r, chunk q (d = 4 q .. 4 q + 3).
  __device__ __forceinline__ static float4 chunk(const char *t, int r, int q) {
    return *reinterpret_cast<const float4 *>(t + r * D * 4 + ((q ^ fsw<D>(r)) << 4));
  }
  // One float: row r, column d.
  __device__ __forceinline__ static float elem(const char *t, int r, int d) {
    return *reinterpret_cast<const float *>(t + r * D * 4 + (((d >> 2) ^ fsw<D>(r)) << 4) + ((d & 3) << 2));
  }
};

}  // namespace tsattn
