// Microscaled rows (OCP MX): elements of 4 bits (e2m1) or 8 (e4m3) in blocks of 32 columns with one e8m0 scale each,
// and the layout of a bank of e2m1 weights that the expert products read.
//
// Rows: codes [R, C * bits / 8] (e2m1: column 2 j in byte j's low half), scales [R, C / 32], C the columns rounded up to
// a stage of 256, zeros in between.
// Banks: v_mfma_scale_f32_16x16x128_f8f6f4 takes 16 rows x 128 columns, lane l the 32 columns l >> 4 of row l & 15 in
// e2m1 and their scale, one byte of a register. A stage is two of them, 8 blocks of a row: step s multiplies the blocks
// 2 q + s, q = l >> 4 (which block meets which step is free as long as both operands agree), so that a lane's two blocks
// of a stage are neighbours in a row's codes and scales. Tile t holds 16 rows: codes [stage][s][lane][16 bytes], so that
// an operand is one run of 1 KB, and scales [lane][stage][s], a lane's scales of two stages in one word (the stages
// rounded up to an even number).
// An e4m3 operand's lane holds the columns 16 q .. and 64 + 16 q .. of the 128: halves of two blocks, while its scale
// register still belongs to block q.
#pragma once
#include "common.hpp"

namespace d3 {

constexpr int MX_BLOCK = 32, MX_STAGE = 256;

__host__ __device__ constexpr int mx_stages(int cols) { return (cols + MX_STAGE - 1) / MX_STAGE; }
// bytes of scales of a lane's row of a bank's tile
__host__ __device__ constexpr int mx_lane_scales(int stages) { return 2 * ((stages + 1) & ~1); }

// 2^(code - 127) for a scale code; 255 is NaN
D3_INLINE float mx_scale(uint32_t code) {
  return __uint_as_float(code == 0u ? 0x00400000u : code == 255u ? 0x7FC00000u : code << 23);
}

}  // namespace d3
