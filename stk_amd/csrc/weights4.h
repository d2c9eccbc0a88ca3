// Weights of 4 bits and a scale (and offset) for every group of inputs, as stk_pack_4bit lays them out.
//
// A piece is 16 outputs x 128 inputs, 1024 bytes, the A operand of four v_mfma_f32_16x16x32: lane l of a wavefront finds its 32
// codes - output l % 16, of every 32 inputs the eight from 8 (l / 16) on - in the 16 bytes from 16 l on, one dword for each step of
// 32 inputs.  Bits [4p + 3, 4p + 7) of a dword are the code of input 2p of the eight, the same bits 16 higher (from bit 32 on: again from 0 on)
// that of input 2p + 1, so that one shift, or turn, and one and-or make a pair of 16-bit values of each; the first pair of
// bfloat16 values needs no shift.  Pieces follow each other along the inputs, then along the outputs, then
// expert by expert.  Scales (16-bit) come in blocks that belong to 16 outputs and the groups of a piece, or one group of whole
// pieces: [expert][16 outputs][block][quarter of the outputs][group][4], so that what a lane needs of a block (it accumulates the four outputs
// of quarter l / 16) is next to each other.  Inputs beyond the last hold code 8, outputs and groups beyond the last scale 0.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace stk {

constexpr int kPieceInputs = 128, kPieceOutputs = 16, kPieceBytes = 1024;

__host__ __device__ inline int64_t pieces_in(int64_t inputs) { return (inputs + kPieceInputs - 1) / kPieceInputs; }
__host__ __device__ inline int64_t pieces_out(int64_t outputs) { return (outputs + kPieceOutputs - 1) / kPieceOutputs; }
__host__ __device__ inline int64_t groups_of(int64_t inputs, int64_t group) { return (inputs + group - 1) / group; }
__host__ __device__ inline int64_t groups_in_block(int64_t group) { return group < kPieceInputs ? kPieceInputs / group : 1; }
__host__ __device__ inline int64_t scale_blocks(int64_t inputs, int64_t group) { return (groups_of(inputs, group) + groups_in_block(group) - 1) / groups_in_block(group); }
// Every multiple of 128 from the inputs on means one group of them all.  What is below the C ABI sees the smallest such size: the kernels
// count a group's pieces in 32 bits, and the sums above are not to overflow.
inline int64_t group_within(int64_t inputs, int64_t group) { return group % kPieceInputs == 0 && group >= inputs ? pieces_in(inputs) * kPieceInputs : group; }
// Where the scale of output o (0 .. 15) of the tile-th 16 outputs and group g is.
__host__ __device__ inline int64_t scale_at(int64_t tile, int o, int64_t g, int64_t inputs, int64_t group) {
  const int64_t sub = groups_in_block(group);
  return ((tile * scale_blocks(inputs, group) + g / sub) * 4 + o / 4) * 4 * sub + g % sub * 4 + o % 4;
}

constexpr int kCodesTurn = 3;   // what a dword of codes from bit 0 on is turned to the left by
// The code of output o % 16 and input i % 128 of a piece.
__host__ __device__ inline int code_of(const uint32_t* piece, int o, int i) {
  const int lane = (o & 15) + 16 * ((i >> 3) & 3), dword = (i >> 5) & 3, j = i & 7, bit = 4 * (j >> 1) + 16 * (j & 1);
  const uint32_t w = piece[4 * lane + dword];
  return (int)((w >> kCodesTurn | w << (32 - kCodesTurn)) >> bit & 15u);
}

}  // namespace stk
