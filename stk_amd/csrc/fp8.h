// 8-bit floating-point values (e4m3: 4 bits of exponent, 3 of mantissa, at most 448, no infinities) with a scale for every block of 128, as
// the products take them.
//
// Rows: codes [row][blocks x 128], zeros beyond the last input, and an exponent byte (2^(byte - 127)) for each row and block, [block / 4][row][block % 4], so
// that a dword holds those of four neighbouring blocks and neighbouring rows' dwords are neighbours.
//
// Pieces: the operand that all rows share, 16 of its lines x 128 inputs in 2048 bytes, in the order of a wavefront's two 16-byte accesses:
// access h, lane l has inputs 64 h + 16 (l / 16) .. + 15 of line l % 16.  (Which input goes where in v_mfma_scale_f32_16x16x128 does not
// matter as long as both operands agree, and all inputs of a block have one scale.)  The four pieces of 64 lines lie next to each other, then
// follow those of the next block, of the next 64 lines, of the next expert.  Lines are dealt to the pieces of 64 so that the four sums that each
// of a row's four lanes has of two pieces make 64 neighbouring bytes of a 16-bit result: line 32 u + 8 q + 4 v + r of the 64 is line 4 q + r
// of piece 2 u + v.  Lines are padded to a multiple of 64 with zeros.
// Scales of pieces: exponent bytes [block / 4][place of the line][block % 4] ("power"), or fp32 [ceil(lines / 128)][blocks] ("float").
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace stk {

constexpr int kBlock8 = 128, kPieceLines8 = 16, kPieceBytes8 = 2048, kGroupLines8 = 64;
enum Scales8 : int { kPowerScales = 0, kFloatScales = 1 };

__host__ __device__ inline int64_t blocks8(int64_t size) { return (size + kBlock8 - 1) / kBlock8; }
__host__ __device__ inline int64_t exponent_stride8(int64_t size) { return (blocks8(size) + 3) / 4 * 4; }
__host__ __device__ inline int64_t row_stride8(int64_t size) { return blocks8(size) * kBlock8; }
__host__ __device__ inline int64_t padded_lines8(int64_t lines) { return (lines + kGroupLines8 - 1) / kGroupLines8 * kGroupLines8; }
__host__ __device__ inline int64_t piece_bytes8(int64_t lines, int64_t size) { return padded_lines8(lines) / kPieceLines8 * blocks8(size) * kPieceBytes8; }
__host__ __device__ inline int64_t scale_bytes8(int64_t lines, int64_t size, int kind) {
  return kind == kPowerScales ? padded_lines8(lines) * exponent_stride8(size) : blocks8(lines) * blocks8(size) * 4;
}
// Place of a line among those of its pieces, and the line of a place.
__host__ __device__ inline int64_t place8(int64_t line) { return (line & ~(int64_t)63) + ((line >> 5) & 1) * 32 + ((line >> 2) & 1) * 16 + ((line >> 3) & 3) * 4 + (line & 3); }
__host__ __device__ inline int line_of_place8(int place) { return (place & ~63) + ((place >> 5) & 1) * 32 + ((place >> 2) & 3) * 8 + ((place >> 4) & 1) * 4 + (place & 3); }
// Byte of a line's exponent of a block, from the first of an operand of so many lines.
__host__ __device__ inline int64_t exponent_at8(int64_t line, int64_t block, int64_t lines) { return ((block >> 2) * lines + line) * 4 + (block & 3); }
// Piece p (16 places) of a block, in pieces from the start of an operand.
__host__ __device__ inline int64_t piece8(int64_t p, int64_t block, int64_t blocks) { return ((p >> 2) * blocks + block) * 4 + (p & 3); }
// Byte of (place, input) from the start of an operand's pieces; `blocks` of them along the inputs.
__host__ __device__ inline int64_t piece_at8(int64_t place, int64_t input, int64_t blocks) {
  const int64_t piece = piece8(place / kPieceLines8, input / kBlock8, blocks);
  const int k = (int)(input % kBlock8);
  return piece * kPieceBytes8 + (k >> 6) * 1024 + ((int)(place & 15) + 16 * ((k & 63) >> 4)) * 16 + (k & 15);
}

// The exponent byte of values whose largest magnitude has the fp32 bits `most`: the smallest 2^e with most <= 448 2^e, e >= -126.  448 =
// 1.75 2^8.  An infinity or a NaN: 0 (the codes say that it is one).
__host__ __device__ inline int exponent_byte8(uint32_t most) {
  if (most >= 0x7f800000u) return 0;
  const int e = (int)(most >> 23) - 8 + ((most & 0x7fffffu) > 0x600000u ? 1 : 0);   // 127 more than the exponent
  return e < 1 ? 1 : e;
}
// 1 / 2^(byte - 127), bytes 1 .. 254 (the largest is 247).
__device__ __forceinline__ float inverse_power8(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

constexpr uint32_t kNan8 = 0x7f7f7f7fu;   // four codes
// Codes of four values that are at most 448, rounded to nearest, ties to even.
__device__ __forceinline__ uint32_t codes8(float a, float b, float c, float d) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}
// The same of 16-bit values (a low, b high halves) divided by a power of two, the conversion's own: on an MI355X equal for all values to that at most.
template <bool BF16>
__device__ __forceinline__ uint32_t codes8_of_pairs(uint32_t a, uint32_t b, float scale) {
  typedef short i16x2_t __attribute__((ext_vector_type(2)));
  i16x2_t v = {0, 0};
  if constexpr (BF16) {
    typedef __bf16 pair_t __attribute__((ext_vector_type(2)));
    v = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(v, __builtin_bit_cast(pair_t, a), scale, false);
    v = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(v, __builtin_bit_cast(pair_t, b), scale, true);
  } else {
    typedef _Float16 pair_t __attribute__((ext_vector_type(2)));
    v = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(v, __builtin_bit_cast(pair_t, a), scale, false);
    v = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(v, __builtin_bit_cast(pair_t, b), scale, true);
  }
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ float value8(uint8_t code) { return __builtin_amdgcn_cvt_f32_fp8((int)code, 0); }

}  // namespace stk
