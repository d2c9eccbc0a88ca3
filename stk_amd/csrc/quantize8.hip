// Quantisation to 8-bit floating point with power-of-two scales, and the stored weights' own formats (fp8.h).
//   scale = the smallest 2^e, e >= -126, with max |v| <= 448 2^e over a block;   code = v / scale, rounded to nearest, ties to even
// Division by a power of two is exact, so that a code is defined without a word on how it is computed; what the larger of two possible
// scales loses is one step of the smallest values, since e4m3 keeps its relative precision down to 2^-6.  The matrix units take such
// scales beside the codes, for nothing.  A block with an infinity or a NaN becomes NaN as a whole.
//
// All of it is bound by bytes: what is read once is written in every form that the products of a training step want of it.  16384 x 4096 bfloat16 along and down:
// 53 us for 268 MB, 5.1 TB/s; 64 weights of 1024 x 4096 and their transposes 218 - 226 us for 1.07 GB; rows alone 22 us for 8192 x 4096.
#include "common.h"
#include "fp8.h"
#include "values.h"

namespace stk {

enum Form8 : int { kNoForm = 0, kRowForm = 1, kPieceForm = 2 };

__device__ __forceinline__ uint32_t larger_bits(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int CONTROL>
__device__ __forceinline__ uint32_t moved_bits(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, 0xf, 0xf, true); }
__device__ __forceinline__ uint32_t team16_larger(uint32_t v) {
  v = larger_bits(v, moved_bits<0xb1>(v)), v = larger_bits(v, moved_bits<0x4e>(v));
  return v = larger_bits(v, moved_bits<0x141>(v)), larger_bits(v, moved_bits<0x140>(v));
}

// Codes of eight values under one scale.
__device__ __forceinline__ uint2 eight_codes(const float (&v)[8], uint32_t most, float inverse) {
  if (most >= 0x7f800000u) return make_uint2(kNan8, kNan8);
  return make_uint2(codes8(v[0] * inverse, v[1] * inverse, v[2] * inverse, v[3] * inverse), codes8(v[4] * inverse, v[5] * inverse, v[6] * inverse, v[7] * inverse));
}

// Rows alone: a team of 16 lanes takes 128 values of a row.  With indices: row r is that of the token indices[r] / top_k (there are rows / top_k).
template <int DTYPE>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const typename Value<DTYPE>::stored* __restrict__ x, int64_t rows, int64_t size, int64_t stride,
                                                            uint8_t* __restrict__ codes, uint8_t* __restrict__ exponents, const int32_t* __restrict__ indices, int top_k) {
  typedef typename Value<DTYPE>::stored stored;
  const int64_t blocks = blocks8(size), teams = (int64_t)gridDim.x * 16;
  const int lane = threadIdx.x & 15;
  for (int64_t at = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); at < rows * blocks; at += teams) {
    const int64_t row = at / blocks, block = at % blocks, first = block * kBlock8 + lane * 8;
    int64_t token = row;
    if (indices) {
      const int slot = indices[row];
      token = (unsigned)slot < (unsigned)rows ? slot / top_k : 0;
    }
    const stored* from = x + token * stride + first;
    float v[8];
    if (first + 8 <= size) load8<DTYPE>(v, from);
    else {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = first + j < size ? Value<DTYPE>::widen(from[j]) : 0.f;
    }
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) most = larger_bits(most, __float_as_uint(v[j]) & 0x7fffffffu);
    most = team16_larger(most);
    const int byte = exponent_byte8(most);
    *reinterpret_cast<uint2*>(codes + row * row_stride8(size) + first) = eight_codes(v, most, inverse_power8(byte));
    if (lane == 0) exponents[exponent_at8(row, block, rows)] = (uint8_t)byte;
  }
}

struct Quantize8 {
  const void* x;
  int64_t stride_e, stride_r, stride_c, rows, cols;   // elements
  uint8_t *along, *along_exponents;                   // quantised along the columns, a line for each row
  uint8_t *down, *down_exponents;                     // quantised down the rows, a line for each column
};

// 128 x 128 values, for which the thread of column eighth c and row quad q keeps rows 4 q .. 4 q + 3 and 64 more.  ALONG and DOWN: the forms
// of codes along the rows and down the columns.  JOINT: one scale for the whole block (weights).  A column's four codes of a quad are one
// dword of LDS; a column's 128 bytes then lie next to each other.
template <int DTYPE, int ALONG, int DOWN, bool JOINT>
__global__ __launch_bounds__(256) void quantize_blocks_kernel(Quantize8 p) {
  typedef typename Value<DTYPE>::stored stored;
  constexpr int kPitch = 33;   // dwords of a column: the quads' writes of 16 lanes fall on every second bank
  __shared__ uint32_t turned[DOWN ? 128 * kPitch : 1];
  __shared__ uint32_t most_of[16][128];
  const int eighth = threadIdx.x & 15, quad = threadIdx.x >> 4;
  const int64_t row0 = (int64_t)blockIdx.y * kBlock8, col0 = (int64_t)blockIdx.x * kBlock8;
  const int64_t row_blocks = blocks8(p.rows), col_blocks = blocks8(p.cols);
  const stored* x = static_cast<const stored*>(p.x) + (int64_t)blockIdx.z * p.stride_e;
  const int64_t first = col0 + 8 * eighth;
  float v[8][8];
  if (first + 8 <= p.cols && p.stride_c == 1) {   // (all eight rows on their way together; behind the last one it once more, and then zeros)
    decltype(fetch8<DTYPE>(x)) raw[8];
#pragma unroll
    for (int i = 0; i < 8; i++) raw[i] = fetch8<DTYPE>(x + min(row0 + 64 * (i >> 2) + 4 * quad + (i & 3), p.rows - 1) * p.stride_r + first);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      widen8<DTYPE>(v[i], raw[i]);
#pragma unroll
      for (int j = 0; j < 8; j++) v[i][j] = row0 + 64 * (i >> 2) + 4 * quad + (i & 3) < p.rows ? v[i][j] : 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int64_t row = row0 + 64 * (i >> 2) + 4 * quad + (i & 3);
      const stored* from = x + row * p.stride_r + first * p.stride_c;
#pragma unroll
      for (int j = 0; j < 8; j++) v[i][j] = row < p.rows && first + j < p.cols ? Value<DTYPE>::widen(from[j * p.stride_c]) : 0.f;
    }
  }
  uint32_t row_most[8], col_most[8];
#pragma unroll
  for (int i = 0; i < 8; i++) row_most[i] = col_most[i] = 0;
#pragma unroll
  for (int i = 0; i < 8; i++)
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint32_t u = __float_as_uint(v[i][j]) & 0x7fffffffu;
      row_most[i] = larger_bits(row_most[i], u), col_most[j] = larger_bits(col_most[j], u);
    }
  if constexpr (JOINT) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) most = larger_bits(most, row_most[i]);
    most = team16_larger(most);
    if (eighth == 0) most_of[quad][0] = most;
    __syncthreads();
    most = 0;
    for (int q = 0; q < 16; q++) most = larger_bits(most, most_of[q][0]);
#pragma unroll
    for (int i = 0; i < 8; i++) row_most[i] = col_most[i] = most;
  } else {
    if constexpr (ALONG != kNoForm) {
#pragma unroll
      for (int i = 0; i < 8; i++) row_most[i] = team16_larger(row_most[i]);
    }
    if constexpr (DOWN != kNoForm) {
#pragma unroll
      for (int j = 0; j < 8; j++) most_of[quad][8 * eighth + j] = col_most[j];
      __syncthreads();
      if (threadIdx.x < 128) {
        uint32_t most = 0;
#pragma unroll
        for (int q = 0; q < 16; q++) most = larger_bits(most, most_of[q][threadIdx.x]);
        most_of[0][threadIdx.x] = most;   // (only this thread reads or writes the column)
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; j++) col_most[j] = most_of[0][8 * eighth + j];
    }
  }
  if constexpr (ALONG != kNoForm) {
    uint8_t *codes = p.along, *exponents = p.along_exponents;
    if constexpr (ALONG == kPieceForm) {
      codes += (int64_t)blockIdx.z * piece_bytes8(p.rows, p.cols);
      exponents += (int64_t)blockIdx.z * scale_bytes8(p.rows, p.cols, kPowerScales);
    }
    const int64_t end = ALONG == kPieceForm ? padded_lines8(p.rows) : p.rows;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int64_t row = row0 + 64 * (i >> 2) + 4 * quad + (i & 3);
      if (row >= end) continue;
      const int byte = exponent_byte8(row_most[i]);
      const int64_t line = ALONG == kPieceForm ? place8(row) : row;
      const int64_t to = ALONG == kPieceForm ? piece_at8(line, first, col_blocks) : row * row_stride8(p.cols) + first;
      *reinterpret_cast<uint2*>(codes + to) = eight_codes(v[i], row_most[i], inverse_power8(byte));
      if (eighth == 0) exponents[exponent_at8(line, blockIdx.x, end)] = (uint8_t)byte;
    }
  }
  if constexpr (DOWN != kNoForm) {
    uint8_t *codes = p.down, *exponents = p.down_exponents;
    if constexpr (DOWN == kPieceForm) {
      codes += (int64_t)blockIdx.z * piece_bytes8(p.cols, p.rows);
      exponents += (int64_t)blockIdx.z * scale_bytes8(p.cols, p.rows, kPowerScales);
    }
    const int64_t end = DOWN == kPieceForm ? padded_lines8(p.cols) : p.cols;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int byte = exponent_byte8(col_most[j]);
      const float inverse = inverse_power8(byte);
      const bool nan = col_most[j] >= 0x7f800000u;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t four = codes8(v[4 * h][j] * inverse, v[4 * h + 1][j] * inverse, v[4 * h + 2][j] * inverse, v[4 * h + 3][j] * inverse);
        turned[(8 * eighth + j) * kPitch + 16 * h + quad] = nan ? kNan8 : four;
      }
      if (quad == 0 && first + j < end) exponents[exponent_at8(DOWN == kPieceForm ? place8(first + j) : first + j, blockIdx.y, end)] = (uint8_t)byte;
    }
    __syncthreads();
    // 16 bytes of a column a thread: neighbours within a column of rows, or in the order of a piece
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int at = k * 256 + threadIdx.x;
      int64_t to, line;
      int col, chunk;
      if constexpr (DOWN == kPieceForm) {
        const int piece = at >> 7, h = (at >> 6) & 1, lane = at & 63;   // piece of the eight, access, lane
        col = line_of_place8(piece * 16 + (lane & 15)), chunk = 4 * h + (lane >> 4);
        line = col0 + col;
        to = piece8(col0 / kPieceLines8 + piece, blockIdx.y, row_blocks) * kPieceBytes8 + h * 1024 + lane * 16;
      } else {
        col = at >> 3, chunk = at & 7;
        line = col0 + col;
        to = line * row_stride8(p.rows) + row0 + 16 * chunk;
      }
      if (line >= end) continue;
      Quad q;
#pragma unroll
      for (int i = 0; i < 4; i++) q[i] = turned[col * kPitch + 4 * chunk + i];
      *reinterpret_cast<Quad*>(codes + to) = q;
    }
  }
}

// Given codes [expert][input][output] and scales [expert][input block][output block] -> pieces and their scales.  A thread per code;
// weights are laid out once.
__global__ __launch_bounds__(256) void pack8_kernel(const uint8_t* __restrict__ codes, int64_t experts, int64_t inputs, int64_t outputs, uint8_t* __restrict__ packed) {
  const int64_t blocks = blocks8(inputs), lines = padded_lines8(outputs), per = lines * blocks * kBlock8 / 4, step = (int64_t)gridDim.x * 256;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < experts * per; at += step) {   // neighbours: neighbouring outputs, four inputs each
    const int64_t e = at / per, line = at % lines, input = at % per / lines * 4;
    uint32_t four = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (line < outputs && input + i < inputs) four |= (uint32_t)codes[(e * inputs + input + i) * outputs + line] << (8 * i);
    *reinterpret_cast<uint32_t*>(packed + e * (lines * blocks * kBlock8) + piece_at8(place8(line), input, blocks)) = four;
  }
}
__global__ __launch_bounds__(256) void pack8_scales_kernel(const void* __restrict__ scales, int kind, int64_t experts, int64_t inputs, int64_t outputs, void* __restrict__ packed) {
  const int64_t blocks = blocks8(inputs), down = blocks8(outputs), lines = padded_lines8(outputs), stride = exponent_stride8(inputs);
  const int64_t count = experts * (kind == kPowerScales ? lines * stride : down * blocks), step = (int64_t)gridDim.x * 256;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < count; at += step) {
    if (kind == kPowerScales) {
      const int64_t e = at / (lines * stride), line = at / 4 % lines, b = at / (4 * lines) % (stride / 4) * 4 + at % 4;   // (line and its place lie in the same 64, of one scale)
      static_cast<uint8_t*>(packed)[at] = b < blocks && line / kBlock8 < down ? static_cast<const uint8_t*>(scales)[(e * blocks + b) * down + line / kBlock8] : (uint8_t)127;
    } else {
      const int64_t e = at / (down * blocks), o = at / blocks % down, b = at % blocks;
      static_cast<float*>(packed)[at] = static_cast<const float*>(scales)[(e * blocks + b) * down + o];
    }
  }
}
template <int DTYPE>
__global__ __launch_bounds__(256) void dequantize8_kernel(const uint8_t* __restrict__ packed, const void* __restrict__ scales, int kind, int64_t experts, int64_t inputs,
                                                          int64_t outputs, typename Value<DTYPE>::stored* __restrict__ out) {
  const int64_t blocks = blocks8(inputs), step = (int64_t)gridDim.x * 256;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < experts * inputs * outputs; at += step) {
    const int64_t o = at % outputs, i = at / outputs % inputs, e = at / outputs / inputs, place = place8(o);
    const float code = value8(packed[e * piece_bytes8(outputs, inputs) + piece_at8(place, i, blocks)]);
    float v;
    if (kind == kPowerScales) {
      const int byte = static_cast<const uint8_t*>(scales)[e * scale_bytes8(outputs, inputs, kind) + exponent_at8(place, i / kBlock8, padded_lines8(outputs))];
      v = byte == 255 ? NAN : ldexpf(code, byte - 127);
    } else {
      v = code * static_cast<const float*>(scales)[(e * blocks8(outputs) + o / kBlock8) * blocks + i / kBlock8];
    }
    out[at] = Value<DTYPE>::round(v);
  }
}

static dim3 loop_grid8(int64_t count, int64_t each) {
  const int64_t n = (count + each - 1) / each;
  return dim3((unsigned)(n < 1 << 18 ? n : 1 << 18));
}

// What a tensor's sizes may be: positions within one are counted in 64 bits, blocks and lines in 32.
bool sizes8(int64_t lines, int64_t size) { return lines <= INT32_MAX - 512 && size <= INT32_MAX - 512; }

int quantize_rows8(const char* who, const void* x, int64_t rows, int64_t size, int64_t stride, int dtype, uint8_t* codes, uint8_t* exponents, const int32_t* indices, int top_k,
                   hipStream_t stream) {
  const dim3 grid = loop_grid8(rows * blocks8(size), 16);
  for_dtype(dtype, [&](auto d) {
    typedef typename Value<d()>::stored T;
    hipLaunchKernelGGL((quantize_rows_kernel<d()>), grid, dim3(256), 0, stream, static_cast<const T*>(x), rows, size, stride, codes, exponents, indices, top_k);
  });
  return check_launch(who);
}

template <int ALONG, int DOWN, bool JOINT>
static int quantize_blocks(const char* who, const Quantize8& p, int64_t experts, int dtype, hipStream_t stream) {
  const int64_t down = blocks8(p.rows), across = blocks8(p.cols);
  if (down > 65535 || experts > 65535) return fail(STK_ERR_UNSUPPORTED, "%s: %lld rows, %lld matrices", who, (long long)p.rows, (long long)experts);
  const dim3 grid((unsigned)across, (unsigned)down, (unsigned)experts);
  for_dtype(dtype, [&](auto d) { hipLaunchKernelGGL((quantize_blocks_kernel<d(), ALONG, DOWN, JOINT>), grid, dim3(256), 0, stream, p); });
  return check_launch(who);
}

}  // namespace stk

using namespace stk;

extern "C" int64_t stk_8bit_piece_bytes(int64_t experts, int64_t inputs, int64_t outputs) {
  return experts < 1 || inputs < 1 || outputs < 1 ? 0 : experts * piece_bytes8(outputs, inputs);
}
extern "C" int64_t stk_8bit_scale_bytes(int64_t experts, int64_t inputs, int64_t outputs, int float_scales) {
  return experts < 1 || inputs < 1 || outputs < 1 ? 0 : experts * scale_bytes8(outputs, inputs, float_scales ? kFloatScales : kPowerScales);
}
extern "C" int64_t stk_8bit_row_bytes(int64_t rows, int64_t size) { return rows < 1 || size < 1 ? 0 : rows * row_stride8(size); }
extern "C" int64_t stk_8bit_exponent_bytes(int64_t rows, int64_t size) { return rows < 1 || size < 1 ? 0 : rows * exponent_stride8(size); }

static int weights_check8(const char* who, int64_t experts, int64_t inputs, int64_t outputs) {
  if (experts < 1 || inputs < 1 || outputs < 1) return fail(STK_ERR_DIMS, "%s: %lld matrices of %lld x %lld", who, (long long)experts, (long long)inputs, (long long)outputs);
  if (!sizes8(inputs, outputs) || experts > INT32_MAX) return fail(STK_ERR_UNSUPPORTED, "%s: size exceeds 32-bit range", who);
  return STK_OK;
}

extern "C" int stk_quantize_8bit(const void* w, int64_t stride_e, int64_t stride_i, int64_t stride_o, int64_t experts, int64_t inputs, int64_t outputs, int dtype,
                                 void* packed, void* exponents, void* packed_t, void* exponents_t, stk_stream_t stream) {
  const char* who = "stk_quantize_8bit";
  if (int rc = weights_check8(who, experts, inputs, outputs)) return rc;
  if (!is_value_dtype(dtype)) return fail(STK_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (!w || !packed || !exponents || !packed_t != !exponents_t) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (!aligned16(packed) || (packed_t && !aligned16(packed_t))) return fail(STK_ERR_UNSUPPORTED, "%s: packed weights at a multiple of 16 bytes", who);
  const Quantize8 p = {w, stride_e, stride_i, stride_o, inputs, outputs, static_cast<uint8_t*>(packed_t), static_cast<uint8_t*>(exponents_t),
                       static_cast<uint8_t*>(packed), static_cast<uint8_t*>(exponents)};
  if (packed_t) return quantize_blocks<kPieceForm, kPieceForm, true>(who, p, experts, dtype, static_cast<hipStream_t>(stream));
  return quantize_blocks<kNoForm, kPieceForm, true>(who, p, experts, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int stk_pack_8bit(const uint8_t* codes, const void* scales, int float_scales, int64_t experts, int64_t inputs, int64_t outputs, void* packed,
                             void* packed_scales, stk_stream_t stream) {
  const char* who = "stk_pack_8bit";
  if (int rc = weights_check8(who, experts, inputs, outputs)) return rc;
  if (!codes || !scales || !packed || !packed_scales) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (!aligned16(packed) || !aligned16(packed_scales)) return fail(STK_ERR_UNSUPPORTED, "%s: packed weights at a multiple of 16 bytes", who);
  const int kind = float_scales ? kFloatScales : kPowerScales;
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(pack8_kernel, loop_grid8(experts * piece_bytes8(outputs, inputs) / 4, 256), dim3(256), 0, s, codes, experts, inputs, outputs,
                     static_cast<uint8_t*>(packed));
  const int64_t count = experts * scale_bytes8(outputs, inputs, kind) / (kind == kFloatScales ? 4 : 1);
  hipLaunchKernelGGL(pack8_scales_kernel, loop_grid8(count, 256), dim3(256), 0, s, scales, kind, experts, inputs, outputs, packed_scales);
  return check_launch(who);
}

extern "C" int stk_dequantize_8bit(const void* packed, const void* scales, int float_scales, int64_t experts, int64_t inputs, int64_t outputs, void* out, int dtype,
                                   stk_stream_t stream) {
  const char* who = "stk_dequantize_8bit";
  if (int rc = weights_check8(who, experts, inputs, outputs)) return rc;
  if (!is_value_dtype(dtype)) return fail(STK_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (!packed || !scales || !out) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  for_dtype(dtype, [&](auto d) {
    typedef typename Value<d()>::stored T;
    hipLaunchKernelGGL((dequantize8_kernel<d()>), loop_grid8(experts * inputs * outputs, 256), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const uint8_t*>(packed), scales, float_scales ? kFloatScales : kPowerScales, experts, inputs, outputs, static_cast<T*>(out));
  });
  return check_launch(who);
}

extern "C" int stk_quantize_rows_8bit(const void* x, int64_t rows, int64_t size, int64_t stride, int dtype, void* codes, void* exponents, void* columns,
                                      void* column_exponents, int pieces, stk_stream_t stream) {
  const char* who = "stk_quantize_rows_8bit";
  if (rows < 0 || size < 1 || stride < 0) return fail(STK_ERR_DIMS, "%s: %lld rows of %lld", who, (long long)rows, (long long)size);
  if (!is_value_dtype(dtype)) return fail(STK_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (!sizes8(rows, size)) return fail(STK_ERR_UNSUPPORTED, "%s: size exceeds 32-bit range", who);
  if (rows == 0) return STK_OK;
  if (!x || !codes != !exponents || !columns != !column_exponents || (!codes && !columns)) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if ((codes && !aligned16(codes)) || (columns && !aligned16(columns))) return fail(STK_ERR_UNSUPPORTED, "%s: codes at a multiple of 16 bytes", who);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!columns) return quantize_rows8(who, x, rows, size, stride, dtype, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(exponents), nullptr, 1, s);
  const Quantize8 p = {x, 0, stride, 1, rows, size, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(exponents), static_cast<uint8_t*>(columns),
                       static_cast<uint8_t*>(column_exponents)};
  if (codes) return pieces ? quantize_blocks<kRowForm, kPieceForm, false>(who, p, 1, dtype, s) : quantize_blocks<kRowForm, kRowForm, false>(who, p, 1, dtype, s);
  return pieces ? quantize_blocks<kNoForm, kPieceForm, false>(who, p, 1, dtype, s) : quantize_blocks<kNoForm, kRowForm, false>(who, p, 1, dtype, s);
}
