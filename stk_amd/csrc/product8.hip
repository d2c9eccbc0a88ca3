// Products of rows with 8-bit floating-point weights that have a scale for every block of 128 x 128, and the gradient of such weights.
//   out = act(sum over blocks b of (sum over the inputs i of b of xq[i] wq[i][o]) sx[b] sw[b][o / 128])
// xq, sx: the rows quantised as fp8.h says.  Powers of two go into the matrix instruction's own scale operands, one byte a line and block;
// so does that of a weight's fp32 scale, whose mantissa multiplies the fp32 sum of a block.
//
// The matrix units multiply e4m3 values exactly and add the products of one instruction with some 13 bits below the largest of them (measured on
// an MI355X, all fp8 instructions alike: products below 2^-13 of the largest lose bits, 2e-6 of the sum of magnitudes in the root mean square for
// normal values); what they add to, and everything across blocks, is fp32.  That is two orders below the last place of the 16-bit results.
#include <type_traits>

#include "common.h"
#include "fp8.h"
#include "gemm_core.h"
#include "product8.h"
#include "values.h"

namespace stk {

// A weight's fp32 scale as mantissa 2^(byte - 127): the power goes into the matrix instruction beside that of the rows, so that only a block's scaled sum has
// to have a place in fp32, not the sum under the scale of the rows alone; the mantissa, in [1, 2) (below 2 for scales below the normal numbers), multiplies
// it.  An infinity or a NaN stays mantissa.
struct FloatScale8 {
  int byte;
  float mantissa;
};
__device__ __forceinline__ FloatScale8 float_scale8(float scale) {
  const uint32_t u = __float_as_uint(scale), byte = u >> 23 & 255u;
  if (byte == 255u) return {127, scale};
  return {(int)byte, byte == 0u ? scale * 0x1p127f : __uint_as_float((u & 0x807fffffu) | 0x3f800000u)};
}

// ------------------------------------------------------------------------------------------------ few rows
// 128 values of a row, of which this lane has 64 h + 16 quarter .. + 15, quantised together with the lanes 16, 32 and 48 away.
template <bool BF16>
__device__ __forceinline__ i32x8_t quantise_fragment(const u32x4 (&raw)[4], int& byte) {
  uint32_t most2 = 0;   // largest magnitudes of the lower and upper halves: 16-bit magnitudes are ordered like their bits
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t word = raw[i][j];
      most2 = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, most2), __builtin_bit_cast(u16x2, word & 0x7fff7fffu)));
    }
  uint32_t most = max(most2 >> 16, most2 & 0xffffu);
  const auto by16 = __builtin_amdgcn_permlane16_swap(most, most, false, false);
  most = max(by16[0], by16[1]);
  const auto by32 = __builtin_amdgcn_permlane32_swap(most, most, false, false);
  most = max(by32[0], by32[1]);
  typedef std::conditional_t<BF16, Value<STK_BF16>, Value<STK_F16>> V;
  const uint32_t bits = __float_as_uint(V::widen(__builtin_bit_cast(typename V::stored, (uint16_t)most)));
  byte = exponent_byte8(bits);
  const float scale = __uint_as_float((uint32_t)byte << 23);
  byte = bits >= 0x7f800000u ? 255 : byte;   // (a scale that is not a number)
  i32x8_t out;
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j += 2) out[2 * i + j / 2] = (int)codes8_of_pairs<BF16>(raw[i][j], raw[i][j + 1], scale);
  return out;
}

// Eight values of a row from input i on, zeros beyond the last input: the eight that end with the row, moved down.  (No branch stands between loads, which
// would wait for each of them.)
__device__ __forceinline__ u32x4 row_values8(const uint16_t* row, int i, int inputs) {
  u32x4 v;
  int down;
  if (inputs >= 8) {
    const int from = min(i, inputs - 8);
    v = __builtin_bit_cast(u32x4, *reinterpret_cast<const QuadAt2*>(row + from));
    down = i - from;
  } else {
    uint32_t one[8];
#pragma unroll
    for (int j = 0; j < 8; j++) one[j] = row[min(j, inputs - 1)];
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = (2 * j < inputs ? one[2 * j] : 0u) | (2 * j + 1 < inputs ? one[2 * j + 1] << 16 : 0u);
    down = i;
  }
  if (down & 1) v = u32x4{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
  if (down & 2) v = u32x4{v[1], v[2], v[3], 0u};
  if (down & 4) v = u32x4{v[2], v[3], 0u, 0u};
  return down >= 8 ? u32x4{0u, 0u, 0u, 0u} : v;
}

// Few rows: KW wavefronts share the inputs of NW x NT pieces and up to 16 rows of one expert, a block at a time; their sums meet in LDS.
// Codes go from memory into registers as the matrix instruction takes them; the rows are quantised on the way, some 75 instructions for 16 x 128 of them.
// Bound by the bytes of the weights where there are many: 64 rows to the top 2 of 64 experts of 1024 x 4096 (233 MB) 42 us, 5.5 TB/s; by a launch and one trip to
// memory where there are few: 1 row of 4096 x 4096 6 us.  More rows of a tile in one wavefront (32, 64) were slower than tiles of 16 that read the
// weights from the caches again.
template <int NT>
struct Stage8 {
  u32x4 w[NT][2], v[4];
  int scale[NT];
};
template <bool BF16, int KIND, int KW, int NW, int NT>
__global__ __launch_bounds__(64 * KW * NW, 2) void stream8_kernel(Product8 p) {
  __shared__ f32x4_t shared[KW > 1 ? (KW - 1) * NW * NT * 64 : 1];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), kw = wave / NW, nw = wave % NW;
  const RowTile8 t = row_tile8<16>(p, (int)(blockIdx.z * gridDim.y + blockIdx.y), lane);
  if (t.rows == 0) return;
  const int row = lane & 15, quarter = lane >> 4;
  const int along = (int)blocks8(p.inputs), down = (int)(padded_lines8(p.outputs) / kPieceLines8);
  // the row of this lane; rows beyond those of the tile are its first one, and what they give is not stored
  int64_t from = t.first + (row < t.rows ? row : 0);
  if (p.top_k > 0) {
    const int slot = p.indices[from];
    from = (unsigned)slot < (unsigned)p.rows ? slot / p.top_k : 0;
  }
  const uint16_t* x = static_cast<const uint16_t*>(p.x) + from * p.x_stride;
  int tile[NT];
  const u32x4* weights[NT];
  cint_t scales[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) {
    tile[n] = ((int)blockIdx.x * NW + nw) * NT + n;
    const int64_t piece = min(tile[n], down - 1);
    weights[n] = reinterpret_cast<const u32x4*>(p.packed + ((int64_t)t.expert * down * along + piece8(piece, 0, along)) * kPieceBytes8) + lane;
    // (the lines of a piece have one scale)
    if constexpr (KIND == kPowerScales) scales[n] = const_ints(static_cast<const uint8_t*>(p.scales) + t.expert * scale_bytes8(p.outputs, p.inputs, KIND) + piece * kPieceLines8 * 4);
    else scales[n] = const_ints(static_cast<const float*>(p.scales) + ((int64_t)t.expert * blocks8(p.outputs) + min(tile[n], down - 1) / 8) * along);
  }
  f32x4_t total[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) total[n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  typedef Stage8<NT> S;
  const auto load = [&](S& g, int block) {
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int h = 0; h < 2; h++) g.w[n][h] = __builtin_nontemporal_load(weights[n] + (int64_t)block * (4 * kPieceBytes8 / 16) + 64 * h);
      if constexpr (KIND == kPowerScales) g.scale[n] = scales[n][(int64_t)(block >> 2) * (down * kPieceLines8)] >> (8 * (block & 3));
      else g.scale[n] = scales[n][block];
    }
    const int first = block * kBlock8 + 16 * quarter;
    if ((block + 1) * kBlock8 <= p.inputs) {
#pragma unroll
      for (int h = 0; h < 4; h++) g.v[h] = __builtin_bit_cast(u32x4, *reinterpret_cast<const QuadAt2*>(x + first + 64 * (h >> 1) + 8 * (h & 1)));
    } else {
#pragma unroll
      for (int h = 0; h < 4; h++) g.v[h] = row_values8(x, first + 64 * (h >> 1) + 8 * (h & 1), (int)p.inputs);
    }
  };
  const auto add = [&](const S& g) {
    int byte;
    const i32x8_t values = quantise_fragment<BF16>(g.v, byte);
#pragma unroll
    for (int n = 0; n < NT; n++) {
      i32x8_t w;
#pragma unroll
      for (int i = 0; i < 8; i++) w[i] = (int)g.w[n][i / 4][i % 4];
      if constexpr (KIND == kPowerScales) total[n] = multiply8(w, values, total[n], g.scale[n], byte);
      else {
        const FloatScale8 by = float_scale8(__uint_as_float((uint32_t)g.scale[n]));
        const f32x4_t part = multiply8(w, values, f32x4_t{0.f, 0.f, 0.f, 0.f}, by.byte, byte);
#pragma unroll
        for (int i = 0; i < 4; i++) total[n][i] = fmaf(part[i], by.mantissa, total[n][i]);
      }
    }
  };
  const int share = (along + KW - 1) / KW, begin = min(kw * share, along), end = min(begin + share, along);
  if (begin < end) {
    S a, b;
    load(a, begin);
    for (int block = begin; block < end; block += 2) {
      if (block + 1 < end) load(b, block + 1);
      add(a);
      if (block + 2 < end) load(a, block + 2);
      if (block + 1 < end) add(b);
    }
  }
  if constexpr (KW > 1) {
    if (kw > 0) {
#pragma unroll
      for (int n = 0; n < NT; n++) shared[(((kw - 1) * NW + nw) * NT + n) * 64 + lane] = total[n];
    }
    __syncthreads();
    if (kw > 0) return;
    for (int k = 0; k < KW - 1; k++)
#pragma unroll
      for (int n = 0; n < NT; n++) total[n] += shared[((k * NW + nw) * NT + n) * 64 + lane];
  }
  activate_sums8(total, p.activation);
  int64_t to;
  float by;
  if (!place_of_row8(p, t, row, to, by)) return;
  const int64_t group = (int64_t)(tile[0] / 4) * 64;
  if (tile[0] >= down) return;
  if constexpr (NT == 4) store_pieces8(p, to, by, group, quarter, total);
  else store8<NT>(p, to, by, group + tile[0] % 4 / 2 * 32 + quarter * 8 + (tile[0] & 1) * 4, total);
}

// ------------------------------------------------------------------------------------------------ many rows
// WM x WN wavefronts share 16 MT WM rows and 64 WN outputs, a block of 128 inputs at a time in stages of LDS that are filled without
// registers: pieces of weights as they lie in memory, rows by whole lines, exponents of four blocks in a dword.
// With fp32 scales every matrix instruction is followed by four additions to sums that lie in vector registers: 8192 x 4096 x 4096 in tiles of 256 x 256
// 144 us, 1.9 PFLOP/s, matrix units busy 39 % of the time, wavefronts waiting at barriers, for LDS or for a transfer 47 % of it.  Smaller tiles are for problems
// that do not fill the chip.  By the depth of the inputs, with 4096 outputs, a block costs 0.40 us in 256 tiles of 32 rows, 0.68 in 512 of 64 and 1.0 in 512 of
// 128; where there are few blocks (2501 rows, 1151 x 2944 and its gradients) the matrix units are busy 13 - 15 % of the time.  Three stages are for tiles of 32
// rows, which few units have: 256 rows of 4096 x 4096, quantising included, 20.3 us, and 23.1 by two.
template <int WM, int WN, int MT, int STAGES>
struct Tile8 {
  static constexpr int kWaves = WM * WN, kRows = 16 * MT * WM, kCols = 64 * WN;
  static constexpr int kRowBytes = kRows * kBlock8, kCodes = (kRows + kCols) * kBlock8, kStage = kCodes + (kRows + kCols) * 4;
  static constexpr int kBytes = STAGES * kStage;
};
template <int KIND, int WHAT, int WM, int WN, int MT, int STAGES>
__global__ __launch_bounds__(64 * WM * WN, 2) void tile8_kernel(Product8 p, int row_tiles, int col_tiles) {
  typedef Tile8<WM, WN, MT, STAGES> T;
  static_assert(STAGES == 2 || STAGES == 3, "what the waits below count");
  extern __shared__ char smem[];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  const int row = lane & 15, quarter = lane >> 4, in_fragment = in_fragment8(lane);
  // neighbouring tiles, which share rows or weights, go to one compute die: four row tiles by all columns, column after column
  constexpr int kPanel = 4;
  int at = xcd_chunked(blockIdx.x, gridDim.x), expert = 0;
  if constexpr (WHAT == kGradient8) expert = at / (row_tiles * col_tiles), at %= row_tiles * col_tiles;
  const int panel = at / (kPanel * col_tiles), inside = at % (kPanel * col_tiles), high = min(kPanel, row_tiles - panel * kPanel);
  const int row_tile = panel * kPanel + inside % high, col_tile = inside / high;
  RowTile8 t;
  int begin = 0, end = (int)blocks8(p.inputs);
  if constexpr (WHAT == kGradient8) {
    t = {0, row_tile * T::kRows, (int)min((int64_t)T::kRows, p.x_rows - (int64_t)row_tile * T::kRows)};
    if (p.bins) {
      const int last = end;
      end = min(max(p.bins[expert] / kBlock8, 0), last);
      begin = expert > 0 ? min(max(p.bins[expert - 1] / kBlock8, 0), end) : 0;
    }
  } else {
    t = row_tile8<T::kRows>(p, row_tile, lane);
    t.expert = uniform(t.expert), t.first = uniform(t.first), t.rows = uniform(t.rows);
    if (t.rows == 0) {
      // a tile behind them all: its rows are those behind the last bin
      if (p.zero_behind && p.bins) {
        const int64_t first = (int64_t)min(max(p.bins[p.experts - 1], 0), (int)p.rows) + (int64_t)t.first * T::kRows;
        const int64_t left = min(p.rows - first, (int64_t)T::kRows), col0 = (int64_t)col_tile * T::kCols, cols = min(p.outputs - col0, (int64_t)T::kCols);
        for (int64_t i = threadIdx.x; i < left * cols; i += 64 * T::kWaves) static_cast<uint16_t*>(p.out)[(first + i / cols) * p.out_stride + col0 + i % cols] = 0;
      }
      return;
    }
  }
  const int blocks = (int)blocks8(p.inputs), exponent_stride = (int)exponent_stride8(p.inputs);
  const int64_t places = padded_lines8(p.outputs), col0 = (int64_t)col_tile * T::kCols;
  const auto source_row = [&](int r) { return r < t.rows ? r : 0; };   // of the tile
  // transfers of 1 KiB: eight rows, half a piece; this wavefront's are number wave, wave + kWaves, ...
  constexpr int kRowMoves = T::kRows / 8 / T::kWaves, kColMoves = T::kCols / 8 / T::kWaves, kRowChunks = (T::kRows + 63) / 64, kChunks = kRowChunks + WN;
  static_assert(T::kRows / 8 % T::kWaves == 0 && T::kCols / 8 % T::kWaves == 0, "whole shares");
  const u32x4 row_buffer = buffer8(p.codes + t.first * row_stride8(p.inputs));
  uint32_t row_offset[kRowMoves];
#pragma unroll
  for (int j = 0; j < kRowMoves; j++) {
    const int r = 8 * (wave + T::kWaves * j) + row_of_transfer8(lane);
    row_offset[j] = source_row(r) * (uint32_t)row_stride8(p.inputs) + 16 * chunk_of_transfer8(r, lane);
  }
  const int64_t matrix = WHAT == kGradient8 ? 0 : t.expert;
  gptr_t col_from[kColMoves];
#pragma unroll
  for (int j = 0; j < kColMoves; j++) {
    const int q = wave + T::kWaves * j;
    const int64_t piece = min(col0 / kPieceLines8 + (q >> 1), places / kPieceLines8 - 1);
    col_from[j] = uniform_global(p.packed + (matrix * (places / kPieceLines8) * blocks + piece8(piece, 0, blocks)) * kPieceBytes8 + 1024 * (q & 1));
  }
  // exponents: 64 lines a transfer, first those of the rows; each wavefront makes as many (the last ones twice)
  constexpr int kLines = KIND == kPowerScales ? kChunks : kRowChunks, kScaleMoves = (kLines + T::kWaves - 1) / T::kWaves;
  constexpr int kMoves = kRowMoves + kColMoves + kScaleMoves;
  const uint8_t* scale_from[kScaleMoves];
#pragma unroll
  for (int j = 0; j < kScaleMoves; j++) {
    const int c = min(wave + T::kWaves * j, kLines - 1);
    if (c < kRowChunks) scale_from[j] = p.exponents + ((int64_t)t.first + source_row(64 * c + lane)) * 4;
    else scale_from[j] = static_cast<const uint8_t*>(p.scales) + matrix * places * exponent_stride + min(col0 + 64 * (c - kRowChunks) + lane, places - 1) * 4;
  }
  const uint32_t lds = (uint32_t)(uintptr_t)(STK_LDS char*)smem;
  const auto issue = [&](int block, int stage) {
    const uint32_t to = lds + stage * T::kStage;
#pragma unroll
    for (int j = 0; j < kRowMoves; j++) transfer8<16>(row_buffer, row_offset[j], block * kBlock8, to + (wave + T::kWaves * j) * 1024);
#pragma unroll
    for (int j = 0; j < kColMoves; j++) dma16(col_from[j] + (int64_t)block * (4 * kPieceBytes8), lane * 16, to + T::kRowBytes + (wave + T::kWaves * j) * 1024);
#pragma unroll
    for (int j = 0; j < kScaleMoves; j++) {
      const int c = min(wave + T::kWaves * j, kLines - 1);
      if (T::kRows >= 64 || c >= kRowChunks || lane < T::kRows)
        dma4_from(scale_from[j] + (block >> 2) * (c < kRowChunks ? p.x_rows : places) * 4, to + T::kCodes + (c < kRowChunks ? c * 256 : T::kRows * 4 + (c - kRowChunks) * 256));
    }
  };
  const float* float_scales = static_cast<const float*>(p.scales) + (matrix * blocks8(p.outputs) + min((col0 + 64 * wn) / kBlock8, blocks8(p.outputs) - 1)) * blocks;

  f32x4_t total[MT][4];
#pragma unroll
  for (int m = 0; m < MT; m++)
#pragma unroll
    for (int n = 0; n < 4; n++) total[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int count = end - begin;
#pragma unroll
  for (int s = 0; s < STAGES - 1; s++)
    if (s < count) issue(begin + s, s);
  for (int step = 0, stage = 0; step < count; step++, stage = stage + 1 < STAGES ? stage + 1 : 0) {
    const int block = begin + step;
    // everybody's part of the block is there, and everybody is done with the one whose place is filled now
    if (STAGES > 2 && step + 1 < count) wait_vmcnt<kMoves>();
    else wait_vmcnt<0>();
    __syncthreads();
    if (step + STAGES - 1 < count) issue(block + STAGES - 1, stage > 0 ? stage - 1 : STAGES - 1);
    int row_scale[MT], col_scale[4];
    const int* exponents = reinterpret_cast<const int*>(smem + stage * T::kStage + T::kCodes);
#pragma unroll
    for (int m = 0; m < MT; m++) row_scale[m] = exponents[16 * (m * WM + wm) + row] >> (8 * (block & 3));
    if constexpr (KIND == kPowerScales) {
#pragma unroll
      for (int n = 0; n < 4; n++) col_scale[n] = exponents[T::kRows + 64 * wn + 16 * n + row] >> (8 * (block & 3));
    }
    const FloatScale8 by = float_scale8(KIND == kFloatScales ? __uint_as_float((uint32_t)const_ints(float_scales)[block]) : 1.f);
    const char* rows = smem + stage * T::kStage + wm * kPieceBytes8;
    const char* cols = smem + stage * T::kStage + T::kRowBytes + wn * 4 * kPieceBytes8 + lane * 16;
    const auto fragment = [&](const char* first, const char* second) {
      i32x8_t f;
      const u32x4 a = *reinterpret_cast<const u32x4*>(first), b = *reinterpret_cast<const u32x4*>(second);
#pragma unroll
      for (int i = 0; i < 4; i++) f[i] = (int)a[i], f[4 + i] = (int)b[i];
      return f;
    };
    const auto row_fragment = [&](int m) { return fragment(rows + in_fragment + m * WM * kPieceBytes8, rows + (in_fragment ^ 64) + m * WM * kPieceBytes8); };
    // The fragment of the next 16 rows is on its way while one is multiplied; with fp32 scales the sums of one are scaled while the next is.  (Leaving out what
    // lies behind the last row of a tile would need branches, around which the sums move between registers: twice the instructions.)
    i32x8_t w[4], values[2];
    values[0] = row_fragment(0);
#pragma unroll
    for (int n = 0; n < 4; n++) w[n] = fragment(cols + n * kPieceBytes8, cols + n * kPieceBytes8 + 1024);
#pragma unroll
    for (int m = 0; m < MT; m++) {
      if (m + 1 < MT) values[(m + 1) & 1] = row_fragment(m + 1);
      f32x4_t part[4];
#pragma unroll
      for (int n = 0; n < 4; n++) {
        if constexpr (KIND == kPowerScales) total[m][n] = multiply8(w[n], values[m & 1], total[m][n], col_scale[n], row_scale[m]);
        else part[n] = multiply8(w[n], values[m & 1], f32x4_t{0.f, 0.f, 0.f, 0.f}, by.byte, row_scale[m]);
      }
      if constexpr (KIND == kFloatScales) {
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) total[m][n][i] = fmaf(part[n][i], by.mantissa, total[m][n][i]);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);   // (the accesses to LDS come first)
      __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);
    }
  }
  if constexpr (WHAT == kGradient8) p.out = static_cast<uint16_t*>(p.out) + (int64_t)expert * p.x_rows * p.out_stride;
#pragma unroll
  for (int m = 0; m < MT; m++) {
    if constexpr (WHAT == kRows8) activate_sums8(total[m], p.activation);
    int64_t to;
    float by;
    if (place_of_row8(p, t, 16 * (m * WM + wm) + row, to, by)) store_pieces8(p, to, by, col0 + 64 * wn, quarter, total[m]);
  }
}

// out[t] = sum over the choices j of a token, in their order, of (weights[s]) sums[s], s = t top_k + j; rounded once.  A thread per
// token and four outputs.
__global__ __launch_bounds__(256) void combine8_kernel(const float* __restrict__ sums, const float* __restrict__ weights, int64_t tokens, int top_k, int64_t outputs,
                                                       uint16_t* __restrict__ out, int64_t out_stride, bool bf16) {
  const int64_t across = (outputs + 3) / 4, step = (int64_t)gridDim.x * 256;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < tokens * across; at += step) {
    const int64_t t = at / across, o = at % across * 4;
    const int here = (int)min(outputs - o, (int64_t)4);
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < top_k; j0 += 4) {   // (the rows of four choices are on their way together)
      float by[4], u[4][4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int64_t s = t * top_k + min(j0 + j, top_k - 1);
        by[j] = weights ? weights[s] : 1.f;
        const float* from = sums + s * outputs + o;
        if (here == 4) {
          const f32x4_t q = __builtin_bit_cast(f32x4_t, *reinterpret_cast<const QuadAt4*>(from));
#pragma unroll
          for (int i = 0; i < 4; i++) u[j][i] = q[i];
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++) u[j][i] = from[min(i, here - 1)];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = j0 + j < top_k ? fmaf(by[j], u[j][i], v[i]) : v[i];
    }
    const uint32_t two[2] = {pack8(v[0], v[1], bf16), pack8(v[2], v[3], bf16)};
    uint16_t* to = out + t * out_stride + o;
    if (here == 4) *reinterpret_cast<PairAt2*>(to) = PairAt2{two[0], two[1]};
    else
      for (int i = 0; i < here; i++) to[i] = (uint16_t)(two[i / 2] >> (16 * (i & 1)));
  }
}

// ------------------------------------------------------------------------------------------------ launches
// Tiles of `of` rows that the rows of the experts can be at most, and with rows behind the last expert those that these need.
static int64_t most_tiles8(const Product8& p, int64_t of) {
  const int64_t tiles = (p.rows + of - 1) / of;
  return p.bins ? (p.zero_behind ? tiles + p.experts : std::min(p.rows, tiles + p.experts - 1)) : tiles;
}

template <int KW, int NW, int NT>
static void launch_stream8(const Product8& p, int kind, hipStream_t stream) {
  const int64_t tiles = most_tiles8(p, 16), pieces = padded_lines8(p.outputs) / kPieceLines8, y = tiles < 65535 ? tiles : 65535;
  const dim3 grid((unsigned)((pieces + NW * NT - 1) / (NW * NT)), (unsigned)y, (unsigned)((tiles + y - 1) / y));
  const auto launch = [&](auto bf16, auto k) { hipLaunchKernelGGL((stream8_kernel<bf16(), k(), KW, NW, NT>), grid, dim3(64 * KW * NW), 0, stream, p); };
  const auto by_kind = [&](auto bf16) {
    if (kind == kPowerScales) launch(bf16, std::integral_constant<int, kPowerScales>());
    else launch(bf16, std::integral_constant<int, kFloatScales>());
  };
  if (p.bf16) by_kind(std::true_type());
  else by_kind(std::false_type());
}
template <int WHAT, int WM, int WN, int MT, int STAGES>
static int launch_tiles8(const char* who, const Product8& p, int kind, hipStream_t stream) {
  typedef Tile8<WM, WN, MT, STAGES> T;
  const int64_t row_tiles = WHAT == kGradient8 ? (p.x_rows + T::kRows - 1) / T::kRows : most_tiles8(p, T::kRows), col_tiles = (p.outputs + T::kCols - 1) / T::kCols;
  const int64_t matrices = WHAT == kGradient8 ? p.experts : 1;
  if (row_tiles > INT32_MAX / col_tiles / matrices) return fail(STK_ERR_UNSUPPORTED, "%s: too many tiles", who);
  const dim3 grid((unsigned)(row_tiles * col_tiles * matrices));
  const auto launch = [&](auto k) {
    const auto kernel = tile8_kernel<decltype(k)::value, WHAT, WM, WN, MT, STAGES>;
    set_lds_limit(kernel, T::kBytes);
    hipLaunchKernelGGL(kernel, grid, dim3(64 * T::kWaves), T::kBytes, stream, p, (int)row_tiles, (int)col_tiles);
  };
  if constexpr (WHAT == kGradient8) launch(std::integral_constant<int, kPowerScales>());
  else if (kind == kPowerScales) launch(std::integral_constant<int, kPowerScales>());
  else launch(std::integral_constant<int, kFloatScales>());
  return check_launch(who);
}

// Which kernel.  The tiles reach their rows by 32 bits.
constexpr int64_t kMostTileInputs8 = 1 << 23;
enum ProductKernel8 : int { kStream8_811 = 0, kStream8_412, kStream8_414, kStream8_222, kStream8_144, kTile8_32, kTile8_64, kTile8_128, kTile8_256 };
static ProductKernel8 product_kernel8(int64_t rows, int64_t experts, int64_t inputs, int64_t outputs) {
  const int64_t along = blocks8(inputs), down = padded_lines8(outputs) / kPieceLines8;
  // as if the rows were spread evenly over the experts: where they really are only the device knows
  const int64_t hit = experts < rows ? experts : rows, each = (rows + hit - 1) / hit;
  // Streams read an expert's weights once for every 16 rows, behind the first time from the caches, and quantise the rows for every piece; tiles take a launch
  // that quantises the rows, and 0.4 us for every block where few of them are in the chip.  Rows that are no whole 16-byte pieces cost the streams twice.
  // Streams and the best tiles: 4096 x 4096, 64 rows (1024 units) 11.4 and 18.5 us, 128 rows 18.9 and 18.7, 256 rows 35 and 20.7; 8 experts of 1024 x 1024, 40 rows each
  // (1536) 8.4 and 10.0; 37, 64, 100 rows of 1151 x 2944 (552, 736, 1288) 9.1, 10.0, 13.3 and 9.1, 9.1, 9.3; 64 experts of 1024 x 4096, 20 rows each 81 and 66.
  const int64_t tiles = hit * ((each + 15) / 16) * down;
  if (each > 16 && tiles > (inputs % 8 ? 640 : 1792) && inputs <= kMostTileInputs8) {
    // Larger tiles read less, smaller ones fill the chip.  4096 x 4096, tiles of 32, 64, 128, 256 rows: 256 rows 21, 24, 29, 55 us; 1024 rows 44, 30, 34, 59;
    // 2048 rows 78, 57, 43, 62; 64 experts of 1024 x 4096, 20 rows each 72, 67, 72, 83, 64 rows each 105, 95, 97, 92, 128 rows each 162, 128, 131, 108.
    // Experts of 256 +- 16 rows, half of which need a second tile of 256: 1024, 2048 and 4096 inputs 182, 250 and 438 by 256, 208, 312 and 561 by 128 (exactly
    // 256 rows each: 134, 206, 358 and 192, 308, 550).
    const auto count = [&](int64_t high, int64_t wide) { return hit * ((each + high - 1) / high) * ((outputs + wide - 1) / wide); };
    if (each > 64 && count(256, 256) >= 192) return kTile8_256;
    if (each > 64 && count(128, 128) > 256) return kTile8_128;
    return count(64, 128) > 256 ? kTile8_64 : kTile8_32;
  }
  // The fewer tiles there are the more wavefronts share the inputs of one: 1 row of 4096 x 4096 (256 tiles) 6.2, 8.8, 10.8 us by 8, 4 and 4 for two and four
  // pieces; 20 rows (512) 10.8, 9.5, 11.2; 64 rows (1024) 21.9, 13.8, 11.2.  Where every unit has a workgroup of four wavefronts with four pieces each they share
  // nothing: 64 rows to the top 2 of 64 experts of 4096 x 1024 (4096) 40.1 us and 43.4 with shared inputs.
  if (tiles <= 320) return kStream8_811;
  if (tiles <= 640) return kStream8_412;
  if (tiles >= 4096) return kStream8_144;
  return along >= 8 ? kStream8_414 : kStream8_222;
}
static int64_t workspace8(int64_t rows, int64_t experts, int64_t inputs, int64_t outputs) {
  if (rows < 1 || product_kernel8(rows, experts, inputs, outputs) < kTile8_32) return 0;
  return (rows * (row_stride8(inputs) + exponent_stride8(inputs)) + 255) / 256 * 256;
}
template <int WHAT>
static int launch_tiles8(const char* who, const Product8& p, int kind, ProductKernel8 kernel, hipStream_t stream) {
  switch (kernel) {
    case kTile8_32: return launch_tiles8<WHAT, 2, 2, 1, 3>(who, p, kind, stream);
    case kTile8_64: return launch_tiles8<WHAT, 2, 2, 2, 2>(who, p, kind, stream);
    case kTile8_128: return launch_tiles8<WHAT, 2, 2, 4, 2>(who, p, kind, stream);
    default:
      if constexpr (WHAT == kRows8) {
        if (kind != kPowerScales || p.activation == kGeluErf) return launch_tiles8<WHAT, 2, 4, 8, 2>(who, p, kind, stream);   // (erf's registers do not fit beside 256 sums)
      }
      return launch_wide8<WHAT>(who, p, stream);
  }
}
// The product of 16-bit rows; the workspace holds them quantised where there are many.
static int launch_product8(const char* who, Product8 p, int kind, int dtype, void* workspace, hipStream_t stream) {
  const ProductKernel8 kernel = product_kernel8(p.rows, p.experts, p.inputs, p.outputs);
  if (kernel >= kTile8_32) {
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    uint8_t* exponents = codes + p.rows * row_stride8(p.inputs);
    // (gathered here: for one expert per token that costs nothing, and a tile's rows are neighbours)
    if (int rc = quantize_rows8(who, p.x, p.rows, p.inputs, p.x_stride, dtype, codes, exponents, p.top_k > 0 ? p.indices : nullptr, p.top_k, stream)) return rc;
    p.codes = codes, p.exponents = exponents, p.x_rows = p.rows, p.top_k = 0;
    return launch_tiles8<kRows8>(who, p, kind, kernel, stream);
  }
  if (most_tiles8(p, 16) > (int64_t)65535 * 65535) return fail(STK_ERR_UNSUPPORTED, "%s: %lld rows", who, (long long)p.rows);
  switch (kernel) {
    case kStream8_811: launch_stream8<8, 1, 1>(p, kind, stream); break;
    case kStream8_412: launch_stream8<4, 1, 2>(p, kind, stream); break;
    case kStream8_414: launch_stream8<4, 1, 4>(p, kind, stream); break;
    case kStream8_222: launch_stream8<2, 2, 2>(p, kind, stream); break;
    default: launch_stream8<1, 4, 4>(p, kind, stream); break;
  }
  return check_launch(who);
}
static int product_check8(const char* who, const Product8& p, int dtype) {
  if (dtype != STK_F16 && dtype != STK_BF16) return fail(STK_ERR_UNSUPPORTED, "%s: rows of 16-bit values", who);
  if (p.rows < 0 || p.x_rows < 0 || p.experts < 1 || p.inputs < 1 || p.outputs < 1)
    return fail(STK_ERR_DIMS, "%s: %lld rows, %lld matrices of %lld x %lld", who, (long long)p.rows, (long long)p.experts, (long long)p.inputs, (long long)p.outputs);
  if (!sizes8(p.rows, p.inputs) || !sizes8(p.x_rows, p.outputs) || p.experts > INT32_MAX) return fail(STK_ERR_UNSUPPORTED, "%s: size exceeds 32-bit range", who);
  if (p.activation < kNoActivation || p.activation > kSilu) return fail(STK_ERR_UNSUPPORTED, "%s: activation %d", who, p.activation);
  if (p.rows == 0) return STK_OK;
  if (!p.packed || !p.scales || (!p.out && !p.sums) || (!p.x && !p.codes)) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (p.x_stride < 0 || (p.out && p.out_stride < p.outputs)) return fail(STK_ERR_DIMS, "%s: strides %lld, %lld", who, (long long)p.x_stride, (long long)p.out_stride);
  if (!aligned16(p.packed) || (reinterpret_cast<uintptr_t>(p.scales) & 3) || (reinterpret_cast<uintptr_t>(p.exponents) & 3)) return fail(STK_ERR_UNSUPPORTED, "%s: codes at a multiple of 16 bytes, scales and exponents of 4", who);
  return STK_OK;
}

}  // namespace stk

using namespace stk;

extern "C" int stk_8bit_product_kernel(int64_t rows, int64_t experts, int64_t inputs, int64_t outputs) {
  return rows < 1 || experts < 1 || inputs < 1 || outputs < 1 ? -1 : (int)product_kernel8(rows, experts, inputs, outputs);
}
extern "C" size_t stk_matmul_8bit_workspace_bytes(int64_t x_rows, int64_t rows, int64_t experts, int64_t inputs, int64_t outputs) {
  return x_rows < 1 || experts < 1 || inputs < 1 || outputs < 1 ? 0 : (size_t)workspace8(rows, experts, inputs, outputs);
}
extern "C" size_t stk_matmul_8bit_scatter_workspace_bytes(int64_t slots, int top_k, int64_t experts, int64_t inputs, int64_t outputs) {
  const size_t rows = stk_matmul_8bit_workspace_bytes(slots, slots, experts, inputs, outputs);
  return slots < 1 || outputs < 1 || top_k == 1 ? rows : rows + (size_t)(slots * outputs) * sizeof(float);
}
static int workspace_check8(const char* who, const void* workspace, size_t has, size_t needs) {
  if (needs > 0 && (!workspace || has < needs || !aligned16(workspace))) return fail(STK_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", who, needs);
  return STK_OK;
}

extern "C" int stk_matmul_8bit(const void* x, int64_t rows, int64_t x_stride, const void* packed, const void* scales, int float_scales, int64_t inputs, int64_t outputs,
                               void* out, int64_t out_stride, int activation, int dtype, void* workspace, size_t workspace_bytes, stk_stream_t stream) {
  const char* who = "stk_matmul_8bit";
  Product8 p = {};
  p.x = x, p.x_stride = x_stride, p.x_rows = p.rows = rows, p.packed = static_cast<const uint8_t*>(packed), p.scales = scales, p.experts = 1, p.inputs = inputs;
  p.outputs = outputs, p.out = out, p.out_stride = out_stride, p.activation = activation, p.bf16 = dtype == STK_BF16;
  if (int rc = product_check8(who, p, dtype)) return rc;
  if (rows == 0) return STK_OK;
  if (int rc = workspace_check8(who, workspace, workspace_bytes, stk_matmul_8bit_workspace_bytes(rows, rows, 1, inputs, outputs))) return rc;
  return launch_product8(who, p, float_scales ? kFloatScales : kPowerScales, dtype, workspace, static_cast<hipStream_t>(stream));
}

extern "C" int stk_gather_matmul_8bit(const void* x, int64_t tokens, int64_t x_stride, const int32_t* indices, const int32_t* bins, int top_k, const void* packed,
                                      const void* scales, int float_scales, int64_t experts, int64_t inputs, int64_t outputs, void* out, int64_t out_stride,
                                      int activation, int dtype, void* workspace, size_t workspace_bytes, stk_stream_t stream) {
  const char* who = "stk_gather_matmul_8bit";
  if (tokens < 0 || top_k < 1 || tokens > INT32_MAX / top_k) return fail(STK_ERR_DIMS, "%s: %lld tokens, top_k %d", who, (long long)tokens, top_k);
  Product8 p = {};
  p.x = x, p.x_stride = x_stride, p.x_rows = tokens, p.rows = tokens * top_k, p.packed = static_cast<const uint8_t*>(packed), p.scales = scales, p.experts = experts;
  p.inputs = inputs, p.outputs = outputs, p.indices = indices, p.bins = bins, p.top_k = top_k, p.out = out, p.out_stride = out_stride, p.activation = activation;
  p.bf16 = dtype == STK_BF16;
  if (int rc = product_check8(who, p, dtype)) return rc;
  if (tokens == 0) return STK_OK;
  if (!indices || !bins) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (int rc = workspace_check8(who, workspace, workspace_bytes, stk_matmul_8bit_workspace_bytes(tokens, p.rows, experts, inputs, outputs))) return rc;
  return launch_product8(who, p, float_scales ? kFloatScales : kPowerScales, dtype, workspace, static_cast<hipStream_t>(stream));
}

extern "C" int stk_matmul_8bit_scatter(const void* x, int64_t x_stride, const int32_t* indices, const int32_t* bins, int top_k, int64_t tokens, const float* weights,
                                       const void* packed, const void* scales, int float_scales, int64_t experts, int64_t inputs, int64_t outputs, void* out,
                                       int64_t out_stride, int dtype, void* workspace, size_t workspace_bytes, stk_stream_t stream) {
  const char* who = "stk_matmul_8bit_scatter";
  if (tokens < 0 || top_k < 1 || tokens > INT32_MAX / top_k) return fail(STK_ERR_DIMS, "%s: %lld tokens, top_k %d", who, (long long)tokens, top_k);
  const int64_t slots = tokens * top_k;
  Product8 p = {};
  p.x = x, p.x_stride = x_stride, p.x_rows = p.rows = slots, p.packed = static_cast<const uint8_t*>(packed), p.scales = scales, p.experts = experts, p.inputs = inputs;
  p.outputs = outputs, p.indices = indices, p.bins = bins, p.out = out, p.out_stride = out_stride, p.weights = weights, p.by_slot = true, p.bf16 = dtype == STK_BF16;
  if (int rc = product_check8(who, p, dtype)) return rc;
  if (tokens == 0) return STK_OK;
  if (!indices || !bins) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (int rc = workspace_check8(who, workspace, workspace_bytes, stk_matmul_8bit_scatter_workspace_bytes(slots, top_k, experts, inputs, outputs))) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int kind = float_scales ? kFloatScales : kPowerScales;
  if (top_k == 1) return launch_product8(who, p, kind, dtype, workspace, s);   // a token's only row goes to its place
  p.sums = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + stk_matmul_8bit_workspace_bytes(slots, slots, experts, inputs, outputs));
  if (int rc = launch_product8(who, p, kind, dtype, workspace, s)) return rc;
  const int64_t count = (tokens * ((outputs + 3) / 4) + 255) / 256;
  hipLaunchKernelGGL(combine8_kernel, dim3((unsigned)(count < 1 << 18 ? count : 1 << 18)), dim3(256), 0, s, p.sums, weights, tokens, top_k, outputs,
                     static_cast<uint16_t*>(out), out_stride, p.bf16);
  return check_launch(who);
}

extern "C" int stk_linear_8bit(const void* codes, const void* exponents, int64_t rows, const int32_t* bins, const void* packed, const void* weight_exponents,
                               int64_t experts, int64_t inputs, int64_t outputs, void* out, int64_t out_stride, int dtype, stk_stream_t stream) {
  const char* who = "stk_linear_8bit";
  Product8 p = {};
  p.codes = static_cast<const uint8_t*>(codes), p.exponents = static_cast<const uint8_t*>(exponents), p.x_rows = p.rows = rows;
  p.packed = static_cast<const uint8_t*>(packed), p.scales = weight_exponents, p.experts = experts, p.inputs = inputs, p.outputs = outputs, p.bins = bins;
  p.out = out, p.out_stride = out_stride, p.bf16 = dtype == STK_BF16, p.zero_behind = true;
  if (int rc = product_check8(who, p, dtype)) return rc;
  if (rows == 0) return STK_OK;
  if (!exponents || (!bins && experts > 1)) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (!aligned16(codes)) return fail(STK_ERR_UNSUPPORTED, "%s: codes at a multiple of 16 bytes", who);
  if (inputs > kMostTileInputs8) return fail(STK_ERR_UNSUPPORTED, "%s: %lld inputs", who, (long long)inputs);
  const ProductKernel8 kernel = product_kernel8(rows, experts, inputs, outputs);
  return launch_tiles8<kRows8>(who, p, kPowerScales, kernel < kTile8_32 ? kTile8_32 : kernel, static_cast<hipStream_t>(stream));
}

extern "C" int stk_weight_gradient_8bit(const void* columns, const void* exponents, const void* grad_pieces, const void* grad_exponents, int64_t rows,
                                        const int32_t* bins, int64_t experts, int64_t inputs, int64_t outputs, void* dw, int dtype, stk_stream_t stream) {
  const char* who = "stk_weight_gradient_8bit";
  Product8 p = {};
  p.codes = static_cast<const uint8_t*>(columns), p.exponents = static_cast<const uint8_t*>(exponents), p.x_rows = p.rows = inputs;
  p.packed = static_cast<const uint8_t*>(grad_pieces), p.scales = grad_exponents, p.experts = experts, p.inputs = rows, p.outputs = outputs, p.bins = bins;
  p.out = dw, p.out_stride = outputs, p.bf16 = dtype == STK_BF16;
  if (int rc = product_check8(who, p, dtype)) return rc;
  if (!exponents || (!bins && experts > 1)) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (!aligned16(columns)) return fail(STK_ERR_UNSUPPORTED, "%s: codes at a multiple of 16 bytes", who);
  if (rows > kMostTileInputs8) return fail(STK_ERR_UNSUPPORTED, "%s: %lld rows", who, (long long)rows);
  const auto count = [&](int64_t side) { return experts * ((inputs + side - 1) / side) * ((outputs + 127) / 128); };
  const ProductKernel8 kernel = experts * ((inputs + 255) / 256) * ((outputs + 255) / 256) >= 192 ? kTile8_256 : count(128) >= 192 ? kTile8_128 : count(64) >= 192 ? kTile8_64 : kTile8_32;
  return launch_tiles8<kGradient8>(who, p, kPowerScales, kernel, static_cast<hipStream_t>(stream));
}
