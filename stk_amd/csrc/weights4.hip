// Products with 4-bit weights and group scales, and the weights' own formats.
//   weight of input i and output o = scale[i / group][o] * (code - 8)      or      scale * code + offset[i / group][o]
#include <type_traits>

#include "common.h"
#include "gemm_core.h"
#include "values.h"
#include "wave_scan.h"
#include "weights4.h"

namespace stk {

// Largest and smallest weight of a group -> scale and offset, rounded to the weights' type; then the codes nearest to the weights
// under the rounded ones.  A thread per group and output.
template <int DTYPE, int OUT>
__global__ __launch_bounds__(256) void quantize_kernel(const typename Value<DTYPE>::stored* __restrict__ w, int64_t stride_e, int64_t stride_i, int64_t stride_o,
                                                       int64_t inputs, int64_t outputs, int64_t group, int64_t groups, uint8_t* __restrict__ codes,
                                                       typename Value<OUT>::stored* __restrict__ scales, typename Value<OUT>::stored* __restrict__ offsets) {
  const int64_t o = (int64_t)blockIdx.x * 256 + threadIdx.x, e = blockIdx.z;
  if (o >= outputs) return;
  for (int64_t g = blockIdx.y; g < groups; g += gridDim.y) {
    const int64_t lo = g * group, hi = lo + group < inputs ? lo + group : inputs;
    const auto* at = w + e * stride_e + o * stride_o;
    float least = INFINITY, most = -INFINITY;
    for (int64_t i = lo; i < hi; i++) {
      const float v = Value<DTYPE>::widen(at[i * stride_i]);
      least = fminf(least, v), most = fmaxf(most, v);
    }
    const auto scale16 = Value<OUT>::round(offsets ? (most - least) / 15.f : fmaxf(most, -least) / 7.f);
    const auto offset16 = Value<OUT>::round(least);
    const float scale = Value<OUT>::widen(scale16), from = offsets ? Value<OUT>::widen(offset16) : -8.f * scale;
    const int64_t to = (e * groups + g) * outputs + o;
    scales[to] = scale16;
    if (offsets) offsets[to] = offset16;
    for (int64_t i = lo; i < hi; i++) {
      const float v = scale > 0.f ? rintf((Value<DTYPE>::widen(at[i * stride_i]) - from) / scale) : offsets ? 0.f : 8.f;
      codes[(e * inputs + i) * outputs + o] = (uint8_t)fminf(fmaxf(v, 0.f), 15.f);
    }
  }
}

// A wavefront per piece: lane l gathers the 32 codes of its 16 bytes.
__global__ __launch_bounds__(256) void pack_codes_kernel(const uint8_t* __restrict__ codes, int64_t inputs, int64_t outputs, int64_t pieces, u32x4* __restrict__ packed) {
  const int lane = threadIdx.x & 63;
  const int64_t piece = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (piece >= pieces) return;
  const int64_t along = pieces_in(inputs), down = pieces_out(outputs);
  const int64_t first_i = piece % along * kPieceInputs, first_o = piece / along % down * kPieceOutputs, e = piece / (along * down);
  const int64_t o = first_o + (lane & 15);
  uint32_t words[4];
#pragma unroll
  for (int d = 0; d < 4; d++) {
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int64_t i = first_i + 32 * d + 8 * (lane >> 4) + j;
      const uint32_t code = i < inputs && o < outputs ? codes[(e * inputs + i) * outputs + o] & 15u : 8u;
      word |= code << (4 * (j >> 1) + 16 * (j & 1));
    }
    words[d] = word;
  }
  packed[piece * 64 + lane] = u32x4{words[0], words[1], words[2], words[3]};
}

// Scales [expert][group][output] -> [expert][16 outputs][group][16]; the same for offsets.
__global__ __launch_bounds__(256) void pack_scales_kernel(const uint16_t* __restrict__ scales, int64_t groups, int64_t outputs, int64_t count,
                                                          uint16_t* __restrict__ packed) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= count) return;
  const int64_t down = pieces_out(outputs), g = at / 16 % groups, o = at / 16 / groups % down * 16 + at % 16, e = at / 16 / groups / down;
  packed[at] = o < outputs ? scales[(e * groups + g) * outputs + o] : (uint16_t)0;
}

template <int DTYPE>
__device__ __forceinline__ float weight_of(const uint8_t* packed, const typename Value<DTYPE>::stored* scales, const typename Value<DTYPE>::stored* offsets,
                                           int64_t e, int64_t i, int64_t o, int64_t along, int64_t down, int64_t group, int64_t groups) {
  int byte, shift;
  code_at((int)(o & 15), (int)(i & 127), &byte, &shift);
  const int code = packed[((e * down + o / 16) * along + i / 128) * kPieceBytes + byte] >> shift & 15;
  const int64_t at = ((e * down + o / 16) * groups + i / group) * 16 + o % 16;
  const float scale = Value<DTYPE>::widen(scales[at]);
  return offsets ? scale * (float)code + Value<DTYPE>::widen(offsets[at]) : scale * (float)(code - 8);
}

template <int DTYPE>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint8_t* __restrict__ packed, const typename Value<DTYPE>::stored* __restrict__ scales,
                                                         const typename Value<DTYPE>::stored* __restrict__ offsets, int64_t inputs, int64_t outputs,
                                                         int64_t group, int64_t count, typename Value<DTYPE>::stored* __restrict__ out) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= count) return;
  const int64_t o = at % outputs, i = at / outputs % inputs, e = at / outputs / inputs;
  out[at] = Value<DTYPE>::round(weight_of<DTYPE>(packed, scales, offsets, e, i, o, pieces_in(inputs), pieces_out(outputs), group, groups_of(inputs, group)));
}

__device__ __forceinline__ float activated(float v, int kind) {
  switch (kind) {
    case kRelu: return activate<kRelu>(v);
    case kGeluTanh: return activate<kGeluTanh>(v);
    case kGeluErf: return activate<kGeluErf>(v);
    case kSilu: return activate<kSilu>(v);
    default: return v;
  }
}

// What a product is told.  Without routing: bins null, one expert.  With: row p of the sorted slots belongs to the first expert whose
// bin ends behind p, and to the slot indices[p].
struct Product4 {
  const void* x;
  int64_t x_stride, rows;          // rows: those multiplied (tokens, or slots)
  const uint8_t* packed;
  const void *scales, *offsets;
  int64_t experts, inputs, outputs, group;
  const int32_t *indices, *bins;
  int top_k;                       // gathered: row p reads token indices[p] / top_k; 0: row p itself
  void* out;                       // 16-bit rows in the order of the rows, ...
  int64_t out_stride;
  float* sums;                     // ... or, where given, fp32 rows [slot][outputs]
  int activation;
};

// ---------------------------------------------------------------- products
// A code becomes the 16-bit number 16 + code: its four bits at the top of the mantissa of a number between 16 and 32.  A group's
// products are then sums over x (16 + code), and the sums over x that are too much, -24 x (the code's zero at 8) or -16 x (with
// offsets), are what the accumulator starts from: a product of x with a constant operand, shared by all outputs.  The group's scale
// multiplies the fp32 sum.  That makes 8 instructions for eight weights and one for a group's four outputs, below half of
// what a stream of weights at memory speed leaves time for.
template <bool BF16> struct Codes;
template <> struct Codes<true> {
  static constexpr uint32_t mask = 0x00780078u, magic = 0x41804180u, minus24 = 0xc1c0c1c0u, minus16 = 0xc180c180u;
  static __device__ __forceinline__ uint32_t placed(uint32_t w, int p) { return p == 0 ? w << 3 : w >> (4 * p - 3); }
};
template <> struct Codes<false> {
  static constexpr uint32_t mask = 0x03c003c0u, magic = 0x4c004c00u, minus24 = 0xce00ce00u, minus16 = 0xcc00cc00u;
  static __device__ __forceinline__ uint32_t placed(uint32_t w, int p) { return p == 0 ? w << 6 : p == 1 ? w << 2 : w >> (4 * p - 6); }
};
template <bool BF16>
__device__ __forceinline__ u32x4 numbers(uint32_t w) {
  typedef Codes<BF16> C;
  u32x4 v;
#pragma unroll
  for (int p = 0; p < 4; p++) v[p] = (C::placed(w, p) & C::mask) | C::magic;
  return v;
}
typedef float f32x4_t __attribute__((ext_vector_type(4)));
template <bool BF16>
__device__ __forceinline__ f32x4_t mfma_16x16x32(u32x4 a, u32x4 b, f32x4_t c) {
  if constexpr (BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// Which rows a tile of up to R rows of one expert is: tiles are numbered expert by expert, an expert of c rows has ceil(c / R).
struct RowTile {
  int expert, first, rows;   // (rows 0: no such tile)
};
template <int R>
__device__ __forceinline__ RowTile row_tile(const Product4& p, int tile, int lane) {
  if (!p.bins) {
    const int64_t first = (int64_t)tile * R, left = p.rows - first;
    return {0, (int)first, left <= 0 ? 0 : left < R ? (int)left : R};
  }
  int before = 0;
  for (int e0 = 0; e0 < p.experts; e0 += kWave) {
    const int e = e0 + lane;
    const bool is = e < p.experts;
    // (bins that do not ascend or leave the rows are kept inside them)
    const int hi = is ? min(max(p.bins[e], 0), (int)p.rows) : 0, lo = is && e > 0 ? min(max(p.bins[e - 1], 0), (int)p.rows) : 0;
    const int count = hi > lo ? hi - lo : 0, tiles = (count + R - 1) / R, upto = before + wave_inclusive_scan(tiles, lane);
    const uint64_t mine = __ballot(upto > tile);
    if (mine) {
      const int at = __builtin_ctzll(mine);
      const int inside = tile - __builtin_amdgcn_readlane(upto - tiles, at), c = __builtin_amdgcn_readlane(count, at);
      return {e0 + at, __builtin_amdgcn_readlane(lo, at) + inside * R, min(c - inside * R, R)};
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return {0, 0, 0};
}

// Eight values of a row from input i on, zeros beyond the last input.
__device__ __forceinline__ u32x4 row_values(const uint16_t* row, int i, int inputs) {
  if (i + 8 <= inputs) return __builtin_bit_cast(u32x4, *reinterpret_cast<const QuadAt2*>(row + i));
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const uint32_t one = i + j < inputs ? row[i + j] : 0u;
    v[j / 2] |= one << (16 * (j & 1));
  }
  return v;
}

// KW wavefronts share the inputs of NW x NT x 16 outputs and 16 MT rows of one expert, a piece of weights at a time; their sums meet
// in LDS.  SUB: groups of a piece whose sums are scaled apart (1, or 4: groups of 32 or 64).
template <bool BF16, bool AFFINE, int SUB, int KW, int NW, int NT, int MT>
__global__ __launch_bounds__(64 * KW * NW) void stream_kernel(Product4 p) {
  constexpr int kAtOnce = NT * MT == 1 ? 4 : NT * MT == 2 ? 2 : 1;   // pieces whose loads are in flight together
  extern __shared__ f32x4_t shared[];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), kw = wave % KW, nw = wave / KW;
  const RowTile t = row_tile<16 * MT>(p, blockIdx.y, lane);
  if (t.rows == 0) return;
  const int along = (int)pieces_in(p.inputs), down = (int)pieces_out(p.outputs), groups = (int)groups_of(p.inputs, p.group);
  const int row = lane & 15, quarter = lane >> 4;
  const uint16_t* x[MT];
  bool has[MT];
#pragma unroll
  for (int m = 0; m < MT; m++) {
    const int r = 16 * m + row;
    has[m] = r < t.rows;
    int64_t from = t.first + (has[m] ? r : 0);
    if (p.top_k > 0) {
      const int slot = p.indices[from];
      has[m] = has[m] && (unsigned)slot < (unsigned)p.rows;
      from = has[m] ? slot / p.top_k : 0;
    }
    x[m] = static_cast<const uint16_t*>(p.x) + from * p.x_stride;
  }
  int tile[NT];   // (the last tiles of a workgroup may lie beyond the outputs: computed again and not stored)
  const u32x4* weights[NT];
  const uint16_t *scales[NT], *offsets[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) {
    tile[n] = ((int)blockIdx.x * NW + nw) * NT + n;
    const int64_t at = (int64_t)t.expert * down + min(tile[n], down - 1);
    weights[n] = reinterpret_cast<const u32x4*>(p.packed + at * along * kPieceBytes) + lane;
    scales[n] = static_cast<const uint16_t*>(p.scales) + at * groups * 16 + 4 * quarter;
    offsets[n] = static_cast<const uint16_t*>(p.offsets) + at * groups * 16 + 4 * quarter;
  }
  const int share = (along + KW - 1) / KW, begin = min(kw * share, along), end = min(begin + share, along);
  const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
  f32x4_t total[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int m = 0; m < MT; m++) total[n][m] = zero;
  constexpr uint32_t minus = AFFINE ? Codes<BF16>::minus16 : Codes<BF16>::minus24;
  const u32x4 constant = {minus, minus, minus, minus};
  const int per_group = (int)(p.group / kPieceInputs), steps = (int)(p.group / 32);   // pieces of a group, or steps of one
  for (int piece = begin; piece < end; piece += kAtOnce) {
    u32x4 w[kAtOnce][NT], v[kAtOnce][MT][4];
    u32x2 s[kAtOnce][NT][SUB], o[kAtOnce][NT][AFFINE ? SUB : 1];
#pragma unroll
    for (int u = 0; u < kAtOnce; u++) {
      const int at = min(piece + u, end - 1);
#pragma unroll
      for (int n = 0; n < NT; n++) {
        w[u][n] = __builtin_nontemporal_load(weights[n] + (int64_t)at * 64);
#pragma unroll
        for (int g = 0; g < SUB; g++) {
          const int group = min(SUB == 1 ? at / per_group : (4 * at + g) / steps, groups - 1);
          s[u][n][g] = *reinterpret_cast<const u32x2*>(scales[n] + group * 16);
          if constexpr (AFFINE) o[u][n][g] = *reinterpret_cast<const u32x2*>(offsets[n] + group * 16);
        }
      }
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int d = 0; d < 4; d++) {
          v[u][m][d] = u32x4{0u, 0u, 0u, 0u};
          if (has[m] && piece + u < end) v[u][m][d] = row_values(x[m], at * kPieceInputs + 32 * d + 8 * quarter, (int)p.inputs);
        }
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; u++)
#pragma unroll
      for (int g = 0; g < SUB; g++) {
        f32x4_t start[MT];
#pragma unroll
        for (int m = 0; m < MT; m++) {
          start[m] = zero;
#pragma unroll
          for (int d = 4 / SUB * g; d < 4 / SUB * (g + 1); d++) start[m] = mfma_16x16x32<BF16>(constant, v[u][m][d], start[m]);
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const f32x2_t s0 = unpack2<BF16>(s[u][n][g].x), s1 = unpack2<BF16>(s[u][n][g].y);
          const f32x4_t scale = {s0.x, s0.y, s1.x, s1.y};
          f32x4_t sum[MT];
#pragma unroll
          for (int m = 0; m < MT; m++) sum[m] = start[m];
#pragma unroll
          for (int d = 4 / SUB * g; d < 4 / SUB * (g + 1); d++) {
            const u32x4 a = numbers<BF16>(w[u][n][d]);
#pragma unroll
            for (int m = 0; m < MT; m++) sum[m] = mfma_16x16x32<BF16>(a, v[u][m][d], sum[m]);
          }
#pragma unroll
          for (int m = 0; m < MT; m++)
#pragma unroll
            for (int i = 0; i < 4; i++) total[n][m][i] = fmaf(scale[i], sum[m][i], total[n][m][i]);
          if constexpr (AFFINE) {
            const f32x2_t o0 = unpack2<BF16>(o[u][n][g].x), o1 = unpack2<BF16>(o[u][n][g].y);
            const f32x4_t offset = {o0.x, o0.y, o1.x, o1.y};
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
              for (int i = 0; i < 4; i++) total[n][m][i] = fmaf(offset[i], start[m][i] * -0.0625f, total[n][m][i]);   // start = -16 sum(x)
          }
        }
      }
  }
  if constexpr (KW > 1) {
    if (kw > 0) {
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int m = 0; m < MT; m++) shared[(((kw - 1) * NW + nw) * NT * MT + n * MT + m) * 64 + lane] = total[n][m];
    }
    __syncthreads();
    if (kw > 0) return;
    for (int k = 0; k < KW - 1; k++)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int m = 0; m < MT; m++) total[n][m] += shared[((k * NW + nw) * NT * MT + n * MT + m) * 64 + lane];
  }
#pragma unroll
  for (int m = 0; m < MT; m++) {
    if (16 * m + row >= t.rows) continue;
    int64_t to = t.first + 16 * m + row;
    if (p.sums) {
      to = p.indices[to];
      if (to < 0 || to >= p.rows) continue;
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const int64_t first = (int64_t)tile[n] * 16 + 4 * quarter;
      if (first >= p.outputs) continue;
      const int here = (int)min(p.outputs - first, (int64_t)4);
      if (p.sums) {
        float* at = p.sums + to * p.outputs + first;
        if (here == 4) *reinterpret_cast<QuadAt4*>(at) = __builtin_bit_cast(Quad, total[n][m]);
        else
          for (int i = 0; i < here; i++) at[i] = total[n][m][i];
        continue;
      }
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; i++) y[i] = activated(total[n][m][i], p.activation);
      const uint32_t two[2] = {pack2<BF16>(y[0], y[1]), pack2<BF16>(y[2], y[3])};
      uint16_t* at = static_cast<uint16_t*>(p.out) + to * p.out_stride + first;
      if (here == 4) *reinterpret_cast<PairAt2*>(at) = PairAt2{two[0], two[1]};
      else
        for (int i = 0; i < here; i++) at[i] = (uint16_t)(two[i / 2] >> (16 * (i & 1)));
    }
  }
}

// out[t] = sum over the choices j of a token, in their order, of (weights[s]) sums[s], s = t top_k + j; rounded once.  A thread per
// token and four outputs.
template <bool BF16>
__global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ sums, const float* __restrict__ weights, int64_t tokens, int top_k,
                                                      int64_t outputs, uint16_t* __restrict__ out, int64_t out_stride) {
  const int64_t across = (outputs + 3) / 4, step = (int64_t)gridDim.x * 256;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < tokens * across; at += step) {
    const int64_t t = at / across, o = at % across * 4;
    const int here = (int)min(outputs - o, (int64_t)4);
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < top_k; j++) {
      const int64_t s = t * top_k + j;
      const float by = weights ? weights[s] : 1.f;
      const float* from = sums + s * outputs + o;
      if (here == 4) {
        const f32x4_t u = __builtin_bit_cast(f32x4_t, *reinterpret_cast<const QuadAt4*>(from));
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = fmaf(by, u[i], v[i]);
      } else {
        for (int i = 0; i < here; i++) v[i] = fmaf(by, from[i], v[i]);
      }
    }
    const uint32_t two[2] = {pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3])};
    uint16_t* to = out + t * out_stride + o;
    if (here == 4) *reinterpret_cast<PairAt2*>(to) = PairAt2{two[0], two[1]};
    else
      for (int i = 0; i < here; i++) to[i] = (uint16_t)(two[i / 2] >> (16 * (i & 1)));
  }
}

static int weights_check(const char* who, int64_t experts, int64_t inputs, int64_t outputs, int64_t group, int dtype) {
  if (dtype != STK_F16 && dtype != STK_BF16) return fail(STK_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (experts < 1 || inputs < 1 || outputs < 1 || group < 1)
    return fail(STK_ERR_DIMS, "%s: %lld experts of %lld x %lld, groups of %lld", who, (long long)experts, (long long)inputs, (long long)outputs, (long long)group);
  if (group != 32 && group != 64 && group % kPieceInputs) return fail(STK_ERR_UNSUPPORTED, "%s: groups of 32, 64 or a multiple of 128 inputs, not %lld", who, (long long)group);
  if (inputs > INT32_MAX / 2 || outputs > INT32_MAX / 2 || experts > 65535 || pieces_in(inputs) * pieces_out(outputs) * experts > INT32_MAX)
    return fail(STK_ERR_UNSUPPORTED, "%s: size exceeds 32-bit range", who);
  return STK_OK;
}

static int product_check(const char* who, const Product4& p, int dtype, int64_t x_rows) {
  if (int rc = weights_check(who, p.experts, p.inputs, p.outputs, p.group, dtype)) return rc;
  if (p.rows < 0 || p.rows > INT32_MAX) return fail(STK_ERR_DIMS, "%s: %lld rows", who, (long long)p.rows);
  if (p.activation < 0 || p.activation > kSilu) return fail(STK_ERR_UNSUPPORTED, "%s: activation %d", who, p.activation);
  if (p.x_stride < 0 || (p.out && p.out_stride < p.outputs)) return fail(STK_ERR_DIMS, "%s: strides", who);
  if (p.rows > 0 && (!p.x || !p.packed || !p.scales || (!p.out && !p.sums))) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (!aligned16(p.packed) || (reinterpret_cast<uintptr_t>(p.scales) & 7) || (reinterpret_cast<uintptr_t>(p.offsets) & 7))
    return fail(STK_ERR_UNSUPPORTED, "%s: packed weights at multiples of 16 bytes, scales of 8", who);
  return STK_OK;
}

template <int KW, int NW, int NT, int MT>
static void launch_stream(const Product4& p, bool bf16, int64_t row_tiles, hipStream_t stream) {
  constexpr int lds = (KW - 1) * NW * NT * MT * 1024;
  const int64_t across = (pieces_out(p.outputs) + NW * NT - 1) / (NW * NT);
  const auto launch = [&](auto kernel) {
    set_lds_limit(kernel, lds);
    hipLaunchKernelGGL(kernel, dim3((unsigned)across, (unsigned)row_tiles), dim3(64 * KW * NW), lds, stream, p);
  };
  const bool sub = p.group < kPieceInputs;
  if (bf16) {
    if (p.offsets) sub ? launch(stream_kernel<true, true, 4, KW, NW, NT, MT>) : launch(stream_kernel<true, true, 1, KW, NW, NT, MT>);
    else sub ? launch(stream_kernel<true, false, 4, KW, NW, NT, MT>) : launch(stream_kernel<true, false, 1, KW, NW, NT, MT>);
  } else {
    if (p.offsets) sub ? launch(stream_kernel<false, true, 4, KW, NW, NT, MT>) : launch(stream_kernel<false, true, 1, KW, NW, NT, MT>);
    else sub ? launch(stream_kernel<false, false, 4, KW, NW, NT, MT>) : launch(stream_kernel<false, false, 1, KW, NW, NT, MT>);
  }
}

// Tiles of `of` rows that the rows of the experts can be at most.
static int64_t most_tiles(const Product4& p, int64_t of) {
  const int64_t hit = p.experts < p.rows ? p.experts : p.rows;
  return (p.rows + (of - 1) * hit) / of;
}

static int launch_product(const char* who, const Product4& p, int dtype, hipStream_t stream) {
  const bool bf16 = dtype == STK_BF16;
  const int64_t hit = p.experts < p.rows ? p.experts : p.rows, each = p.rows / hit;   // rows of an expert, about
  const int64_t along = pieces_in(p.inputs);
  if (most_tiles(p, 16) > 65535) return fail(STK_ERR_UNSUPPORTED, "%s: %lld rows", who, (long long)p.rows);
  if (each > 32) launch_stream<1, 4, 2, 4>(p, bf16, most_tiles(p, 64), stream);
  else if (each > 16) launch_stream<2, 2, 2, 2>(p, bf16, most_tiles(p, 32), stream);
  else if (along >= 64) launch_stream<16, 1, 1, 1>(p, bf16, most_tiles(p, 16), stream);
  else if (along >= 32 && hit == 1) launch_stream<8, 1, 1, 1>(p, bf16, most_tiles(p, 16), stream);
  else if (along >= 16) launch_stream<4, 1, 1, 1>(p, bf16, most_tiles(p, 16), stream);
  else launch_stream<2, 2, 1, 1>(p, bf16, most_tiles(p, 16), stream);
  return STK_OK;
}

}  // namespace stk

using namespace stk;

extern "C" int64_t stk_4bit_packed_bytes(int64_t experts, int64_t inputs, int64_t outputs) {
  return experts < 1 || inputs < 1 || outputs < 1 ? 0 : experts * pieces_in(inputs) * pieces_out(outputs) * kPieceBytes;
}
extern "C" int64_t stk_4bit_scales(int64_t experts, int64_t inputs, int64_t outputs, int64_t group_size) {
  return experts < 1 || inputs < 1 || outputs < 1 || group_size < 1 ? 0 : experts * groups_of(inputs, group_size) * pieces_out(outputs) * kPieceOutputs;
}

extern "C" int stk_quantize_4bit(const void* w, int64_t stride_e, int64_t stride_i, int64_t stride_o, int64_t experts, int64_t inputs, int64_t outputs,
                                 int64_t group_size, uint8_t* codes, void* scales, void* offsets, int w_dtype, int dtype, stk_stream_t stream) {
  const char* who = "stk_quantize_4bit";
  if (int rc = weights_check(who, experts, inputs, outputs, group_size, dtype)) return rc;
  if (w_dtype != dtype && w_dtype != STK_F32) return fail(STK_ERR_UNSUPPORTED, "%s: weights of the scales' type or float32", who);
  if (!w || !codes || !scales) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  const int64_t groups = groups_of(inputs, group_size);
  const dim3 grid((unsigned)((outputs + 255) / 256), (unsigned)(groups < 65535 ? groups : 65535), (unsigned)experts);
  const auto launch = [&](auto from, auto to) {
    typedef typename Value<from()>::stored W;
    typedef typename Value<to()>::stored S;
    hipLaunchKernelGGL((quantize_kernel<from(), to()>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const W*>(w), stride_e, stride_i, stride_o,
                       inputs, outputs, group_size, groups, codes, static_cast<S*>(scales), static_cast<S*>(offsets));
  };
  const auto by_type = [&](auto to) {
    if (w_dtype == STK_F32) launch(std::integral_constant<int, STK_F32>(), to);
    else launch(to, to);
  };
  if (dtype == STK_BF16) by_type(std::integral_constant<int, STK_BF16>());
  else by_type(std::integral_constant<int, STK_F16>());
  return check_launch(who);
}

extern "C" int stk_pack_4bit(const uint8_t* codes, const void* scales, const void* offsets, int64_t experts, int64_t inputs, int64_t outputs, int64_t group_size,
                             void* packed, void* packed_scales, void* packed_offsets, stk_stream_t stream) {
  const char* who = "stk_pack_4bit";
  if (int rc = weights_check(who, experts, inputs, outputs, group_size, STK_F16)) return rc;
  if (!codes || !scales || !packed || !packed_scales || !offsets != !packed_offsets) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (!aligned16(packed)) return fail(STK_ERR_UNSUPPORTED, "%s: packed weights at a multiple of 16 bytes", who);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t pieces = experts * pieces_in(inputs) * pieces_out(outputs), count = stk_4bit_scales(experts, inputs, outputs, group_size);
  const int64_t groups = groups_of(inputs, group_size);
  hipLaunchKernelGGL(pack_codes_kernel, dim3((unsigned)((pieces + 3) / 4)), dim3(256), 0, s, codes, inputs, outputs, pieces, static_cast<u32x4*>(packed));
  hipLaunchKernelGGL(pack_scales_kernel, dim3((unsigned)((count + 255) / 256)), dim3(256), 0, s, static_cast<const uint16_t*>(scales), groups, outputs, count,
                     static_cast<uint16_t*>(packed_scales));
  if (offsets)
    hipLaunchKernelGGL(pack_scales_kernel, dim3((unsigned)((count + 255) / 256)), dim3(256), 0, s, static_cast<const uint16_t*>(offsets), groups, outputs, count,
                       static_cast<uint16_t*>(packed_offsets));
  return check_launch(who);
}

extern "C" int stk_dequantize_4bit(const void* packed, const void* scales, const void* offsets, int64_t experts, int64_t inputs, int64_t outputs,
                                   int64_t group_size, void* out, int dtype, stk_stream_t stream) {
  const char* who = "stk_dequantize_4bit";
  if (int rc = weights_check(who, experts, inputs, outputs, group_size, dtype)) return rc;
  if (!packed || !scales || !out) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  const int64_t count = experts * inputs * outputs;
  const auto launch = [&](auto d) {
    typedef typename Value<d()>::stored T;
    hipLaunchKernelGGL((dequantize_kernel<d()>), dim3((unsigned)((count + 255) / 256)), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const uint8_t*>(packed), static_cast<const T*>(scales), static_cast<const T*>(offsets), inputs, outputs, group_size, count,
                       static_cast<T*>(out));
  };
  if (dtype == STK_BF16) launch(std::integral_constant<int, STK_BF16>());
  else launch(std::integral_constant<int, STK_F16>());
  return check_launch(who);
}

extern "C" size_t stk_matmul_4bit_workspace_bytes(int64_t rows, int64_t experts, int64_t inputs, int64_t outputs) { return 0; }

extern "C" int stk_matmul_4bit(const void* x, int64_t rows, int64_t x_stride, const void* packed, const void* scales, const void* offsets, int64_t inputs,
                               int64_t outputs, int64_t group_size, void* out, int64_t out_stride, int activation, int dtype, void*, size_t, stk_stream_t stream) {
  const char* who = "stk_matmul_4bit";
  const Product4 p = {x, x_stride, rows, static_cast<const uint8_t*>(packed), scales, offsets, 1, inputs, outputs, group_size, nullptr, nullptr, 0,
                      out, out_stride, nullptr, activation};
  if (int rc = product_check(who, p, dtype, rows)) return rc;
  if (rows == 0) return STK_OK;
  if (int rc = launch_product(who, p, dtype, static_cast<hipStream_t>(stream))) return rc;
  return check_launch(who);
}

extern "C" int stk_gather_matmul_4bit(const void* x, int64_t tokens, int64_t x_stride, const int32_t* indices, const int32_t* bins, int top_k, const void* packed,
                                      const void* scales, const void* offsets, int64_t experts, int64_t inputs, int64_t outputs, int64_t group_size, void* out,
                                      int64_t out_stride, int activation, int dtype, void*, size_t, stk_stream_t stream) {
  const char* who = "stk_gather_matmul_4bit";
  if (tokens < 0 || top_k < 1) return fail(STK_ERR_DIMS, "%s: %lld tokens, top_k %d", who, (long long)tokens, top_k);
  const Product4 p = {x, x_stride, tokens * top_k, static_cast<const uint8_t*>(packed), scales, offsets, experts, inputs, outputs, group_size, indices, bins, top_k,
                      out, out_stride, nullptr, activation};
  if (int rc = product_check(who, p, dtype, tokens)) return rc;
  if (tokens == 0) return STK_OK;
  if (!indices || !bins) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (int rc = launch_product(who, p, dtype, static_cast<hipStream_t>(stream))) return rc;
  return check_launch(who);
}

extern "C" size_t stk_matmul_4bit_scatter_workspace_bytes(int64_t slots, int64_t experts, int64_t inputs, int64_t outputs) {
  return slots < 1 || outputs < 1 ? 0 : (size_t)(slots * outputs) * sizeof(float);
}

extern "C" int stk_matmul_4bit_scatter(const void* x, int64_t x_stride, const int32_t* indices, const int32_t* bins, int top_k, int64_t tokens,
                                       const float* weights, const void* packed, const void* scales, const void* offsets, int64_t experts, int64_t inputs,
                                       int64_t outputs, int64_t group_size, void* out, int64_t out_stride, int dtype, void* workspace, size_t workspace_bytes,
                                       stk_stream_t stream) {
  const char* who = "stk_matmul_4bit_scatter";
  if (tokens < 0 || top_k < 1) return fail(STK_ERR_DIMS, "%s: %lld tokens, top_k %d", who, (long long)tokens, top_k);
  const int64_t slots = tokens * top_k;
  const Product4 p = {x, x_stride, slots, static_cast<const uint8_t*>(packed), scales, offsets, experts, inputs, outputs, group_size, indices, bins, 0,
                      nullptr, 0, static_cast<float*>(workspace), 0};
  if (slots > 0 && (!workspace || workspace_bytes < stk_matmul_4bit_scatter_workspace_bytes(slots, experts, inputs, outputs)))
    return fail(STK_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", who, stk_matmul_4bit_scatter_workspace_bytes(slots, experts, inputs, outputs));
  if (int rc = product_check(who, p, dtype, slots)) return rc;
  if (tokens == 0) return STK_OK;
  if (!indices || !bins || !out || out_stride < outputs) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (int rc = launch_product(who, p, dtype, s)) return rc;
  const int64_t groups = (tokens * ((outputs + 3) / 4) + 255) / 256;
  const dim3 grid((unsigned)(groups < 65536 ? groups : 65536));
  const auto combine = dtype == STK_BF16 ? combine_kernel<true> : combine_kernel<false>;
  hipLaunchKernelGGL(combine, grid, dim3(256), 0, s, static_cast<const float*>(workspace), weights, tokens, top_k, outputs, static_cast<uint16_t*>(out), out_stride);
  return check_launch(who);
}
