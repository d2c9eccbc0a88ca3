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
// under the rounded ones.  A group with a NaN, or whose rounded scale or offset is no finite number, has a scale of NaN: minimum and
// maximum pass over a NaN, and an infinite scale would make codes of 0 of every weight.  A thread per group and output.
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
    bool finite = true;
    for (int64_t i = lo; i < hi; i++) {
      const float v = Value<DTYPE>::widen(at[i * stride_i]);
      least = fminf(least, v), most = fmaxf(most, v);
      finite = finite && v == v;
    }
    auto scale16 = Value<OUT>::round(offsets ? (most - least) / 15.f : fmaxf(most, -least) / 7.f);
    const auto offset16 = Value<OUT>::round(least);
    finite = finite && Value<OUT>::widen(scale16) < INFINITY && !(offsets && fabsf(Value<OUT>::widen(offset16)) == INFINITY);
    if (!finite) scale16 = Value<OUT>::round(NAN);
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

// A wavefront per piece: lane l gathers the 32 codes of its 16 bytes.  The eight wavefronts of a workgroup take neighbouring outputs: 128 bytes
// of each row of codes.
__global__ __launch_bounds__(512) void pack_codes_kernel(const uint8_t* __restrict__ codes, int64_t inputs, int64_t outputs, int64_t pieces, u32x4* __restrict__ packed) {
  const int lane = threadIdx.x & 63;
  const int64_t along = pieces_in(inputs), down = pieces_out(outputs);
  for (int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 6); at < pieces; at += (int64_t)gridDim.x * 8) {
    const int64_t tile = at % down, k = at / down % along, e = at / (down * along);
    const int64_t first = k * kPieceInputs, o = tile * kPieceOutputs + (lane & 15);
    uint32_t words[4];
#pragma unroll
    for (int d = 0; d < 4; d++) {
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int64_t i = first + 32 * d + 8 * (lane >> 4) + j;
        const uint32_t code = i < inputs && o < outputs ? codes[(e * inputs + i) * outputs + o] & 15u : 8u;
        word |= code << (4 * (j >> 1) + 16 * (j & 1));
      }
      words[d] = word << kCodesTurn | word >> (32 - kCodesTurn);
    }
    packed[((e * down + tile) * along + k) * 64 + lane] = u32x4{words[0], words[1], words[2], words[3]};
  }
}

// Scales [expert][group][output] -> the order of weights4.h; the same for offsets.
__global__ __launch_bounds__(256) void pack_scales_kernel(const uint16_t* __restrict__ scales, int64_t inputs, int64_t outputs, int64_t group, int64_t count,
                                                          uint16_t* __restrict__ packed) {
  const int64_t sub = groups_in_block(group), blocks = scale_blocks(inputs, group), groups = groups_of(inputs, group), down = pieces_out(outputs);
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < count; at += (int64_t)gridDim.x * 256) {
    const int64_t within = at % (16 * sub), block = at / (16 * sub) % blocks, tile = at / (16 * sub) / blocks;
    const int64_t o = tile % down * 16 + within / (4 * sub) * 4 + within % 4, g = block * sub + within / 4 % sub, e = tile / down;
    packed[at] = o < outputs && g < groups ? scales[(e * groups + g) * outputs + o] : (uint16_t)0;
  }
}

template <int DTYPE>
__device__ __forceinline__ float weight_of(const uint8_t* packed, const typename Value<DTYPE>::stored* scales, const typename Value<DTYPE>::stored* offsets,
                                           int64_t e, int64_t i, int64_t o, int64_t inputs, int64_t outputs, int64_t group) {
  const int64_t along = pieces_in(inputs), down = pieces_out(outputs);
  const int code = code_of(reinterpret_cast<const uint32_t*>(packed + ((e * down + o / 16) * along + i / 128) * kPieceBytes), (int)(o & 15), (int)(i & 127));
  const int64_t at = scale_at(e * down + o / 16, (int)(o & 15), i / group, inputs, group);
  const float scale = Value<DTYPE>::widen(scales[at]);
  return offsets ? scale * (float)code + Value<DTYPE>::widen(offsets[at]) : scale * (float)(code - 8);
}

template <int DTYPE>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint8_t* __restrict__ packed, const typename Value<DTYPE>::stored* __restrict__ scales,
                                                         const typename Value<DTYPE>::stored* __restrict__ offsets, int64_t inputs, int64_t outputs,
                                                         int64_t group, int64_t count, typename Value<DTYPE>::stored* __restrict__ out) {
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < count; at += (int64_t)gridDim.x * 256) {
    const int64_t o = at % outputs, i = at / outputs % inputs, e = at / outputs / inputs;
    out[at] = Value<DTYPE>::round(weight_of<DTYPE>(packed, scales, offsets, e, i, o, inputs, outputs, group));
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
// multiplies the fp32 sum.  That makes 7 instructions for eight weights (8 in float16) and one for a group's four outputs, below half of
// what a stream of weights at memory speed leaves time for.
template <bool BF16> struct Codes;
template <> struct Codes<true> {
  static constexpr uint32_t mask = 0x00780078u, magic = 0x41804180u, minus24 = 0xc1c0c1c0u, minus16 = 0xc180c180u;
  static __device__ __forceinline__ uint32_t placed(uint32_t w, int p) { return p == 0 ? w : p == 3 ? __builtin_amdgcn_alignbit(w, w, 12) : w >> (4 * p); }
};
template <> struct Codes<false> {
  static constexpr uint32_t mask = 0x03c003c0u, magic = 0x4c004c00u, minus24 = 0xce00ce00u, minus16 = 0xcc00cc00u;
  static __device__ __forceinline__ uint32_t placed(uint32_t w, int p) { return p == 0 ? w << 3 : p == 3 ? __builtin_amdgcn_alignbit(w, w, 9) : w >> (4 * p - 3); }
};
// The mask and the magic number in registers that the compiler takes for variables: with constants it makes two instructions of an
// and-or, which has no room for two literals.
template <bool BF16>
struct Decoder {
  uint32_t mask = Codes<BF16>::mask, magic = Codes<BF16>::magic;
  __device__ __forceinline__ Decoder() { asm("" : "+s"(mask), "+v"(magic)); }
  __device__ __forceinline__ u32x4 operator()(uint32_t w) const {
    u32x4 v;
#pragma unroll
    for (int p = 0; p < 4; p++) v[p] = (Codes<BF16>::placed(w, p) & mask) | magic;
    return v;
  }
};
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

// total = activation(total); the kind is the same for all, so that the functions of many values overlap.  A sum that is NaN stays one: an
// infinity among the rows is NaN here, and relu by the comparison with 0 from the other side would make 0 of it.
template <int KIND, int NT, int MT>
__device__ __forceinline__ void activate_each(f32x4_t (&total)[NT][MT]) {
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float v = total[n][m][i];
        total[n][m][i] = KIND == kRelu ? (v <= 0.f ? 0.f : v) : activate<KIND>(v);
      }
}
template <int NT, int MT>
__device__ __forceinline__ void activate_sums(f32x4_t (&total)[NT][MT], int kind) {
  switch (kind) {
    case kRelu: activate_each<kRelu>(total); break;
    case kGeluTanh: activate_each<kGeluTanh>(total); break;
    case kGeluErf: activate_each<kGeluErf>(total); break;
    case kSilu: activate_each<kSilu>(total); break;
    default: break;
  }
}

// The sums of a wavefront: total[n][m][i] belongs to output 16 tile[n] + 4 quarter + i and row 16 m + row of the tile.
template <bool BF16, int NT, int MT>
__device__ __forceinline__ void store(const Product4& p, const RowTile& t, const int (&tile)[NT], f32x4_t (&total)[NT][MT], int row, int quarter) {
  activate_sums(total, p.activation);
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
      const f32x4_t y = total[n][m];
      const uint32_t two[2] = {pack2<BF16>(y[0], y[1]), pack2<BF16>(y[2], y[3])};
      uint16_t* at = static_cast<uint16_t*>(p.out) + to * p.out_stride + first;
      if (here == 4) *reinterpret_cast<PairAt2*>(at) = PairAt2{two[0], two[1]};
      else
        for (int i = 0; i < here; i++) at[i] = (uint16_t)(two[i / 2] >> (16 * (i & 1)));
    }
  }
}

// The products of one group of a piece, scaled and added to the totals.  v(m, d): the fragment of rows 16 m .. 16 m + 15 for step d.
template <bool BF16, bool AFFINE, int SUB, int NT, int MT, class V>
__device__ __forceinline__ void add_group(const Decoder<BF16>& numbers, f32x4_t (&total)[NT][MT], int k, const u32x4 (&w)[NT], const u32x2 (&s)[NT][SUB], const u32x2 (&o)[NT][AFFINE ? SUB : 1], V&& v) {
  constexpr uint32_t minus = AFFINE ? Codes<BF16>::minus16 : Codes<BF16>::minus24;
  const u32x4 constant = {minus, minus, minus, minus};
  constexpr int kSteps = 4 / SUB;
  u32x4 x[kSteps][MT];
  f32x4_t start[MT];
#pragma unroll
  for (int m = 0; m < MT; m++) {
    start[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < kSteps; d++) {
      x[d][m] = v(m, kSteps * k + d);
      start[m] = mfma_16x16x32<BF16>(constant, x[d][m], start[m]);
    }
  }
#pragma unroll
  for (int n = 0; n < NT; n++) {
    f32x4_t sum[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) sum[m] = start[m];
#pragma unroll
    for (int d = 0; d < kSteps; d++) {
      const u32x4 a = numbers(w[n][kSteps * k + d]);
#pragma unroll
      for (int m = 0; m < MT; m++) sum[m] = mfma_16x16x32<BF16>(a, x[d][m], sum[m]);
    }
    const f32x2_t s0 = unpack2<BF16>(s[n][k].x), s1 = unpack2<BF16>(s[n][k].y);
    const f32x4_t scale = {s0.x, s0.y, s1.x, s1.y};
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int i = 0; i < 4; i++) total[n][m][i] = fmaf(scale[i], sum[m][i], total[n][m][i]);
    if constexpr (AFFINE) {
      const f32x2_t o0 = unpack2<BF16>(o[n][k].x), o1 = unpack2<BF16>(o[n][k].y);
      const f32x4_t offset = {o0.x, o0.y, o1.x, o1.y};
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) total[n][m][i] = fmaf(offset[i], start[m][i] * -0.0625f, total[n][m][i]);   // start = -16 sum(x)
    }
  }
}

// What a wavefront holds of a piece: the codes of NT x 16 outputs, their scales and offsets, and MT x 16 rows of x.
template <int NT, int MT, int SUB, bool AFFINE>
struct Stage {
  u32x4 w[NT], v[MT > 0 ? MT : 1][4];
  u32x2 s[NT][SUB], o[NT][AFFINE ? SUB : 1];
};

// Few rows: KW wavefronts share the inputs of NW x NT x 16 outputs and up to 16 rows of one expert, a piece of weights at a time; their sums meet
// in LDS.  Two pieces are on their way at a time (three or four: the same or slower, registers cost wavefronts).  SUB: groups of a piece whose
// sums are scaled apart (4, 2 or 1: groups of 32, 64, more).  Rows beyond those of the tile are read from its first one: what they give
// stays in columns that are not stored.  The 2 of the launch bounds keeps the compiler from accumulation registers, which it would take beside
// 130 others: two wavefronts instead of three (4x1x4 on the 128 slots of 64 experts of 4096 x 1024: 31.5 us, 29.6 so).
// Bound by the bytes of the weights where many experts are hit (64 tokens, top 2 of 64 experts of 1024 x 4096: 121 MB in 26.1 us,
// 4.65 TB/s of the 5.16 of a copy; of 4096 x 1024 with the sum over the choices 29.5, two launches), and by the launch and one trip to
// memory for a single row (4096 x 4096, 8.7 MB: 5.3 us).  Four tiles with groups of 32 want more than the 256 registers that there are: with
// offsets 12 to 14 go to scratch memory (55 us for the same tokens, 58 for 4096 x 1024), in bfloat16 without offsets 1x4x4 loses 113, which
// cost it 99 us where float16 takes 34.5.
template <bool BF16, bool AFFINE, int SUB, int KW, int NW, int NT>
__global__ __launch_bounds__(64 * KW * NW, 2) void stream_kernel(Product4 p) {
  constexpr int MT = 1, DEPTH = 2;
  extern __shared__ f32x4_t shared[];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), kw = wave % KW, nw = wave / KW;
  const RowTile t = row_tile<16 * MT>(p, (int)(blockIdx.z * gridDim.y + blockIdx.y), lane);
  if (t.rows == 0) return;
  const int along = (int)pieces_in(p.inputs), down = (int)pieces_out(p.outputs), blocks = (int)scale_blocks(p.inputs, p.group);
  const int row = lane & 15, quarter = lane >> 4;
  int tile[NT];   // (the last tiles of a workgroup may lie beyond the outputs: computed again and not stored)
  const u32x4* weights[NT];
  const uint16_t *scales[NT], *offsets[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) {
    tile[n] = ((int)blockIdx.x * NW + nw) * NT + n;
    const int64_t at = (int64_t)t.expert * down + min(tile[n], down - 1);
    weights[n] = reinterpret_cast<const u32x4*>(p.packed + at * along * kPieceBytes) + lane;
    scales[n] = static_cast<const uint16_t*>(p.scales) + (at * blocks * 4 + quarter) * (4 * SUB);
    offsets[n] = static_cast<const uint16_t*>(p.offsets) + (at * blocks * 4 + quarter) * (4 * SUB);
  }
  const uint16_t* x[MT];
  int64_t from[MT];
  int slot[MT];
#pragma unroll
  for (int m = 0; m < MT; m++) {
    from[m] = t.first + (16 * m + row < t.rows ? 16 * m + row : 0);
    slot[m] = p.top_k > 0 ? p.indices[from[m]] : 0;
  }
  const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
  f32x4_t total[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int m = 0; m < MT; m++) total[n][m] = zero;
  const int per_block = SUB > 1 ? 1 : (int)(p.group / kPieceInputs);   // pieces with the same scales
  const Decoder<BF16> numbers;
  typedef Stage<NT, MT, SUB, AFFINE> S;

  const auto load_weights = [&](S& g, int piece) {
    const int block = SUB > 1 || per_block == 1 ? piece : piece / per_block;
#pragma unroll
    for (int n = 0; n < NT; n++) {
      g.w[n] = __builtin_nontemporal_load(weights[n] + (int64_t)piece * 64);
#pragma unroll
      for (int k = 0; k < SUB; k++) {
        g.s[n][k] = reinterpret_cast<const u32x2*>(scales[n] + (int64_t)block * (16 * SUB))[k];
        if constexpr (AFFINE) g.o[n][k] = reinterpret_cast<const u32x2*>(offsets[n] + (int64_t)block * (16 * SUB))[k];
      }
    }
  };
  const auto load_rows = [&](S& g, int piece) {
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int d = 0; d < 4; d++) g.v[m][d] = __builtin_bit_cast(u32x4, *reinterpret_cast<const QuadAt2*>(x[m] + piece * kPieceInputs + 32 * d));
  };
  const auto add = [&](const S& g) {
#pragma unroll
    for (int k = 0; k < SUB; k++) add_group<BF16, AFFINE, SUB>(numbers, total, k, g.w, g.s, g.o, [&](int m, int d) { return g.v[m][d]; });
  };

  const int share = (along + KW - 1) / KW, begin = min(kw * share, along), end = min(begin + share, along);
  const int whole = max(begin, min(end, (int)(p.inputs / kPieceInputs)));   // the pieces in front of it have all their inputs
  S stage[DEPTH];
  int piece = begin;
  if (piece < whole) load_weights(stage[0], piece);
  // (the slots were asked for in front of the weights: waiting for them does not wait for those)
#pragma unroll
  for (int m = 0; m < MT; m++) {
    if (p.top_k > 0) from[m] = (unsigned)slot[m] < (unsigned)p.rows ? slot[m] / p.top_k : 0;
    x[m] = static_cast<const uint16_t*>(p.x) + from[m] * p.x_stride + 8 * quarter;
  }
  if (piece < whole) {
    load_rows(stage[0], piece);
#pragma unroll
    for (int u = 1; u < DEPTH; u++) load_weights(stage[u], min(piece + u, whole - 1)), load_rows(stage[u], min(piece + u, whole - 1));
    for (; piece + 2 * DEPTH <= whole; piece += DEPTH)
#pragma unroll
      for (int u = 0; u < DEPTH; u++) add(stage[u]), load_weights(stage[u], piece + DEPTH + u), load_rows(stage[u], piece + DEPTH + u);
#pragma unroll
    for (int u = 0; u < DEPTH; u++) {
      if (piece + u < whole) add(stage[u]);
      if (piece + DEPTH + u < whole) load_weights(stage[u], piece + DEPTH + u), load_rows(stage[u], piece + DEPTH + u);
    }
#pragma unroll
    for (int u = 0; u < DEPTH; u++)
      if (piece + DEPTH + u < whole) add(stage[u]);
  }
  if (end > whole) {   // the last piece, whose inputs end inside it
    load_weights(stage[0], whole);
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int d = 0; d < 4; d++) stage[0].v[m][d] = row_values(x[m], whole * kPieceInputs + 32 * d, (int)p.inputs - 8 * quarter);
    add(stage[0]);
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
  store<BF16>(p, t, tile, total, row, quarter);
}

// Many rows: four wavefronts, side by side on 64 NT outputs, share 16 MT rows of one expert, whose values pass through LDS in pieces of
// 128 inputs (two of them, one being multiplied and one being written).  A code then becomes a number once for 16 MT rows.
template <bool BF16, bool AFFINE, int SUB, int NT, int MT>
__global__ __launch_bounds__(256) void tile_kernel(Product4 p) {
  __shared__ u32x4 values[2][16 * MT * 16];   // [row][eight inputs], the place within a row swizzled by the row
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const RowTile t = row_tile<16 * MT>(p, (int)(blockIdx.z * gridDim.y + blockIdx.y), lane);
  if (t.rows == 0) return;
  const int along = (int)pieces_in(p.inputs), down = (int)pieces_out(p.outputs), blocks = (int)scale_blocks(p.inputs, p.group);
  const int whole = (int)(p.inputs / kPieceInputs), row = lane & 15, quarter = lane >> 4;
  // what this thread carries to LDS: eight inputs, number `eight` of a piece, of every 16th row
  const int eight = threadIdx.x & 15, carried = threadIdx.x >> 4;
  const uint16_t* x[MT];
#pragma unroll
  for (int m = 0; m < MT; m++) {
    int64_t from = t.first + (16 * m + carried < t.rows ? 16 * m + carried : 0);
    if (p.top_k > 0) {
      const int slot = p.indices[from];
      from = (unsigned)slot < (unsigned)p.rows ? slot / p.top_k : 0;
    }
    x[m] = static_cast<const uint16_t*>(p.x) + from * p.x_stride;
  }
  int tile[NT];
  const u32x4* weights[NT];
  const uint16_t *scales[NT], *offsets[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) {
    tile[n] = ((int)blockIdx.x * 4 + wave) * NT + n;
    const int64_t at = (int64_t)t.expert * down + min(tile[n], down - 1);
    weights[n] = reinterpret_cast<const u32x4*>(p.packed + at * along * kPieceBytes) + lane;
    scales[n] = static_cast<const uint16_t*>(p.scales) + (at * blocks * 4 + quarter) * (4 * SUB);
    offsets[n] = static_cast<const uint16_t*>(p.offsets) + (at * blocks * 4 + quarter) * (4 * SUB);
  }
  const int per_block = SUB > 1 ? 1 : (int)(p.group / kPieceInputs);
  const Decoder<BF16> numbers;
  u32x4 carry[MT];
  Stage<NT, 0, SUB, AFFINE> ahead;   // the weights of the next piece
  const auto load_weights = [&](int piece) {
    const int block = SUB > 1 || per_block == 1 ? piece : piece / per_block;
#pragma unroll
    for (int n = 0; n < NT; n++) {
      ahead.w[n] = weights[n][(int64_t)piece * 64];
#pragma unroll
      for (int k = 0; k < SUB; k++) {
        ahead.s[n][k] = reinterpret_cast<const u32x2*>(scales[n] + (int64_t)block * (16 * SUB))[k];
        if constexpr (AFFINE) ahead.o[n][k] = reinterpret_cast<const u32x2*>(offsets[n] + (int64_t)block * (16 * SUB))[k];
      }
    }
  };
  const auto load_rows = [&](int piece) {
    const int i = piece * kPieceInputs + 8 * eight;
#pragma unroll
    for (int m = 0; m < MT; m++)
      carry[m] = piece < whole ? __builtin_bit_cast(u32x4, *reinterpret_cast<const QuadAt2*>(x[m] + i)) : row_values(x[m], i, (int)p.inputs);
  };
  const auto write_rows = [&](u32x4* to) {
#pragma unroll
    for (int m = 0; m < MT; m++) to[(16 * m + carried) * 16 + (eight ^ carried)] = carry[m];
  };
  f32x4_t total[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int m = 0; m < MT; m++) total[n][m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  load_rows(0);
  load_weights(0);
  write_rows(values[0]);
  __syncthreads();
  for (int piece = 0; piece < along; piece++) {
    const auto here = ahead;
    if (piece + 1 < along) load_rows(piece + 1), load_weights(piece + 1);
    const u32x4* from = values[piece & 1];
#pragma unroll
    for (int k = 0; k < SUB; k++)
      add_group<BF16, AFFINE, SUB>(numbers, total, k, here.w, here.s, here.o, [&](int m, int d) { return from[(16 * m + row) * 16 + ((4 * d + quarter) ^ row)]; });
    if (piece + 1 < along) write_rows(values[(piece + 1) & 1]);
    __syncthreads();
  }
  store<BF16>(p, t, tile, total, row, quarter);
}

// The same with everything on its way to LDS without registers, the next piece of x arriving while one is multiplied, codes and scales
// (each wavefront reads its own) in one place that is filled again once they are in registers: rows whose values come in whole 16-byte pieces
// at multiples of 16 bytes.  What counts is how many wavefronts are on a compute unit: 16384 rows over 64 experts (1024 x 4096, 137 GFLOP,
// 302 MB) take 216 - 223 us, 615 - 635 TFLOP/s, with three workgroups of 32 x 256 on a unit, 242 with two of 48 x 256; in the case of offsets
// 266 with two stages of codes, 238 so; 263 with three pieces on their way, 300 through registers (the kernel above); 2048
// rows of 4096 x 4096 run at 790.  Vector instructions, of which making numbers of codes is a half, are issued three quarters of the time and
// the matrix units are busy 35 % (counters); one MFMA of five at 64 outputs a wavefront, one of three at 32, is for the sums of x.  What is lost
// at the ends of a tile shows in short rows of inputs: the rate with 1024 is three quarters of that with 4096.  A raised priority of the wavefronts
// while they multiply is worth 2 % either way; workgroups that walk over tiles, with the next one's first piece on its way, were slower (250).
static __device__ u32x4 no_values;   // (what lies behind the last input)
// 16 bytes per lane from any addresses into the LDS bytes from lds_base on, lane after lane.
__device__ __forceinline__ void dma16_any(const void* from, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(uniform((int)lds_base)), "v"((uint64_t)from) : "memory", "m0");
}
template <int NT, int MT>
struct Stage16 {
  static constexpr int kRows = MT * 4096, kCodes = 4 * NT * 1024, kScales = 4 * 512;   // bytes
  static constexpr int bytes(bool affine) { return 2 * kRows + kCodes + (affine ? 2 : 1) * kScales; }
};
template <bool BF16, bool AFFINE, int SUB, int NT, int MT>
__global__ __launch_bounds__(256, 3) void ring_kernel(Product4 p) {
  typedef Stage16<NT, MT> R;
  constexpr int kPrivate = 2 * R::kRows;
  extern __shared__ char smem[];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const RowTile t = row_tile<16 * MT>(p, (int)(blockIdx.z * gridDim.y + blockIdx.y), lane);
  if (t.rows == 0) return;
  const int along = (int)pieces_in(p.inputs), down = (int)pieces_out(p.outputs), blocks = (int)scale_blocks(p.inputs, p.group);
  const int row = lane & 15, quarter = lane >> 4;
  // a transfer carries four rows; this lane eight inputs of one of them, put where that row's swizzle wants them
  const char* x[MT];
  int first_input[MT];
#pragma unroll
  for (int m = 0; m < MT; m++) {
    const int r = 4 * (m * 4 + wave) + quarter;
    int64_t from = t.first + (r < t.rows ? r : 0);
    if (p.top_k > 0) {
      const int slot = p.indices[from];
      from = (unsigned)slot < (unsigned)p.rows ? slot / p.top_k : 0;
    }
    first_input[m] = 8 * (row ^ (r & 15));
    x[m] = reinterpret_cast<const char*>(static_cast<const uint16_t*>(p.x) + from * p.x_stride + first_input[m]);
  }
  int tile[NT];
  gptr_t weights[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) {
    tile[n] = ((int)blockIdx.x * 4 + wave) * NT + n;
    weights[n] = uniform_global(p.packed + ((int64_t)t.expert * down + min(tile[n], down - 1)) * along * kPieceBytes);
  }
  const int per_block = SUB > 1 ? 1 : (int)(p.group / kPieceInputs);
  // lanes that carry scales: 2 SUB for each 16 outputs
  const int mine = min(((int)blockIdx.x * 4 + wave) * NT + lane / (2 * SUB), down - 1);
  const int64_t scale_from = ((int64_t)t.expert * down + mine) * blocks * (32 * SUB) + lane % (2 * SUB) * 16;
  const uint32_t lds = (uint32_t)(uintptr_t)(STK_LDS char*)smem;
  const auto issue_rows = [&](int piece, int stage) {
    const uint32_t to = lds + stage * R::kRows;
    const bool last = (piece + 1) * kPieceInputs > p.inputs;
#pragma unroll
    for (int m = 0; m < MT; m++) {
      const char* from = x[m] + (int64_t)piece * (2 * kPieceInputs);
      if (last && piece * kPieceInputs + first_input[m] >= p.inputs) from = reinterpret_cast<const char*>(&no_values);
      dma16_any(from, to + (m * 4 + wave) * 1024);
    }
  };
  const auto issue_codes = [&](int piece) {
    const uint32_t to = lds + kPrivate;
#pragma unroll
    for (int n = 0; n < NT; n++) dma16(weights[n] + (int64_t)piece * kPieceBytes, lane * 16, to + (wave * NT + n) * 1024);
    if (lane < NT * 2 * SUB) {
      const int64_t at = scale_from + (int64_t)(SUB > 1 || per_block == 1 ? piece : piece / per_block) * (32 * SUB);
      dma16_any(static_cast<const char*>(p.scales) + at, to + R::kCodes + wave * 512);
      if constexpr (AFFINE) dma16_any(static_cast<const char*>(p.offsets) + at, to + R::kCodes + R::kScales + wave * 512);
    }
  };
  const Decoder<BF16> numbers;
  f32x4_t total[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int m = 0; m < MT; m++) total[n][m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  issue_codes(0), issue_rows(0, 0);
  for (int piece = 0; piece < along; piece++) {
    wait_vmcnt<0>();
    __syncthreads();   // everybody's part of the piece is there, and everybody is done with the one whose place is filled now
    if (piece + 1 < along) issue_rows(piece + 1, (piece + 1) & 1);
    const char *from = smem + (piece & 1) * R::kRows, *own = smem + kPrivate;
    u32x4 w[NT];
    u32x2 s[NT][SUB], o[NT][AFFINE ? SUB : 1];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      w[n] = reinterpret_cast<const u32x4*>(own + (wave * NT + n) * 1024)[lane];
#pragma unroll
      for (int k = 0; k < SUB; k++) {
        s[n][k] = reinterpret_cast<const u32x2*>(own + R::kCodes + wave * 512 + n * 32 * SUB)[quarter * SUB + k];
        if constexpr (AFFINE) o[n][k] = reinterpret_cast<const u32x2*>(own + R::kCodes + R::kScales + wave * 512 + n * 32 * SUB)[quarter * SUB + k];
      }
    }
    // a wavefront's codes and scales are its own: once they are in registers the next ones may arrive in their place
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
#pragma unroll
    for (int n = 0; n < NT; n++) asm volatile("" : "+v"(w[n]));
    if (piece + 1 < along) issue_codes(piece + 1);
    const u32x4* values = reinterpret_cast<const u32x4*>(from);
#pragma unroll
    for (int k = 0; k < SUB; k++)
      add_group<BF16, AFFINE, SUB>(numbers, total, k, w, s, o, [&](int m, int d) { return values[(16 * m + row) * 16 + ((4 * d + quarter) ^ row)]; });
  }
  store<BF16>(p, t, tile, total, row, quarter);
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
    const uint32_t two[2] = {pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3])};
    uint16_t* to = out + t * out_stride + o;
    if (here == 4) *reinterpret_cast<PairAt2*>(to) = PairAt2{two[0], two[1]};
    else
      for (int i = 0; i < here; i++) to[i] = (uint16_t)(two[i / 2] >> (16 * (i & 1)));
  }
}

// Workgroups of a kernel that loops over `count` things, `each` of them a workgroup at a time.
static dim3 loop_grid(int64_t count, int64_t each) {
  const int64_t groups = (count + each - 1) / each;
  return dim3((unsigned)(groups < 1 << 18 ? groups : 1 << 18));
}

// (leaves the group in the kernels' terms)
static int weights_check(const char* who, int64_t experts, int64_t inputs, int64_t outputs, int64_t& group, int dtype) {
  if (dtype != STK_F16 && dtype != STK_BF16) return fail(STK_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (experts < 1 || inputs < 1 || outputs < 1 || group < 1)
    return fail(STK_ERR_DIMS, "%s: %lld experts of %lld x %lld, groups of %lld", who, (long long)experts, (long long)inputs, (long long)outputs, (long long)group);
  if (group != 32 && group != 64 && group % kPieceInputs) return fail(STK_ERR_UNSUPPORTED, "%s: groups of 32, 64 or a multiple of 128 inputs, not %lld", who, (long long)group);
  if (inputs > 1 << 26 || outputs > 1 << 26 || experts > 65535 || pieces_in(inputs) * pieces_out(outputs) > INT32_MAX / experts)
    return fail(STK_ERR_UNSUPPORTED, "%s: size exceeds 32-bit range", who);
  group = group_within(inputs, group);
  return STK_OK;
}

static int product_check(const char* who, Product4& p, int dtype) {
  if (int rc = weights_check(who, p.experts, p.inputs, p.outputs, p.group, dtype)) return rc;
  if (p.rows < 0 || p.rows > INT32_MAX) return fail(STK_ERR_DIMS, "%s: %lld rows", who, (long long)p.rows);
  if (p.activation < 0 || p.activation > kSilu) return fail(STK_ERR_UNSUPPORTED, "%s: activation %d", who, p.activation);
  if (p.x_stride < 0 || (p.out && p.out_stride < p.outputs)) return fail(STK_ERR_DIMS, "%s: strides", who);
  if (p.rows > 0 && (!p.x || !p.packed || !p.scales || (!p.out && !p.sums))) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (!aligned16(p.packed) || !aligned16(p.scales) || !aligned16(p.offsets)) return fail(STK_ERR_UNSUPPORTED, "%s: packed weights and scales at multiples of 16 bytes", who);
  return STK_OK;
}

// Tiles of `of` rows that the rows of the experts can be at most.
static int64_t most_tiles(const Product4& p, int64_t of) {
  const int64_t hit = p.experts < p.rows ? p.experts : p.rows;
  return (p.rows + (of - 1) * hit) / of;
}
// Row tiles lie along y, and beyond what y holds along z (those that there are not end at once).
static dim3 grid_of(int64_t across, int64_t row_tiles) {
  const int64_t layers = (row_tiles + 65534) / 65535;
  return dim3((unsigned)across, (unsigned)((row_tiles + layers - 1) / layers), (unsigned)layers);
}
// fn(bf16, affine, groups of a piece) as constants.
template <class Fn>
static void for_form(const Product4& p, bool bf16, Fn&& fn) {
  const auto by_group = [&](auto type, auto affine) {
    if (p.group == 32) fn(type, affine, std::integral_constant<int, 4>());
    else if (p.group == 64) fn(type, affine, std::integral_constant<int, 2>());
    else fn(type, affine, std::integral_constant<int, 1>());
  };
  const auto by_offsets = [&](auto type) {
    if (p.offsets) by_group(type, std::true_type());
    else by_group(type, std::false_type());
  };
  if (bf16) by_offsets(std::true_type());
  else by_offsets(std::false_type());
}
template <int KW, int NW, int NT>
static void launch_stream(const Product4& p, bool bf16, hipStream_t stream) {
  for_form(p, bf16, [&](auto type, auto affine, auto sub) {
    constexpr int lds = (KW - 1) * NW * NT * 1024;
    const auto kernel = stream_kernel<decltype(type)::value, decltype(affine)::value, decltype(sub)::value, KW, NW, NT>;
    set_lds_limit(kernel, lds);
    const int64_t across = (pieces_out(p.outputs) + NW * NT - 1) / (NW * NT);
    hipLaunchKernelGGL(kernel, grid_of(across, most_tiles(p, 16)), dim3(64 * KW * NW), lds, stream, p);
  });
}
template <int NT, int MT>
static void launch_tiles(const Product4& p, bool bf16, hipStream_t stream) {
  for_form(p, bf16, [&](auto type, auto affine, auto sub) {
    const auto kernel = tile_kernel<decltype(type)::value, decltype(affine)::value, decltype(sub)::value, NT, MT>;
    const int64_t across = (pieces_out(p.outputs) + 4 * NT - 1) / (4 * NT);
    hipLaunchKernelGGL(kernel, grid_of(across, most_tiles(p, 16 * MT)), dim3(256), 0, stream, p);
  });
}

template <int NT, int MT>
static void launch_ring(const Product4& p, bool bf16, hipStream_t stream) {
  for_form(p, bf16, [&](auto type, auto affine, auto sub) {
    constexpr int lds = Stage16<NT, MT>::bytes(decltype(affine)::value);
    const auto kernel = ring_kernel<decltype(type)::value, decltype(affine)::value, decltype(sub)::value, NT, MT>;
    set_lds_limit(kernel, lds);
    const int64_t across = (pieces_out(p.outputs) + 4 * NT - 1) / (4 * NT);
    hipLaunchKernelGGL(kernel, grid_of(across, most_tiles(p, 16 * MT)), dim3(256), lds, stream, p);
  });
}

// Which kernel.  With T tiles of 16 rows and 16 outputs, and pieces along the inputs, the streams want some thousand wavefronts and then
// as many outputs for one as possible: a fragment of x serves all of them.  Rows in some number share codes instead (ring, or tile
// where x is no whole 16-byte pieces).  The choice between streams and ring was measured in bfloat16 with groups of 128 and no offsets and
// decides for every form; the ring's tiles were measured in the forms named below.  us at T, pieces, in the order of the rule, KW x NW x NT (cold):
//                                             8x1x1  4x1x2  2x2x2  4x1x4  1x4x4   ring, rows x outputs:  16x128  32x128  32x256
//   256, 32   (1 row, 4096 x 4096)              6.9    9.2   12.0   11.1   23.0                            20.5    24.8    33.9
//   512, 32   (32 rows, the same)              14.0   10.8   15.0   12.6   27.6                            20.2    25.0    34.5
//   1024, 32  (64 rows)                        22.3   15.2   15.2   12.8   27.6                            20.6    25.0    34.4
//   4096, 32  (256 rows)                       72.7   43.3   42.2   29.9   28.6                            25.8    25.2    34.3
//   2048, 8   (16 rows, 8 experts, 1024 x 4096) 19.4  10.0    9.7   10.2   12.0                            10.6    11.6    14.4
//   7168, 8   (28 rows for 28 of 64 experts)   52.4   21.6   18.1   19.0   17.1                            15.3    17.1    18.9
//   16384, 8  (256 rows, 64 experts)            140   48.7   38.8   41.4   31.2                            32.2    38.4    39.7
//   4096, 32  (256 rows, 64 experts, 4096 x 1024) 55.8 34.2  35.6   30.6   31.3                            38.9    39.9    39.1
//   (512 rows over 8 experts, 1024 x 4096)      102   33.7   29.3   26.4   24.0                            18.3    17.3    19.4
// and with many rows (other times on other devices: 3 % apart)              ring, rows x outputs:     32x128  48x128  32x256  48x256
//   2048 rows over 64 experts, 1024 x 4096                                                            52      50      47      47
//   16384 rows over 64 experts, 1024 x 4096                                                           235     230     216     243
//   the same with groups of 64                                                                        245     225     222     223
//   the same with offsets                                                                             255     255     238     253
//   the same with offsets and groups of 64                                                            290     292     279     275
//   the same with groups of 32, and with offsets                                                      269, 363        273, 357
//   8192 rows over 64 experts, 4096 x 1024                                                            119     125     109     122
//   the same with offsets                                                                             130     129     119     135
//   512, 1000, 2048 rows, 4096 x 4096                                                                 33, 51, 92      36, 50, 86
// (64 x 256 needs more registers than two workgroups of a compute unit have: 270 us on the 16384 rows.)
enum ProductKernel : int {
  kStream8x1x1 = 0, kStream4x1x2, kStream4x1x4, kStream2x2x2, kStream1x4x4,   // few rows: KW x NW x NT
  kTile32x128, kRing32x256, kRing32x128, kRing16x128                          // many: rows x outputs
};
static ProductKernel product_kernel(int64_t rows, int64_t experts, int64_t inputs, int64_t outputs, bool whole) {
  const int64_t along = pieces_in(inputs), down = pieces_out(outputs);
  // as if the rows were spread evenly over the experts: where they really are only the device knows
  const int64_t hit = experts < rows ? experts : rows, each = (rows + hit - 1) / hit;
  const int64_t tiles = hit * ((each + 15) / 16) * down, across8 = (down + 7) / 8, across16 = (down + 15) / 16;
  if (along >= 24 ? each > 16 && tiles > 3000 : each >= 8 && tiles >= 1536) {
    if (!whole) return kTile32x128;
    if (each >= 24 && hit * ((each + 31) / 32) * across16 >= 512) return kRing32x256;
    if (each >= 12 && hit * ((each + 31) / 32) * across8 >= 256) return kRing32x128;
    return kRing16x128;
  }
  if (tiles <= 320) return kStream8x1x1;
  if (tiles <= 640) return kStream4x1x2;
  if (along >= 24) return kStream4x1x4;
  return tiles <= 4096 ? kStream2x2x2 : kStream1x4x4;
}
static int launch_product(const char* who, const Product4& p, int dtype, hipStream_t stream) {
  const bool bf16 = dtype == STK_BF16;
  if (most_tiles(p, 16) > (int64_t)65535 * 65535) return fail(STK_ERR_UNSUPPORTED, "%s: %lld rows", who, (long long)p.rows);
  switch (product_kernel(p.rows, p.experts, p.inputs, p.outputs, p.inputs % 8 == 0 && p.x_stride % 8 == 0 && aligned16(p.x))) {
    case kStream8x1x1: launch_stream<8, 1, 1>(p, bf16, stream); break;
    case kStream4x1x2: launch_stream<4, 1, 2>(p, bf16, stream); break;
    case kStream4x1x4: launch_stream<4, 1, 4>(p, bf16, stream); break;
    case kStream2x2x2: launch_stream<2, 2, 2>(p, bf16, stream); break;
    case kStream1x4x4: launch_stream<1, 4, 4>(p, bf16, stream); break;
    case kTile32x128: launch_tiles<2, 2>(p, bf16, stream); break;
    case kRing32x256: launch_ring<4, 2>(p, bf16, stream); break;
    case kRing32x128: launch_ring<2, 2>(p, bf16, stream); break;
    case kRing16x128: launch_ring<2, 1>(p, bf16, stream); break;
  }
  return STK_OK;
}

}  // namespace stk

using namespace stk;

extern "C" int64_t stk_4bit_packed_bytes(int64_t experts, int64_t inputs, int64_t outputs) {
  return experts < 1 || inputs < 1 || outputs < 1 ? 0 : experts * pieces_in(inputs) * pieces_out(outputs) * kPieceBytes;
}
extern "C" int64_t stk_4bit_scales(int64_t experts, int64_t inputs, int64_t outputs, int64_t group_size) {
  if (experts < 1 || inputs < 1 || outputs < 1 || group_size < 1) return 0;
  const int64_t group = group_within(inputs, group_size);
  return experts * scale_blocks(inputs, group) * groups_in_block(group) * pieces_out(outputs) * kPieceOutputs;
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
  hipLaunchKernelGGL(pack_codes_kernel, loop_grid(pieces, 8), dim3(512), 0, s, codes, inputs, outputs, pieces, static_cast<u32x4*>(packed));
  hipLaunchKernelGGL(pack_scales_kernel, loop_grid(count, 256), dim3(256), 0, s, static_cast<const uint16_t*>(scales), inputs, outputs, group_size, count,
                     static_cast<uint16_t*>(packed_scales));
  if (offsets)
    hipLaunchKernelGGL(pack_scales_kernel, loop_grid(count, 256), dim3(256), 0, s, static_cast<const uint16_t*>(offsets), inputs, outputs, group_size, count,
                       static_cast<uint16_t*>(packed_offsets));
  return check_launch(who);
}

extern "C" int stk_dequantize_4bit(const void* packed, const void* scales, const void* offsets, int64_t experts, int64_t inputs, int64_t outputs,
                                   int64_t group_size, void* out, int dtype, stk_stream_t stream) {
  const char* who = "stk_dequantize_4bit";
  if (int rc = weights_check(who, experts, inputs, outputs, group_size, dtype)) return rc;
  if (!packed || !scales || !out) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (!aligned16(packed)) return fail(STK_ERR_UNSUPPORTED, "%s: packed weights at a multiple of 16 bytes", who);
  const int64_t count = experts * inputs * outputs;
  const auto launch = [&](auto d) {
    typedef typename Value<d()>::stored T;
    hipLaunchKernelGGL((dequantize_kernel<d()>), loop_grid(count, 256), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const uint8_t*>(packed), static_cast<const T*>(scales), static_cast<const T*>(offsets), inputs, outputs, group_size, count,
                       static_cast<T*>(out));
  };
  if (dtype == STK_BF16) launch(std::integral_constant<int, STK_BF16>());
  else launch(std::integral_constant<int, STK_F16>());
  return check_launch(who);
}

extern "C" int stk_matmul_4bit(const void* x, int64_t rows, int64_t x_stride, const void* packed, const void* scales, const void* offsets, int64_t inputs,
                               int64_t outputs, int64_t group_size, void* out, int64_t out_stride, int activation, int dtype, stk_stream_t stream) {
  const char* who = "stk_matmul_4bit";
  Product4 p = {x, x_stride, rows, static_cast<const uint8_t*>(packed), scales, offsets, 1, inputs, outputs, group_size, nullptr, nullptr, 0,
                      out, out_stride, nullptr, activation};
  if (int rc = product_check(who, p, dtype)) return rc;
  if (rows == 0) return STK_OK;
  if (int rc = launch_product(who, p, dtype, static_cast<hipStream_t>(stream))) return rc;
  return check_launch(who);
}

extern "C" int stk_gather_matmul_4bit(const void* x, int64_t tokens, int64_t x_stride, const int32_t* indices, const int32_t* bins, int top_k, const void* packed,
                                      const void* scales, const void* offsets, int64_t experts, int64_t inputs, int64_t outputs, int64_t group_size, void* out,
                                      int64_t out_stride, int activation, int dtype, stk_stream_t stream) {
  const char* who = "stk_gather_matmul_4bit";
  if (tokens < 0 || top_k < 1 || tokens > INT32_MAX / top_k) return fail(STK_ERR_DIMS, "%s: %lld tokens, top_k %d", who, (long long)tokens, top_k);
  Product4 p = {x, x_stride, tokens * top_k, static_cast<const uint8_t*>(packed), scales, offsets, experts, inputs, outputs, group_size, indices, bins, top_k,
                      out, out_stride, nullptr, activation};
  if (int rc = product_check(who, p, dtype)) return rc;
  if (tokens == 0) return STK_OK;
  if (!indices || !bins) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (int rc = launch_product(who, p, dtype, static_cast<hipStream_t>(stream))) return rc;
  return check_launch(who);
}

extern "C" int stk_4bit_product_kernel(int64_t rows, int64_t experts, int64_t inputs, int64_t outputs, int whole_pieces) {
  return rows < 1 || experts < 1 || inputs < 1 || outputs < 1 ? -1 : (int)product_kernel(rows, experts, inputs, outputs, whole_pieces != 0);
}

extern "C" size_t stk_matmul_4bit_scatter_workspace_bytes(int64_t slots, int64_t outputs) {
  return slots < 1 || outputs < 1 ? 0 : (size_t)(slots * outputs) * sizeof(float);
}

extern "C" int stk_matmul_4bit_scatter(const void* x, int64_t x_stride, const int32_t* indices, const int32_t* bins, int top_k, int64_t tokens,
                                       const float* weights, const void* packed, const void* scales, const void* offsets, int64_t experts, int64_t inputs,
                                       int64_t outputs, int64_t group_size, void* out, int64_t out_stride, int dtype, void* workspace, size_t workspace_bytes,
                                       stk_stream_t stream) {
  const char* who = "stk_matmul_4bit_scatter";
  if (tokens < 0 || top_k < 1 || tokens > INT32_MAX / top_k) return fail(STK_ERR_DIMS, "%s: %lld tokens, top_k %d", who, (long long)tokens, top_k);
  const int64_t slots = tokens * top_k;
  Product4 p = {x, x_stride, slots, static_cast<const uint8_t*>(packed), scales, offsets, experts, inputs, outputs, group_size, indices, bins, 0,
                      nullptr, 0, static_cast<float*>(workspace), 0};
  if (slots > 0 && (!workspace || workspace_bytes < stk_matmul_4bit_scatter_workspace_bytes(slots, outputs)))
    return fail(STK_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", who, stk_matmul_4bit_scatter_workspace_bytes(slots, outputs));
  if (int rc = product_check(who, p, dtype)) return rc;
  if (tokens == 0) return STK_OK;
  if (!indices || !bins || !out || out_stride < outputs) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (int rc = launch_product(who, p, dtype, s)) return rc;
  const dim3 grid = loop_grid(tokens * ((outputs + 3) / 4), 256);
  const auto combine = dtype == STK_BF16 ? combine_kernel<true> : combine_kernel<false>;
  hipLaunchKernelGGL(combine, grid, dim3(256), 0, s, static_cast<const float*>(workspace), weights, tokens, top_k, outputs, static_cast<uint16_t*>(out), out_stride);
  return check_launch(who);
}
