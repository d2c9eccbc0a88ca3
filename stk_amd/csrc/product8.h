// What the kernels of the products with 8-bit floating-point weights have in common (product8.hip, product8_wide.hip).
#pragma once
#include <type_traits>

#include "common.h"
#include "fp8.h"
#include "gemm_core.h"
#include "values.h"
#include "wave_scan.h"

namespace stk {

bool sizes8(int64_t lines, int64_t size);
int quantize_rows8(const char* who, const void* x, int64_t rows, int64_t size, int64_t stride, int dtype, uint8_t* codes, uint8_t* exponents, const int32_t* indices, int top_k, hipStream_t stream);

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// What a product is told.  Without routing: bins null, one expert.  With: row p of the sorted slots belongs to the first expert whose bin
// ends behind p, and to the slot indices[p].
struct Product8 {
  const void* x;                             // 16-bit rows, ...
  int64_t x_stride;
  const uint8_t *codes, *exponents;          // ... or quantised ones
  int64_t x_rows, rows;                      // rows there are (of quantised ones: lines); those multiplied (slots)
  const uint8_t* packed;
  const void* scales;
  int64_t experts, inputs, outputs;
  const int32_t *indices, *bins;
  int top_k;                                 // 16-bit rows gathered: row p reads token indices[p] / top_k; 0, and quantised ones: row p itself
  void* out;                                 // 16-bit rows in the order of the rows, or with `by_slot` of the slots, times `weights` of these, ...
  int64_t out_stride;
  bool by_slot;
  const float* weights;
  float* sums;                               // ... or, where given, fp32 rows [slot][outputs]
  int activation;
  bool bf16, zero_behind;                    // zero_behind: rows behind the last bin become zeros
};

// Which rows a tile of up to R rows of one expert is: tiles are numbered expert by expert, an expert of c rows has ceil(c / R).
struct RowTile8 {
  int expert, first, rows;   // (rows 0: no such tile, but the first-th behind them all)
};
template <int R, class Bins>
__device__ __forceinline__ RowTile8 row_tile8(const Product8& p, Bins bins, int tile, int lane) {
  int before = 0;
  for (int e0 = 0; e0 < p.experts; e0 += 64) {
    const int e = e0 + lane;
    const bool is = e < p.experts;
    // (bins that do not ascend or leave the rows are kept inside them)
    const int hi = is ? min(max((int)bins[e], 0), (int)p.rows) : 0, lo = is && e > 0 ? min(max((int)bins[e - 1], 0), (int)p.rows) : 0;
    const int count = hi > lo ? hi - lo : 0, tiles = (count + R - 1) / R, upto = before + wave_inclusive_scan(tiles, lane);
    const uint64_t mine = __ballot(upto > tile);
    if (mine) {
      const int at = __builtin_ctzll(mine);
      const int inside = tile - __builtin_amdgcn_readlane(upto - tiles, at), c = __builtin_amdgcn_readlane(count, at);
      return {e0 + at, __builtin_amdgcn_readlane(lo, at) + inside * R, min(c - inside * R, R)};
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return {0, tile - before, 0};
}
template <int R>
__device__ __forceinline__ RowTile8 row_tile8(const Product8& p, int tile, int lane) {
  if (p.bins) return row_tile8<R>(p, p.bins, tile, lane);
  const int64_t first = (int64_t)tile * R, left = p.rows - first;
  return {0, (int)first, left <= 0 ? 0 : left < R ? (int)left : R};
}

__device__ __forceinline__ f32x4_t multiply8(i32x8_t weights, i32x8_t rows, f32x4_t sum, int weight_scale, int row_scale) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(weights, rows, sum, 0, 0, 0, weight_scale, 0, row_scale);
}

// total = activation(total); a NaN stays one (relu by the comparison from the other side would make 0 of it).
template <int KIND, int N>
__device__ __forceinline__ void activate_each8(f32x4_t (&total)[N]) {
#pragma unroll
  for (int n = 0; n < N; n++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float v = total[n][i];
      total[n][i] = KIND == kRelu ? (v <= 0.f ? 0.f : v) : activate<KIND>(v);
    }
}
template <int N>
__device__ __forceinline__ void activate_sums8(f32x4_t (&total)[N], int kind) {
  switch (kind) {
    case kRelu: activate_each8<kRelu>(total); break;
    case kGeluTanh: activate_each8<kGeluTanh>(total); break;
    case kGeluErf: activate_each8<kGeluErf>(total); break;
    case kSilu: activate_each8<kSilu>(total); break;
    default: break;
  }
}
__device__ __forceinline__ uint32_t pack8(float a, float b, bool bf16) { return bf16 ? pack2<true>(a, b) : pack2<false>(a, b); }

// Where row r of a tile is stored, or false.
__device__ __forceinline__ bool place_of_row8(const Product8& p, const RowTile8& t, int r, int64_t& to, float& by) {
  if (r >= t.rows) return false;
  to = t.first + r, by = 1.f;
  if (p.sums || p.by_slot) {
    to = p.indices[to];
    if (to < 0 || to >= p.rows) return false;
    if (!p.sums && p.weights) by = p.weights[to];
  }
  return true;
}
// 4 N neighbouring outputs of a row from `first` on.
template <int N>
__device__ __forceinline__ void store8(const Product8& p, int64_t to, float by, int64_t first, const f32x4_t (&v)[N]) {
  const int here = (int)min(p.outputs - first, (int64_t)(4 * N));
  if (here <= 0) return;
  if (p.sums) {
    float* at = p.sums + to * p.outputs + first;
    if (here == 4 * N) {
#pragma unroll
      for (int n = 0; n < N; n++) *reinterpret_cast<QuadAt4*>(at + 4 * n) = __builtin_bit_cast(Quad, v[n]);
    } else {
#pragma unroll
      for (int i = 0; i < 4 * N; i++)
        if (i < here) at[i] = v[i / 4][i % 4];
    }
    return;
  }
  uint32_t two[2 * N];
#pragma unroll
  for (int i = 0; i < 2 * N; i++) two[i] = pack8(v[i / 2][2 * (i & 1)] * by, v[i / 2][2 * (i & 1) + 1] * by, p.bf16);
  uint16_t* at = static_cast<uint16_t*>(p.out) + to * p.out_stride + first;
  if (here == 4 * N) {
    if constexpr (N == 1) *reinterpret_cast<PairAt2*>(at) = PairAt2{two[0], two[1]};
    else *reinterpret_cast<QuadAt2*>(at) = QuadAt2{two[0], two[1], two[2], two[3]};
  } else {
#pragma unroll
    for (int i = 0; i < 4 * N; i++)
      if (i < here) at[i] = (uint16_t)(two[i / 2] >> (16 * (i & 1)));
  }
}
// The sums of a row's lane of the four pieces of 64 outputs, whose first is `first`.
__device__ __forceinline__ void store_pieces8(const Product8& p, int64_t to, float by, int64_t first, int quarter, const f32x4_t (&v)[4]) {
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const f32x4_t two[2] = {v[2 * u], v[2 * u + 1]};
    store8<2>(p, to, by, first + 32 * u + 8 * quarter, two);
  }
}

// Rows of a tile in LDS: eight of 128 bytes a transfer (1 KiB), whole lines of memory.  The 16-byte chunk c of row r is at slot c ^ (r / 2 % 8), which
// spreads what the 16 rows of a fragment read at a time over all banks.  What lane l of a transfer takes is a matter of its address:
__device__ __forceinline__ int row_of_transfer8(int lane) { return lane >> 3; }
__device__ __forceinline__ int chunk_of_transfer8(int row, int lane) { return (lane & 7) ^ ((row >> 1) & 7); }
// The first 16 bytes of a lane of a fragment of 16 rows; the other 16 are at this ^ 64.
__device__ __forceinline__ int in_fragment8(int lane) { return (lane & 15) * kBlock8 + (((lane >> 4) ^ ((lane >> 1) & 7)) << 4); }

// What the gradient of the weights is told beside: dw[e][i][o] = the sum over the rows r of expert e of xq[r][i] gq[r][o].  codes: the columns of x
// (a line for each input, row blocks along it), packed: those of g as pieces; outputs, out: those of dw, x_rows its inputs, `inputs` the rows.
// Otherwise a product of rows.
enum What8 : int { kRows8 = 0, kGradient8 = 1 };

// 4 bytes per lane from any addresses into the LDS bytes from lds_base on, lane after lane.
__device__ __forceinline__ void dma4_from(const void* from, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(uniform((int)lds_base)), "v"((uint64_t)from) : "memory", "m0");
}

// 16, or 4, bytes from `offset` + `start` on in a buffer: everything from an address on, as far as 32 bits reach.  (The wait: a scalar register that the VALU
// wrote may be read by a memory access five states later, and the compiler does not see that this is one.)
__device__ __forceinline__ u32x4 buffer8(const uint8_t* from) {
  const uint64_t a = (uint64_t)uniform_global(from);
  return u32x4{(uint32_t)a, (uint32_t)(a >> 32) & 0xffffu, 0xffffffffu, 0x00020000u};
}
template <int BYTES>
__device__ __forceinline__ void transfer8(u32x4 buffer, uint32_t offset, uint32_t start, uint32_t to) {
  if constexpr (BYTES == 16) asm volatile("s_mov_b32 m0, %3\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %0, %2 offen lds" : : "s"(buffer), "v"(offset), "s"(start), "s"(to) : "memory", "m0");
  else asm volatile("s_mov_b32 m0, %3\n\ts_nop 3\n\tbuffer_load_dword %1, %0, %2 offen lds" : : "s"(buffer), "v"(offset), "s"(start), "s"(to) : "memory", "m0");
}

// Tiles of 256 x 256 with power-of-two scales (product8_wide.hip).
template <int WHAT>
int launch_wide8(const char* who, const Product8& p, hipStream_t stream);

}  // namespace stk
