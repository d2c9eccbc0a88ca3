// Products of many rows with 8-bit weights that have power-of-two scales, and the gradient of such weights: tiles of 256 x 256.
//
// Four wavefronts, one on each SIMD, have 128 x 128 sums each, which fill the accumulation registers: 32 KiB that a wavefront reads from LDS feed 64 matrix
// instructions.  A step is one block of 128 inputs, 32 KiB of rows and 32 KiB of weights in one of two stages of LDS, which are filled without
// registers.  A wavefront keeps its weights of a step in registers, where the next step's replace them one by one behind their last use, and takes
// rows two fragments of 16 ahead, so that the matrix instructions wait for neither.  A wavefront alone on its SIMD issues an instruction every four
// or five clocks and a matrix instruction takes 32, so what stands between two of them is at most a transfer (two instructions) and the accesses
// to LDS.  Two barriers a step say that a part of a stage has been read by everybody and may be filled, and that one has arrived; between its
// transfer and its first use lies a step or more, and what is waited for is counted, never everything.
//
// Workgroups stay: each takes tile after tile, and the transfers of the next tile's first blocks run during the last steps of one and while its sums
// are stored.
//
// Measured (MI355X): the gradient of 4096 x 4096 weights from 16384 rows 217 - 237 us on different machines, 2.3 - 2.5 PFLOP/s, where the library's product without
// block scales takes 230; the matrix units are busy for 59 % of the clocks, which fall to 2.1 GHz under them (alone, out of registers, they reach
// 3.5 PFLOP/s at 1.7).  With the transfers cut off a step takes two thirds of that: what bounds it is their way through the caches into LDS, 66 KiB
// a step and unit, 9 TB/s.  The product of the same sizes, four tiles for each workgroup, takes 243 - 270 us: all of them store at the same time.  With
// eight blocks of inputs (64 experts of 1024 x 4096, 256 rows each) storing and applying gelu takes a third of 175 us.
#include <type_traits>

#include "common.h"
#include "fp8.h"
#include "gemm_core.h"
#include "product8.h"
#include "wave_scan.h"

namespace stk {

constexpr int kWideTile = 256, kWideSide = kWideTile * kBlock8, kWideExponents = 2 * kWideTile * 4, kWideBins = 2048;
constexpr int kWideBytes = 4 * kWideSide + 2 * kWideExponents + kWideBins * 4;

// sum += weights rows, the sum in accumulation registers.  As text, so that a sum stays in its registers: left to the compiler the 256 of them move
// about and spill.  The compiler does not see into the text, so that waits for what may stand directly in front of it are part of it: two states between
// a VALU write and a matrix instruction that reads the register, five between a VALU write of a scalar register (it may come back from a
// spilled one) and a memory access that reads it, one between m0 and a transfer.  settle8 stands behind writes of the execution mask, and finish8 between
// matrix instructions and whatever reads their sums.
#define STK_SUM8 "v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]"
#define STK_SUM8_OPERANDS "v"(weights), "v"(rows), "v"(weight_scale), "v"(row_scale)
__device__ __forceinline__ void accumulate8(f32x4_t& sum, const i32x8_t& weights, const i32x8_t& rows, int weight_scale, int row_scale) {
  asm volatile("s_nop 1\n\t" STK_SUM8 : "+a"(sum) : STK_SUM8_OPERANDS);
}
// The same with a transfer into the LDS bytes from `to` + AT on: 16 or 4 bytes of each lane, from `offset` + `start` on in a buffer.
template <int AT, int BYTES>
__device__ __forceinline__ void accumulate8_fetch(f32x4_t& sum, const i32x8_t& weights, const i32x8_t& rows, int weight_scale, int row_scale, u32x4 buffer, uint32_t offset,
                                                  uint32_t start, uint32_t to) {
  if constexpr (BYTES == 16)
    asm volatile("s_add_i32 m0, %8, %9\n\ts_nop 2\n\t" STK_SUM8 "\n\tbuffer_load_dwordx4 %6, %5, %7 offen lds"
                 : "+a"(sum) : STK_SUM8_OPERANDS, "s"(buffer), "v"(offset), "s"(start), "s"(to), "n"(AT) : "memory", "m0", "scc");
  else
    asm volatile("s_add_i32 m0, %8, %9\n\ts_nop 2\n\t" STK_SUM8 "\n\tbuffer_load_dword %6, %5, %7 offen lds"
                 : "+a"(sum) : STK_SUM8_OPERANDS, "s"(buffer), "v"(offset), "s"(start), "s"(to), "n"(AT) : "memory", "m0", "scc");
}
__device__ __forceinline__ void settle8() { asm volatile("s_nop 4"); }
__device__ __forceinline__ void finish8() { asm volatile("s_nop 15\n\ts_nop 15"); }
// lgkmcnt(0), said so that the compiler knows: after a read through the scalar unit it would wait for all of LDS at the next step's first fragment.
__device__ __forceinline__ void scalars_read8() { __builtin_amdgcn_s_waitcnt(0xc07f); }
// Eight results to the buffer's byte `offset` + AT.  (As text, so that it is one instruction and the compiler does not wait for it.)
template <int AT>
__device__ __forceinline__ void store_eight8(u32x4 eight, uint32_t offset, u32x4 buffer) {
  asm volatile("s_nop 4\n\tbuffer_store_dwordx4 %0, %1, %2, 0 offen offset:%3\n\ts_nop 0" : : "v"(eight), "v"(offset), "s"(buffer), "n"(AT) : "memory");
}

template <int WHAT, int ACTIVATION>
__global__ __launch_bounds__(256, 1) void wide8_kernel(Product8 p, int row_tiles, int col_tiles) {
  extern __shared__ char smem[];   // rows of two stages, weights of two, exponents of two (of the rows, of the weights), bins
  constexpr int kExponentsAt = 4 * kWideSide, kBinsAt = kExponentsAt + 2 * kWideExponents;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
  const int row = lane & 15, quarter = lane >> 4;
  const int blocks = (int)blocks8(p.inputs), exponent_stride = (int)exponent_stride8(p.inputs);
  const int64_t places = padded_lines8(p.outputs);
  const uint32_t row_lines = (uint32_t)p.x_rows * 4, col_lines = (uint32_t)places * 4;   // bytes of the exponents of four blocks
  const uint32_t lds = (uint32_t)(uintptr_t)(STK_LDS char*)smem;
  typedef const STK_LDS int* lds_ints;
  const lds_ints near_bins = (lds_ints)(STK_LDS char*)(smem + kBinsAt);
  const bool near = p.bins && p.experts <= kWideBins;
  if (near) {
    for (int e = threadIdx.x; e < p.experts; e += 256) reinterpret_cast<int*>(smem + kBinsAt)[e] = p.bins[e];
    __syncthreads();
  }
  const auto rows_of = [&](int tile) {
    RowTile8 t = near ? row_tile8<kWideTile>(p, near_bins, tile, lane) : row_tile8<kWideTile>(p, tile, lane);
    t.expert = uniform(t.expert), t.first = uniform(t.first), t.rows = uniform(t.rows);
    return t;
  };
  // how many tiles there are: an expert's only where it has rows
  if (WHAT == kRows8 && p.bins) row_tiles = INT32_MAX - rows_of(INT32_MAX).first;
  const int tiles = row_tiles * col_tiles * (WHAT == kGradient8 ? (int)p.experts : 1);
  // Each compute die has a stretch of the tiles, its workgroups neighbours, which share rows or weights: four row tiles by all columns, column after column.
  const int die = blockIdx.x & 7, dies = min(8, (int)gridDim.x), turn = ((int)gridDim.x - die + 7) >> 3;
  const int stretch_end = (int)((int64_t)tiles * (die + 1) / dies);
  int mine = (int)((int64_t)tiles * die / dies) + (int)(blockIdx.x >> 3);
  struct Work {
    RowTile8 t;
    int col_tile, begin, end, at;
  };
  const auto work_of = [&](int at) {
    Work w;
    w.at = at;
    int expert = 0;
    if constexpr (WHAT == kGradient8) expert = at / (row_tiles * col_tiles), at %= row_tiles * col_tiles;
    constexpr int kPanel = 4;
    const int panel = at / (kPanel * col_tiles), inside = at % (kPanel * col_tiles), high = min(kPanel, row_tiles - panel * kPanel);
    const int row_tile = panel * kPanel + inside % high;
    w.col_tile = inside / high, w.begin = 0, w.end = blocks;
    if constexpr (WHAT == kGradient8) {
      w.t = {expert, row_tile * kWideTile, (int)min((int64_t)kWideTile, p.x_rows - (int64_t)row_tile * kWideTile)};
      if (p.bins) {
        const auto bin = [&](int e) { return near ? uniform(near_bins[e]) : const_ints(p.bins)[e]; };
        w.end = min(max(bin(expert) / kBlock8, 0), blocks);
        w.begin = expert > 0 ? min(max(bin(expert - 1) / kBlock8, 0), w.end) : 0;
      }
    } else w.t = rows_of(row_tile);
    return w;
  };

  // ------------------------------------------------------------ transfers, two steps ahead: 1 KiB, or 256 bytes of exponents, each
  Work next = {};            // the tile whose transfers come next
  int next_block = 0;        // ... and the block
  uint32_t row_offset[8] = {}, col_offset[8] = {}, row_exponents = 0, col_exponents = 0;
  u32x4 row_buffer = buffer8(p.codes), col_buffer = buffer8(p.packed), row_exponent_buffer = buffer8(p.exponents), col_exponent_buffer = buffer8(static_cast<const uint8_t*>(p.scales));
  const auto aim = [&](int at) {   // at this tile, or the next one that has any
    for (; at < stretch_end; at += turn) {
      next = work_of(at);
      if (next.begin < next.end) break;
    }
    if (at >= stretch_end) {   // nothing is left: transfers of nothing, from where the last ones were
      next.at = stretch_end;
      row_buffer[2] = col_buffer[2] = row_exponent_buffer[2] = col_exponent_buffer[2] = 0;
      return;
    }
    next_block = next.begin;
    const RowTile8 t = next.t;
    const int64_t line = row_stride8(p.inputs);
    const auto source = [&](int r) { return (uint32_t)(r < t.rows ? r : 0); };   // of the tile
    const int64_t matrix = WHAT == kGradient8 ? 0 : t.expert, col0 = (int64_t)next.col_tile * kWideTile;
#pragma unroll
    for (int j = 0; j < 8; j++) {   // numbers wave, wave + 4, ...: eight rows, half a piece
      const int r = 8 * (wave + 4 * j) + row_of_transfer8(lane);
      row_offset[j] = source(r) * (uint32_t)line + 16 * chunk_of_transfer8(r, lane);
      const int64_t group = min(col0 + 64 * (j >> 1), places - 64) - col0;
      col_offset[j] = (uint32_t)(group / 64 * blocks * (4 * kPieceBytes8)) + (wave + 4 * (j & 1)) * 1024 + lane * 16;
    }
    row_exponents = source(64 * wave + lane) * 4;
    col_exponents = (uint32_t)(min(col0 + 64 * wave + lane, places - 1) - col0) * 4;
    row_buffer = buffer8(p.codes + t.first * line), row_exponent_buffer = buffer8(p.exponents + (int64_t)t.first * 4);
    col_buffer = buffer8(p.packed + (matrix * (places / kPieceLines8) * blocks + piece8(col0 / kPieceLines8, 0, blocks)) * kPieceBytes8);
    col_exponent_buffer = buffer8(static_cast<const uint8_t*>(p.scales) + matrix * places * exponent_stride + col0 * 4);
  };
  const auto fetched = [&]() {   // everything of a block
    if (next.at < stretch_end && ++next_block == next.end) {
      next_block--;
      aim(next.at + turn);
      scalars_read8();
    }
  };
  // Transfers of a wavefront: weights, exponents and upper rows of a block during a step, its lower rows at the start of the next.
  constexpr int kColsOf = 8, kExponentsOf = 2, kUpperOf = 4, kLowerOf = 4, kFirstOf = kColsOf + kExponentsOf + kUpperOf;
  constexpr uint32_t kOutRange = 1u << 31;

  // ------------------------------------------------------------ one step
  f32x4_t total[8][8];
  i32x8_t weights[8], values[4];
  int row_scale[8], col_scale[8];
  int stage = 0;
  const auto fragment = [&](const char* first, const char* second) {
    i32x8_t f;
    const u32x4 a = *reinterpret_cast<const u32x4*>(first), b = *reinterpret_cast<const u32x4*>(second);
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = (int)a[i], f[4 + i] = (int)b[i];
    return f;
  };
  const int in_fragment = in_fragment8(lane) + wm * kPieceBytes8;
  const auto row_fragment = [&](int of, int m) {
    const char* from = smem + of * kWideSide + 2 * m * kPieceBytes8;
    return fragment(from + in_fragment, from + (in_fragment ^ 64));
  };
  const auto col_fragment = [&](int of, int n) {
    const char* from = smem + 2 * kWideSide + of * kWideSide + lane * 16 + wn * 8 * kPieceBytes8 + n * kPieceBytes8;
    return fragment(from, from + 1024);
  };
  const auto read_scales = [&](int of, int side) {   // as they are: of four blocks
    const int* from = reinterpret_cast<const int*>(smem + kExponentsAt + of * kWideExponents) + row;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (side == 0) row_scale[i] = (from + 16 * wm)[32 * i];
      else col_scale[i] = (from + kWideTile + 128 * wn)[16 * i];
    }
  };
  int stores = 0;   // by at least how many instructions the sums were stored in front of a step (0, 16 or 32)
  const auto step = [&](int block) {
    int by_row[8], by_col[8];
#pragma unroll
    for (int i = 0; i < 8; i++) by_row[i] = row_scale[i] >> (8 * (block & 3)), by_col[i] = col_scale[i] >> (8 * (block & 3));
    settle8();
    uint32_t to_rows = lds + (stage ^ 1) * kWideSide + wave * 1024, start = next_block * kBlock8;   // of the next step's lower rows
    uint32_t to_cols = 0, to_exponents = 0, start_cols = 0, start_row_exponents = 0, start_col_exponents = 0;
    static_for<4>([&](auto pair) {
      constexpr int P = decltype(pair)::value;
      // 1: everybody has read the upper rows and, in the step before, the weights and exponents; the lower rows are there.
      // 3: everybody has read the lower rows; the next weights, exponents and upper rows are there.
      // Younger than these are as many transfers each time, and in the first step of a tile the stores of the last one, which need not have ended.
      if constexpr (P == 1 || P == 3) {
        constexpr int kYounger = P == 1 ? kFirstOf + kLowerOf : kLowerOf + kColsOf + kExponentsOf;
        if (stores == 32) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(kYounger + 32) : "memory");
        else if (stores == 16) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(kYounger + 16) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(kYounger) : "memory");
      }
      static_for<8>([&](auto at) {
        constexpr int N = decltype(at)::value, M = 2 * P;
        const i32x8_t &upper = values[2 * (P & 1)], &lower = values[2 * (P & 1) + 1];
        // (as many transfers to each pair of fragments as the next has: more at a time wait for each other)
        constexpr int kCol = P == 1 && N < 5 ? N : P == 2 && N < 3 ? 5 + N : -1, kRow = P == 3 && N >= 4 ? N - 4 : P == 0 && N >= 4 ? N : -1;
        if constexpr (kCol >= 0)
          accumulate8_fetch<4096 * kCol, 16>(total[M][N], weights[N], upper, by_col[N], by_row[M], col_buffer, col_offset[kCol], start_cols, to_cols);
        else if constexpr (kRow >= 0)
          accumulate8_fetch<4096 * kRow, 16>(total[M][N], weights[N], upper, by_col[N], by_row[M], row_buffer, row_offset[kRow], start, to_rows);
        else if constexpr (P == 2 && (N == 4 || N == 6))
          accumulate8_fetch<N / 6 * kWideTile * 4, 4>(total[M][N], weights[N], upper, by_col[N], by_row[M], N == 6 ? col_exponent_buffer : row_exponent_buffer,
                                                      N == 6 ? col_exponents : row_exponents, N == 6 ? start_col_exponents : start_row_exponents, to_exponents);
        else accumulate8(total[M][N], weights[N], upper, by_col[N], by_row[M]);
        if constexpr (N < 2) values[2 * (~P & 1) + N] = P < 3 ? row_fragment(stage, M + 2 + N) : row_fragment(stage ^ 1, N);
        accumulate8(total[M + 1][N], weights[N], lower, by_col[N], by_row[M + 1]);
        if constexpr (P == 3) {
          weights[N] = col_fragment(stage ^ 1, N);
          if constexpr (N == 2 || N == 3) read_scales(stage ^ 1, N - 2);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (P == 0) {
        fetched();
        to_rows = lds + stage * kWideSide + wave * 1024, to_cols = to_rows + 2 * kWideSide, to_exponents = lds + kExponentsAt + stage * kWideExponents + wave * 256;
        start = next_block * kBlock8, start_cols = next_block * (4 * kPieceBytes8);
        start_row_exponents = (next_block >> 2) * row_lines, start_col_exponents = (next_block >> 2) * col_lines;
      }
    });
    stage ^= 1, stores = 0;
  };

  aim(mine);
  for (int s = 0; s < 2; s++) {
    const uint32_t to = lds + s * kWideSide + wave * 1024, to_exponents = lds + kExponentsAt + s * kWideExponents + wave * 256;
#pragma unroll
    for (int j = 0; j < 8; j++) transfer8<16>(col_buffer, col_offset[j], next_block * (4 * kPieceBytes8), to + 2 * kWideSide + 4096 * j);
    transfer8<4>(row_exponent_buffer, row_exponents, (next_block >> 2) * row_lines, to_exponents);
    transfer8<4>(col_exponent_buffer, col_exponents, (next_block >> 2) * col_lines, to_exponents + kWideTile * 4);
#pragma unroll
    for (int j = 0; j < 4; j++) transfer8<16>(row_buffer, row_offset[j], next_block * kBlock8, to + 4096 * j);
    if (s == 1) break;   // (the lower rows of the second block: in the first step)
#pragma unroll
    for (int j = 4; j < 8; j++) transfer8<16>(row_buffer, row_offset[j], next_block * kBlock8, to + 4096 * j);
    fetched();
  }
  wait_vmcnt<kLowerOf + kFirstOf>();
  __syncthreads();
#pragma unroll
  for (int n = 0; n < 8; n++) weights[n] = col_fragment(0, n);
  read_scales(0, 0), read_scales(0, 1);
  values[0] = row_fragment(0, 0), values[1] = row_fragment(0, 1);
  const bool even = !p.sums && !p.by_slot && (reinterpret_cast<uintptr_t>(p.out) & 3) == 0 && p.out_stride % 2 == 0 && p.out_stride <= 1 << 22;   // (256 rows of 8 MiB are kOutRange)
  for (; mine < stretch_end; mine += turn) {
    const Work w = mine == next.at ? next : work_of(mine);
#pragma unroll
    for (int m = 0; m < 8; m++)
#pragma unroll
      for (int n = 0; n < 8; n++) total[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    scalars_read8();
    for (int block = w.begin; block < w.end; block++) step(block);
    finish8();
    Product8 to_where = p;
    if constexpr (WHAT == kGradient8) to_where.out = static_cast<uint16_t*>(p.out) + (int64_t)w.t.expert * p.x_rows * p.out_stride;
    const int64_t first = (int64_t)w.col_tile * kWideTile + 128 * wn;
    // Whole lines of 64 outputs go out by 32-bit offsets, rows that are not there by one that is out of range, four instructions for 16 rows.
    const bool whole = first + 128 <= p.outputs && even;
    uint16_t* rows_out = static_cast<uint16_t*>(to_where.out) + (int64_t)w.t.first * p.out_stride + first;
    u32x4 out_buffer = buffer8(reinterpret_cast<const uint8_t*>(whole ? rows_out : static_cast<uint16_t*>(p.out)));
    out_buffer[2] = kOutRange;
#pragma unroll
    for (int m = 0; m < 8; m++) {
#pragma unroll
      for (int n = 0; n < 8; n++) asm volatile("" : "+a"(total[m][n]));   // (16 rows at a time leave the accumulation registers)
      const int r = 16 * (2 * m + wm) + row;
      if (r - row >= w.t.rows) break;   // (none of the 16)
      f32x4_t sums[2][4];
#pragma unroll
      for (int g = 0; g < 2; g++) {
#pragma unroll
        for (int n = 0; n < 4; n++) sums[g][n] = total[m][4 * g + n];
        if constexpr (ACTIVATION != kNoActivation) activate_each8<ACTIVATION>(sums[g]);
      }
      if (whole) {
        const uint32_t offset = r < w.t.rows ? (uint32_t)(r * (int)p.out_stride + 8 * quarter) * 2 : kOutRange;
        const auto store = [&](auto at) {
          constexpr int I = decltype(at)::value;
          const f32x4_t &a = sums[I >> 1][2 * (I & 1)], &b = sums[I >> 1][2 * (I & 1) + 1];
          const u32x4 eight = {pack8(a[0], a[1], p.bf16), pack8(a[2], a[3], p.bf16), pack8(b[0], b[1], p.bf16), pack8(b[2], b[3], p.bf16)};
          store_eight8<64 * I>(eight, offset, out_buffer);
        };
        static_for<4>(store);
      } else {
        int64_t to;
        float by;
        if (place_of_row8(to_where, w.t, r, to, by)) store_pieces8(to_where, to, by, first, quarter, sums[0]), store_pieces8(to_where, to, by, first + 64, quarter, sums[1]);
      }
    }
    stores = !whole ? 0 : w.t.rows > 16 * (14 + wm) ? 32 : w.t.rows > 16 * (6 + wm) ? 16 : 0;   // (four for every 16 rows)
  }
  wait_vmcnt<0>();
  // rows behind the last expert's
  if (WHAT == kRows8 && p.zero_behind && p.bins) {
    const int64_t begin = min(max(p.bins[p.experts - 1], 0), (int)p.rows);
    for (int64_t r = begin + blockIdx.x; r < p.rows; r += gridDim.x)
      for (int64_t i = threadIdx.x; i < p.outputs; i += 256) static_cast<uint16_t*>(p.out)[r * p.out_stride + i] = 0;
  }
}

template <int WHAT>
int launch_wide8(const char* who, const Product8& p, hipStream_t stream) {
  const int64_t row_tiles = ((WHAT == kGradient8 ? p.x_rows : p.rows) + kWideTile - 1) / kWideTile, col_tiles = (p.outputs + kWideTile - 1) / kWideTile;
  // with routing each expert may add a tile that is not full
  const int64_t most = WHAT == kGradient8 ? row_tiles * p.experts : p.bins ? std::min(p.rows, row_tiles + p.experts - 1) : row_tiles;
  if (most > INT32_MAX / col_tiles) return fail(STK_ERR_UNSUPPORTED, "%s: too many tiles", who);
  const int64_t tiles = most * col_tiles;
  const dim3 grid((unsigned)std::min(tiles, (int64_t)compute_units()));
  const auto launch = [&](auto activation) {
    const auto kernel = wide8_kernel<WHAT, decltype(activation)::value>;
    set_lds_limit(kernel, kWideBytes);
    hipLaunchKernelGGL(kernel, grid, dim3(256), kWideBytes, stream, p, (int)row_tiles, (int)col_tiles);
  };
  if constexpr (WHAT == kGradient8) launch(std::integral_constant<int, kNoActivation>());
  else {
    switch (p.activation) {
      case kRelu: launch(std::integral_constant<int, kRelu>()); break;
      case kGeluTanh: launch(std::integral_constant<int, kGeluTanh>()); break;
      case kSilu: launch(std::integral_constant<int, kSilu>()); break;
      default: launch(std::integral_constant<int, kNoActivation>());
    }
  }
  return check_launch(who);
}
template int launch_wide8<kRows8>(const char*, const Product8&, hipStream_t);
template int launch_wide8<kGradient8>(const char*, const Product8&, hipStream_t);

}  // namespace stk
