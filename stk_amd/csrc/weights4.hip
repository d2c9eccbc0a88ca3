// Products with 4-bit weights and group scales, and the weights' own formats.
//   weight of input i and output o = scale[i / group][o] * (code - 8)      or      scale * code + offset[i / group][o]
#include <type_traits>

#include "common.h"
#include "gemm_core.h"
#include "values.h"
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

__device__ __forceinline__ int expert_of(const int32_t* bins, int experts, int64_t row) {
  int lo = 0, hi = experts - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (bins[mid] > row) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// A thread per row and output.
template <int DTYPE>
__global__ __launch_bounds__(256) void product_kernel(Product4 p) {
  typedef typename Value<DTYPE>::stored T;
  const int64_t o = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (o >= p.outputs) return;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const int64_t slot = p.indices ? p.indices[row] : row, e = p.bins ? expert_of(p.bins, (int)p.experts, row) : 0;
    if (slot < 0 || slot >= p.rows) continue;
    const T* x = static_cast<const T*>(p.x) + (p.top_k > 0 ? slot / p.top_k : row) * p.x_stride;
    float sum = 0.f;
    for (int64_t i = 0; i < p.inputs; i++)
      sum += Value<DTYPE>::widen(x[i]) * weight_of<DTYPE>(p.packed, static_cast<const T*>(p.scales), static_cast<const T*>(p.offsets), e, i, o,
                                                          pieces_in(p.inputs), pieces_out(p.outputs), p.group, groups_of(p.inputs, p.group));
    if (p.sums) p.sums[slot * p.outputs + o] = sum;
    else static_cast<T*>(p.out)[row * p.out_stride + o] = Value<DTYPE>::round(activated(sum, p.activation));
  }
}

// out[t] = sum over the choices j of a token, in their order, of (weights[s]) sums[s], s = t top_k + j; rounded once.
template <int DTYPE>
__global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ sums, const float* __restrict__ weights, int64_t tokens, int top_k,
                                                      int64_t outputs, typename Value<DTYPE>::stored* __restrict__ out, int64_t out_stride) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, t = at / outputs, o = at % outputs;
  if (t >= tokens) return;
  float v = 0.f;
  for (int j = 0; j < top_k; j++) {
    const int64_t s = t * top_k + j;
    v += weights ? weights[s] * sums[s * outputs + o] : sums[s * outputs + o];
  }
  out[t * out_stride + o] = Value<DTYPE>::round(v);
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

static void launch_product(const Product4& p, int dtype, hipStream_t stream) {
  const dim3 grid((unsigned)((p.outputs + 255) / 256), (unsigned)(p.rows < 65535 ? p.rows : 65535));
  if (dtype == STK_BF16) hipLaunchKernelGGL((product_kernel<STK_BF16>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((product_kernel<STK_F16>), grid, dim3(256), 0, stream, p);
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
  launch_product(p, dtype, static_cast<hipStream_t>(stream));
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
  launch_product(p, dtype, static_cast<hipStream_t>(stream));
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
  if (tokens * outputs / 256 >= INT32_MAX) return fail(STK_ERR_UNSUPPORTED, "%s: size exceeds 32-bit range", who);
  hipStream_t s = static_cast<hipStream_t>(stream);
  launch_product(p, dtype, s);
  const unsigned grid = (unsigned)((tokens * outputs + 255) / 256);
  if (dtype == STK_BF16)
    hipLaunchKernelGGL((combine_kernel<STK_BF16>), dim3(grid), dim3(256), 0, s, static_cast<const float*>(workspace), weights, tokens, top_k, outputs,
                       static_cast<Value<STK_BF16>::stored*>(out), out_stride);
  else
    hipLaunchKernelGGL((combine_kernel<STK_F16>), dim3(grid), dim3(256), 0, s, static_cast<const float*>(workspace), weights, tokens, top_k, outputs,
                       static_cast<Value<STK_F16>::stored*>(out), out_stride);
  return check_launch(who);
}
