// Values of the three element types as fp32 numbers, for the kernels that work on rows and not on tiles.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/stk_amd.h"

namespace stk {

// Value<DTYPE>: how an element is stored, and how it becomes an fp32 number and back (rounded to nearest, ties to even).
template <int DTYPE> struct Value;
template <> struct Value<STK_F16> {
  typedef _Float16 stored;
  static __device__ __forceinline__ float widen(stored v) { return (float)v; }
  static __device__ __forceinline__ stored round(float v) { return (stored)v; }
};
template <> struct Value<STK_BF16> {
  typedef __bf16 stored;
  static __device__ __forceinline__ float widen(stored v) { return (float)v; }
  static __device__ __forceinline__ stored round(float v) { return (stored)v; }
};
template <> struct Value<STK_F32> {
  typedef float stored;
  static __device__ __forceinline__ float widen(stored v) { return v; }
  static __device__ __forceinline__ stored round(float v) { return v; }
};

// Eight consecutive values as fp32 numbers and back.  The address needs the alignment of one value: the memory unit takes 16-byte
// accesses at any address.
typedef uint32_t Quad __attribute__((ext_vector_type(4)));
typedef uint32_t QuadAt2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t QuadAt4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t PairAt2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float Pair __attribute__((ext_vector_type(2)));
typedef _Float16 HalfPair __attribute__((ext_vector_type(2)));
template <int DTYPE> struct Eight { Quad q[DTYPE == STK_F32 ? 2 : 1]; };
template <int DTYPE>
__device__ __forceinline__ Eight<DTYPE> fetch8(const typename Value<DTYPE>::stored* p) {
  if constexpr (DTYPE == STK_F32) return {{*reinterpret_cast<const QuadAt4*>(p), *reinterpret_cast<const QuadAt4*>(p + 4)}};
  else return {{*reinterpret_cast<const QuadAt2*>(p)}};
}
template <int DTYPE>
__device__ __forceinline__ void widen8(float (&v)[8], const Eight<DTYPE>& from) {
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const uint32_t word = from.q[0][j];   // (a bit cast of a vector's element itself takes element 0)
    if constexpr (DTYPE == STK_F32) {
      const uint32_t behind = from.q[1][j];
      v[j] = __uint_as_float(word), v[4 + j] = __uint_as_float(behind);
    } else if constexpr (DTYPE == STK_BF16) {
      v[2 * j] = __uint_as_float(word << 16), v[2 * j + 1] = __uint_as_float(word & 0xffff0000u);
    } else {
      const HalfPair h = __builtin_bit_cast(HalfPair, word);
      v[2 * j] = (float)h.x, v[2 * j + 1] = (float)h.y;
    }
  }
}
template <int DTYPE>
__device__ __forceinline__ void load8(float (&v)[8], const typename Value<DTYPE>::stored* p) { widen8<DTYPE>(v, fetch8<DTYPE>(p)); }
template <int DTYPE>
__device__ __forceinline__ void store8(typename Value<DTYPE>::stored* p, const float (&v)[8]) {
  if constexpr (DTYPE == STK_F32) {
    Quad a, b;
#pragma unroll
    for (int j = 0; j < 4; j++) a[j] = __float_as_uint(v[j]), b[j] = __float_as_uint(v[4 + j]);
    *reinterpret_cast<QuadAt4*>(p) = a, *reinterpret_cast<QuadAt4*>(p + 4) = b;
  } else {
    Quad a;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      typedef typename Value<DTYPE>::stored Two __attribute__((ext_vector_type(2)));
      a[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(Pair{v[2 * j], v[2 * j + 1]}, Two));
    }
    *reinterpret_cast<QuadAt2*>(p) = a;
  }
}

// Sums over teams of 16 lanes, in every lane, and over the wavefront, as a scalar: data-parallel moves, no LDS.
template <int CONTROL, int ROWS = 0xf>
__device__ __forceinline__ float moved(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CONTROL, ROWS, 0xf, true));
}
__device__ __forceinline__ float team16_sum(float v) {
  v += moved<0xb1>(v);    // lanes 1 0 3 2 of each four
  v += moved<0x4e>(v);    // lanes 2 3 0 1
  v += moved<0x141>(v);   // halves of 16 lanes mirrored
  v += moved<0x140>(v);   // 16 lanes mirrored
  return v;
}
__device__ __forceinline__ float wave64_sum(float v) {
  v = team16_sum(v);
  v += moved<0x142, 0xa>(v);   // lane 15 of a row to the next row
  v += moved<0x143, 0xc>(v);   // lane 31 to the upper half
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
}

// Calls fn(std::integral_constant<int, dtype>()) for one of the three types.
template <class Fn>
inline void for_dtype(int dtype, Fn&& fn) {
  if (dtype == STK_F16) fn(std::integral_constant<int, STK_F16>());
  else if (dtype == STK_BF16) fn(std::integral_constant<int, STK_BF16>());
  else fn(std::integral_constant<int, STK_F32>());
}
inline bool is_value_dtype(int dtype) { return dtype == STK_F16 || dtype == STK_BF16 || dtype == STK_F32; }

}  // namespace stk
