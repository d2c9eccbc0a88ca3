// Values of the three element types as fp32 numbers, for the kernels that work on rows and not on tiles.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

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

// Calls fn(std::integral_constant<int, dtype>()) for one of the three types.
template <class Fn>
inline void for_dtype(int dtype, Fn&& fn) {
  if (dtype == STK_F16) fn(std::integral_constant<int, STK_F16>());
  else if (dtype == STK_BF16) fn(std::integral_constant<int, STK_BF16>());
  else fn(std::integral_constant<int, STK_F32>());
}
inline bool is_value_dtype(int dtype) { return dtype == STK_F16 || dtype == STK_BF16 || dtype == STK_F32; }

}  // namespace stk
