// stk_layer_norm and its gradients.  With mu and v the mean and the variance of a row of n values, r = 1 / sqrt(v + eps) and
// z = (x - mu) r,
//   y = z w + b
//   dx = r (g - mean(g) - z mean(g z)),  g = dy w        dw = sum over rows of dy z        db = sum over rows of dy
// Statistics and sums are fp32; the variance is that of the differences from the mean (never E[x^2] - mu^2, which cancels
// where the mean is large).
#include <type_traits>

#include "common.h"
#include "values.h"

namespace stk {

// Sum over the 256 threads of a workgroup; every thread gets it.
__device__ __forceinline__ float workgroup_sum(float v, float* part) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return part[0] + part[1] + part[2] + part[3];
}

template <int DTYPE, int PARAM>
__global__ __launch_bounds__(256) void layer_norm_kernel(const typename Value<DTYPE>::stored* __restrict__ x, int64_t x_stride, int64_t n,
                                                         const typename Value<PARAM>::stored* __restrict__ weight,
                                                         const typename Value<PARAM>::stored* __restrict__ bias, float eps,
                                                         typename Value<DTYPE>::stored* __restrict__ out, int64_t out_stride,
                                                         float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float part[4];
  const int64_t row = blockIdx.x;
  x += row * x_stride, out += row * out_stride;
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 256) s += Value<DTYPE>::widen(x[i]);
  const float mu = workgroup_sum(s, part) / (float)n;
  float q = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 256) {
    const float d = Value<DTYPE>::widen(x[i]) - mu;
    q += d * d;
  }
  const float r = 1.f / sqrtf(workgroup_sum(q, part) / (float)n + eps);
  for (int64_t i = threadIdx.x; i < n; i += 256) {
    float y = (Value<DTYPE>::widen(x[i]) - mu) * r;
    if (weight) y *= Value<PARAM>::widen(weight[i]);
    if (bias) y += Value<PARAM>::widen(bias[i]);
    out[i] = Value<DTYPE>::round(y);
  }
  if (threadIdx.x == 0 && mean) mean[row] = mu, rstd[row] = r;
}

template <int DTYPE, int PARAM>
__global__ __launch_bounds__(256) void layer_norm_dx_kernel(const typename Value<DTYPE>::stored* __restrict__ grad, int64_t grad_stride,
                                                            const typename Value<DTYPE>::stored* __restrict__ x, int64_t x_stride,
                                                            const float* __restrict__ mean, const float* __restrict__ rstd,
                                                            const typename Value<PARAM>::stored* __restrict__ weight, int64_t n,
                                                            typename Value<DTYPE>::stored* __restrict__ dx, int64_t dx_stride) {
  __shared__ float part[4];
  const int64_t row = blockIdx.x;
  x += row * x_stride, grad += row * grad_stride, dx += row * dx_stride;
  const float mu = mean[row], r = rstd[row];
  float a = 0.f, b = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 256) {
    const float g = Value<DTYPE>::widen(grad[i]) * (weight ? Value<PARAM>::widen(weight[i]) : 1.f);
    a += g, b += g * ((Value<DTYPE>::widen(x[i]) - mu) * r);
  }
  a = workgroup_sum(a, part) / (float)n;
  b = workgroup_sum(b, part) / (float)n;
  for (int64_t i = threadIdx.x; i < n; i += 256) {
    const float g = Value<DTYPE>::widen(grad[i]) * (weight ? Value<PARAM>::widen(weight[i]) : 1.f);
    dx[i] = Value<DTYPE>::round(r * (g - a - (Value<DTYPE>::widen(x[i]) - mu) * r * b));
  }
}

// Rows are dealt to kParamShares shares; a thread sums a column over the rows of a share.
constexpr int kParamShares = 128;
template <int DTYPE>
__global__ __launch_bounds__(256) void layer_norm_param_kernel(const typename Value<DTYPE>::stored* __restrict__ grad, int64_t grad_stride,
                                                               const typename Value<DTYPE>::stored* __restrict__ x, int64_t x_stride,
                                                               const float* __restrict__ mean, const float* __restrict__ rstd, int64_t rows, int64_t n,
                                                               float* __restrict__ sums) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < rows; row += kParamShares) {
    const float g = Value<DTYPE>::widen(grad[row * grad_stride + i]);
    dw += g * ((Value<DTYPE>::widen(x[row * x_stride + i]) - mean[row]) * rstd[row]), db += g;
  }
  sums[(2 * blockIdx.y) * n + i] = dw, sums[(2 * blockIdx.y + 1) * n + i] = db;
}
template <int PARAM>
__global__ __launch_bounds__(256) void layer_norm_param_sum_kernel(const float* __restrict__ sums, int shares, int64_t n, typename Value<PARAM>::stored* __restrict__ dweight,
                                                                   typename Value<PARAM>::stored* __restrict__ dbias) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float dw = 0.f, db = 0.f;
  for (int s = 0; s < shares; s++) dw += sums[(int64_t)(2 * s) * n + i], db += sums[(int64_t)(2 * s + 1) * n + i];
  if (dweight) dweight[i] = Value<PARAM>::round(dw);
  if (dbias) dbias[i] = Value<PARAM>::round(db);
}

static int norm_check(const char* who, int64_t rows, int64_t size, int dtype, int param_dtype) {
  if (!is_value_dtype(dtype)) return fail(STK_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (param_dtype != dtype && param_dtype != STK_F32) return fail(STK_ERR_UNSUPPORTED, "%s: weight and bias have the rows' type or float32", who);
  if (rows < 0 || size < 1) return fail(STK_ERR_DIMS, "%s: %lld rows of %lld", who, (long long)rows, (long long)size);
  if (rows > INT32_MAX || size > INT32_MAX) return fail(STK_ERR_UNSUPPORTED, "%s: size exceeds 32-bit range", who);
  return STK_OK;
}

template <class Fn>
static void for_types(int dtype, int param_dtype, Fn&& fn) {
  for_dtype(dtype, [&](auto d) {
    if (param_dtype == STK_F32) fn(d, std::integral_constant<int, STK_F32>());
    else fn(d, d);
  });
}

}  // namespace stk

using namespace stk;

extern "C" int stk_layer_norm(const void* x, int64_t rows, int64_t size, int64_t x_stride, const void* weight, const void* bias, float eps, void* out,
                              int64_t out_stride, float* mean, float* rstd, int dtype, int param_dtype, stk_stream_t stream) {
  const char* who = "stk_layer_norm";
  if (int rc = norm_check(who, rows, size, dtype, param_dtype)) return rc;
  if (rows == 0) return STK_OK;
  if (!x || !out || !mean != !rstd) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (x_stride < 0 || out_stride < size) return fail(STK_ERR_DIMS, "%s: strides %lld, %lld", who, (long long)x_stride, (long long)out_stride);
  for_types(dtype, param_dtype, [&](auto d, auto p) {
    typedef typename Value<d()>::stored T;
    typedef typename Value<p()>::stored P;
    hipLaunchKernelGGL((layer_norm_kernel<d(), p()>), dim3((unsigned)rows), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const T*>(x), x_stride,
                       size, static_cast<const P*>(weight), static_cast<const P*>(bias), eps, static_cast<T*>(out), out_stride, mean, rstd);
  });
  return check_launch(who);
}

extern "C" size_t stk_layer_norm_backward_workspace_bytes(int64_t rows, int64_t size) {
  if (rows <= 0 || size <= 0) return 0;
  return (size_t)(2 * kParamShares * size) * sizeof(float);
}

extern "C" int stk_layer_norm_backward(const void* grad, int64_t grad_stride, const void* x, int64_t x_stride, const float* mean, const float* rstd,
                                       const void* weight, int64_t rows, int64_t size, void* dx, int64_t dx_stride, void* dweight, void* dbias, int dtype,
                                       int param_dtype, void* workspace, size_t workspace_bytes, stk_stream_t stream) {
  const char* who = "stk_layer_norm_backward";
  if (int rc = norm_check(who, rows, size, dtype, param_dtype)) return rc;
  const bool params = dweight || dbias;
  if (!params && (!dx || rows == 0)) return STK_OK;
  if (rows > 0 && (!grad || !x || !mean || !rstd)) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (grad_stride < 0 || x_stride < 0 || (dx && dx_stride < size)) return fail(STK_ERR_DIMS, "%s: strides", who);
  if (params && rows > 0 && (!workspace || workspace_bytes < stk_layer_norm_backward_workspace_bytes(rows, size)))
    return fail(STK_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", who, stk_layer_norm_backward_workspace_bytes(rows, size));
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* sums = static_cast<float*>(workspace);
  for_types(dtype, param_dtype, [&](auto d, auto p) {
    typedef typename Value<d()>::stored T;
    typedef typename Value<p()>::stored P;
    const T *g = static_cast<const T*>(grad), *xs = static_cast<const T*>(x);
    if (dx && rows > 0)
      hipLaunchKernelGGL((layer_norm_dx_kernel<d(), p()>), dim3((unsigned)rows), dim3(256), 0, s, g, grad_stride, xs, x_stride, mean, rstd,
                         static_cast<const P*>(weight), size, static_cast<T*>(dx), dx_stride);
    if (params) {
      const unsigned columns = (unsigned)((size + 255) / 256);
      if (rows > 0)   // (without rows there is no workspace either: the sums are those of no share)
        hipLaunchKernelGGL((layer_norm_param_kernel<d()>), dim3(columns, kParamShares), dim3(256), 0, s, g, grad_stride, xs, x_stride, mean, rstd, rows, size, sums);
      hipLaunchKernelGGL((layer_norm_param_sum_kernel<p()>), dim3(columns), dim3(256), 0, s, sums, rows > 0 ? kParamShares : 0, size,
                         static_cast<P*>(dweight), static_cast<P*>(dbias));
    }
  });
  return check_launch(who);
}
