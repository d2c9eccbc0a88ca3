// stk_top_experts: a router's softmax over the experts' scores of a token and the top_k largest of them, and the gradient of
// the chosen weights with respect to the scores.
//   weights_j = p[chosen_j],  p = softmax(scores)            or, normalized, p[chosen_j] / sum over j
//   ds_i = sum_j g_j weights_j (1[i = chosen_j] - q_i),       q = p, or the normalized weights at their places
// Chosen in descending order of the scores, ties to the lower expert; a NaN ranks above every number.  All in fp32.
#include <type_traits>

#include "common.h"
#include "values.h"
#include "wave_scan.h"

namespace stk {

constexpr int kRouterExperts = 1024;   // what stk_route takes
constexpr int kRouterTopK = 64;
constexpr int kRouterValues = kRouterExperts / kWave;

// Whole numbers in the order of the scores: -0 like 0, NaN on top; 0 ranks below every score.
__device__ __forceinline__ uint32_t rank_of(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t u = __float_as_uint(v + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float score_of(uint32_t rank) { return __uint_as_float(rank & 0x80000000u ? rank ^ 0x80000000u : ~rank); }

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const uint32_t o = __shfl_xor(v, d, kWave);
    v = o > v ? o : v;
  }
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
  return v;
}

// A wavefront per token; lane l holds the experts l, l + 64, ...
template <int DTYPE>
__global__ __launch_bounds__(256) void top_experts_kernel(const typename Value<DTYPE>::stored* __restrict__ scores, int64_t stride, int64_t tokens, int experts,
                                                          int top_k, int normalize, int32_t* __restrict__ chosen, float* __restrict__ weights) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= tokens) return;
  uint32_t rank[kRouterValues], best = 0;
#pragma unroll
  for (int j = 0; j < kRouterValues; j++) {
    const int e = lane + 64 * j;
    rank[j] = e < experts ? rank_of(Value<DTYPE>::widen(scores[t * stride + e])) : 0u;
    best = rank[j] > best ? rank[j] : best;
  }
  const float top = score_of(wave_max(best));
  const bool none = top == -INFINITY;   // every expert is masked
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < kRouterValues; j++)
    if (rank[j]) sum += expf(score_of(rank[j]) - top);
  sum = wave_sum(sum);
  float mine = 0.f;   // of choice `lane`
  int mine_at = 0;
  for (int k = 0; k < top_k; k++) {
    best = 0;
#pragma unroll
    for (int j = 0; j < kRouterValues; j++) best = rank[j] > best ? rank[j] : best;
    best = wave_max(best);
    int at = experts;
#pragma unroll
    for (int j = kRouterValues - 1; j >= 0; j--)
      if (rank[j] == best) at = lane + 64 * j;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      const int o = __shfl_xor(at, d, kWave);
      at = o < at ? o : at;
    }
#pragma unroll
    for (int j = 0; j < kRouterValues; j++)
      if (lane + 64 * j == at) rank[j] = 0;
    if (lane == k) mine = none ? 0.f : expf(score_of(best) - top), mine_at = at;
  }
  const float by = normalize ? wave_sum(mine) : sum;
  if (lane < top_k) {
    chosen[t * top_k + lane] = mine_at;
    weights[t * top_k + lane] = none ? 0.f : mine / by;
  }
}

template <int DTYPE>
__global__ __launch_bounds__(256) void top_experts_backward_kernel(const typename Value<DTYPE>::stored* __restrict__ scores, int64_t stride,
                                                                   const int32_t* __restrict__ chosen,
                                                                   const float* __restrict__ weights, const float* __restrict__ grad, int64_t tokens, int experts,
                                                                   int top_k, int normalize, typename Value<DTYPE>::stored* __restrict__ out,
                                                                   int64_t out_stride) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= tokens) return;
  const float w = lane < top_k ? weights[t * top_k + lane] : 0.f, g = lane < top_k ? grad[t * top_k + lane] : 0.f;
  const int at = lane < top_k ? chosen[t * top_k + lane] : -1;
  const float onto = g * w, inner = wave_sum(onto);
  // p of the first choice is exp(0) / sum: with its score and weight those of the others need no sum of their own (the logarithm
  // of the sum would not do: added to a score of -1e38 it is lost).  A weight of 0: every expert is masked.
  const float first = __shfl(w, 0, kWave);
  float top = 0.f;
  if (!normalize) top = Value<DTYPE>::widen(scores[t * stride + min(max(__shfl(at, 0, kWave), 0), experts - 1)]);
  for (int e = lane; e - lane < experts; e += kWave) {   // (all lanes stay: they exchange the choices)
    float q = 0.f, d = 0.f;
    if (!normalize && e < experts) q = first == 0.f ? 0.f : expf(Value<DTYPE>::widen(scores[t * stride + e]) - top) * first;
    for (int k = 0; k < top_k; k++) {
      const int at_k = __shfl(at, k, kWave);
      const float onto_k = __shfl(onto, k, kWave), w_k = __shfl(w, k, kWave);
      if (at_k == e) d = onto_k, q = normalize ? w_k : q;
    }
    if (e < experts) out[t * out_stride + e] = Value<DTYPE>::round(d - q * inner);
  }
}

static int router_check(const char* who, int64_t tokens, int64_t experts, int top_k, int dtype) {
  if (!is_value_dtype(dtype)) return fail(STK_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (tokens < 0 || experts < 1 || top_k < 1 || top_k > experts)
    return fail(STK_ERR_DIMS, "%s: the top %d of %lld experts, %lld tokens", who, top_k, (long long)experts, (long long)tokens);
  if (experts > kRouterExperts || top_k > kRouterTopK) return fail(STK_ERR_UNSUPPORTED, "%s: at most %d experts, the top %d", who, kRouterExperts, kRouterTopK);
  if (tokens * top_k > INT32_MAX) return fail(STK_ERR_UNSUPPORTED, "%s: size exceeds 32-bit range", who);
  return STK_OK;
}

}  // namespace stk

using namespace stk;

extern "C" int stk_top_experts(const void* scores, int64_t tokens, int64_t experts, int64_t stride, int top_k, int normalize, int32_t* chosen, float* weights,
                               int dtype, stk_stream_t stream) {
  const char* who = "stk_top_experts";
  if (int rc = router_check(who, tokens, experts, top_k, dtype)) return rc;
  if (tokens == 0) return STK_OK;
  if (!scores || !chosen || !weights) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (stride < 0) return fail(STK_ERR_DIMS, "%s: stride %lld", who, (long long)stride);
  for_dtype(dtype, [&](auto d) {
    typedef typename Value<d()>::stored T;
    hipLaunchKernelGGL((top_experts_kernel<d()>), dim3((unsigned)((tokens + 3) / 4)), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const T*>(scores), stride, tokens, (int)experts, top_k, normalize, chosen, weights);
  });
  return check_launch(who);
}

extern "C" int stk_top_experts_backward(const void* scores, int64_t stride, const int32_t* chosen, const float* weights, const float* grad,
                                        int64_t tokens, int64_t experts, int top_k, int normalize, void* dscores, int64_t dscores_stride, int dtype,
                                        stk_stream_t stream) {
  const char* who = "stk_top_experts_backward";
  if (int rc = router_check(who, tokens, experts, top_k, dtype)) return rc;
  if (tokens == 0) return STK_OK;
  if (!chosen || !weights || !grad || !dscores || (!normalize && !scores)) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (stride < 0 || dscores_stride < experts) return fail(STK_ERR_DIMS, "%s: strides %lld, %lld", who, (long long)stride, (long long)dscores_stride);
  for_dtype(dtype, [&](auto d) {
    typedef typename Value<d()>::stored T;
    hipLaunchKernelGGL((top_experts_backward_kernel<d()>), dim3((unsigned)((tokens + 3) / 4)), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const T*>(scores), stride, chosen, weights, grad, tokens, (int)experts, top_k, normalize, static_cast<T*>(dscores),
                       dscores_stride);
  });
  return check_launch(who);
}
