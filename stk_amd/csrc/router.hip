// stk_top_experts: a router's softmax over the experts' scores of a token and the top_k largest of them, and the gradient of
// the chosen weights with respect to the scores.
//   weights_j = p[chosen_j],  p = softmax(scores)            or, normalized, p[chosen_j] / sum over j
//   ds_i = sum_j g_j weights_j (1[i = chosen_j] - q_i),       q = p, or the normalized weights at their places
// Chosen in descending order of the scores, ties to the lower expert; a NaN ranks above every number.  All in fp32.
//
// A round of the choice is a maximum over the team's keys, in which score and expert are one number, by data-parallel moves.  Bytes are few
// (32768 tokens x 64 float32 scores, top 2: 8.9 MB forward, 2 us at the rate of a copy); the launches take 5.9 us forward and 6.7 backward
// there (a wavefront a token took 23.4 and 10.5), 12.5 and 13 for 16384 x 256 top 8 in bfloat16 (32.8 and 21.2), 2.5 for 64 tokens, and a
// training step waits for the host.
#include <type_traits>

#include "common.h"
#include "values.h"
#include "wave_scan.h"

namespace stk {

constexpr int kRouterExperts = 1024;   // what stk_route takes
constexpr int kRouterTopK = 64;

// Keys of (score, expert) in the order of choice: the larger score, or of two that are alike the lower expert, is the larger key.  Scores
// become whole numbers in their order (-0 like 0, NaN on top); the experts stand behind them, turned round.  A 16-bit score leaves room for
// both in 32 bits.  0 is below every key.
template <int DTYPE>
struct Key {
  typedef std::conditional_t<DTYPE == STK_F32, uint64_t, uint32_t> type;
  static constexpr int shift = DTYPE == STK_F32 ? 32 : 16;
  static constexpr uint32_t all = DTYPE == STK_F32 ? 0xffffffffu : 0xffffu, sign = DTYPE == STK_F32 ? 0x80000000u : 0x8000u;
  static __device__ __forceinline__ type of(typename Value<DTYPE>::stored score, int expert) {
    const float v = Value<DTYPE>::widen(score);
    uint32_t u;
    if constexpr (DTYPE == STK_F32) u = __float_as_uint(score);
    else u = __builtin_bit_cast(uint16_t, score);
    u = v == 0.f ? sign : u & sign ? ~u & all : u | sign;
    if (v != v) u = all;
    return (type)u << shift | (type)(0xffffu - expert);
  }
  static __device__ __forceinline__ float score(type key) {
    const uint32_t u = (uint32_t)(key >> shift), bits = u & sign ? u ^ sign : ~u & all;
    if constexpr (DTYPE == STK_F32) return __uint_as_float(bits);
    else return Value<DTYPE>::widen(__builtin_bit_cast(typename Value<DTYPE>::stored, (uint16_t)bits));
  }
  static __device__ __forceinline__ int expert(type key) { return 0xffff - (int)(key & 0xffffu); }
};

template <int CONTROL, class T>
__device__ __forceinline__ T moved_key(T v) {
  if constexpr (sizeof(T) == 4) return __builtin_amdgcn_update_dpp(0, v, CONTROL, 0xf, 0xf, true);
  else
    return (uint64_t)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CONTROL, 0xf, 0xf, true) << 32 |
           (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, 0xf, 0xf, true);
}
template <class T>
__device__ __forceinline__ T larger(T a, T b) { return a > b ? a : b; }

// The largest of a team's keys, in every lane.
template <int LANES, class T>
__device__ __forceinline__ T team_max(T v) {
  v = larger(v, moved_key<0xb1>(v)), v = larger(v, moved_key<0x4e>(v)), v = larger(v, moved_key<0x141>(v)), v = larger(v, moved_key<0x140>(v));
  if constexpr (LANES == 64) {
    T best = 0;
#pragma unroll
    for (int r = 0; r < 64; r += 16) {
      T one;
      if constexpr (sizeof(T) == 4) one = __builtin_amdgcn_readlane(v, r);
      else one = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), r) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, r);
      best = larger(best, one);
    }
    v = best;
  }
  return v;
}
template <int LANES>
__device__ __forceinline__ float team_sum(float v) { return LANES == 16 ? team16_sum(v) : wave64_sum(v); }

// exp(x), x <= 0, from the hardware's power of two (1 unit in the last place): x log2(e) is rounded, and what that loses is put back
// to first order.
__device__ __forceinline__ float exponential(float x) {
  constexpr float kLog2e = 1.44269504088896341f, kLog2eRest = 1.92596299112661746887e-8f, kLn2 = 0.693147180559945309f;
  const float t = x * kLog2e, rest = fmaf(x, kLog2eRest, fmaf(x, kLog2e, -t)), y = __builtin_amdgcn_exp2f(t);
  return t < -149.f ? 0.f : fmaf(y, rest * kLn2, y);   // (below every fp32 number, also for x = -infinity, which makes NaN of the rest)
}

// A token belongs to a team of 16 or 64 lanes, V experts a lane: neighbours, which are one access, where that fills the team, otherwise
// every 16th or 64th, so that the lanes' single accesses lie next to each other (16384 x 1000 float32 scores, neighbours
// throughout: backward 90 us, 22 so; forward 39, 30).
template <int DTYPE, int LANES, int V>
__global__ __launch_bounds__(256) void top_experts_kernel(const typename Value<DTYPE>::stored* __restrict__ scores, int64_t stride, int64_t tokens, int experts,
                                                          int top_k, int normalize, int32_t* __restrict__ chosen, float* __restrict__ weights) {
  typedef Key<DTYPE> K;
  typedef typename K::type key_t;
  typedef typename Value<DTYPE>::stored stored;
  const bool whole = experts == LANES * V;
  const int lane = threadIdx.x % LANES, first = whole ? lane * V : lane, step = whole ? 1 : LANES;   // the experts first + step j
  for (int64_t t = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; t < tokens; t += (int64_t)gridDim.x * (256 / LANES)) {
    const stored* from = scores + t * stride;
    stored mine[V];
    if (whole) {
      __builtin_memcpy(mine, from + first, sizeof(mine));
    } else {
#pragma unroll
      for (int j = 0; j < V; j++) mine[j] = from[min(first + step * j, experts - 1)];
    }
    key_t key[V], best = 0;
#pragma unroll
    for (int j = 0; j < V; j++) {
      key[j] = first + step * j < experts ? K::of(mine[j], first + step * j) : 0;
      best = larger(best, key[j]);
    }
    best = team_max<LANES>(best);
    const float top = K::score(best);
    const bool none = top == -INFINITY;   // every expert is masked
    float sum = 0.f;
    if (!normalize) {
#pragma unroll
      for (int j = 0; j < V; j++) sum += first + step * j < experts ? exponential(Value<DTYPE>::widen(mine[j]) - top) : 0.f;
      sum = team_sum<LANES>(sum);
      // (the sum of a row with a NaN or +infinity is one: top - top is NaN there)
    }
    // choice k is kept by lane k % LANES, in its place k / LANES
    constexpr int kKept = kRouterTopK / LANES;
    float weight[kKept];
    int at[kKept];
    float all = 0.f;
#pragma unroll
    for (int r = 0; r < kKept; r++) {
      if (r * LANES >= top_k) break;
      weight[r] = 0.f, at[r] = 0;
      const int here = min(top_k - r * LANES, LANES);
      for (int k = 0; k < here; k++) {
        const bool is = lane == k;
        at[r] = is ? K::expert(best) : at[r];
        weight[r] = is ? K::score(best) : weight[r];
        if (r * LANES + k + 1 == top_k) break;
        key_t next = 0;
#pragma unroll
        for (int j = 0; j < V; j++) {
          key[j] = key[j] == best ? 0 : key[j];
          next = larger(next, key[j]);
        }
        best = team_max<LANES>(next);
      }
      weight[r] = lane < here && !none ? exponential(weight[r] - top) : 0.f;
      all += weight[r];
    }
    if (normalize) sum = team_sum<LANES>(all);
#pragma unroll
    for (int r = 0; r < kKept; r++)
      if (r * LANES + lane < top_k) {
        chosen[t * top_k + r * LANES + lane] = at[r];
        weights[t * top_k + r * LANES + lane] = none ? 0.f : weight[r] / sum;
      }
  }
}

// The gradient of a token's row goes through LDS: every lane writes its experts' shares, the chosen experts' own terms are put on
// top, the lanes store what is there.
template <int DTYPE, int LANES, int V>
__global__ __launch_bounds__(256) void top_experts_backward_kernel(const typename Value<DTYPE>::stored* __restrict__ scores, int64_t stride,
                                                                   const int32_t* __restrict__ chosen, const float* __restrict__ weights,
                                                                   const float* __restrict__ grad, int64_t tokens, int experts, int top_k, int normalize,
                                                                   typename Value<DTYPE>::stored* __restrict__ out, int64_t out_stride) {
  typedef typename Value<DTYPE>::stored stored;
  __shared__ float rows[256 / LANES][LANES * V];
  const bool whole = experts == LANES * V;
  const int lane = threadIdx.x % LANES, first = whole ? lane * V : lane, step = whole ? 1 : LANES;
  float* row = rows[threadIdx.x / LANES];
  constexpr int kKept = kRouterTopK / LANES;
  for (int64_t t = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; t < tokens; t += (int64_t)gridDim.x * (256 / LANES)) {
    float w[kKept], onto[kKept], inner = 0.f;
    int at[kKept];
#pragma unroll
    for (int r = 0; r < kKept; r++) {
      const int k = r * LANES + lane;
      w[r] = onto[r] = 0.f, at[r] = -1;
      if (k < top_k) {
        w[r] = weights[t * top_k + k], at[r] = chosen[t * top_k + k];
        onto[r] = grad[t * top_k + k] * w[r];
      }
      inner += onto[r];
    }
    inner = team_sum<LANES>(inner);
    if (normalize) {
#pragma unroll
      for (int j = 0; j < V; j++) row[first + step * j] = 0.f;
    } else {
      // p of the first choice is exp(0) / sum: with its score and weight those of the others need no sum of their own (the logarithm
      // of the sum would not do: added to a score of -1e38 it is lost).  A weight of 0: every expert is masked.
      const stored* from = scores + t * stride;
      const float largest = weights[t * top_k];
      const float top = Value<DTYPE>::widen(from[min(max(chosen[t * top_k], 0), experts - 1)]);
      stored mine[V];
      if (whole) {
        __builtin_memcpy(mine, from + first, sizeof(mine));
      } else {
#pragma unroll
        for (int j = 0; j < V; j++) mine[j] = from[min(first + step * j, experts - 1)];
      }
#pragma unroll
      for (int j = 0; j < V; j++) row[first + step * j] = largest == 0.f ? 0.f : -(exponential(Value<DTYPE>::widen(mine[j]) - top) * largest * inner);
    }
    // (a team lies in one wavefront, whose LDS accesses are made in order)
    asm volatile("" : : : "memory");
#pragma unroll
    for (int r = 0; r < kKept; r++)
      if ((unsigned)at[r] < (unsigned)experts) row[at[r]] = normalize ? onto[r] - w[r] * inner : onto[r] + row[at[r]];
    asm volatile("" : : : "memory");
    stored result[V];
#pragma unroll
    for (int j = 0; j < V; j++) result[j] = Value<DTYPE>::round(row[first + step * j]);
    if (whole) {
      __builtin_memcpy(out + t * out_stride + first, result, sizeof(result));
    } else {
#pragma unroll
      for (int j = 0; j < V; j++)
        if (first + step * j < experts) out[t * out_stride + first + step * j] = result[j];
    }
    asm volatile("" : : : "memory");
  }
}

template <class Fn>
static void for_experts(int64_t experts, Fn&& fn) {
  typedef std::integral_constant<int, 16> Sixteen;
  typedef std::integral_constant<int, 64> Wave;
  if (experts <= 16) fn(Sixteen(), std::integral_constant<int, 1>());
  else if (experts <= 32) fn(Sixteen(), std::integral_constant<int, 2>());
  else if (experts <= 64) fn(Sixteen(), std::integral_constant<int, 4>());
  else if (experts <= 128) fn(Sixteen(), std::integral_constant<int, 8>());
  else if (experts <= 256) fn(Sixteen(), std::integral_constant<int, 16>());
  else if (experts <= 512) fn(Wave(), std::integral_constant<int, 8>());
  else fn(Wave(), std::integral_constant<int, 16>());
}
static dim3 router_grid(int64_t tokens, int lanes) {
  const int64_t groups = (tokens + 256 / lanes - 1) / (256 / lanes);
  return dim3((unsigned)(groups < 1 << 20 ? groups : 1 << 20));
}

static int router_check(const char* who, int64_t tokens, int64_t experts, int top_k, int dtype) {
  if (!is_value_dtype(dtype)) return fail(STK_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (tokens < 0 || experts < 1 || top_k < 1 || top_k > experts)
    return fail(STK_ERR_DIMS, "%s: the top %d of %lld experts, %lld tokens", who, top_k, (long long)experts, (long long)tokens);
  if (experts > kRouterExperts || top_k > kRouterTopK) return fail(STK_ERR_UNSUPPORTED, "%s: at most %d experts, the top %d", who, kRouterExperts, kRouterTopK);
  if (tokens > INT32_MAX / top_k) return fail(STK_ERR_UNSUPPORTED, "%s: size exceeds 32-bit range", who);
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
    for_experts(experts, [&](auto lanes, auto v) {
      constexpr int D = decltype(d)::value, L = decltype(lanes)::value, V = decltype(v)::value;
      hipLaunchKernelGGL((top_experts_kernel<D, L, V>), router_grid(tokens, L), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const T*>(scores), stride,
                         tokens, (int)experts, top_k, normalize, chosen, weights);
    });
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
    for_experts(experts, [&](auto lanes, auto v) {
      constexpr int D = decltype(d)::value, L = decltype(lanes)::value, V = decltype(v)::value;
      hipLaunchKernelGGL((top_experts_backward_kernel<D, L, V>), router_grid(tokens, L), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const T*>(scores),
                         stride, chosen, weights, grad, tokens, (int)experts, top_k, normalize, static_cast<T*>(dscores), dscores_stride);
    });
  });
  return check_launch(who);
}
