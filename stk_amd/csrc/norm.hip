// stk_layer_norm and its gradients.  With mu and v the mean and the variance of a row of n values, r = 1 / sqrt(v + eps) and
// z = (x - mu) r,
//   y = z w + b
//   dx = r (g - mean(g) - z mean(g z)),  g = dy w        dw = sum over rows of dy z        db = sum over rows of dy
// Statistics and sums are fp32; the variance is that of the differences from the mean (never E[x^2] - mu^2, which cancels
// where the mean is large).  The sum for the mean is one of differences too, from the row's first value: equal values have a mean of exactly
// that value and no deviation.  (With the sum of the values themselves the mean of 1000 values 1000.0 is off by a unit, and 1 / sqrt(eps)
// makes 0.02 of that in every result.  Adding the mean of the differences from a first mean is as good, and another sum over the
// row: 32768 x 8192 in 240 us.)
//
// A row belongs to a team of 16, 64, 256, 512 or 1024 lanes that holds it in registers, pieces of eight values a lane, so that it is read once.
// The last piece of a row whose length is no multiple of eight is moved back over its neighbour; the values it shares with
// it are left out of the sums and stored twice.
//
// Bound by bytes: 32768 x 8192 in bfloat16 take 208 us forward (1.07 GB, 5.2 TB/s, a copy reaches 5.2) and 316 backward (1.61 GB, 5.1 TB/s).
// 16384 x 1024 takes 16 and 21 + 4 for the sums over the shares, less than the 43 us that the host needs for a step of autograd; 64 rows
// are a launch (3.6 us).  Not bound by bytes: the backward pass of float32 rows of 1025 to 2048 values (5003 x 1151: 28 us for 69 MB, a team
// of 64 lanes with 32 values each takes 247 registers), and the kernels that loop over rows too long for registers (below).
#include <type_traits>

#include "common.h"
#include "values.h"

namespace stk {

// A team of LANES lanes on rows of up to 8 PIECES LANES values, THREADS / LANES of them a workgroup; TAIL: the length is no
// multiple of eight.
template <int LANES_, int PIECES_, int THREADS, bool TAIL_>
struct Team {
  static constexpr int LANES = LANES_, PIECES = PIECES_;
  static constexpr bool TAIL = TAIL_;
  static constexpr int kThreads = THREADS, kTeams = kThreads / LANES, kWaves = LANES / 64;
  int lane, team;
  int first[PIECES], skip[PIECES];   // first value of a piece, and how many values at its front are none of its own (8: no piece)
  __device__ __forceinline__ explicit Team(int n) {
    lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
      const int at = 8 * (lane + LANES * i);
      first[i] = TAIL && at < n && at + 8 > n ? n - 8 : at;
      skip[i] = at < n ? at - first[i] : 8;
    }
  }
  __device__ __forceinline__ bool has(int i) const { return skip[i] < 8; }
  __device__ __forceinline__ bool owns(int i, int j) const { return TAIL ? j >= skip[i] : has(i); }
  // Sums over the lanes of a team, in every one of them.  `part`: LDS of a workgroup of several wavefronts, [N * kWaves], not the same
  // in two calls that follow each other (of which only one barrier is between).
  template <int N>
  __device__ __forceinline__ void sums(float (&v)[N], float* part) const {
#pragma unroll
    for (int k = 0; k < N; k++) v[k] = LANES == 16 ? team16_sum(v[k]) : wave64_sum(v[k]);
    if constexpr (LANES > 64) {
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int k = 0; k < N; k++) part[k * kWaves + (threadIdx.x >> 6)] = v[k];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < N; k++) {
        v[k] = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) v[k] += part[k * kWaves + w];
      }
    }
  }
  __device__ __forceinline__ float sum(float v, float* part) const {
    float one[1] = {v};
    sums(one, part);
    return one[0];
  }
};

template <class T, int DTYPE, int PARAM>
__global__ __launch_bounds__(T::kThreads) void layer_norm_kernel(const typename Value<DTYPE>::stored* __restrict__ x, int64_t x_stride, int64_t rows, int n,
                                                                 const typename Value<PARAM>::stored* __restrict__ weight,
                                                                 const typename Value<PARAM>::stored* __restrict__ bias, float eps,
                                                                 typename Value<DTYPE>::stored* __restrict__ out, int64_t out_stride,
                                                                 float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float part[2][T::kWaves > 1 ? T::kWaves : 1];
  const T t(n);
  const float over_n = 1.f / (float)n;
  for (int64_t row = (int64_t)blockIdx.x * T::kTeams + t.team; row < rows; row += (int64_t)gridDim.x * T::kTeams) {
    const auto* from = x + row * x_stride;
    const float pivot = Value<DTYPE>::widen(from[0]);
    float v[T::PIECES][8], s = 0.f, q = 0.f;
#pragma unroll
    for (int i = 0; i < T::PIECES; i++)
      if (t.has(i)) load8<DTYPE>(v[i], from + t.first[i]);
#pragma unroll
    for (int i = 0; i < T::PIECES; i++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        v[i][j] -= pivot;
        s += t.owns(i, j) ? v[i][j] : 0.f;
      }
    const float off = t.sum(s, part[0]) * over_n;
#pragma unroll
    for (int i = 0; i < T::PIECES; i++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        v[i][j] -= off;
        q += t.owns(i, j) ? v[i][j] * v[i][j] : 0.f;
      }
    const float r = 1.f / sqrtf(t.sum(q, part[1]) * over_n + eps);
    auto* to = out + row * out_stride;
#pragma unroll
    for (int i = 0; i < T::PIECES; i++)
      if (t.has(i)) {
        float w[8], b[8];
        if (weight) load8<PARAM>(w, weight + t.first[i]);
        if (bias) load8<PARAM>(b, bias + t.first[i]);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          v[i][j] *= r;
          if (weight) v[i][j] *= w[j];
          if (bias) v[i][j] += b[j];
        }
        store8<DTYPE>(to + t.first[i], v[i]);
      }
    if (t.lane == 0 && mean) mean[row] = pivot + off, rstd[row] = r;
  }
}

// dx of a workgroup's rows, and its share of the sums over rows: sums[2 blockIdx] those of dy z, sums[2 blockIdx + 1] those of dy.
template <class T, int DTYPE, int PARAM, bool PARAMS>
__global__ __launch_bounds__(T::kThreads) void layer_norm_backward_kernel(const typename Value<DTYPE>::stored* __restrict__ grad, int64_t grad_stride,
                                                                          const typename Value<DTYPE>::stored* __restrict__ x, int64_t x_stride,
                                                                          const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                          const typename Value<PARAM>::stored* __restrict__ weight, int64_t rows, int n,
                                                                          typename Value<DTYPE>::stored* __restrict__ dx, int64_t dx_stride,
                                                                          float* __restrict__ sums) {
  __shared__ float part[2][2 * (T::kWaves > 1 ? T::kWaves : 1)];
  __shared__ float together[PARAMS && T::LANES <= 64 ? 2 * 8 * T::LANES * T::PIECES : 1];
  const T t(n);
  const float over_n = 1.f / (float)n;
  float dw[T::PIECES][8], db[T::PIECES][8];
#pragma unroll
  for (int i = 0; i < T::PIECES; i++)
#pragma unroll
    for (int j = 0; j < 8; j++) dw[i][j] = db[i][j] = 0.f;
  const int64_t step = (int64_t)gridDim.x * T::kTeams;
  Eight<DTYPE> x_ahead[T::PIECES], g_ahead[T::PIECES];   // of the next row, on their way once this one's registers are free
  float mu_ahead = 0.f, r_ahead = 0.f;
  const auto fetch = [&](int64_t row) {
    mu_ahead = mean[row], r_ahead = rstd[row];
#pragma unroll
    for (int i = 0; i < T::PIECES; i++)
      if (t.has(i)) x_ahead[i] = fetch8<DTYPE>(x + row * x_stride + t.first[i]), g_ahead[i] = fetch8<DTYPE>(grad + row * grad_stride + t.first[i]);
  };
  int64_t row = (int64_t)blockIdx.x * T::kTeams + t.team;
  if (row < rows) fetch(row);
  int turn = 0;
  for (; row < rows; row += step, turn ^= 1) {
    const float mu = mu_ahead, r = r_ahead;
    float z[T::PIECES][8], g[T::PIECES][8], m[2] = {0.f, 0.f};   // m: mean(g) and mean(g z)
#pragma unroll
    for (int i = 0; i < T::PIECES; i++) widen8<DTYPE>(z[i], x_ahead[i]), widen8<DTYPE>(g[i], g_ahead[i]);
#pragma unroll
    for (int i = 0; i < T::PIECES; i++) {
      float w[8];
      if (weight && t.has(i)) load8<PARAM>(w, weight + t.first[i]);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        z[i][j] = (z[i][j] - mu) * r;
        if constexpr (PARAMS) dw[i][j] += t.owns(i, j) ? g[i][j] * z[i][j] : 0.f, db[i][j] += t.owns(i, j) ? g[i][j] : 0.f;
        if (weight) g[i][j] *= w[j];
        m[0] += t.owns(i, j) ? g[i][j] : 0.f, m[1] += t.owns(i, j) ? g[i][j] * z[i][j] : 0.f;
      }
    }
    if (dx) {
      t.sums(m, part[turn]);
      m[0] *= over_n, m[1] *= over_n;
#pragma unroll
      for (int i = 0; i < T::PIECES; i++)
        if (t.has(i)) {
#pragma unroll
          for (int j = 0; j < 8; j++) g[i][j] = r * (g[i][j] - m[0] - z[i][j] * m[1]);
          store8<DTYPE>(dx + row * dx_stride + t.first[i], g[i]);
        }
    }
    if (row + step < rows) fetch(row + step);
  }
  if constexpr (PARAMS) {
    float* to = sums + (int64_t)blockIdx.x * 2 * n;
    if constexpr (T::LANES > 64) {
#pragma unroll
      for (int i = 0; i < T::PIECES; i++)
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (t.owns(i, j)) to[t.first[i] + j] = dw[i][j], to[n + t.first[i] + j] = db[i][j];
    } else {   // one team after the other adds its own to those in LDS, in the order of the teams
      for (int k = 0; k < T::kTeams; k++) {
        if (t.team == k) {
#pragma unroll
          for (int i = 0; i < T::PIECES; i++)
#pragma unroll
            for (int j = 0; j < 8; j++)
              if (t.owns(i, j)) {
                float *w = together + t.first[i] + j, *b = w + 8 * T::LANES * T::PIECES;
                *w = k ? *w + dw[i][j] : dw[i][j], *b = k ? *b + db[i][j] : db[i][j];
              }
        }
        __syncthreads();
      }
      for (int i = threadIdx.x; i < n; i += T::kThreads) to[i] = together[i], to[n + i] = together[8 * T::LANES * T::PIECES + i];
    }
  }
}

// dweight and dbias from the shares' sums: 32 columns of a workgroup, 32 threads a column that take every 32nd share each.
template <int PARAM>
__global__ __launch_bounds__(1024) void layer_norm_param_kernel(const float* __restrict__ sums, int shares, int n, typename Value<PARAM>::stored* __restrict__ dweight,
                                                                typename Value<PARAM>::stored* __restrict__ dbias) {
  __shared__ float part[32][33];
  const int column = threadIdx.x & 31, turn = threadIdx.x >> 5, at = blockIdx.x * 32 + column;   // (columns of dweight, then of dbias)
  const bool mine = at < 2 * n;
  float v = 0.f;
  if (mine) {
    int s = turn;
    for (; s + 7 * 32 < shares; s += 8 * 32) {
      float u[8];
#pragma unroll
      for (int k = 0; k < 8; k++) u[k] = sums[(int64_t)(s + 32 * k) * 2 * n + at];
#pragma unroll
      for (int k = 0; k < 8; k++) v += u[k];
    }
    for (; s < shares; s += 32) v += sums[(int64_t)s * 2 * n + at];
  }
  part[turn][column] = v;
  __syncthreads();
  if (turn > 0 || !mine) return;
  for (int k = 1; k < 32; k++) v += part[k][column];
  if (at < n) {
    if (dweight) dweight[at] = Value<PARAM>::round(v);
  } else if (dbias) {
    dbias[at - n] = Value<PARAM>::round(v);
  }
}

// ---------------------------------------------------------------- rows of fewer than eight values, or too long for registers
// A value at a time, a row read three times forward, x and dy again for each of dx and the sums: a training pass of 3000 x 20000 in
// bfloat16 takes 569 us (239 forward), 4.9 times what its bytes would; 8192 x 16384, which fit, 375.

// Sum over the 256 threads of a workgroup; every thread gets it.
__device__ __forceinline__ float workgroup_sum(float v, float* part) {
  v = wave64_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return part[0] + part[1] + part[2] + part[3];
}

template <int DTYPE, int PARAM>
__global__ __launch_bounds__(256) void layer_norm_any_kernel(const typename Value<DTYPE>::stored* __restrict__ x, int64_t x_stride, int64_t rows, int n,
                                                             const typename Value<PARAM>::stored* __restrict__ weight,
                                                             const typename Value<PARAM>::stored* __restrict__ bias, float eps,
                                                             typename Value<DTYPE>::stored* __restrict__ out, int64_t out_stride, float* __restrict__ mean,
                                                             float* __restrict__ rstd) {
  __shared__ float part[4];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const auto* from = x + row * x_stride;
    auto* to = out + row * out_stride;
    const float pivot = Value<DTYPE>::widen(from[0]);
    float s = 0.f, q = 0.f;
    for (int i = threadIdx.x; i < n; i += 256) s += Value<DTYPE>::widen(from[i]) - pivot;
    const float mu = pivot + workgroup_sum(s, part) / (float)n;
    for (int i = threadIdx.x; i < n; i += 256) {
      const float d = Value<DTYPE>::widen(from[i]) - mu;
      q += d * d;
    }
    const float r = 1.f / sqrtf(workgroup_sum(q, part) / (float)n + eps);
    for (int i = threadIdx.x; i < n; i += 256) {
      float y = (Value<DTYPE>::widen(from[i]) - mu) * r;
      if (weight) y *= Value<PARAM>::widen(weight[i]);
      if (bias) y += Value<PARAM>::widen(bias[i]);
      to[i] = Value<DTYPE>::round(y);
    }
    if (threadIdx.x == 0 && mean) mean[row] = mu, rstd[row] = r;
  }
}

template <int DTYPE, int PARAM>
__global__ __launch_bounds__(256) void layer_norm_any_dx_kernel(const typename Value<DTYPE>::stored* __restrict__ grad, int64_t grad_stride,
                                                                const typename Value<DTYPE>::stored* __restrict__ x, int64_t x_stride,
                                                                const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                const typename Value<PARAM>::stored* __restrict__ weight, int64_t rows, int n,
                                                                typename Value<DTYPE>::stored* __restrict__ dx, int64_t dx_stride) {
  __shared__ float part[4];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const auto *xs = x + row * x_stride, *gs = grad + row * grad_stride;
    const float mu = mean[row], r = rstd[row];
    float a = 0.f, b = 0.f;
    for (int i = threadIdx.x; i < n; i += 256) {
      const float g = Value<DTYPE>::widen(gs[i]) * (weight ? Value<PARAM>::widen(weight[i]) : 1.f);
      a += g, b += g * ((Value<DTYPE>::widen(xs[i]) - mu) * r);
    }
    a = workgroup_sum(a, part) / (float)n;
    b = workgroup_sum(b, part) / (float)n;
    for (int i = threadIdx.x; i < n; i += 256) {
      const float g = Value<DTYPE>::widen(gs[i]) * (weight ? Value<PARAM>::widen(weight[i]) : 1.f);
      dx[row * dx_stride + i] = Value<DTYPE>::round(r * (g - a - (Value<DTYPE>::widen(xs[i]) - mu) * r * b));
    }
  }
}

// A thread sums a column over every `shares`-th row.
template <int DTYPE>
__global__ __launch_bounds__(256) void layer_norm_any_sums_kernel(const typename Value<DTYPE>::stored* __restrict__ grad, int64_t grad_stride,
                                                                  const typename Value<DTYPE>::stored* __restrict__ x, int64_t x_stride,
                                                                  const float* __restrict__ mean, const float* __restrict__ rstd, int64_t rows, int n,
                                                                  float* __restrict__ sums) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float g = Value<DTYPE>::widen(grad[row * grad_stride + i]);
    dw += g * ((Value<DTYPE>::widen(x[row * x_stride + i]) - mean[row]) * rstd[row]), db += g;
  }
  float* to = sums + (int64_t)blockIdx.y * 2 * n;
  to[i] = dw, to[n + i] = db;
}

// ---------------------------------------------------------------- host
static int norm_check(const char* who, int64_t rows, int64_t size, int dtype, int param_dtype) {
  if (!is_value_dtype(dtype)) return fail(STK_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (param_dtype != dtype && param_dtype != STK_F32) return fail(STK_ERR_UNSUPPORTED, "%s: weight and bias have the rows' type or float32", who);
  if (rows < 0 || size < 1) return fail(STK_ERR_DIMS, "%s: %lld rows of %lld", who, (long long)rows, (long long)size);
  if (size > INT32_MAX / 4) return fail(STK_ERR_UNSUPPORTED, "%s: size exceeds 32-bit range", who);
  return STK_OK;
}

template <class Fn>
static void for_types(int dtype, int param_dtype, Fn&& fn) {
  for_dtype(dtype, [&](auto d) {
    if (param_dtype == STK_F32) fn(d, std::integral_constant<int, STK_F32>());
    else fn(d, d);
  });
}

// The teams for rows of `size` values, forward and backward with the workgroups that share the rows of a backward pass (each leaves
// 2 n fp32 sums); rows of other sizes: the kernels above that loop over a row.  float32 rows take the same teams, which were measured in
// bfloat16 only.  Backward 1024,2 has 128 registers a lane and spills 6 to 11 more (28 with bfloat16 parameters).  Times in us of
// alternatives as lanes, pieces x threads @ workgroups, bfloat16, cold:
//   16384 x 1024   forward 64,2 15.5, 256,1 22.6          backward 64,2 x512 @512 23.2, x256 @1024 23.2, @512 25.1, 256,1 x256 @1024 34.2
//   16384 x 2048   forward 256,1 31.9, 64,4 33.6          backward 64,4 x512 @256 47.8, 256,1 x256 @1024 49.0, 64,4 x512 @512 52.9
//   16384 x 4096   forward 256,2 55.6, 512,1 57.9         backward 512,1 @512 81.8, 256,2 @512 90.8, 512,1 @256 105
//   32768 x 8192   forward 512,2 203, 256,4 256, 1024,1 268   backward 1024,1 @256 316, @512 323, 256,4 @512 399, 512,2 @256 491
//   8192 x 16384   forward 1024,2 116, 512,4 142          backward 1024,2 @256 169, 512,4 @256 234
//   65536 x 512    forward 64,1 31.3                      backward 64,1 x512 @512 42.6, x256 @1024 42.9, @512 45.5
//   65536 x 64     forward 16,1 9.4, 64,1 23.0            backward 16,1 x256 @1024 12.5, @512 13.6, 64,1 x256 @1024 27
constexpr int kRegisterRow = 16384;
static bool fits_registers(int64_t size) { return size >= 8 && size <= kRegisterRow; }
template <class T, int SHARES = 0> struct Type {
  typedef T type;
  static constexpr int shares = SHARES;
};
template <bool TAIL, class Fn>
static void forward_team(int64_t size, Fn&& fn) {
  if (size <= 128) fn(Type<Team<16, 1, 256, TAIL>>());
  else if (size <= 512) fn(Type<Team<64, 1, 256, TAIL>>());
  else if (size <= 1024) fn(Type<Team<64, 2, 256, TAIL>>());
  else if (size <= 2048) fn(Type<Team<256, 1, 256, TAIL>>());
  else if (size <= 4096) fn(Type<Team<256, 2, 256, TAIL>>());
  else if (size <= 8192) fn(Type<Team<512, 2, 512, TAIL>>());
  else fn(Type<Team<1024, 2, 1024, TAIL>>());
}
template <bool TAIL, class Fn>
static void backward_team(int64_t size, Fn&& fn) {
  if (size <= 128) fn(Type<Team<16, 1, 256, TAIL>, 1024>());
  else if (size <= 512) fn(Type<Team<64, 1, 512, TAIL>, 512>());
  else if (size <= 1024) fn(Type<Team<64, 2, 512, TAIL>, 512>());
  else if (size <= 2048) fn(Type<Team<64, 4, 512, TAIL>, 256>());
  else if (size <= 4096) fn(Type<Team<512, 1, 512, TAIL>, 512>());
  else if (size <= 8192) fn(Type<Team<1024, 1, 1024, TAIL>, 256>());
  else fn(Type<Team<1024, 2, 1024, TAIL>, 256>());
}
// Shares of the sums over rows.
constexpr int kLoopShares = 128;
static int64_t shares_of(int64_t rows, int64_t size) {
  if (!fits_registers(size)) return rows < kLoopShares ? rows : kLoopShares;
  int64_t shares = 0;
  backward_team<false>(size, [&](auto t) {
    typedef decltype(t) B;
    const int64_t most = (rows + B::type::kTeams - 1) / B::type::kTeams;
    shares = most < B::shares ? most : B::shares;
  });
  return shares;
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
  hipStream_t s = static_cast<hipStream_t>(stream);
  for_types(dtype, param_dtype, [&](auto d, auto p) {
    constexpr int D = decltype(d)::value, P = decltype(p)::value;
    const auto* xs = static_cast<const typename Value<D>::stored*>(x);
    auto* to = static_cast<typename Value<D>::stored*>(out);
    const auto *w = static_cast<const typename Value<P>::stored*>(weight), *b = static_cast<const typename Value<P>::stored*>(bias);
    const auto launch = [&](auto team) {
      typedef typename decltype(team)::type T;
      const int64_t groups = (rows + T::kTeams - 1) / T::kTeams;
      hipLaunchKernelGGL((layer_norm_kernel<T, D, P>), dim3((unsigned)(groups < 65536 ? groups : 65536)), dim3(T::kThreads), 0, s, xs, x_stride, rows, (int)size, w, b, eps,
                         to, out_stride, mean, rstd);
    };
    if (!fits_registers(size))
      hipLaunchKernelGGL((layer_norm_any_kernel<D, P>), dim3((unsigned)(rows < 65536 ? rows : 65536)), dim3(256), 0, s, xs, x_stride, rows, (int)size, w, b, eps, to,
                         out_stride, mean, rstd);
    else if (size % 8) forward_team<true>(size, launch);
    else forward_team<false>(size, launch);
  });
  return check_launch(who);
}

extern "C" size_t stk_layer_norm_backward_workspace_bytes(int64_t rows, int64_t size) {
  if (rows <= 0 || size <= 0) return 0;
  return (size_t)(2 * shares_of(rows, size) * size) * sizeof(float);
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
  const int shares = (int)shares_of(rows, size), n = (int)size;   // (no rows, no shares: the sums are zeros)
  for_types(dtype, param_dtype, [&](auto d, auto p) {
    constexpr int D = decltype(d)::value, P = decltype(p)::value;
    typedef typename Value<P>::stored Param;
    const auto *g = static_cast<const typename Value<D>::stored*>(grad), *xs = static_cast<const typename Value<D>::stored*>(x);
    auto* to = static_cast<typename Value<D>::stored*>(dx);
    const Param* w = static_cast<const Param*>(weight);
    const auto launch = [&](auto team) {
      typedef typename decltype(team)::type T;
      const int64_t groups = (rows + T::kTeams - 1) / T::kTeams;
      if (params)
        hipLaunchKernelGGL((layer_norm_backward_kernel<T, D, P, true>), dim3((unsigned)shares), dim3(T::kThreads), 0, s, g, grad_stride, xs, x_stride, mean, rstd, w, rows, n,
                           to, dx_stride, sums);
      else
        hipLaunchKernelGGL((layer_norm_backward_kernel<T, D, P, false>), dim3((unsigned)(groups < 65536 ? groups : 65536)), dim3(T::kThreads), 0, s, g, grad_stride, xs,
                           x_stride, mean, rstd, w, rows, n, to, dx_stride, nullptr);
    };
    if (rows > 0 && fits_registers(size)) {
      if (size % 8) backward_team<true>(size, launch);
      else backward_team<false>(size, launch);
    } else if (rows > 0) {
      if (dx)
        hipLaunchKernelGGL((layer_norm_any_dx_kernel<D, P>), dim3((unsigned)(rows < 65536 ? rows : 65536)), dim3(256), 0, s, g, grad_stride, xs, x_stride, mean, rstd, w,
                           rows, n, to, dx_stride);
      if (params)
        hipLaunchKernelGGL((layer_norm_any_sums_kernel<D>), dim3((unsigned)((size + 255) / 256), (unsigned)shares), dim3(256), 0, s, g, grad_stride, xs, x_stride, mean,
                           rstd, rows, n, sums);
    }
    if (params)
      hipLaunchKernelGGL((layer_norm_param_kernel<P>), dim3((unsigned)((2 * size + 31) / 32)), dim3(1024), 0, s, sums, shares, n, static_cast<Param*>(dweight),
                         static_cast<Param*>(dbias));
  });
  return check_launch(who);
}
