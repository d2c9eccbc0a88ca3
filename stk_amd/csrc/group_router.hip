// stk_group_top_experts: a router's choice among groups of experts, and the gradient of the chosen weights with respect to the scores.
//   p = softmax(scores) or sigmoid(scores);   c = p + bias  (a score of -infinity: c = -infinity)
//   value of a group = the sum of its `best` largest c;   the top_groups groups of the largest values, ties to the lower group
//   chosen: the top_k experts of these groups with the largest c - without a bias the largest scores - in descending order, ties to the lower expert
//   weights_j = scale p[chosen_j]      or, normalized, divided by the sum of p over the chosen ones
// Gradient, with u_j = g_j weights_j and q_j = weights_j / scale:
//   sigmoid                ds[chosen_j] = (u_j - [normalized] q_j sum u) (1 - p_j)
//   softmax, normalized    ds[chosen_j] = u_j - q_j sum u
//   softmax                ds_i = (u_j where i = chosen_j) - p_i sum u
//
// Which experts are chosen is to be a matter of the inputs, not of how exp is computed.  Everything is computed in fp32, whose error in c is below
// 2^-19 (softmax: the sum's error counts) or 2^-21 (sigmoid) of the largest p and |bias|, and keys (below) lose another 2^-19; where two values that decide
// the choice or its order are closer than twice the error and that, 2^-17 or 2^-18, and are not of equal inputs (which are equal whatever the precision), the
// token is done again in 64 bits: one token in some hundred.  A workgroup collects its own and a wavefront takes each.  Where the order of c is that of
// the scores (no bias, and one expert decides for its group) the groups are compared by these.
//
// A token belongs to a team of 16 or 64 lanes, and expert i to its lane i % LANES, place i / LANES.  A round of the choice is a maximum over
// keys of 32 bits: the ordered bits of c with the place in the lowest four, so that a lane's maximum says whose it is; what that takes off c is
// within the margin of the 64-bit check.  A lane remembers the last of its keys that was chosen, t, and the largest key below is t plus the largest
// key - t modulo 2^32: an instruction and a half for each key and round.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "values.h"
#include "wave_scan.h"

namespace stk {

constexpr int kFewTokens = 2048;
constexpr int kGroupRouterExperts = 1024, kGroupRouterTopK = 32, kGroupRouterGroups = 64;

struct GroupRouter {
  const void* scores;
  int64_t stride, tokens;
  int experts, groups, top_groups, best, top_k;
  int sigmoid, normalize;
  float scale;
  const float* bias;
  uint32_t group_size, group_magic;   // i / group_size = i group_magic >> 22
  int32_t* chosen;
  float* weights;
};

// Value of a lane of the team (of a whole wavefront: the same lane for all).
template <class T, class Fn>
__device__ __forceinline__ T by_words(T v, Fn&& move) {
  constexpr int N = sizeof(T) / 4;
  uint32_t w[N];
  __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
  for (int i = 0; i < N; i++) w[i] = move(w[i]);
  __builtin_memcpy(&v, w, sizeof(T));
  return v;
}
template <int LANES, class T>
__device__ __forceinline__ T from_lane(T v, int lane) {
  if constexpr (LANES == 64) return by_words(v, [&](uint32_t w) { return (uint32_t)__builtin_amdgcn_readlane((int)w, lane); });
  else return __shfl(v, lane, LANES);
}
template <int LANES>
__device__ __forceinline__ bool any_of_team(bool v) {
  const uint64_t all = __ballot(v);
  if constexpr (LANES == 64) return all != 0;
  else return (all >> (threadIdx.x & 48) & 0xffffu) != 0;
}
template <int LANES>
__device__ __forceinline__ uint64_t ballot_of_team(bool v) {
  const uint64_t all = __ballot(v);
  if constexpr (LANES == 64) return all;
  else return all >> (threadIdx.x & 48) & 0xffffu;
}
template <int CONTROL>
__device__ __forceinline__ uint32_t moved_key32(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, 0xf, 0xf, true); }
// The same value for all lanes: pairs, quads, eights and sixteens meet by permutations that cost no trip to LDS, then the rows of a wavefront in their order.
template <int LANES, class T, class Fn>
__device__ __forceinline__ T reduce_team(T v, Fn&& fn) {
  v = fn(v, by_words(v, moved_key32<0xb1>)), v = fn(v, by_words(v, moved_key32<0x4e>));
  v = fn(v, by_words(v, moved_key32<0x141>)), v = fn(v, by_words(v, moved_key32<0x140>));
  if constexpr (LANES == 64) v = fn(fn(from_lane<64>(v, 0), from_lane<64>(v, 16)), fn(from_lane<64>(v, 32), from_lane<64>(v, 48)));
  return v;
}
template <int LANES>
__device__ __forceinline__ uint32_t largest_key(uint32_t v) {
  v = max(v, moved_key32<0xb1>(v)), v = max(v, moved_key32<0x4e>(v)), v = max(v, moved_key32<0x141>(v)), v = max(v, moved_key32<0x140>(v));
  if constexpr (LANES == 64) {
    uint32_t best = 0;
#pragma unroll
    for (int r = 0; r < 64; r += 16) best = max(best, (uint32_t)__builtin_amdgcn_readlane((int)v, r));
    v = best;
  }
  return v;
}

// Numbers in their order as whole numbers: -0 like 0, NaN on top, nothing at 0.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v);
  return v != v ? 0xffffffffu : v == 0.f ? 0x80000000u : u & 0x80000000u ? ~u : u | 0x80000000u;
}
// No NaN, and the way back.
__device__ __forceinline__ uint32_t ordered_number(float v) {
  const int u = (int)__float_as_uint(v + 0.f);
  return (uint32_t)u ^ ((uint32_t)(u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float number_of(uint32_t key) { return __uint_as_float(key ^ (~(uint32_t)((int)key >> 31) | 0x80000000u)); }
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v), sign = 1ull << 63;
  return v != v ? ~0ull : v == 0. ? sign : u & sign ? ~u : u | sign;
}

// exp(x), x <= 0, from the hardware's power of two (1 unit in the last place): x log2(e) is rounded, and what that loses is put back
// to first order.
__device__ __forceinline__ float exponential_of(float x) {
  constexpr float kLog2e = 1.44269504088896341f, kLog2eRest = 1.92596299112661746887e-8f, kLn2 = 0.693147180559945309f;
  const float t = x * kLog2e, rest = fmaf(x, kLog2eRest, fmaf(x, kLog2e, -t)), y = __builtin_amdgcn_exp2f(t);
  return t < -149.f ? 0.f : fmaf(y, rest * kLn2, y);
}
__device__ __forceinline__ double exponential_of(double x) { return exp(x); }
// exp(a - b), a - b <= 0, in the range of 64 bits: what a - b rounds away and what the exponent of fp32 has no room for are kept.
__device__ __forceinline__ double exponential_of_difference(float a, float b) {
#pragma clang fp contract(off)   // (t - whole is to be that of the rounded t)
  constexpr float kLog2e = 1.44269504088896341f, kLog2eRest = 1.92596299112661746887e-8f, kLn2 = 0.693147180559945309f;
  const float x = a - b, was = x - a, lost = (a - (x - was)) - (b + was);
  const float t = x * kLog2e, rest = fmaf(lost, kLog2e, fmaf(x, kLog2eRest, fmaf(x, kLog2e, -t))), whole = rintf(t), y = __builtin_amdgcn_exp2f(t - whole);
  return t < -1080.f ? 0. : ldexp((double)fmaf(y, rest * kLn2, y), (int)whole);
}
__device__ __forceinline__ double exponential_of_difference(double a, double b) { return exp(a - b); }
// 1 / (1 + exp(-s)) from the exponential of -|s|.
template <class F>
__device__ __forceinline__ F sigmoid_of(F s) {
  const F t = exponential_of(s < 0 ? s : -s);
  return (s < 0 ? t : F(1)) / (F(1) + t);
}
// The same for the choice, to within 2^-21.
__device__ __forceinline__ float sigmoid_near(float s) {
  const float t = exponential_of(-fabsf(s));
  return (s < 0 ? t : 1.f) * __builtin_amdgcn_rcpf(1.f + t);
}

// The two largest of a group.
template <class F>
struct Two {
  F first, second;
};
// Whether a comes in front of b: NaN in front of every number.
template <class F>
__device__ __forceinline__ bool in_front(F a, F b) { return a > b || (a != a && b == b); }
template <class F>
__device__ __forceinline__ void put(Two<F>& t, F v) {
  const bool top = in_front(v, t.first);
  t.second = top ? t.first : in_front(v, t.second) ? v : t.second;
  t.first = top ? v : t.first;
}

// One token in the precision of F.  from: its scores; mine: those of this lane's experts lane + LANES j.  row: LDS of the team for the c of every expert,
// and the groups' values behind them.  at, weight: what lane k < top_k is to write.  false (F = float only): two of the values that decide are too
// close for it.
template <class F, int DTYPE, int LANES, int V>
__device__ __forceinline__ bool choose(const GroupRouter& r, const typename Value<DTYPE>::stored* from, const float (&mine)[V], const float (&bias)[V], F* row, int lane, int& at, float& weight) {
  constexpr bool kFast = std::is_same<F, float>::value;
  const F kNone = -INFINITY;
  F c[V];
  F top = 0, total = 1, largest_p = 0, largest_b = 0;
  bool strange = false;
  // (behind the last expert are scores of -infinity, whose share is 0)
  if (!r.sigmoid) {
    F most = kNone;
#pragma unroll
    for (int j = 0; j < V; j++) most = in_front((F)mine[j], most) ? (F)mine[j] : most;
    top = reduce_team<LANES>(most, [](F a, F b) { return in_front(a, b) ? a : b; });
    total = 0;
    const F shift = top == kNone ? F(0) : top;   // (a row of masked experts)
#pragma unroll
    for (int j = 0; j < V; j++) total += exponential_of((F)mine[j] - shift);
    total = reduce_team<LANES>(total, [](F a, F b) { return a + b; });
  }
  const auto share = [&](F s) { return top == kNone ? F(0) : exponential_of(s - top) / total; };   // a softmax's p of a score
  // without a bias experts are in the order of the scores, in which sigmoids of 1 are told apart, and so are groups of which the best expert decides
  const bool by_score = r.bias == nullptr, groups_by_score = by_score && r.best == 1;
  if (groups_by_score) {
#pragma unroll
    for (int j = 0; j < V; j++) {
      c[j] = (F)mine[j];
      if constexpr (kFast) strange |= !(mine[j] < INFINITY);
    }
  } else {
    if (r.sigmoid) {
#pragma unroll
      for (int j = 0; j < V; j++) {
        if constexpr (kFast) c[j] = sigmoid_near(mine[j]);
        else c[j] = sigmoid_of((F)mine[j]);
      }
    } else {
      const F one_by = top == kNone ? F(0) : F(1) / total, shift = top == kNone ? F(0) : top;
#pragma unroll
      for (int j = 0; j < V; j++) {
        if constexpr (kFast) c[j] = exponential_of(mine[j] - shift) * one_by;
        else c[j] = share((F)mine[j]);
      }
    }
    uint32_t most_p = 0, most_b = 0;   // as bits: of magnitudes, NaN and infinities are the largest
#pragma unroll
    for (int j = 0; j < V; j++) {
      if constexpr (kFast) most_p = max(most_p, __float_as_uint(c[j])), most_b = max(most_b, __float_as_uint(bias[j]) & 0x7fffffffu);
      const F sum = c[j] + (F)bias[j];
      c[j] = mine[j] == -INFINITY ? kNone : sum;
    }
    // (from 2^126 on a group's sum may leave fp32)
    if constexpr (kFast) strange = max(most_p, most_b) >= 0x7e800000u, largest_p = __uint_as_float(most_p), largest_b = __uint_as_float(most_b);
  }
  if (r.top_groups < r.groups) {
#pragma unroll
    for (int j = 0; j < V; j++) row[lane + LANES * j + ((lane + LANES * j) >> 5)] = c[j];   // (groups of 32 start on different banks)
  }
  asm volatile("" : : : "memory");   // (a team lies in one wavefront, whose LDS accesses are made in order)
  F margin = 0;
  if constexpr (kFast) {
    // infinities and NaN among them: the fp32 comparisons below say nothing
    if (any_of_team<LANES>(strange)) return false;
    largest_p = reduce_team<LANES>(largest_p, [](F a, F b) { return fmaxf(a, b); });
    if (r.bias) largest_b = reduce_team<LANES>(largest_b, [](F a, F b) { return fmaxf(a, b); });
    // (the absolute part: a p below the normal numbers counts as 0 here, off by up to 2^-126, and a group has two)
    margin = fmaf(largest_p + largest_b, r.sigmoid ? 0x1p-18f : 0x1p-17f, 0x1p-125f);
  }
  // ------------------------------------------------------------ groups
  uint64_t kept = ~0ull;
  if (r.top_groups < r.groups) {
    // a group's lanes look through it together
    int along = 1;
    while (2 * along * r.groups <= LANES) along *= 2;
    const int group = lane / along, size = (int)r.group_size;
    Two<F> two = {kNone, kNone};
    if constexpr (kFast) {
      // (no NaN here; four of them are on their way from LDS together)
      const int base = min(group, r.groups - 1) * size, end = group < r.groups ? size : 0;
      for (int i0 = lane % along; i0 < end; i0 += 4 * along) {
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const int i = i0 + q * along, e = base + min(i, size - 1);
          v[q] = row[e + (e >> 5)];
          if (i >= end) v[q] = kNone;
        }
#pragma unroll
        for (int q = 0; q < 4; q++) two.second = fmaxf(two.second, fminf(two.first, v[q])), two.first = fmaxf(two.first, v[q]);
      }
    } else if (group < r.groups) {
      for (int i = lane % along; i < size; i += along) {
        const int e = group * size + i;
        put(two, row[e + (e >> 5)]);
      }
    }
    for (int d = 1; d < along; d *= 2) {
      const Two<F> other = {__shfl_xor(two.first, d, LANES), __shfl_xor(two.second, d, LANES)};
      put(two, other.first), put(two, other.second);
    }
    const F value = group < r.groups ? r.best == 2 ? two.first + two.second : two.first : kNone;
    const bool first_lane = lane % along == 0 && group < r.groups;
    kept = 0;
    if constexpr (kFast) {
      // (ordered values of numbers are above 0, infinities below included)
      uint32_t key = first_lane ? ordered(value) : 0u;
      float last = kNone;
      for (int k = 0; k < r.top_groups; k++) {
        const uint32_t best = largest_key<LANES>(key);
        const int who = __builtin_ctzll(ballot_of_team<LANES>(key == best));
        kept |= 1ull << (who / along);
        if (k == r.top_groups - 1) last = from_lane<LANES>(value, who);
        if (lane == who) key = 0u;
      }
      // one that is not kept and may count as much
      if (any_of_team<LANES>(!groups_by_score && key != 0u && last - value <= 2 * margin)) return false;
    } else {
      int rank = 0;
      for (int g = 0; g < r.groups; g++) {
        const F other = from_lane<LANES>(value, g * along);
        rank += in_front(other, value) || ((other == value || (other != other && value != value)) && g < group) ? 1 : 0;
      }
      // bits of the groups: those of their first lanes
      const uint64_t bits = ballot_of_team<LANES>(first_lane && rank < r.top_groups);
      for (int g = 0; g < r.groups; g++) kept |= (bits >> (g * along) & 1ull) << g;
    }
  }
  // ------------------------------------------------------------ experts
  typedef std::conditional_t<kFast, uint32_t, uint64_t> key_t;
  key_t key[V];
#pragma unroll
  for (int j = 0; j < V; j++) {
    const uint32_t e = lane + LANES * j;
    const F v = by_score ? (F)mine[j] : c[j];
    if constexpr (kFast) key[j] = (ordered_number(v) & ~15u) | (15u - j);
    else key[j] = ordered(v);
    if ((int)e >= r.experts) key[j] = 0u;
  }
  if (r.top_groups < r.groups) {
#pragma unroll
    for (int j = 0; j < V; j++) {   // (behind the last expert it is 0 already)
      const uint32_t g = (lane + LANES * j) * r.group_magic >> 22;
      if constexpr (kFast && LANES == 16) key[j] &= (uint32_t)__builtin_amdgcn_sbfe((int)kept, g, 1);   // (at most 16 groups)
      else key[j] = kept >> (g & 63u) & 1ull ? key[j] : 0u;
    }
  }
  at = 0;
  uint32_t mark = 0;   // the last of this lane's keys that was chosen
  for (int k = 0; k < r.top_k; k++) {
    key_t best = 0;
    int place = 0, who;
    if constexpr (kFast) {
#pragma unroll
      for (int j = 0; j < V; j++) best = max(best, key[j] - mark);
      best += mark;
      if (best - 1u >= mark - 1u) best = 0u;   // (none below: the largest of all came round)
      const key_t all = largest_key<LANES>(best);
      who = __builtin_ctzll(ballot_of_team<LANES>(best == all));
      place = 15 - (int)(all & 15u);
      if (lane == who) mark = all;
    } else {
#pragma unroll
      for (int j = 0; j < V; j++) best = max(best, key[j]);
      // the largest by halves of 32 bits; of equal ones the lowest expert: the lowest place, then the lowest lane
      const uint32_t high = largest_key<LANES>((uint32_t)(best >> 32)), low = largest_key<LANES>((uint32_t)(best >> 32) == high ? (uint32_t)best : 0u);
      const key_t all = (key_t)high << 32 | low;
      int first = V;
#pragma unroll
      for (int j = V - 1; j >= 0; j--) first = key[j] == all ? j : first;
      place = 16 - (int)largest_key<LANES>(first < V ? 16u - first : 0u);
      who = __builtin_ctzll(ballot_of_team<LANES>(first == place));
#pragma unroll
      for (int j = 0; j < V; j++) key[j] = lane == who && j == place ? 0u : key[j];
    }
    if (lane == k) at = who + LANES * place;
  }
  const bool is = lane < r.top_k;
  const F s_at = is ? (F)Value<DTYPE>::widen(from[at]) : kNone;
  F share_of_one = 1, t_at = 1;   // sigmoid: 1 / (1 + t), t = exp(-|s|)
  if (r.sigmoid) t_at = exponential_of(s_at < 0 ? s_at : -s_at), share_of_one = F(1) / (F(1) + t_at);
  if constexpr (kFast) {
    const float b_at = r.bias ? r.bias[at] : 0.f, c_at = by_score ? s_at : s_at == kNone ? kNone : (r.sigmoid ? (s_at < 0 ? t_at : 1.f) * share_of_one : share(s_at)) + b_at;
    // the order of the chosen
    const float next_c = __shfl_down(c_at, 1, LANES), next_s = __shfl_down(s_at, 1, LANES), next_b = __shfl_down(b_at, 1, LANES);
    // (16 numbers share a key: of scores below the normal numbers these are 2^-145 apart at most, whatever their size)
    const auto too_close = [&](float a, float b) { return fabsf(a - b) <= (by_score ? fmaf(fminf(fabsf(a), fabsf(b)), 0x1p-18f, 0x1p-145f) : margin); };
    if (any_of_team<LANES>(lane < r.top_k - 1 && too_close(c_at, next_c) && !(s_at == next_s && b_at == next_b))) return false;
    // the last of them and those that are not chosen (whose keys tell c to 2^-19 of it)
    const float c_last = from_lane<LANES>(c_at, r.top_k - 1);
    uint32_t rest = 0;   // the lane's largest that is not chosen
#pragma unroll
    for (int j = 0; j < V; j++) rest = max(rest, key[j] - mark);
    rest += mark;
    if (any_of_team<LANES>(rest - 1u < mark - 1u && too_close(number_of(rest & ~15u), c_last))) {   // of equal inputs?
      const float s_last = from_lane<LANES>(s_at, r.top_k - 1), b_last = from_lane<LANES>(b_at, r.top_k - 1);
      bool wrong = false;
#pragma unroll
      for (int j = 0; j < V; j++)
        if (key[j] - 1u < mark - 1u && too_close(number_of(key[j] & ~15u), c_last)) {
          const int e = lane + LANES * j;
          wrong |= !(Value<DTYPE>::widen(from[e]) == s_last && (by_score || r.bias[e] == b_last));
        }
      if (any_of_team<LANES>(wrong)) return false;
    }
  }
  // The weights.  p leaves fp32 at scores of -87 (of a softmax: below the largest), and a sum of such p with it; p / exp(base), with the largest of the
  // chosen scores (of sigmoids: or 0) as base, has the same shares and does not.  A row whose chosen p are 0 in 64 bits has no weights.
  constexpr float kNothing = -745.14f;   // exp of less rounds to 0 in 64 bits
  const auto add = [](F a, F b) { return a + b; };
  F base = r.sigmoid ? F(0) : top;
  bool nothing = false;
  if (r.normalize) {
    const F most = reduce_team<LANES>(s_at, [](F a, F b) { return in_front(a, b) ? a : b; });
    nothing = (r.sigmoid ? most : most - top) < kNothing;
    base = !r.sigmoid || most < 0 ? most : F(0);
  }
  nothing = (nothing || base == kNone) && total == total;   // (masked experts; a softmax with a NaN or +infinity in its row is NaN throughout)
  const F from_base = r.sigmoid && !(s_at < 0) ? F(0) : s_at;
  const double power = exponential_of_difference(from_base, base);
  F whole = r.sigmoid ? F(1) : total;
  if (r.normalize) {
    const F sum = reduce_team<LANES>((F)power * share_of_one, add);
    whole = total == total ? sum : total;
  }
  F by;   // (1 / whole, in fp32 to one unit in the last place)
  if constexpr (kFast) by = share_of_one * __builtin_amdgcn_rcpf(whole);
  else by = share_of_one / whole;
  weight = nothing ? 0.f : (float)(power * ((double)by * (double)r.scale));
  return true;
}

template <int DTYPE, int LANES, int V>
__device__ __forceinline__ void load_scores(float (&mine)[V], const typename Value<DTYPE>::stored* from, int lane, int experts) {
#pragma unroll
  for (int j = 0; j < V; j++) mine[j] = Value<DTYPE>::widen(from[min(lane + LANES * j, experts - 1)]);   // (all on their way together)
#pragma unroll
  for (int j = 0; j < V; j++) mine[j] = lane + LANES * j < experts ? mine[j] : -INFINITY;
}
template <int LANES, int V>
__device__ __forceinline__ void load_bias(float (&bias)[V], const GroupRouter& r, int lane) {
#pragma unroll
  for (int j = 0; j < V; j++) bias[j] = 0.f;
  if (r.bias) {
#pragma unroll
    for (int j = 0; j < V; j++) bias[j] = r.bias[min(lane + LANES * j, r.experts - 1)];
  }
}
__device__ __forceinline__ void write_choice(const GroupRouter& r, int64_t t, int lane, int at, float weight) {
  if (lane < r.top_k) r.chosen[t * r.top_k + lane] = at, r.weights[t * r.top_k + lane] = weight;
}
template <int DTYPE, int LANES, int V>
__global__ __launch_bounds__(256) void group_top_experts_kernel(GroupRouter r) {
  typedef typename Value<DTYPE>::stored stored;
  constexpr int kTeams = 256 / LANES, kExperts = LANES * V, kRow = kExperts + kExperts / 32 + 1, kWide = (kExperts + 63) / 64;
  __shared__ union {
    float fast[kTeams][kRow];
    double wide[4][64 * kWide + 2 * kWide + 1];
  } rows;
  __shared__ int again[kTeams], agains;
  const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES, wave = threadIdx.x / 64, place = threadIdx.x & 63;
  const int64_t first = (int64_t)blockIdx.x * kTeams;   // (a grid for all tokens: what a loop keeps of the lanes' experts takes more registers than the choice)
  if (threadIdx.x == 0) agains = 0;
  __syncthreads();
  if (first + team < r.tokens) {
    const stored* from = static_cast<const stored*>(r.scores) + (first + team) * r.stride;
    float mine[V], bias[V], weight;
    int at;
    load_scores<DTYPE, LANES>(mine, from, lane, r.experts), load_bias<LANES>(bias, r, lane);
    if (choose<float, DTYPE, LANES, V>(r, from, mine, bias, rows.fast[team], lane, at, weight)) write_choice(r, first + team, lane, at, weight);
    else if (lane == 0) again[atomicAdd(&agains, 1)] = team;
  }
  __syncthreads();
  for (int i = wave; i < agains; i += 4) {
    const int64_t t = first + again[i];
    const stored* from = static_cast<const stored*>(r.scores) + t * r.stride;
    float mine[kWide], bias[kWide], weight;
    int at;
    load_scores<DTYPE, 64>(mine, from, place, r.experts), load_bias<64>(bias, r, place);
    choose<double, DTYPE, 64, kWide>(r, from, mine, bias, rows.wide[wave], place, at, weight);
    write_choice(r, t, place, at, weight);
    asm volatile("" : : : "memory");   // (a team lies in one wavefront, whose LDS accesses are made in order)
  }
}

// The gradient of a token's row goes through LDS: zeros or what every expert gets, the chosen experts' own terms on top, then out.
template <int DTYPE, int LANES, int V>
__global__ __launch_bounds__(256) void group_top_experts_backward_kernel(GroupRouter r, const float* __restrict__ grad, typename Value<DTYPE>::stored* __restrict__ out,
                                                                         int64_t out_stride) {
  typedef typename Value<DTYPE>::stored stored;
  __shared__ float rows[256 / LANES][LANES * V];
  const int lane = threadIdx.x % LANES;
  float* row = rows[threadIdx.x / LANES];
  const auto add = [](float a, float b) { return a + b; };
  const int64_t t = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (t >= r.tokens) return;
  const stored* from = static_cast<const stored*>(r.scores) + t * r.stride;
  float w = 0.f, u = 0.f;
  int at = -1;
  if (lane < r.top_k) {
    w = r.weights[t * r.top_k + lane], at = r.chosen[t * r.top_k + lane];
    u = grad[t * r.top_k + lane] * w;
  }
  const float all = reduce_team<LANES>(u, add);
  float mine[V];
#pragma unroll
  for (int j = 0; j < V; j++) mine[j] = 0.f;
  if (!r.sigmoid && !r.normalize) {
    float most = -INFINITY, total = 0.f;
    load_scores<DTYPE, LANES>(mine, from, lane, r.experts);
#pragma unroll
    for (int j = 0; j < V; j++) most = in_front(mine[j], most) ? mine[j] : most;
    most = reduce_team<LANES>(most, [](float a, float b) { return in_front(a, b) ? a : b; });
#pragma unroll
    for (int j = 0; j < V; j++) {
      mine[j] = most == -INFINITY ? 0.f : exponential_of(mine[j] - most);
      total += mine[j];
    }
    total = reduce_team<LANES>(total, add);
#pragma unroll
    for (int j = 0; j < V; j++) mine[j] = most == -INFINITY ? 0.f : -(mine[j] / total) * all;
  }
#pragma unroll
  for (int j = 0; j < V; j++) row[lane + LANES * j] = mine[j];
  asm volatile("" : : : "memory");   // (a team lies in one wavefront, whose LDS accesses are made in order)
  if ((unsigned)at < (unsigned)r.experts) {
    float own = r.normalize ? u - w / r.scale * all : u;
    if (r.sigmoid) own *= sigmoid_of(-Value<DTYPE>::widen(from[at]));
    row[at] += own;
  }
  asm volatile("" : : : "memory");
#pragma unroll
  for (int j = 0; j < V; j++)
    if (lane + LANES * j < r.experts) out[t * out_stride + lane + LANES * j] = Value<DTYPE>::round(row[lane + LANES * j]);
}

// Teams of 16 lanes have a lane for every choice, and for every group, where these are few.  Where there are few tokens a wavefront each is sooner done:
// the top 8 of 256 in groups for 2048 tokens 12.1 us, with teams 13.1; for 16384 teams 21 (16.8 MB of scores are 3.4 us: bound by what the choice
// executes, some 1500 instructions for a wavefront's four tokens, and by the tokens that are done again, 7 us where a workgroup has one).
template <class Fn>
static void for_team(const GroupRouter& r, Fn&& fn) {
  typedef std::integral_constant<int, 16> Sixteen;
  typedef std::integral_constant<int, 64> Wave;
  if (r.top_k <= 16 && r.groups <= 16 && r.experts <= 256 && r.tokens > kFewTokens) {
    if (r.experts <= 64) fn(Sixteen(), std::integral_constant<int, 4>());
    else if (r.experts <= 128) fn(Sixteen(), std::integral_constant<int, 8>());
    else if (r.experts <= 192) fn(Sixteen(), std::integral_constant<int, 12>());
    else fn(Sixteen(), std::integral_constant<int, 16>());
  } else if (r.experts <= 256) fn(Wave(), std::integral_constant<int, 4>());
  else if (r.experts <= 512) fn(Wave(), std::integral_constant<int, 8>());
  else fn(Wave(), std::integral_constant<int, 16>());
}
// fn(first token, how many, grid): as many launches as it takes, since one may have less than 2^32 threads.
constexpr int64_t kTokensOfLaunch = 1 << 24;
template <class Fn>
static void for_launches(int64_t tokens, int lanes, Fn&& fn) {
  for (int64_t first = 0; first < tokens; first += kTokensOfLaunch) {
    const int64_t here = std::min(tokens - first, kTokensOfLaunch);
    fn(first, here, dim3((unsigned)((here + 256 / lanes - 1) / (256 / lanes))));
  }
}
// r without its first tokens.
template <class T>
static GroupRouter part_of(GroupRouter r, int64_t first, int64_t here) {
  r.scores = static_cast<const T*>(r.scores) + first * r.stride, r.tokens = here;
  r.chosen += first * r.top_k, r.weights += first * r.top_k;
  return r;
}
static int group_router_check(const char* who, GroupRouter& r, int64_t experts, int dtype) {
  if (!is_value_dtype(dtype)) return fail(STK_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (r.tokens < 0 || experts < 1 || r.groups < 1 || experts % r.groups) return fail(STK_ERR_DIMS, "%s: %lld experts in %d groups", who, (long long)experts, r.groups);
  if (experts > kGroupRouterExperts || r.top_k > kGroupRouterTopK || r.groups > kGroupRouterGroups)
    return fail(STK_ERR_UNSUPPORTED, "%s: at most %d experts, %d groups, the top %d", who, kGroupRouterExperts, kGroupRouterGroups, kGroupRouterTopK);
  const int64_t size = experts / r.groups;
  if (r.top_groups < 1 || r.top_groups > r.groups || r.top_k < 1 || r.top_k > r.top_groups * size)
    return fail(STK_ERR_DIMS, "%s: the top %d experts of the top %d groups of %lld", who, r.top_k, r.top_groups, (long long)size);
  if (r.best < 1 || r.best > 2 || r.best > size) return fail(STK_ERR_DIMS, "%s: a group's value from its best %d of %lld experts", who, r.best, (long long)size);
  if (!(r.scale - r.scale == 0.f) || r.scale == 0.f) return fail(STK_ERR_DIMS, "%s: scale %g", who, (double)r.scale);
  if (r.tokens > INT32_MAX / r.top_k) return fail(STK_ERR_UNSUPPORTED, "%s: size exceeds 32-bit range", who);
  r.experts = (int)experts, r.group_size = (uint32_t)size, r.group_magic = (uint32_t)(((1u << 22) + size - 1) / size);
  return STK_OK;
}

}  // namespace stk

using namespace stk;

extern "C" int stk_group_top_experts(const void* scores, int64_t tokens, int64_t experts, int64_t stride, int groups, int top_groups, int best, int top_k,
                                     int sigmoid, const float* bias, int normalize, float scale, int32_t* chosen, float* weights, int dtype, stk_stream_t stream) {
  const char* who = "stk_group_top_experts";
  GroupRouter r = {scores, stride, tokens, 0, groups, top_groups, best, top_k, sigmoid, normalize, scale, bias, 0, 0, chosen, weights};
  if (int rc = group_router_check(who, r, experts, dtype)) return rc;
  if (tokens == 0) return STK_OK;
  if (!scores || !chosen || !weights) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (stride < 0) return fail(STK_ERR_DIMS, "%s: stride %lld", who, (long long)stride);
  for_dtype(dtype, [&](auto d) {
    typedef typename Value<d()>::stored T;
    for_team(r, [&](auto lanes, auto v) {
      constexpr int D = decltype(d)::value, L = decltype(lanes)::value, V = decltype(v)::value;
      for_launches(tokens, L, [&](int64_t first, int64_t here, dim3 grid) {
        hipLaunchKernelGGL((group_top_experts_kernel<D, L, V>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), part_of<T>(r, first, here));
      });
    });
  });
  return check_launch(who);
}

extern "C" int stk_group_top_experts_backward(const void* scores, int64_t stride, const int32_t* chosen, const float* weights, const float* grad, int64_t tokens,
                                              int64_t experts, int top_k, int sigmoid, int normalize, float scale, void* dscores, int64_t dscores_stride, int dtype,
                                              stk_stream_t stream) {
  const char* who = "stk_group_top_experts_backward";
  GroupRouter r = {scores, stride, tokens, 0, 1, 1, 1, top_k, sigmoid, normalize, scale, nullptr, 0, 0, const_cast<int32_t*>(chosen), const_cast<float*>(weights)};
  if (int rc = group_router_check(who, r, experts, dtype)) return rc;
  if (tokens == 0) return STK_OK;
  if (!scores || !chosen || !weights || !grad || !dscores) return fail(STK_ERR_DIMS, "%s: missing pointer", who);
  if (stride < 0 || dscores_stride < experts) return fail(STK_ERR_DIMS, "%s: strides %lld, %lld", who, (long long)stride, (long long)dscores_stride);
  for_dtype(dtype, [&](auto d) {
    typedef typename Value<d()>::stored T;
    for_team(r, [&](auto lanes, auto v) {
      constexpr int D = decltype(d)::value, L = decltype(lanes)::value, V = decltype(v)::value;
      for_launches(tokens, L, [&](int64_t first, int64_t here, dim3 grid) {
        hipLaunchKernelGGL((group_top_experts_backward_kernel<D, L, V>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), part_of<T>(r, first, here),
                           grad + first * r.top_k, static_cast<T*>(dscores) + first * dscores_stride, dscores_stride);
      });
    });
  });
  return check_launch(who);
}
