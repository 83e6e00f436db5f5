// Routing of tokens to experts and the plan of their rows (tx_experts_route).
//
// Per token: scores s = softmax(l) or 1 / (1 + e^-l) of its logits l, the choice by c = s + bias (the
// largest first, ties to the lower index), with groups only among the groups whose best one or two c have
// the largest sums; the weights are the chosen experts' s, divided by their sum where asked, times scale.
// The plan lists the pairs token * top_k + j by expert, ascending inside an expert: a stable counting sort.
//
// kLanes lanes take a token, each with `per_lane` (at most V) consecutive experts.  A lane sorts its
// candidates once, as 32-bit keys whose lowest bits name the expert of the lane, and each round takes the
// largest head: 2 instructions a comparison, and no search for what won.  The bits that the name covers are
// looked at where they matter: the choice is that of exact arithmetic, and a token with two neighbours in
// the order that the keys do not tell apart (or, where c is computed, closer than fp32's error) is chosen
// again by choose_exact: in fp32, and where that cannot tell either, with scores in 64 bits.
//
// The plan: a warp takes tokens side by side and counts its pairs by expert as it goes, which gives a pair
// its rank among the warp's; place_kernel adds what lies before, of the warps and blocks before it.  A few
// tokens are one block, which does both.
//
// Bound: instructions and their latency, and place_kernel (10 to 12 us), each block of which sums the counts of
// all runs.  Measured: 65536 tokens of 128 bf16 logits, 8 of each, 24.6 us (HBM would take 3.8; 28.7 with
// place_kernel launched behind the runs and its pairs loaded behind the counts); 16384 tokens of 256, 8 of each
// from 4 in 8 groups, with a bias, 31 us (2.9), from 4 in 8 by softmax with a bias, where every doubt takes
// the exact choice, 102, from 20 in 64 groups that cut through lanes 313; 8 tokens of 64, one launch, 9.2.  With
// a round for each chosen expert, in place of the lanes' eight largest together, the first took 50 us, the second
// 48; the rounds that are left: 16384 tokens, 12 of 256 in groups, 65 us, 16 of 128 41; 8192 tokens, 8 of
// 1024 105, 32 of 1024 289.
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/tessattn.h"
#include "common.cuh"
#include "kernels.h"

namespace tx {
namespace {

constexpr uint32_t kFull = 0xffffffffu, kNone = 0xffffffffu;
constexpr uint32_t kMaxK = 32;
constexpr int kMostWarps = 32;  // of a block

// Values as unsigned integers of the same order.  Closed experts are -inf, below kLowest; of a token with a NaN
// the experts are chosen by choose_exact.
constexpr uint32_t kLowest = 0x00800000u;  // the key of fp32's lowest value
__device__ __forceinline__ uint32_t key_of(float c) {
  const uint32_t u = __float_as_uint(c + 0.f);  // -0 as 0
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

constexpr float kLog2e = 1.44269504088896341f;
// The hardware exponential (2^-22) and reciprocal (2^-23).
__device__ __forceinline__ float quick_exp(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * kLog2e));
  return y;
}
__device__ __forceinline__ float quick_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sigmoid(float l) { return quick_rcp(1.f + quick_exp(-l)); }
// e^x of x <= 0 in 64 bits without a branch, so that a lane's many overlap: x = k ln 2 + r, with ln 2 as the
// nearest double and what that leaves, the Taylor series of e^r to r^13 (|r| < 0.35: 4e-18 is left), and 2^k in
// two steps, of which the second rounds where the value is subnormal.  (e^-746 is 0.)
__device__ __forceinline__ double exp_of(double x) {
  const double z = fmax(x, -746.0), k = rint(z * 1.4426950408889634);
  const double r = fma(k, -2.3190468138462996e-17, fma(k, -0.6931471805599453, z));
  double y = 1.0 / 6227020800.0;
  y = fma(y, r, 1.0 / 479001600.0);
  y = fma(y, r, 1.0 / 39916800.0);
  y = fma(y, r, 1.0 / 3628800.0);
  y = fma(y, r, 1.0 / 362880.0);
  y = fma(y, r, 1.0 / 40320.0);
  y = fma(y, r, 1.0 / 5040.0);
  y = fma(y, r, 1.0 / 720.0);
  y = fma(y, r, 1.0 / 120.0);
  y = fma(y, r, 1.0 / 24.0);
  y = fma(y, r, 1.0 / 6.0);
  y = fma(y, r, 0.5);
  y = fma(y, r, 1.0);
  y = fma(y, r, 1.0);
  y = __longlong_as_double(__double_as_longlong(y) + ((long long)((int)k + 600) << 52)) * 0x1p-600;
  return x != x ? x : y;
}
// 1 / (1 + e^-l): the reciprocal by Newton's steps from the hardware's.
__device__ __forceinline__ double sigmoid(double l) {
  const double t = exp_of(-fabs(l)), d = 1.0 + t;  // 1 .. 2
  double y = (double)quick_rcp((float)d);
  y = fma(y, fma(-d, y, 1.0), y);
  y = fma(y, fma(-d, y, 1.0), y);
  return l < 0 ? t * y : y;
}

template <int kLanes, typename S>
__device__ __forceinline__ S lanes_sum(S v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
template <int kLanes>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
template <int kLanes>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  if constexpr (kLanes == 32) {
    return __reduce_max_sync(kFull, v);
  } else {
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(kFull, v, o));
    return v;
  }
}

__device__ __forceinline__ float logit_at(const RouteProblem &p, size_t token, uint32_t e) {
  const size_t at = token * p.ld + e;
  return p.logits_dtype == TX_BF16 ? bf16_bits_to_f32(static_cast<const uint16_t *>(p.logits)[at])
                                   : static_cast<const float *>(p.logits)[at];
}

// What two fp32 scores together may be off by.  Softmax: the sum over V values and lanes, the exponential's
// 4 units of 2^-24 and its argument's rounding, the reciprocal and the product make (V + 16) 2^-24 of a score,
// and none is above 1 / sum.  Sigmoid: 2^-21.4 (a quarter of the exponential's error, the sum's and the
// reciprocal's rounding).
template <int V>
__device__ __forceinline__ float score_tolerance(bool softmax, float inv_sum) {
  return softmax ? (float)((V + 16) * 1.1920929e-7f) * inv_sum : 7.2e-7f;
}

// A group's sum is off by the rounding of both its terms, 2^-24 of each (s + bias) however little of them the
// sum leaves, and of itself, besides what the scores are off by.  So two sums are told apart beyond 3 of the
// scores' tolerances and 4 roundings of the larger terms: kSumRoundings of |best| + |second|.
constexpr float kSumRoundings = 2.4e-7f;
__device__ __forceinline__ float terms_of(float best, float second, bool both) {
  return fabsf(best) + (both ? fabsf(second) : 0.f);
}

// keep_groups for groups that cut through lanes: one after the other over all lanes.
template <int kLanes, int V>
__device__ __noinline__ uint32_t keep_any_groups(const RouteProblem &p, uint32_t sub, uint32_t slot,
                                                 const float (&c)[V], float tol, bool *near) {
  const float none = -INFINITY;
  const uint32_t per = p.experts / p.groups;
  auto sum_of = [&](uint32_t g, float *terms) {
    float a = none, b = none;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t e = sub * p.per_lane + i;
      const float v = i < (int)p.per_lane && e >= g * per && e < (g + 1) * per ? c[i] : none;
      b = fmaxf(b, fminf(a, v));
      a = fmaxf(a, v);
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) {
      const float x = __shfl_xor_sync(kFull, a, o), y = __shfl_xor_sync(kFull, b, o);
      b = fmaxf(fminf(a, x), fmaxf(b, y));
      a = fmaxf(a, x);
    }
    const bool both = p.group_best > 1 && b > none;
    *terms = terms_of(a, b, both);
    return both ? a + b : a;
  };
  // The lane keeps the sums of groups sub, sub + kLanes, ...: 64 groups at most.
  constexpr int kSums = 64 / kLanes;
  float sums[kSums], size[kSums];
  uint32_t before[kSums];
#pragma unroll
  for (int m = 0; m < kSums; ++m) {
    sums[m] = none;
    size[m] = 0.f;
    before[m] = 0;
  }
  for (uint32_t g = 0; g < p.groups; ++g) {
    float terms;
    const float s = sum_of(g, &terms);
#pragma unroll
    for (int m = 0; m < kSums; ++m)
      if (g == sub + m * kLanes) {
        sums[m] = s;
        size[m] = terms;
      }
  }
  for (uint32_t h = 0; h < p.groups; ++h) {
    float other = none;
#pragma unroll
    for (int m = 0; m < kSums; ++m)
      if (h / kLanes == m) other = sums[m];
    other = __shfl_sync(kFull, other, slot * kLanes + h % kLanes);
#pragma unroll
    for (int m = 0; m < kSums; ++m)
      before[m] += other > sums[m] || (other == sums[m] && h < sub + m * kLanes);
  }
  // What a sum that is kept may come down to, and one that is left out up to.
#pragma unroll
  for (int m = 0; m < kSums; ++m) {
    const float off = size[m] * (0.5f * kSumRoundings);
    if (sums[m] > none) sums[m] += before[m] < p.top_groups ? -off : off;
  }
  uint32_t mask = 0;
  float low = INFINITY, high = none;  // the lowest of those kept, the highest of those left out
  for (uint32_t g = 0; g < p.groups; ++g) {
    float s = none;
    uint32_t n = 0;
#pragma unroll
    for (int m = 0; m < kSums; ++m)
      if (g / kLanes == m) {
        s = sums[m];
        n = before[m];
      }
    s = __shfl_sync(kFull, s, slot * kLanes + g % kLanes);
    n = __shfl_sync(kFull, n, slot * kLanes + g % kLanes);
    if (n < p.top_groups) {
      low = fminf(low, s);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint32_t e = sub * p.per_lane + i;
        if (e >= g * per && e < (g + 1) * per) mask |= 1u << i;
      }
    } else {
      high = fmaxf(high, s);
    }
  }
  if (high > none) *near |= !(low - high > 3.f * tol);
  return mask;
}
// Whether the lane's experts lie in a group that stays, bit i for its i-th; c[i] is -inf where closed or
// NaN, top the largest logit of softmax scores.  near: whether a sum that stays and one that does not are
// closer than fp32 tells, unless that is settled here.
template <int kLanes, int V>
__device__ __forceinline__ uint32_t keep_groups(const RouteProblem &p, uint32_t sub, uint32_t slot,
                                                const float (&c)[V], float tol, size_t token, float top,
                                                bool *near) {
  const float none = -INFINITY;
  if (p.group_lanes) {
    // A group is group_lanes lanes: the best two of a lane, then of its group, then the group's place among
    // the others.
    float a = none, b = none;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      b = fmaxf(b, fminf(a, c[i]));
      a = fmaxf(a, c[i]);
    }
    const uint32_t g = sub / p.group_lanes, at = sub - g * p.group_lanes;
    const uint32_t base = slot * kLanes + g * p.group_lanes;
    float best = a, second = b;
    for (uint32_t t = 1; t < p.group_lanes; ++t) {
      const uint32_t from = at + t < p.group_lanes ? at + t : at + t - p.group_lanes;
      const float x = __shfl_sync(kFull, a, (base + from) & 31);
      const float y = __shfl_sync(kFull, b, (base + from) & 31);
      second = fmaxf(fminf(best, x), fmaxf(second, y));
      best = fmaxf(best, x);
    }
    const bool both = p.group_best > 1 && second > none;
    const float sum = both ? best + second : best;
    // (Of two groups the one with the larger terms sees the other.)
    const float close = 3.f * tol + terms_of(best, second, both) * kSumRoundings;
    auto near_to = [&](float other) { return !(fabsf(other - sum) > close); };
    uint32_t before = 0;
    bool touch = false;
    for (uint32_t h = 0; h < p.groups; ++h) {
      const float other = __shfl_sync(kFull, sum, slot * kLanes + h * p.group_lanes);
      before += other > sum || (other == sum && h < g);
      touch |= h != g && near_to(other);
    }
    bool kept = before < p.top_groups;
    if (__any_sync(kFull, touch && g < p.groups && sum > none)) {
      bool doubt = false;
      for (uint32_t h = 0; h < p.groups; ++h) {
        const float other = __shfl_sync(kFull, sum, slot * kLanes + h * p.group_lanes);
        const bool stays = __shfl_sync(kFull, (int)kept, slot * kLanes + h * p.group_lanes);
        doubt |= g < p.groups && sum > none && stays != kept && near_to(other);
      }
      if (p.softmax && p.bias) {
        *near |= doubt;  // the scores' sum is needed in 64 bits
      } else if (__any_sync(kFull, doubt)) {
        // The sums again in 64 bits, of the few experts that may be among a group's best two (softmax scores
        // but for their common factor).
        const float cut = (second > none ? second : best) - 2.f * tol - fabsf(second) * 2.4e-7f;
        uint32_t left = 0;
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (c[i] > none && !(c[i] < cut)) left |= 1u << i;
        double a2 = none, b2 = none;
        while (__any_sync(kFull, left != 0)) {
          if (left) {
            const uint32_t e = sub * p.per_lane + __ffs(left) - 1;
            left &= left - 1;
            const double l = logit_at(p, token, e);
            const double v = p.softmax ? exp_of(l - (double)top)
                                       : sigmoid(l) + (p.bias ? (double)p.bias[e] : 0.0);
            b2 = fmax(b2, fmin(a2, v));
            a2 = fmax(a2, v);
          }
          __syncwarp();
        }
        double best2 = a2, second2 = b2;
        for (uint32_t t = 1; t < p.group_lanes; ++t) {
          const uint32_t from = at + t < p.group_lanes ? at + t : at + t - p.group_lanes;
          const double x = __shfl_sync(kFull, a2, (base + from) & 31);
          const double y = __shfl_sync(kFull, b2, (base + from) & 31);
          second2 = fmax(fmin(best2, x), fmax(second2, y));
          best2 = fmax(best2, x);
        }
        const double sum2 = p.group_best > 1 && second2 > none ? best2 + second2 : best2;
        before = 0;
        for (uint32_t h = 0; h < p.groups; ++h) {
          const double other = __shfl_sync(kFull, sum2, slot * kLanes + h * p.group_lanes);
          before += other > sum2 || (other == sum2 && h < g);
        }
        kept = before < p.top_groups;
      }
    }
    return kept ? kFull : 0;
  }
  return keep_any_groups<kLanes, V>(p, sub, slot, c, tol, near);
}

// The choice of the warp's tokens with whole values: of the logits as they are, or of scores in 64 bits.  Reads
// the logits again and leaves the chosen experts in `chosen`, kNone behind the last.  Few tokens come here, and
// then the code does for the first time: loops over values in local memory, little unrolled.
template <int kLanes, int V, bool kScored>
__device__ __noinline__ void choose_exact(const RouteProblem &p, uint32_t *chosen, uint32_t token,
                                          bool valid, uint32_t sub, uint32_t slot) {
  double c[V];  // -inf: closed
  uint32_t nan = 0;
  float top = -INFINITY;
  const uint32_t first = sub * p.per_lane;
#pragma unroll 4
  for (int i = 0; i < V; ++i) {
    const uint32_t e = first + i;
    const float l = valid && i < (int)p.per_lane && e < p.experts ? logit_at(p, token, e) : -INFINITY;
    top = fmaxf(top, l);
    c[i] = l;
  }
  if constexpr (kScored) {
    top = lanes_max<kLanes>(top);
    double sum = 0.0;
#pragma unroll 4
    for (int i = 0; i < V; ++i) {
      const double s = p.softmax ? exp_of(c[i] - (double)top) : sigmoid(c[i]);
      const bool is = c[i] != -INFINITY;
      sum += is && s == s ? s : 0.0;
      c[i] = is ? s : c[i];
    }
    const double inv = p.softmax ? 1.0 / lanes_sum<kLanes>(sum) : 1.0;
#pragma unroll 1
    for (int i = 0; i < V; ++i)
      if (c[i] != -INFINITY) {
        const double b = p.bias ? (double)p.bias[first + i] : 0.0;
        c[i] = b == -INFINITY ? b : c[i] * inv + b;
      }
  }
  // NaN ranks below every number: -inf from here on, with a mark.
#pragma unroll 1
  for (int i = 0; i < V; ++i)
    if (c[i] != c[i]) {
      nan |= 1u << i;
      c[i] = -INFINITY;
    }
  uint32_t kept = kFull;
  if (p.groups > 1) {
    // One group after the other: its best two over all lanes.  The lane keeps the sums of groups sub,
    // sub + kLanes, ...: 64 at most.
    const uint32_t per = p.experts / p.groups;
    constexpr int kSums = 64 / kLanes;
    double sums[kSums];
#pragma unroll 1
    for (uint32_t g = 0; g < p.groups; ++g) {
      double a = -INFINITY, b = -INFINITY;
#pragma unroll 4
      for (uint32_t e = max(g * per, first); e < min((g + 1) * per, first + p.per_lane); ++e) {
        const double v = c[e - first];
        b = fmax(b, fmin(a, v));
        a = fmax(a, v);
      }
#pragma unroll 1
      for (int o = kLanes / 2; o > 0; o >>= 1) {
        const double x = __shfl_xor_sync(kFull, a, o), y = __shfl_xor_sync(kFull, b, o);
        b = fmax(fmin(a, x), fmax(b, y));
        a = fmax(a, x);
      }
      if (g % kLanes == sub) sums[g / kLanes] = p.group_best > 1 && b > -INFINITY ? a + b : a;
    }
    kept = 0;
#pragma unroll 1
    for (uint32_t g = 0; g < p.groups; ++g) {
      const double own = __shfl_sync(kFull, sums[g / kLanes], slot * kLanes + g % kLanes);
      uint32_t before = 0;
#pragma unroll 1
      for (uint32_t h = sub; h < p.groups; h += kLanes)
        before += sums[h / kLanes] > own || (sums[h / kLanes] == own && h < g);
      __syncwarp();
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) before += __shfl_xor_sync(kFull, before, o);
      if (before < p.top_groups)
#pragma unroll 1
        for (uint32_t e = max(g * per, first); e < min((g + 1) * per, first + p.per_lane); ++e)
          kept |= 1u << (e - first);
    }
  }
  // Without a bias scores rise with their logits, and those tell more.
  if (kScored && !p.bias)
#pragma unroll 1
    for (int i = 0; i < V; ++i)
      if (c[i] != -INFINITY) c[i] = logit_at(p, token, first + i);
  // Taken experts lose their bit; the NaN that are left rank behind all numbers, by index.
  uint32_t open = 0;
#pragma unroll 1
  for (int i = 0; i < V; ++i)
    if (c[i] > -INFINITY || (nan >> i & 1)) open |= 1u << i;
  open &= kept;
#pragma unroll 1
  for (uint32_t j = 0; j < p.top_k; ++j) {
    double best = -INFINITY;
    uint32_t at = kNone;  // what is left, numbers first, then the lower index
#pragma unroll 4
    for (int i = 0; i < V; ++i)
      if ((open >> i & 1) && (at == kNone || c[i] > best)) {
        best = c[i];
        at = first + i;
      }
#pragma unroll 1
    for (int o = kLanes / 2; o > 0; o >>= 1) {
      const double other = __shfl_xor_sync(kFull, best, o);
      const uint32_t at2 = __shfl_xor_sync(kFull, at, o);
      if (other > best || (other == best && at2 < at)) {
        best = other;
        at = at2;
      }
    }
    if (sub == 0) chosen[j] = at;
    if (at >= first && at < first + p.per_lane) open &= ~(1u << (at - first));
  }
  __syncwarp();
}

// Sorts V keys, the largest first: Batcher's odd-even merge network.
template <int V>
__device__ __forceinline__ void sort_keys(uint32_t (&k)[V]) {
#pragma unroll
  for (int p = 1; p < V; p *= 2)
#pragma unroll
    for (int q = p; q >= 1; q /= 2)
#pragma unroll
      for (int j = q % p; j <= V - 1 - q; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < V && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t a = k[i + j], b = k[i + j + q];
            k[i + j] = max(a, b);
            k[i + j + q] = min(a, b);
          }
}

// The 8 largest of V keys in their order, largest first: halves sorted, and the larger of each key of one and
// its counterpart from the other's end, which rise and then fall.
__device__ __forceinline__ void sort_bitonic(uint32_t (&t)[8]) {
#pragma unroll
  for (int d = 4; d; d /= 2)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!(i & d)) {
        const uint32_t a = t[i], b = t[i + d];
        t[i] = max(a, b);
        t[i + d] = min(a, b);
      }
}
template <int V>
__device__ __forceinline__ void top_keys(const uint32_t (&k)[V], uint32_t (&t)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = k[i];
  sort_keys(t);
  if constexpr (V == 16) {
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = k[8 + i];
    sort_keys(b);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = max(t[i], b[7 - i]);
    sort_bitonic(t);
  }
}
// t[i] for an i that is known only here.
__device__ __forceinline__ uint32_t pick(const uint32_t (&t)[8], uint32_t i) {
  const uint32_t a = i & 1 ? t[1] : t[0], b = i & 1 ? t[3] : t[2], c = i & 1 ? t[5] : t[4],
                 d = i & 1 ? t[7] : t[6];
  const uint32_t x = i & 2 ? b : a, y = i & 2 ? d : c;
  return i & 4 ? y : x;
}

// The logits of a lane's experts, as they lie.
template <int V>
struct Logits {
  uint32_t w[V];
  // -inf where there is none; here: whether the token has logits
  __device__ __forceinline__ void load(const RouteProblem &p, size_t token, uint32_t sub, bool here) {
    const uint32_t e0 = sub * p.per_lane;
    const size_t at = token * p.ld + e0;
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = 0xff800000u;
    if constexpr (V >= 4) {
      if (p.vec && p.logits_dtype == TX_F32) {  // per_lane == V, on 16-byte boundaries
#pragma unroll
        for (int i = 0; i < V; i += 4)
          if (here && e0 + i < p.experts) {
            const uint4 q = *reinterpret_cast<const uint4 *>(static_cast<const float *>(p.logits) + at + i);
            w[i] = q.x; w[i + 1] = q.y; w[i + 2] = q.z; w[i + 3] = q.w;
          }
        return;
      }
    }
    if constexpr (V >= 8) {
      if (p.vec) {
#pragma unroll
        for (int i = 0; i < V; i += 8)
          if (here && e0 + i < p.experts) {
            const uint4 q =
                *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.logits) + at + i);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const uint32_t u = t == 0 ? q.x : t == 1 ? q.y : t == 2 ? q.z : q.w;
              w[i + 2 * t] = u << 16;
              w[i + 2 * t + 1] = u & 0xffff0000u;
            }
          }
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (here && i < (int)p.per_lane && e0 + i < p.experts)
        w[i] = p.logits_dtype == TX_BF16
                   ? (uint32_t) static_cast<const uint16_t *>(p.logits)[at + i] << 16
                   : static_cast<const uint32_t *>(p.logits)[at + i];
  }
};

// ---- the plan -------------------------------------------------------------------------------
// Exclusive sums of count[experts] into offset[experts + 1] (which may be count); parts is scratch of a
// word for each warp.  All threads of the block call it.
__device__ void scan_counts(const uint32_t *count, uint32_t *offset, uint32_t experts, uint32_t *parts) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x / 32;
  uint32_t carry = 0;
  for (uint32_t e0 = 0; e0 < experts; e0 += blockDim.x) {
    const uint32_t e = e0 + threadIdx.x, own = e < experts ? count[e] : 0;
    uint32_t v = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(kFull, v, o);
      if ((int)lane >= o) v += u;
    }
    if (lane == 31) parts[warp] = v;
    __syncthreads();
    uint32_t before = lane < warps ? parts[lane] : 0, all = before;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(kFull, all, o);
      if ((int)lane >= o) all += u;
    }
    before = carry + __shfl_sync(kFull, all - before, warp);
    if (e < experts) offset[e] = before + v - own;
    carry += __shfl_sync(kFull, all, 31);
    __syncthreads();
  }
  if (threadIdx.x == 0) offset[experts] = carry;
  __syncthreads();
}
// The tokens of warp `warp` in the run of block `block`: [*first, *end).
__device__ __forceinline__ void warp_tokens(const RouteProblem &p, uint32_t block, uint32_t warp,
                                            uint32_t *first, uint32_t *end) {
  const uint64_t run = (uint64_t)block * p.run, last = min(run + p.run, (uint64_t)p.tokens);
  *first = (uint32_t)min(run + (uint64_t)warp * p.run_warp, last);
  *end = (uint32_t)min((uint64_t)*first + p.run_warp, last);
}
// A warp's pairs, whose ranks lie in p.places: before[e] is added to those of expert e, and, where that is
// their row, the row filled.
template <bool kRows>
__device__ __forceinline__ void place_pairs(const RouteProblem &p, uint32_t first, uint32_t end,
                                            const uint32_t *before) {
  const uint64_t b = (uint64_t)end * p.top_k;
#pragma unroll 4
  for (uint64_t i = (uint64_t)first * p.top_k + (threadIdx.x & 31); i < b; i += 32) {
    const int32_t e = p.chosen[i], rank = p.places[i];
    if (e >= 0) {
      const uint32_t at = before[e] + (uint32_t)rank;
      p.places[i] = (int32_t)at;
      if (kRows) p.order[at] = (int32_t)i;
    }
  }
}

// Shared memory: by_warp [kWarps][experts], offset [experts + 1], a word for each warp, the bias, for every
// token in work its chosen experts and their keys, one more than there may be, and the lanes' sorted keys.
constexpr uint32_t kSlotWords = 2 * (kMaxK + 1);

// kTop8: up to 8 experts a token.  Every lane's 8 largest meet those of the other lanes in steps of a shuffle for each (8 maxima and a sort of 8), after which every lane has the
// token's 8, without a round for each or a branch.  Their keys name the expert in all lanes.
template <int kLanes, int V, bool kScored, int kWarps, bool kTop8>
__global__ void __launch_bounds__(32 * kWarps, 1)
    route_kernel(const __grid_constant__ RouteProblem p) {
  constexpr uint32_t kThreads = 32 * kWarps;
  constexpr uint32_t kTokens = 32 / kLanes;  // of a warp at a time
  // The low bits of a key: V - 1 - i for expert i of the lane, or, where the keys' lowest 16 bits are alike
  // (bf16 logits compared as they are), kNameAll - e for expert e.  The latter lose nothing and put equals
  // in their order.  Of kTop8 the others' name is kName - e.
  constexpr uint32_t kName = kTop8 ? kLanes * V - 1 : V - 1, kNameAll = 0xffff;
  constexpr int kMine = ((kTop8 ? 8 : kMaxK) + kLanes - 1) / kLanes;  // chosen experts a lane weighs
  constexpr bool kListed = V > 8;        // sorted keys behind the first in shared memory
  extern __shared__ __align__(16) uint8_t smem[];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % kLanes;
  const uint32_t slot = lane / kLanes, group_mask = (kLanes == 32 ? kFull : (1u << kLanes) - 1)
                                                   << (slot * kLanes);
  uint32_t *by_warp = reinterpret_cast<uint32_t *>(smem), *words = by_warp + warp * p.experts;
  uint32_t *offset = by_warp + kWarps * p.experts;
  uint32_t *parts = offset + p.experts + 1;
  float *bias = reinterpret_cast<float *>(parts + kWarps);
  uint32_t *chosen = reinterpret_cast<uint32_t *>(bias + (kScored ? kLanes * V : 0)) +
                     (warp * kTokens + slot) * kSlotWords;
  uint32_t *chosen_key = chosen + kMaxK + 1;
  uint32_t *list = chosen - (warp * kTokens + slot) * kSlotWords + kWarps * kTokens * kSlotWords +
                   warp * V * 32 + lane;
  if (p.order)
    for (uint32_t e = lane; e < p.experts; e += 32) words[e] = 0;
  if constexpr (kScored) {
    // By the lane last, so that lanes side by side meet banks side by side.
    for (uint32_t e = threadIdx.x; e < kLanes * V; e += kThreads) {
      const uint32_t at = e % kLanes * p.per_lane + e / kLanes;
      bias[e] = p.bias && e / kLanes < p.per_lane && at < p.experts ? p.bias[at] : 0.f;
    }
    __syncthreads();
  }
  __syncwarp();
  asm volatile("griddepcontrol.launch_dependents;");
  uint32_t first, end;
  warp_tokens(p, blockIdx.x, warp, &first, &end);
  bool told = !kScored && p.logits_dtype == TX_BF16;
  // Where the next token to load stands in its sequence, and how many rows of that are valid.
  uint32_t next = first + slot, row = 0, seq = 0, length = 0;
  if (p.lengths && next < end) {
    seq = next / p.seq;
    row = next - seq * p.seq;
    length = (uint32_t)max(p.lengths[seq], 0);
  }
  // A block that is alone, each warp with one round of tokens, places its pairs from registers.
  const bool once = gridDim.x == 1 && p.run_warp <= kTokens;
  uint32_t kept_e[kMine], kept_rank[kMine];
  Logits<V> raw;
  bool valid = next < end && (!p.lengths || row < length);
  raw.load(p, next, sub, valid);
  for (uint32_t t0 = first; t0 < end; t0 += kTokens) {
    const uint32_t token = t0 + slot;
    const bool here = token < end, had = valid;
    float tol = 0.f, all_top = 0.f, all_sum = 1.f;  // of all logits, where the weights need them
    uint32_t key[V];
    bool near = false, far = false;  // neighbours to put in order; a choice to make again
    {
      float c[V];
#pragma unroll
      for (int i = 0; i < V; ++i) c[i] = __uint_as_float(raw.w[i]);
      if (p.softmax && (kScored || !p.renormalise)) {
        all_top = c[0];
#pragma unroll
        for (int i = 1; i < V; ++i) all_top = fmaxf(all_top, c[i]);
        all_top = lanes_max<kLanes>(all_top);
        float sum = 0.f;
        if (!p.renormalise) {
#pragma unroll
          for (int i = 0; i < V; ++i) sum += c[i] == -INFINITY ? 0.f : expf(c[i] - all_top);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) sum += c[i] == -INFINITY ? 0.f : quick_exp(c[i] - all_top);
        }
        all_sum = lanes_sum<kLanes>(sum);
      }
      if constexpr (kTop8 && !kScored) {
        // fp32 logits that were bf16 are many equals: they are told apart as well.
        uint32_t low = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) low |= __float_as_uint(c[i]);
        told = !__any_sync(kFull, low & kNameAll);
      }
      if constexpr (!kScored) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          far |= c[i] != c[i];
          key[i] = told ? (key_of(c[i]) & ~kNameAll) | (kNameAll - sub * p.per_lane - i)
                        : (key_of(c[i]) & ~kName) | (kName - (kTop8 ? sub * p.per_lane : 0) - i);
        }
      } else {
        const float inv = p.softmax ? quick_rcp(all_sum) : 1.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float s = p.softmax ? quick_exp(c[i] - all_top) * inv : sigmoid(c[i]);
          c[i] = c[i] == -INFINITY ? -INFINITY : s + bias[i * kLanes + sub];  // closed by either's -inf
          far |= c[i] != c[i];
        }
        tol = score_tolerance<V>(p.softmax, inv);
        uint32_t kept = kFull;
        if (p.groups > 1) kept = keep_groups<kLanes, V>(p, sub, slot, c, tol, token, all_top, &far);
#pragma unroll
        for (int i = 0; i < V; ++i)
          key[i] = kept >> i & 1
                       ? (key_of(c[i]) & ~kName) | (kName - (kTop8 ? sub * p.per_lane : 0) - i)
                       : 0;
      }
    }
    // The next tokens' logits travel meanwhile.
    auto load_next = [&] {
      next += kTokens;
      if (p.lengths && next < end) {
        row += kTokens;
        if (row >= p.seq) {
          seq = next / p.seq;
          row = next - seq * p.seq;
          length = (uint32_t)max(p.lengths[seq], 0);
        }
      }
      valid = next < end && (!p.lengths || row < length);
      raw.load(p, next, sub, valid);
    };
    uint32_t e[kMine];
    if constexpr (kTop8) {
      uint32_t t[8], own[8];
      top_keys<V>(key, t);
#pragma unroll
      for (int i = 0; i < 8; ++i) own[i] = t[i];
#pragma unroll
      for (int o = 1; o < kLanes; o *= 2) {
        uint32_t b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = __shfl_xor_sync(kFull, t[i], o);
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = max(t[i], b[7 - i]);
        sort_bitonic(t);
      }
      load_next();
      const uint32_t names = told ? kNameAll : kName;
#pragma unroll
      for (int m = 0; m < kMine; ++m) {
        const uint32_t j = sub + m * kLanes, mine = pick(t, j & 7);
        e[m] = j < p.top_k && mine >= kLowest ? names - (mine & names) : kNone;
      }
      if (!told) {
        // The largest behind the 8.
        uint32_t ninth = 0;
#pragma unroll
        for (int i = 7; i >= 0; --i) ninth = own[i] < t[7] ? max(ninth, own[i]) : ninth;
        ninth = lanes_max<kLanes>(ninth);
        auto key_at = [&](uint32_t j) { return j < 8 ? pick(t, j) : ninth; };
        auto close = [&](uint32_t a, uint32_t b) {  // whether the order of a and b below it is in doubt
          const float w = value_of(a & ~kName), v = value_of(b & ~kName);
          return b >= kLowest && !(w - v > tol + fabsf(w) * ((kName + 1) * 1.3e-7f));
        };
#pragma unroll
        for (int m = 0; m < kMine; ++m) {
          const uint32_t j = sub + m * kLanes;
          near |= e[m] != kNone && close(key_at(j), key_at(j + 1));
        }
        // (Where a lane's 8 are all among the token's, its next are not known.)
        near |= V > 8 && own[7] >= t[7] && t[7] >= kLowest;
        if (__any_sync(kFull, near)) {
          // All that may belong among the chosen are put in the order of their logits, where scores grow with
          // them, or of sigmoids in 64 bits.  Softmax scores with a bias need the sum in 64 bits too.
          constexpr uint32_t kMost = 16;
          constexpr int kEach = (kMost + kLanes - 1) / kLanes;
          const uint32_t last = key_at(p.top_k - 1);
          uint32_t count = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const bool is = own[i] >= kLowest && (own[i] >= last || last < kLowest || close(last, own[i]));
            const uint32_t all = __ballot_sync(kFull, is) & group_mask;
            const uint32_t at = count + __popc(all & ((1u << lane) - 1));
            if (is && at < kMost) chosen[at] = kName - (own[i] & kName);
            count += __popc(all);
            if (i == 7) far |= V > 8 && is;
          }
          far |= count > kMost || (near && kScored && p.softmax && p.bias);
          __syncwarp();
          if (!__any_sync(kFull, far)) {
            double c[kEach];
            uint32_t of[kEach], place[kEach], *high = chosen_key, *low = chosen_key + kMost;
#pragma unroll
            for (int m = 0; m < kEach; ++m) {
              const uint32_t j = sub + m * kLanes;
              of[m] = j < count ? chosen[j] : kNone;
              place[m] = 0;
              if (of[m] == kNone) continue;
              c[m] = logit_at(p, token, of[m]);
              if (kScored && p.bias) c[m] = sigmoid(c[m]) + (double)p.bias[of[m]];
              high[j] = (uint32_t)((uint64_t)__double_as_longlong(c[m]) >> 32);
              low[j] = (uint32_t)__double_as_longlong(c[m]);
            }
            __syncwarp();
            for (uint32_t j = 0; j < count; ++j) {
              const double other = __longlong_as_double((long long)((uint64_t)high[j] << 32 | low[j]));
              const uint32_t other_e = chosen[j];
#pragma unroll
              for (int m = 0; m < kEach; ++m)
                place[m] += of[m] != kNone && (other > c[m] || (other == c[m] && other_e < of[m]));
            }
            __syncwarp();
#pragma unroll
            for (int m = 0; m < kEach; ++m)
              if (of[m] != kNone) chosen[place[m]] = of[m];
            __syncwarp();
#pragma unroll
            for (int m = 0; m < kMine; ++m)
              if (e[m] != kNone) e[m] = chosen[sub + m * kLanes];
            __syncwarp();
          }
        }
      }
    } else {
      load_next();
      sort_keys(key);
      if constexpr (kListed) {
#pragma unroll
        for (int i = 1; i < V; ++i)
          if (i <= (int)p.top_k) list[i * 32] = key[i];
      }
      // The lowest lane with the largest head, names apart, has the next expert.
      const uint32_t names = told ? 0 : kName;
      uint32_t taken = 0;
      for (uint32_t j = 0; j < p.top_k + !told; ++j) {
        const uint32_t head = key[0], named = head | names, top = lanes_max<kLanes>(named);
        if (lane == __ffs(__ballot_sync(kFull, named == top) & group_mask) - 1) {
          chosen[j] = told ? kNameAll - (head & kNameAll) : sub * p.per_lane + kName - (head & kName);
          chosen_key[j] = head;
          if constexpr (kListed) {
            key[0] = ++taken < V ? list[taken * 32] : 0;
          } else {
#pragma unroll
            for (int i = 0; i + 1 < V; ++i) key[i] = key[i + 1];
            key[V - 1] = 0;
          }
        }
      }
      __syncwarp();
#pragma unroll
      for (int m = 0; m < kMine; ++m) {
        const uint32_t j = sub + m * kLanes;
        e[m] = kNone;
        if (j >= p.top_k) continue;
        const uint32_t own = chosen_key[j];
        if (own >= kLowest) e[m] = chosen[j];
        if (told || own < kLowest) continue;
        const uint32_t after = chosen_key[j + 1];
        const float w = value_of(own & ~kName), v = value_of(after & ~kName);
        if (after >= kLowest && !(w - v > tol + fabsf(w) * (V * 2.4e-7f))) {
          // Equal in logit and bias they are in the right order, but behind the last there may be another.
          const uint32_t f = chosen[j + 1];
          far |= j + 1 == p.top_k || logit_at(p, token, e[m]) != logit_at(p, token, f) ||
                  (p.bias && p.bias[e[m]] != p.bias[f]);
        }
      }
    }
    if (__any_sync(kFull, far)) {
      __syncwarp();
      choose_exact<kLanes, V, kScored>(p, chosen, token, had, sub, slot);
#pragma unroll
      for (int m = 0; m < kMine; ++m)
        if (sub + m * kLanes < p.top_k) e[m] = chosen[sub + m * kLanes];
      __syncwarp();
    }
    // Weights.  With a common factor taken out first: e^l by the largest l, and for the sigmoid
    // e^min(l, 0) / (1 + e^-|l|) by the largest of the numerators; renormalised it cancels.
    float x[kMine], top = -INFINITY;
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      x[m] = e[m] != kNone ? logit_at(p, token, e[m]) : -INFINITY;
      if (e[m] != kNone) top = fmaxf(top, p.softmax ? x[m] : fminf(x[m], 0.f));
    }
    top = p.renormalise ? lanes_max<kLanes>(top) : p.softmax ? all_top : 0.f;
    float s[kMine], sum = 0.f;
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      s[m] = 0.f;
      if (e[m] == kNone) continue;
      s[m] = p.softmax ? expf(x[m] - top)
                       : expf(fminf(x[m], 0.f) - top) * quick_rcp(1.f + expf(-fabsf(x[m])));
      sum += s[m];
    }
    const float factor = p.scale * quick_rcp(p.renormalise ? lanes_sum<kLanes>(sum) : all_sum);
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const uint32_t j = sub + m * kLanes;
      if (!here || j >= p.top_k) continue;
      const size_t at = (size_t)token * p.top_k + j;
      p.chosen[at] = e[m] == kNone ? -1 : (int32_t)e[m];
      p.weights[at] = e[m] == kNone ? 0.f : s[m] * factor;
    }
    if (!p.order) continue;
    // The rank of a pair among the warp's of its expert: words[e] holds those of the tokens before in its
    // lower bits, and bit 24 + t for token t of these.  (A token has an expert once.)
#pragma unroll
    for (int m = 0; m < kMine; ++m)
      if (e[m] != kNone) atomicOr(words + e[m], 1u << (24 + slot));
    __syncwarp();
    uint32_t word[kMine];
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const uint32_t j = sub + m * kLanes;
      word[m] = e[m] != kNone ? words[e[m]] : 0;
      const uint32_t rank = (word[m] & 0xffffffu) + __popc(word[m] >> 24 & ((1u << slot) - 1));
      kept_e[m] = here ? e[m] : kNone;
      kept_rank[m] = rank;
      if (here && j < p.top_k && !(once && e[m] != kNone))
        p.places[(size_t)token * p.top_k + j] = e[m] == kNone ? -1 : (int32_t)rank;
    }
    __syncwarp();
#pragma unroll
    for (int m = 0; m < kMine; ++m)
      if (e[m] != kNone && !(word[m] >> 24 & ((1u << slot) - 1)))
        words[e[m]] = (word[m] & 0xffffffu) + __popc(word[m] >> 24);
    __syncwarp();
  }
  if (!p.order) return;
  __syncthreads();
  // The counts of the warps before each warp, and of the block.
  for (uint32_t e = threadIdx.x; e < p.experts; e += kThreads) {
    uint32_t run = 0;
#pragma unroll 8
    for (uint32_t w = 0; w < kWarps; ++w) {
      const uint32_t n = by_warp[w * p.experts + e];
      by_warp[w * p.experts + e] = run;
      run += n;
    }
    offset[e] = run;
    if (gridDim.x > 1) p.counts[(size_t)e * gridDim.x + blockIdx.x] = run;
  }
  __syncthreads();
  if (gridDim.x > 1) {
    place_pairs<false>(p, first, end, words);
    return;
  }
  scan_counts(offset, offset, p.experts, parts);
  for (uint32_t e = threadIdx.x; e <= p.experts; e += kThreads) p.offsets[e] = (int32_t)offset[e];
  for (uint32_t e = lane; e < p.experts; e += 32) words[e] += offset[e];
  __syncwarp();
  if (!once) {
    place_pairs<true>(p, first, end, words);
  } else if (first < end) {
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      if (kept_e[m] == kNone) continue;
      const uint32_t at = words[kept_e[m]] + kept_rank[m];
      const size_t pair = (size_t)(first + slot) * p.top_k + sub + m * kLanes;
      p.places[pair] = (int32_t)at;
      p.order[at] = (int32_t)pair;
    }
  }
}

// Places the pairs of run blockIdx.x, ranked within it, behind those of the runs before it.
constexpr int kPlaceThreads = 1024;
__global__ void __launch_bounds__(kPlaceThreads, 1)
    place_kernel(const __grid_constant__ RouteProblem p) {
  __shared__ uint32_t total[1024], base[1024], offset[1025], parts[32];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, runs = gridDim.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // for the runs, see run_warps
  const uint64_t first = min((uint64_t)blockIdx.x * p.run, (uint64_t)p.tokens) * p.top_k;
  const uint64_t end = min((uint64_t)(blockIdx.x + 1) * p.run, (uint64_t)p.tokens) * p.top_k;
  // The block's first pairs travel while the counts are summed.
  constexpr int kHeld = 4;
  int32_t held_e[kHeld], held_rank[kHeld];
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
    const uint64_t i = first + threadIdx.x + h * kPlaceThreads;
    held_e[h] = i < end ? __ldcg(p.chosen + i) : -1;
    held_rank[h] = i < end ? __ldcg(p.places + i) : 0;
  }
  // A warp sums the counts of an expert over the runs, and of those before this one; the loads of four
  // experts are on their way at once.
  for (uint32_t e0 = warp * 4; e0 < p.experts; e0 += kPlaceThreads / 8) {
    uint32_t all[4] = {}, before[4] = {};
#pragma unroll 5
    for (uint32_t b = lane; b < runs; b += 32) {
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t n = e0 + i < p.experts ? __ldcg(p.counts + (size_t)(e0 + i) * runs + b) : 0;
        all[i] += n;
        before[i] += b < blockIdx.x ? n : 0;
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t a = __reduce_add_sync(kFull, all[i]), b = __reduce_add_sync(kFull, before[i]);
      if (lane == 0 && e0 + i < p.experts) {
        total[e0 + i] = a;
        base[e0 + i] = b;
      }
    }
  }
  __syncthreads();
  scan_counts(total, offset, p.experts, parts);
  if (blockIdx.x == 0)
    for (uint32_t e = threadIdx.x; e <= p.experts; e += kPlaceThreads) p.offsets[e] = (int32_t)offset[e];
  for (uint32_t e = threadIdx.x; e < p.experts; e += kPlaceThreads) base[e] += offset[e];
  __syncthreads();
  auto place = [&](uint64_t i, int32_t e, int32_t rank) {
    if (e < 0) return;
    const uint32_t at = base[e] + (uint32_t)rank;
    p.places[i] = (int32_t)at;
    p.order[at] = (int32_t)i;
  };
#pragma unroll
  for (int h = 0; h < kHeld; ++h)
    place(first + threadIdx.x + h * kPlaceThreads, held_e[h], held_rank[h]);
#pragma unroll 4
  for (uint64_t i = first + threadIdx.x + kHeld * kPlaceThreads; i < end; i += kPlaceThreads)
    place(i, p.chosen[i], p.places[i]);
}

template <int kLanes, int V, bool kScored, int kWarps, bool kTop8>
cudaError_t run_warps(RouteProblem p, cudaStream_t stream) {
  constexpr uint32_t kTokens = 32 / kLanes;
  const uint32_t run = std::min(p.run, p.tokens);
  p.run_warp = ((run + kWarps - 1) / kWarps + kTokens - 1) / kTokens * kTokens;
  const size_t size = p.logits_dtype == TX_BF16 ? 2 : 4;
  p.vec = p.per_lane == V && V * size % 16 == 0 && p.experts % (16 / size) == 0 &&
          p.ld * size % 16 == 0 && (uintptr_t)p.logits % 16 == 0;
  const uint32_t bytes = ((kWarps + 1) * p.experts + 1 + kWarps + (kScored ? kLanes * V : 0) +
                          kWarps * kTokens * kSlotWords + (V > 8 && !kTop8 ? kWarps * V * 32 : 0)) *
                         4;
  static std::atomic<uint64_t> seen{0};
  cudaError_t e = allow_smem((const void *)route_kernel<kLanes, V, kScored, kWarps, kTop8>, 232448, seen);
  if (e != cudaSuccess) return e;
  route_kernel<kLanes, V, kScored, kWarps, kTop8><<<p.blocks, 32 * kWarps, bytes, stream>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess || p.blocks == 1 || !p.order) return e;
  // Launched while the runs finish (griddepcontrol), it waits for them on the device.
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(p.blocks);
  config.blockDim = dim3(kPlaceThreads);
  config.stream = stream;
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, place_kernel, p);
}
// Few warps where a round of theirs takes all tokens: a block of 32 is slower to start and to add up (8 tokens
// of 64 experts: 8.2 against 9.5 us).
template <int kLanes, int V, bool kScored, bool kTop8>
cudaError_t run(const RouteProblem &p, cudaStream_t stream) {
  // 64 registers a thread with 32 warps, 128 with 16.  64 are few: 17 of the 18 forms of 32 warps keep some in
  // local memory (4 to 616 bytes stored; the two of the large cases above 132 and 12).
  constexpr int kWarps = V <= 8 || kTop8 ? kMostWarps : kMostWarps / 2;
  if (p.tokens <= 4 * (32 / kLanes)) return run_warps<kLanes, V, kScored, 4, kTop8>(p, stream);
  return run_warps<kLanes, V, kScored, kWarps, kTop8>(p, stream);
}
template <int kLanes, int V>
cudaError_t run_top8(const RouteProblem &p, cudaStream_t stream) {
  return p.bias || p.groups > 1 ? run<kLanes, V, true, true>(p, stream)
                                : run<kLanes, V, false, true>(p, stream);
}
template <int kLanes, int V>
cudaError_t run_rounds(const RouteProblem &p, cudaStream_t stream) {
  return p.bias || p.groups > 1 ? run<kLanes, V, true, false>(p, stream)
                                : run<kLanes, V, false, false>(p, stream);
}

}  // namespace

// Tokens of a block.  A block takes about 16384 / experts tokens at once (half of that where they take more
// than 8 each), and while these are all, one block is the faster way: 64 tokens of 256 experts 12.3 us, in two
// launches 15.4; 128 tokens 16.4 and 15.7; 128 of 1024 experts 109 and 43.  Otherwise a block for each SM, of
// no less than such a number of tokens or 32.
size_t route_plan(RouteProblem *p, int num_sms) {
  const uint32_t once = std::min(std::max((p->top_k <= 8 ? 16384 : 8192) / p->experts, 16u), 256u);
  p->run = std::max<uint32_t>(p->order && p->tokens <= once ? once : std::min(once, 32u),
                              (uint32_t)(((uint64_t)p->tokens + num_sms - 1) / num_sms));
  p->blocks = (p->tokens + p->run - 1) / p->run;
  return p->order && p->blocks > 1 ? (size_t)p->blocks * p->experts * 4 : 0;
}

cudaError_t launch_experts_route(RouteProblem p, cudaStream_t stream) {
  // Experts of a lane.  With groups a group has to be whole lanes; where no number of experts a lane does
  // that, group_lanes is 0.
  auto cut = [&](uint32_t most) {
    p.per_lane = most;
    p.group_lanes = 0;
    if (p.groups < 2) return;
    const uint32_t per = p.experts / p.groups;
    for (uint32_t v = std::min(most, per); v && !p.group_lanes; --v)
      if (per % v == 0 && p.experts / v <= 32) {
        p.per_lane = v;
        p.group_lanes = per / v;
      }
  };
  auto lanes = [&] { return (p.experts + p.per_lane - 1) / p.per_lane; };
  if (p.top_k <= 8 && p.experts <= 512) {
    cut(p.experts <= 32 ? 8 : 16);
    if (p.experts <= 32 && lanes() <= 4) return run_top8<4, 8>(p, stream);
    if (lanes() <= 4) return run_top8<4, 16>(p, stream);
    if (lanes() <= 8) return run_top8<8, 16>(p, stream);
    if (lanes() <= 16) return run_top8<16, 16>(p, stream);
    return run_top8<32, 16>(p, stream);
  }
  // Rounds: 8 experts a lane where 32 lanes can hold them.
  const uint32_t most = p.experts <= 256 ? 8 : p.experts <= 512 ? 16 : 32;
  cut(most);
  if (most == 32) return run_rounds<32, 32>(p, stream);
  if (most == 16) return run_rounds<32, 16>(p, stream);
  if (lanes() <= 4) return run_rounds<4, 8>(p, stream);
  if (lanes() <= 8) return run_rounds<8, 8>(p, stream);
  if (lanes() <= 16) return run_rounds<16, 8>(p, stream);
  return run_rounds<32, 8>(p, stream);
}

}  // namespace tx
