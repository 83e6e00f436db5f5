// Routing of tokens to experts and the plan of their rows (tx_experts_route).
//
// Per token: scores s = softmax(l) or 1 / (1 + e^-l) of its logits l, the choice by c = s + bias (the
// largest first, ties to the lower index), with groups only among the groups whose best one or two c have
// the largest sums; the weights are the chosen experts' s, divided by their sum where asked, times scale.
// The plan lists the pairs token * top_k + j by expert, ascending inside an expert: a stable counting sort.
//
// The choice is that of exact arithmetic: without bias and groups c grows with l, so the logits themselves
// are compared; otherwise c is taken in fp32, and a token with two candidates closer than fp32's error at
// a border that decides (and not equal in logit and bias) takes its scores again in 64 bits.  In 64 bits
// alone the exponentials would cost several times the rest.
//
// kLanes lanes take a token, each with V consecutive experts.  A block takes a run of tokens and counts its
// pairs by expert; the second kernel sums the counts of the runs before its own and places its pairs.
// A few tokens are one block, which does both.
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/tessattn.h"
#include "common.cuh"
#include "kernels.h"

namespace tx {
namespace {

constexpr uint32_t kFull = 0xffffffffu;
constexpr int kWarps = 16, kThreads = 32 * kWarps;
constexpr uint32_t kMaxK = 32;

// Values as unsigned integers of the same order: 0 is closed, 1 is NaN (below every number).
__device__ __forceinline__ uint32_t key_of(float c) {
  const uint32_t u = __float_as_uint(c + 0.f);  // -0 as 0
  if (c != c) return 1;
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(double c) {
  const uint64_t u = (uint64_t)__double_as_longlong(c + 0.0);
  if (c != c) return 1;
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ float sigmoid(float l) { return 1.f / (1.f + expf(-l)); }
__device__ __forceinline__ double sigmoid(double l) { return 1.0 / (1.0 + exp(-l)); }
__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

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
template <typename S>
struct KeyOf {
  using type = uint32_t;
};
template <>
struct KeyOf<double> {
  using type = uint64_t;
};

__device__ __forceinline__ float logit_at(const RouteProblem &p, size_t token, uint32_t e) {
  const size_t at = token * p.ld + e;
  return p.logits_dtype == TX_BF16 ? bf16_bits_to_f32(static_cast<const uint16_t *>(p.logits)[at])
                                   : static_cast<const float *>(p.logits)[at];
}

// What a token's lanes share in shared memory.
struct Shared {
  uint32_t *chosen;  // [kMaxK]
  void *c;           // [experts] of S (groups only)
  void *sum;         // [groups] of S
  uint32_t *kept;    // [groups]
};

// The choice of one token among candidates c: key[i] of expert sub * V + i, 0 where closed.  Leaves the
// chosen experts in sh.chosen (kNone behind the last) and returns whether fp32 could not decide.
constexpr uint32_t kNone = 0xffffffffu;

template <int kLanes, int V, typename S>
__device__ bool choose(const RouteProblem &p, const Shared &sh, size_t token, uint32_t sub,
                       typename KeyOf<S>::type (&key)[V], const S (&c)[V], float tol) {
  using Key = typename KeyOf<S>::type;
  bool unsure = false;
  if (p.groups > 1) {
    const uint32_t per = p.experts / p.groups;
    S *cs = static_cast<S *>(sh.c), *sum = static_cast<S *>(sh.sum);
    const S none = -(S)INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (sub * V + i < p.experts) cs[sub * V + i] = key[i] > 1 ? c[i] : none;
    __syncwarp();
    for (uint32_t g = sub; g < p.groups; g += kLanes) {
      S a = none, b = none;
      for (uint32_t e = g * per; e < (g + 1) * per; ++e) {
        const S v = cs[e];
        if (v > a) {
          b = a;
          a = v;
        } else if (v > b) {
          b = v;
        }
      }
      sum[g] = p.group_best > 1 && b > none ? a + b : a;
    }
    __syncwarp();
    for (uint32_t g = sub; g < p.groups; g += kLanes) {
      uint32_t before = 0;
      for (uint32_t h = 0; h < p.groups; ++h)
        before += sum[h] > sum[g] || (sum[h] == sum[g] && h < g);
      sh.kept[g] = before < p.top_groups;
    }
    __syncwarp();
    if (tol > 0.f) {
      S low = (S)INFINITY, high = none;  // the lowest sum kept, the highest left out
      for (uint32_t g = 0; g < p.groups; ++g) {
        if (sh.kept[g])
          low = low < sum[g] ? low : sum[g];
        else
          high = high > sum[g] ? high : sum[g];
      }
      const S size = (low < 0 ? -low : low) * (S)2.4e-7f;
      unsure |= high > none && low - high <= 3 * (S)tol + size;
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (sub * V + i < p.experts && !sh.kept[(sub * V + i) / per]) key[i] = 0;
  }
  Key last = 0;
  uint32_t last_e = kNone;
  bool done = false;  // (the rounds are the warp's; a token that needs no more of them idles)
  for (uint32_t j = 0;; ++j) {
    Key top = 0;
    uint32_t at = 0;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (key[i] > top) {
        top = key[i];
        at = sub * V + i;
      }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) {
      const Key k2 = __shfl_xor_sync(kFull, top, o);
      const uint32_t at2 = __shfl_xor_sync(kFull, at, o);
      if (k2 > top || (k2 == top && at2 < at)) {
        top = k2;
        at = at2;
      }
    }
    bool same = false;
    if (sizeof(S) == 4 && tol > 0.f && j && !done && top > 1) {
      const float v = value_of((uint32_t)top), w = value_of((uint32_t)last);
      if (!(w - v > tol + 1.2e-7f * fabsf(w))) {
        same = logit_at(p, token, at) == logit_at(p, token, last_e) &&
               (!p.bias || p.bias[at] == p.bias[last_e]);
        unsure |= !same;
      }
    }
    if (j < p.top_k && sub == 0) sh.chosen[j] = top ? at : kNone;
    // Past the last one only equals of it may be followed by a candidate too close to tell.
    done |= !top || (j >= p.top_k && !same);
    if (j + 1 >= p.top_k && !(sizeof(S) == 4 && tol > 0.f)) break;
    if (j >= p.top_k && __all_sync(kFull, done)) break;
    if (!done) {
      last = top;
      last_e = at;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (sub * V + i == at) key[i] = 0;
    }
  }
  __syncwarp();
  return unsure;
}

template <int kLanes, int V, typename S>
__device__ bool score_and_choose(const RouteProblem &p, const Shared &sh, size_t token, uint32_t sub,
                                 const float (&l)[V], const bool (&open)[V]) {
  S s[V];
  float tol = 0.f;
  if (p.softmax) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (open[i]) top = fmaxf(top, l[i]);
    top = lanes_max<kLanes>(top);
    S sum = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s[i] = open[i] ? exp_of((S)l[i] - (S)top) : (S)0;
      sum += s[i];
    }
    sum = lanes_sum<kLanes>(sum);
    const S inv = (S)1 / sum;
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] *= inv;
    // A score is off by (V + 12) 2^-24 of itself at most, and none is above 1 / sum: the sum over V
    // values and lanes, the exponential (2 units), its argument's rounding, the reciprocal and product.
    tol = (float)((V + 12) * 1.1920929e-7f) * (float)inv;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = open[i] ? sigmoid((S)l[i]) : (S)0;
    tol = 7.2e-7f;  // two scores, each off by 2^-21.4
  }
  using Key = typename KeyOf<S>::type;
  Key key[V];
  S c[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    c[i] = s[i];
    if (p.bias && sub * V + i < p.experts) c[i] += (S)__ldg(p.bias + sub * V + i);
    key[i] = open[i] ? key_of(c[i]) : 0;
  }
  return choose<kLanes, V, S>(p, sh, token, sub, key, c, sizeof(S) == 4 ? tol : 0.f);
}

// ---- the plan -------------------------------------------------------------------------------
// Exclusive sums of count[experts] into offset[experts + 1]; all threads of the block call it.
__device__ void scan_counts(const uint32_t *count, uint32_t *offset, uint32_t experts) {
  if (threadIdx.x < 32) {
    uint32_t carry = 0;
    for (uint32_t e0 = 0; e0 < experts; e0 += 32) {
      const uint32_t e = e0 + threadIdx.x, own = e < experts ? count[e] : 0;
      uint32_t v = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(kFull, v, o);
        if ((int)threadIdx.x >= o) v += u;
      }
      if (e < experts) offset[e] = carry + v - own;
      carry += __shfl_sync(kFull, v, 31);
    }
    if (threadIdx.x == 0) offset[experts] = carry;
  }
  __syncthreads();
}

// Places the pairs [first, end): base[e] is where this run's pairs of expert e start.
__device__ void place_pairs(const RouteProblem &p, uint64_t first, uint64_t end, const uint32_t *base,
                            uint32_t *by_warp /* [kWarps][experts] */) {
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint64_t per = ((end - first + kWarps - 1) / kWarps + 31) / 32 * 32;
  const uint64_t a = first + warp * per, b = min(end, a + per);
  uint32_t *mine = by_warp + (size_t)warp * p.experts;
  for (uint32_t i = threadIdx.x; i < kWarps * p.experts; i += kThreads) by_warp[i] = 0;
  __syncthreads();
  for (uint64_t i = a; i < b; i += 32) {
    const int32_t e = i + lane < b ? p.chosen[i + lane] : -1;
    const uint32_t peers = __match_any_sync(kFull, e);
    if (e >= 0 && lane == __ffs(peers) - 1) mine[e] += __popc(peers);
    __syncwarp();
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < p.experts; e += kThreads) {
    uint32_t run = base[e];
    for (uint32_t w = 0; w < kWarps; ++w) {
      uint32_t *at = by_warp + (size_t)w * p.experts + e;
      const uint32_t n = *at;
      *at = run;
      run += n;
    }
  }
  __syncthreads();
  for (uint64_t i = a; i < b; i += 32) {
    const int32_t e = i + lane < b ? p.chosen[i + lane] : -1;
    const uint32_t peers = __match_any_sync(kFull, e);
    uint32_t at = 0;
    if (e >= 0) at = mine[e] + __popc(peers & ((1u << lane) - 1));
    __syncwarp();
    if (e >= 0 && lane == __ffs(peers) - 1) mine[e] += __popc(peers);
    __syncwarp();
    if (i + lane < b) {
      p.places[i + lane] = e >= 0 ? (int32_t)at : -1;
      if (e >= 0) p.order[at] = (int32_t)(i + lane);
    }
  }
}

// kLanes lanes a token, V experts a lane.  Shared memory: the chosen of every token in work, with groups
// their candidates and sums, the block's counts by expert, and for a plan in one block its places.
template <int kLanes, int V>
__global__ void __launch_bounds__(kThreads) route_kernel(const __grid_constant__ RouteProblem p) {
  constexpr uint32_t kTokens = 32 / kLanes;  // of a warp at a time
  extern __shared__ __align__(16) uint8_t smem[];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % kLanes;
  const uint32_t slot = warp * kTokens + lane / kLanes;
  uint32_t *count = reinterpret_cast<uint32_t *>(smem);
  uint32_t *offset = count + p.experts;
  uint32_t *chosen = offset + p.experts + 1;
  Shared sh;
  sh.chosen = chosen + slot * kMaxK;
  uint8_t *more = smem + p.off_groups;
  const uint32_t group_bytes = p.groups > 1 ? p.experts * 8 + p.groups * 12 + (p.groups & 1) * 4 : 0;
  sh.c = more + (size_t)slot * group_bytes;
  sh.sum = more + (size_t)slot * group_bytes + p.experts * 8;
  sh.kept = reinterpret_cast<uint32_t *>(more + (size_t)slot * group_bytes + p.experts * 8 +
                                         p.groups * 8);
  for (uint32_t e = threadIdx.x; e < p.experts; e += kThreads) count[e] = 0;
  __syncthreads();
  const uint32_t first = min((uint64_t)blockIdx.x * p.run, (uint64_t)p.tokens);
  const uint32_t end = min((uint64_t)first + p.run, (uint64_t)p.tokens);
  for (uint32_t t0 = first + warp * kTokens; t0 < end; t0 += kWarps * kTokens) {
    const uint32_t token = t0 + lane / kLanes;
    const bool here = token < end;
    bool valid = here;
    if (here && p.lengths) valid = (int64_t)(token % p.seq) < (int64_t)p.lengths[token / p.seq];
    float l[V];
    bool open[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t e = sub * V + i;
      open[i] = valid && e < p.experts;
      l[i] = open[i] ? logit_at(p, token, e) : -INFINITY;
      open[i] = open[i] && l[i] != -INFINITY;
      if (open[i] && p.bias) open[i] = __ldg(p.bias + e) != -INFINITY;
    }
    if (p.bias || p.groups > 1) {
      const bool unsure = score_and_choose<kLanes, V, float>(p, sh, token, sub, l, open);
      if (__any_sync(kFull, unsure)) score_and_choose<kLanes, V, double>(p, sh, token, sub, l, open);
    } else {
      uint32_t key[V];
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = open[i] ? key_of(l[i]) : 0;
      choose<kLanes, V, float>(p, sh, token, sub, key, l, 0.f);
    }
    // Weights.  With a common factor taken out first: e^l by the largest l, and for the sigmoid
    // e^min(l, 0) / (1 + e^-|l|) by the largest of the numerators; renormalised it cancels.
    float top = -INFINITY, total = 1.f;
    if (p.softmax && !p.renormalise) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (open[i]) top = fmaxf(top, l[i]);
      top = lanes_max<kLanes>(top);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (open[i]) sum += expf(l[i] - top);
      total = lanes_sum<kLanes>(sum);
    } else if (p.renormalise) {
      for (uint32_t j = sub; j < p.top_k; j += kLanes)
        if (sh.chosen[j] != kNone) {
          const float x = logit_at(p, token, sh.chosen[j]);
          top = fmaxf(top, p.softmax ? x : fminf(x, 0.f));
        }
      top = lanes_max<kLanes>(top);
    } else {
      top = 0.f;
    }
    auto score = [&](uint32_t e) {
      const float x = logit_at(p, token, e);
      return p.softmax ? expf(x - top) : expf(fminf(x, 0.f) - top) / (1.f + expf(-fabsf(x)));
    };
    if (p.renormalise) {
      float sum = 0.f;
      for (uint32_t j = sub; j < p.top_k; j += kLanes)
        if (sh.chosen[j] != kNone) sum += score(sh.chosen[j]);
      total = lanes_sum<kLanes>(sum);
    }
    if (here) {
      for (uint32_t j = sub; j < p.top_k; j += kLanes) {
        const uint32_t e = sh.chosen[j];
        const size_t at = (size_t)token * p.top_k + j;
        p.chosen[at] = e == kNone ? -1 : (int32_t)e;
        p.weights[at] = e == kNone ? 0.f : score(e) / total * p.scale;
        if (p.order && e != kNone) atomicAdd(count + e, 1u);
      }
    }
    __syncwarp();
  }
  if (!p.order) return;
  __syncthreads();
  if (gridDim.x > 1) {
    for (uint32_t e = threadIdx.x; e < p.experts; e += kThreads)
      p.counts[(size_t)blockIdx.x * p.experts + e] = count[e];
    return;
  }
  scan_counts(count, offset, p.experts);
  for (uint32_t e = threadIdx.x; e <= p.experts; e += kThreads) p.offsets[e] = (int32_t)offset[e];
  place_pairs(p, 0, (uint64_t)p.tokens * p.top_k, offset,
              reinterpret_cast<uint32_t *>(smem + p.off_places));
}

// Places the pairs of run blockIdx.x behind those of the runs before it.
__global__ void __launch_bounds__(kThreads) place_kernel(const __grid_constant__ RouteProblem p) {
  extern __shared__ __align__(16) uint8_t smem[];
  uint32_t *total = reinterpret_cast<uint32_t *>(smem), *base = total + p.experts;
  uint32_t *offset = base + p.experts;
  for (uint32_t e = threadIdx.x; e < p.experts; e += kThreads) total[e] = base[e] = 0;
  __syncthreads();
  // Threads side by side take experts, the rest of them runs.
  uint32_t wide = 32;
  while (wide < p.experts && wide < kThreads) wide *= 2;
  const uint32_t part = threadIdx.x / wide, parts = kThreads / wide;
  for (uint32_t e = threadIdx.x % wide; e < p.experts; e += wide) {
    uint32_t all = 0, before = 0;
#pragma unroll 8
    for (uint32_t b = part; b < gridDim.x; b += parts) {
      const uint32_t n = __ldcg(p.counts + (size_t)b * p.experts + e);
      all += n;
      if (b < blockIdx.x) before += n;
    }
    atomicAdd(total + e, all);
    atomicAdd(base + e, before);
  }
  __syncthreads();
  scan_counts(total, offset, p.experts);
  for (uint32_t e = threadIdx.x; e < p.experts; e += kThreads) base[e] += offset[e];
  if (blockIdx.x == 0)
    for (uint32_t e = threadIdx.x; e <= p.experts; e += kThreads) p.offsets[e] = (int32_t)offset[e];
  __syncthreads();
  const uint64_t first = min((uint64_t)blockIdx.x * p.run, (uint64_t)p.tokens);
  const uint64_t end = min(first + p.run, (uint64_t)p.tokens);
  place_pairs(p, first * p.top_k, end * p.top_k, base, offset + p.experts + 1);
}

template <int kLanes, int V>
cudaError_t run(RouteProblem p, cudaStream_t stream) {
  constexpr uint32_t kTokens = kWarps * (32 / kLanes);  // a block's at a time
  uint32_t bytes = (2 * p.experts + 1 + kTokens * kMaxK) * 4;
  bytes = (bytes + 15) / 16 * 16;
  p.off_groups = bytes;
  if (p.groups > 1) bytes += kTokens * (p.experts * 8 + p.groups * 12 + (p.groups & 1) * 4);
  // One block plans from the same memory once its tokens are routed.
  p.off_places = p.off_groups;
  const uint32_t places = kWarps * p.experts * 4;
  if (p.blocks == 1 && p.order) bytes = std::max(bytes, p.off_places + places);
  static std::atomic<uint64_t> seen{0}, seen_place{0};
  cudaError_t e = allow_smem((const void *)route_kernel<kLanes, V>, 232448, seen);
  if (e != cudaSuccess) return e;
  route_kernel<kLanes, V><<<p.blocks, kThreads, bytes, stream>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess || p.blocks == 1 || !p.order) return e;
  if ((e = allow_smem((const void *)place_kernel, 232448, seen_place)) != cudaSuccess) return e;
  place_kernel<<<p.blocks, kThreads, (3 * p.experts + 1) * 4 + places, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

// Runs of tokens: one while a single block is the faster way, else a block for each SM.
void route_plan(RouteProblem *p, int num_sms) {
  p->run = std::max<uint32_t>(128, (uint32_t)(((uint64_t)p->tokens + num_sms - 1) / num_sms));
  p->blocks = (p->tokens + p->run - 1) / p->run;
}

cudaError_t launch_experts_route(const RouteProblem &p, cudaStream_t stream) {
  if (p.experts <= 16) return run<4, 4>(p, stream);
  if (p.experts <= 32) return run<8, 4>(p, stream);
  if (p.experts <= 64) return run<8, 8>(p, stream);
  if (p.experts <= 128) return run<16, 8>(p, stream);
  if (p.experts <= 256) return run<32, 8>(p, stream);
  if (p.experts <= 512) return run<32, 16>(p, stream);
  return run<32, 32>(p, stream);
}

}  // namespace tx
