// Parts shared by the linear layers on tcgen05 (linear_fused.cu, experts_linear.cu): bounded waits,
// activations of the epilogue, and the entry point that makes tensor maps.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "../../include/tessattn.h"
#include "common.cuh"
#include "tcgen05.cuh"

namespace tx {
namespace lfused {

using namespace ptx;

constexpr long long kDrainCycles = 2000000000ll;

// kCluster: threads or products of the other CTA of a pair arrive at the barrier.
template <bool kCluster>
__device__ __forceinline__ bool test_bar(uint32_t bar, uint32_t parity) {
  if constexpr (kCluster)
    return mbar_test_cluster(bar, parity);
  else
    return mbar_test(bar, parity);
}
template <bool kCluster = false>
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile int *abort_flag,
                                         int *status, int site, long long limit) {
  if (test_bar<kCluster>(bar, parity)) return true;
  const long long t0 = clock64();
  while (true) {
    if (test_bar<kCluster>(bar, parity)) return true;
    if (*abort_flag) return false;
    if (clock64() - t0 > limit) {
      *abort_flag = 1;
      report_status(status, kStatusTimeout | (site << 8));
      return false;
    }
  }
}
// since: where several are drained in turn, when the first began.
template <bool kCluster = false>
__device__ __forceinline__ void drain_bar(uint32_t bar, uint32_t parity, long long since) {
  while (!test_bar<kCluster>(bar, parity) && clock64() - since < kDrainCycles) {
  }
}
template <bool kCluster = false>
__device__ __forceinline__ void drain_bar(uint32_t bar, uint32_t parity) {
  drain_bar<kCluster>(bar, parity, clock64());
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// TX_ACT_GELU for fp32 results, and where the value is multiplied (gated products): a kernel of its own, or
// chosen as the tile ends.
constexpr int kGeluF32 = TX_ACT_SILU + 1;

// The hardware exponential and reciprocal (2^-22 of the value each) in place of exp and a
// division: the epilogue's arithmetic is what bounds a layer of small k.
template <int kAct>
__device__ __forceinline__ float activate(float y) {
  constexpr float kLog2e = 1.44269504088896341f;
  if constexpr (kAct == TX_ACT_RELU) {
    return y < 0.f ? 0.f : y;
  } else if constexpr (kAct == kGeluF32) {
    // Q(z) = erfc(z / sqrt 2) / 2 = e^(-z^2 / 2) t p(t), t = 1 / (1 + 0.3 z), z = |y|, p a fit of degree 7
    // (least squares of the relative error, reweighted to equal ripples: 5e-8 up to z = 10); gelu =
    // y (1 - Q) for y > 0 and y Q below, so the negative side does not cancel.  The Newton step takes
    // the reciprocal's error from t.  2^-21.7 |y| in all, and 2^-18 of the value down to y = -8
    // (erfcf takes 53 us for 8192 x 1536 x 384 where this takes 35 and the form below 31).
    const float z = fminf(fabsf(y), 16.f), d = fmaf(z, 0.3f, 1.f);
    float t = rcp(d);
    t = fmaf(t, fmaf(-d, t, 1.f), t);
    float q = fmaf(t, 0.0375477113f, -0.165076032f);
    q = fmaf(t, q, 0.220082358f);
    q = fmaf(t, q, -0.0665214509f);
    q = fmaf(t, q, 0.13549459f);
    q = fmaf(t, q, 0.0977567211f);
    q = fmaf(t, q, 0.12111108f);
    q = fmaf(t, q, 0.119605049f);
    q *= t * ex2(z * (z * (-0.5f * kLog2e)));
    return y * (y > 0.f ? 1.f - q : q);
  } else if constexpr (kAct == TX_ACT_GELU) {
    // 1 - erf(z), z = |y| / sqrt 2, as 1 / (1 + a1 z + ... + a6 z^6)^16 (Abramowitz and Stegun
    // 7.1.28, absolute error 3e-7), the coefficients here for |y|; gelu = y (1 - tail / 2) for
    // y > 0 and y tail / 2 below.  One special function (7.1.26 takes an exponential as well: 26.7
    // against 25.0 us at 8192 x 1536 x 384).  The 16th power takes the reciprocal's rounding
    // with it: 1.4e-6 |y| in all, which below y = -4 is more than the rounding to bf16 (0.4 % of the
    // value there, 5 % at -5), so an fp32 result takes the form above.
    const float z = fabsf(y);
    float q = fmaf(z, 5.38297500e-06f, 4.88906374e-05f);
    q = fmaf(z, q, 3.80035750e-05f);
    q = fmaf(z, q, 3.27762630e-03f);
    q = fmaf(z, q, 2.11410062e-02f);
    q = fmaf(z, q, 4.98673469e-02f);
    q = rcp(fmaf(z, q, 1.f));
    q *= q;
    q *= q;
    q *= q;
    const float tail = 0.5f * (q * q);
    return y * (y > 0.f ? 1.f - tail : tail);
  } else if constexpr (kAct == TX_ACT_GELU_TANH) {  // (1 + tanh u) / 2 = 1 / (1 + e^(-2u))
    const float u = y * fmaf(0.044715f, y * y, 1.f);
    return y * rcp(1.f + ex2(u * (-1.5957691216057308f * kLog2e)));
  } else if constexpr (kAct == TX_ACT_SILU) {
    return y * rcp(1.f + ex2(y * -kLog2e));
  } else {
    return y;
  }
}

inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void *ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return (PFN_cuTensorMapEncodeTiled_v12000)ptr;
  }();
  return fn;
}
}  // namespace lfused
}  // namespace tx
