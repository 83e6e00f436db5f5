// Linear layer with bias, activation and residual in its epilogue (tx_linear_fused):
//   out = act(x w^T + bias) + residual,  x [m, k] and w [n, k] bf16, fp32 sums,
// any m, n and k, rows of x and w on 16-byte boundaries.
//
// linear_kernel: 128 x BN tiles on tcgen05 (kind::f16), K through a ring of 64-column stages
// filled by TMA (128-byte swizzle; rows past m or n and columns past k arrive as zeros), two
// accumulators in tensor memory so that eight epilogue warps finish one tile while the next is
// multiplied; persistent, one CTA per SM.  Results leave through shared memory and TMA stores
// (whole 128-byte rows; a thread that stored its own row directly wrote 16 bytes to each of 32
// rows per instruction), and a residual of the output's type comes in the same way, a box ahead.
// Bound: for large k the tiles' way from L2 to shared memory (9.8 TB/s at 128 x 256), for small k
// the epilogue.  Measured: 33500 x 1024 x 2048 into an fp32 residual 170 us, 827 TFLOP/s; 8192 x
// 1536 x 384 with GELU 25 us, 387 TFLOP/s; 777 x 1000 x 1001 12.3 us.
// Few tiles of long k: k is cut over CTAs, whose partial sums the last to arrive adds up.
// gemv_kernel: a few rows (m <= 8) only stream w once: one or four warps per output column, w
// straight from global memory into registers, the sums over lanes by shuffles.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "../../include/tessattn.h"
#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace tx {
namespace lfused {

using namespace ptx;

constexpr int kBM = 128;
constexpr uint32_t kBK = 64;
constexpr int kThreads = 320;  // warp 0 TMA, warp 1 MMA, warps 2-9 epilogue
constexpr int kMaxStages = 8;
constexpr uint32_t kPart = 8;  // K stages (512 columns) of one partial sum
constexpr uint32_t kBufBytes = 32 * 128;  // staging: 32 rows x 128 bytes, two per epilogue warp
constexpr long long kDrainCycles = 2000000000ll;

template <int kBN>
struct Cfg {
  static constexpr uint32_t kABytes = kBM * 128, kBBytes = kBN * 128;
  static constexpr uint32_t kStageBytes = kABytes + kBBytes;
  static constexpr uint32_t kStaging = kBN >= 128 ? 8 * 2 * kBufBytes : 0;
  static constexpr int kFit = (int)((232448 - 1024 - kStaging) / kStageBytes);
  static constexpr int kStages = kFit < kMaxStages ? kFit : kMaxStages;
  static constexpr uint32_t kOffStaging = kStages * kStageBytes;
  static constexpr uint32_t kOffMisc = kOffStaging + kStaging;
  static constexpr uint32_t kSmemBytes = kOffMisc + 512;
  static constexpr uint32_t kTmemCols = 2 * kBN;
  static constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) |
                                     ((uint32_t)(kBN >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
};
enum : uint32_t { kBarFull = 0, kBarEmpty = kMaxStages, kBarAcc = 2 * kMaxStages,
                  kBarFree = kBarAcc + 2, kBarDrain = kBarFree + 2,
                  kBarRes = kBarDrain + 1,  // + 2 * epilogue warp + buffer: residual landed
                  kNumBars = kBarRes + 16 };
enum : uint32_t { kOffTmem = 8 * kNumBars, kOffAbort = kOffTmem + 4 };
static_assert(kOffAbort + 4 <= 512, "misc area");
enum : int { kSiteEmpty = 1, kSiteFull = 2, kSiteAcc = 3, kSiteFree = 4, kSiteRes = 5 };

__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile int *abort_flag,
                                         int *status, int site, long long limit) {
  if (mbar_test(bar, parity)) return true;
  const long long t0 = clock64();
  while (true) {
    if (mbar_test(bar, parity)) return true;
    if (*abort_flag) return false;
    if (clock64() - t0 > limit) {
      *abort_flag = 1;
      report_status(status, kStatusTimeout | (site << 8));
      return false;
    }
  }
}
__device__ __forceinline__ void drain_bar(uint32_t bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_test(bar, parity) && clock64() - t0 < kDrainCycles) {
  }
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

// TX_ACT_GELU for fp32 results: a kernel of its own.
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

__device__ __forceinline__ float residual_at(const LinearFusedProblem &p, size_t i) {
  return p.residual_dtype == 1 ? bf16_bits_to_f32(static_cast<const uint16_t *>(p.residual)[i])
                               : static_cast<const float *>(p.residual)[i];
}
__device__ __forceinline__ void store_at(const LinearFusedProblem &p, size_t i, float v) {
  if (p.out_dtype == 1)
    static_cast<uint16_t *>(p.out)[i] = f32_to_bf16_bits(v);
  else
    static_cast<float *>(p.out)[i] = v;
}

// How the epilogue reaches global memory, chosen by the launcher.
enum : int {
  kDirect = 0,   // element by element or 16 bytes at a time, a thread per row
  kStaged = 1,   // results through shared memory and TMA stores, the residual read directly
  kStagedRes = 2 // the residual too: loaded by TMA into the buffer its sum leaves from
};

// kLong: k takes more than one partial sum.  Kernels of their own, since the sums' registers and
// the rolled loop in one kernel left spills in the first (178 against 169 us at 33500 x 1024 x 2048).
template <int kBN, int kAct, bool kLong>
__global__ void __launch_bounds__(kThreads, 1)
    linear_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                  const __grid_constant__ CUtensorMap tm_res,
                  const __grid_constant__ CUtensorMap tm_out,
                  const __grid_constant__ LinearFusedProblem p) {
  using C = Cfg<kBN>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_addr(smem), bars = sbase + C::kOffMisc;
  auto bar = [&](uint32_t i) { return bars + 8u * i; };
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + C::kOffMisc + kOffAbort);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t nt = (p.n + kBN - 1) / kBN, mt = (p.m + kBM - 1) / kBM, tiles = nt * mt;
  const uint32_t nk_all = (p.k + kBK - 1) / kBK;
  // With a split k (64 columns, long k) a CTA has one tile and one part of k.
  constexpr bool kSplits = kLong && kBN == 64;
  const uint32_t splits = kSplits ? p.splits : 1, split = kSplits ? blockIdx.x % splits : 0;
  const uint32_t tile_first = kSplits ? blockIdx.x / splits : blockIdx.x;
  const uint32_t tile_step = kSplits && splits > 1 ? tiles : gridDim.x;
  const uint32_t kb_first = kSplits ? nk_all * split / splits : 0;
  const uint32_t nk = kSplits ? nk_all * (split + 1) / splits : nk_all;
  const uint32_t parts = (nk - kb_first + kPart - 1) / kPart;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(bar(kBarFull + s), 1);
      mbar_init(bar(kBarEmpty + s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar(kBarAcc + b), 1);
      mbar_init(bar(kBarFree + b), 256);
    }
    mbar_init(bar(kBarDrain), 1);
    for (int b = 0; b < 16; ++b) mbar_init(bar(kBarRes + b), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     bars + kOffTmem),
                 "r"(C::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<uint32_t *>(smem + C::kOffMisc + kOffTmem);

  if (warp == 0) {
    if (lane == 0) {
      uint32_t fills = 0;
      bool ok = true;
      for (uint32_t tile = tile_first; ok && tile < tiles; tile += tile_step) {
        const int m0 = (int)(tile / nt * kBM), n0 = (int)(tile % nt * kBN);
        for (uint32_t kb = kb_first; kb < nk; ++kb) {
          const uint32_t s = fills % C::kStages, round = fills / C::kStages;
          if (round && !(ok = wait_bar(bar(kBarEmpty + s), (round - 1) & 1, abort_flag, p.status,
                                       kSiteEmpty, p.wait_cycles)))
            break;
          const uint32_t dst = sbase + s * C::kStageBytes;
          mbar_expect_tx(bar(kBarFull + s), C::kStageBytes);
          tma_load_2d(dst, &tm_x, bar(kBarFull + s), (int)(kb * kBK), m0);
          tma_load_2d(dst + C::kABytes, &tm_w, bar(kBarFull + s), (int)(kb * kBK), n0);
          ++fills;
        }
      }
      // No copy may land after the CTA has gone.
      for (uint32_t s = 0; s < (uint32_t)C::kStages && s < fills; ++s)
        drain_bar(bar(kBarFull + s), ((fills - 1 - s) / C::kStages) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t step = 0, done = 0;  // K stages, partial sums
      bool ok = true;
      for (uint32_t tile = tile_first; ok && tile < tiles; tile += tile_step) {
        for (uint32_t kb = kb_first; ok && kb < nk; ++done) {
          const uint32_t b = done & 1, acc = tmem + b * kBN;
          if (done >= 2 && !(ok = wait_bar(bar(kBarFree + b), ((done >> 1) - 1) & 1, abort_flag,
                                           p.status, kSiteFree, p.wait_cycles)))
            break;
          tc_fence_after();
          const uint32_t end = min(kb + kPart, nk);
          for (uint32_t first = kb; kb < end; ++kb, ++step) {
            const uint32_t s = step % C::kStages;
            if (!(ok = wait_bar(bar(kBarFull + s), (step / C::kStages) & 1, abort_flag, p.status,
                                kSiteFull, p.wait_cycles)))
              break;
            tc_fence_after();
            const uint32_t st = sbase + s * C::kStageBytes;
            const uint64_t ad = sw128_desc(st, 16, 1024), bd = sw128_desc(st + C::kABytes, 16, 1024);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              umma(acc, ad + ks * 2, bd + ks * 2, C::kIdesc, kb > first || ks > 0);
            umma_commit(bar(kBarEmpty + s));
          }
          if (ok) umma_commit(bar(kBarAcc + b));
        }
      }
      umma_commit(bar(kBarDrain));
      drain_bar(bar(kBarDrain), 0);
    }
    __syncwarp();
  } else {
    // Warp w finishes columns [half * kCols, +kCols) of the 32 rows of its tensor-memory quarter.
    constexpr uint32_t kCols = kBN / 2;
    const uint32_t quarter = (uint32_t)warp & 3, half = (uint32_t)(warp - 2) >> 2;
    const uint32_t staging = sbase + C::kOffStaging + (uint32_t)(warp - 2) * 2 * kBufBytes;
    const uint32_t res_bar = kBarRes + 2 * (uint32_t)(warp - 2);
    const int mode = kBN >= 128 ? p.epilogue : kDirect;
    const bool f32_out = p.out_dtype == 0;
    uint32_t done = 0, sent = 0;               // partial sums taken, boxes stored
    uint32_t res_loads = 0, res_used = 0;      // residual boxes asked for and consumed
    bool ok = true;
    // Residual box number `res_loads` (columns from n, rows from m) into its buffer, once the
    // store that last left from there has been read.
    auto load_residual = [&](uint32_t n, uint32_t m) {
      const uint32_t b = res_loads & 1;
      if (lane == 0) {
        bulk_wait_read<0>();
        mbar_expect_tx(bar(res_bar + b), kBufBytes);
        tma_load_2d(staging + b * kBufBytes, &tm_res, bar(res_bar + b), (int)n, (int)m);
      }
      ++res_loads;
    };
    for (uint32_t tile = tile_first; ok && tile < tiles; tile += tile_step) {
      const uint32_t m0 = tile / nt * kBM + quarter * 32, m = m0 + lane;
      const uint32_t n0 = tile % nt * kBN + half * kCols;
      const uint32_t box = f32_out ? 32 : 64;  // columns of a 128-byte staging row
      const bool rows = m0 < p.m && n0 < p.n;  // this warp has something to write
      if (mode == kStagedRes && rows) load_residual(n0, m0);
      // Bias, activation, residual and store of columns [c, c + 32) of this warp's share.
      auto finish = [&](uint32_t c, float *v) {
        const uint32_t n = n0 + c;
        if (rows && n < p.n && ok) {
        const bool whole = n + 32 <= p.n;
        if (p.bias) {
          if (whole && p.bias_vec) {
#pragma unroll
            for (int t = 0; t < 8; ++t) {
              const float4 q = __ldg(reinterpret_cast<const float4 *>(p.bias + n) + t);
              v[4 * t] += q.x; v[4 * t + 1] += q.y;
              v[4 * t + 2] += q.z; v[4 * t + 3] += q.w;
            }
          } else {
#pragma unroll
            for (int t = 0; t < 32; ++t)
              if (n + t < p.n) v[t] += __ldg(p.bias + n + t);
          }
        }
#pragma unroll
        for (int t = 0; t < 32; ++t) v[t] = activate<kAct>(v[t]);
        if (p.residual && mode != kStagedRes && m < p.m) {
          const size_t at = (size_t)m * p.ldr + n;
          if (whole && p.res_vec && p.residual_dtype == 0) {
#pragma unroll
            for (int t = 0; t < 8; ++t) {
              const float4 q = reinterpret_cast<const float4 *>(
                  static_cast<const float *>(p.residual) + at)[t];
              v[4 * t] += q.x; v[4 * t + 1] += q.y;
              v[4 * t + 2] += q.z; v[4 * t + 3] += q.w;
            }
          } else if (whole && p.res_vec) {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const uint4 q = reinterpret_cast<const uint4 *>(
                  static_cast<const uint16_t *>(p.residual) + at)[t];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                v[8 * t + 2 * e] += bf16_lo(u4_at(q, e));
                v[8 * t + 2 * e + 1] += bf16_hi(u4_at(q, e));
              }
            }
          } else {
#pragma unroll
            for (int t = 0; t < 32; ++t)
              if (n + t < p.n) v[t] += residual_at(p, at + t);
          }
        }
        if (mode == kDirect) {
          const size_t at = (size_t)m * p.ldo + n;
          if (m >= p.m) {
          } else if (whole && p.out_vec && f32_out) {
#pragma unroll
            for (int t = 0; t < 8; ++t)
              reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at)[t] = make_float4(
                  v[4 * t], v[4 * t + 1], v[4 * t + 2], v[4 * t + 3]);
          } else if (whole && p.out_vec) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
              reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out) + at)[t] =
                  make_uint4(pack_bf16x2(v[8 * t], v[8 * t + 1]),
                             pack_bf16x2(v[8 * t + 2], v[8 * t + 3]),
                             pack_bf16x2(v[8 * t + 4], v[8 * t + 5]),
                             pack_bf16x2(v[8 * t + 6], v[8 * t + 7]));
          } else {
#pragma unroll
            for (int t = 0; t < 32; ++t)
              if (n + t < p.n) store_at(p, at + t, v[t]);
          }
        } else if constexpr (kBN >= 128) {
          // A staging row is 128 bytes of this lane's output row, its 16-byte pieces swizzled as
          // the tensor map has them; bf16 takes two 32-column steps to fill one.
          const bool starts = f32_out || c % 64 == 0, ends = f32_out || c % 64 == 32;
          uint32_t b;
          if (mode == kStagedRes) {
            b = res_used & 1;
            if (starts) {
              // The next box, if this tile has one, travels while this one is finished.
              if (c + box < kCols && n + box < p.n) load_residual(n + box, m0);
              ok = __all_sync(0xffffffffu, wait_bar(bar(res_bar + b), (res_used >> 1) & 1,
                                                    abort_flag, p.status, kSiteRes, p.wait_cycles));
            }
          } else {
            b = sent & 1;
            if (starts) {
              if (lane == 0) bulk_wait_read<1>();
              __syncwarp();
            }
          }
          const uint32_t row = staging + b * kBufBytes + (uint32_t)lane * 128, sw = lane & 7;
          if (f32_out) {
#pragma unroll
            for (uint32_t q = 0; q < 8; ++q) {
              const uint32_t at = row + ((q ^ sw) << 4);
              if (mode == kStagedRes) {
                const uint4 o = ld_shared_v4(at);
                v[4 * q] += __uint_as_float(o.x);
                v[4 * q + 1] += __uint_as_float(o.y);
                v[4 * q + 2] += __uint_as_float(o.z);
                v[4 * q + 3] += __uint_as_float(o.w);
              }
              st_shared_v4(at, __float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]),
                           __float_as_uint(v[4 * q + 2]), __float_as_uint(v[4 * q + 3]));
            }
          } else {
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q) {
              const uint32_t at = row + (((q + (c % 64) / 8) ^ sw) << 4);
              if (mode == kStagedRes) {
                const uint4 o = ld_shared_v4(at);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  v[8 * q + 2 * e] += bf16_lo(u4_at(o, e));
                  v[8 * q + 2 * e + 1] += bf16_hi(u4_at(o, e));
                }
              }
              st_shared_v4(at, pack_bf16x2(v[8 * q], v[8 * q + 1]),
                           pack_bf16x2(v[8 * q + 2], v[8 * q + 3]),
                           pack_bf16x2(v[8 * q + 4], v[8 * q + 5]),
                           pack_bf16x2(v[8 * q + 6], v[8 * q + 7]));
            }
          }
          if (ends || n + 32 >= p.n) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tm_out, staging + b * kBufBytes, (int)(n - c % box), (int)m0);
              bulk_commit();
            }
            ++sent;
            if (mode == kStagedRes) ++res_used;
          }
        }
        }
        __syncwarp();
      };
      const uint32_t lanes = (quarter * 32u) << 16;
      if constexpr (kLong) {
        // Partial sums of 512 K are added in fp32 registers: the accumulator cuts off bits at each of
        // its additions, always towards zero, and over 2048 K in one go that left an error of 2e-6
        // of the result, eight times that of fp32 products in fp32.  The accumulator is free again
        // before the epilogue (putting the sum back into it for the rolled loop below: 169 -> 194 us
        // at 33500 x 1024 x 2048).
        float v[kCols];
        for (uint32_t part = 0; part < parts; ++part, ++done) {
          const uint32_t b = done & 1, t0 = tmem + b * kBN + half * kCols + lanes;
          if (!(ok = __all_sync(0xffffffffu, wait_bar(bar(kBarAcc + b), (done >> 1) & 1, abort_flag,
                                                      p.status, kSiteAcc, p.wait_cycles))))
            break;
          tc_fence_after();
#pragma unroll
          for (uint32_t c = 0; c < kCols; c += 16) {
            uint32_t a[16];
            tmem_load(t0 + c, a);
#pragma unroll
            for (int t = 0; t < 16; ++t)
              v[c + t] = part ? v[c + t] + __uint_as_float(a[t]) : __uint_as_float(a[t]);
          }
          tc_fence_before();
          mbar_arrive(bar(kBarFree + b));
        }
        bool mine = true;
        if constexpr (kSplits) {
          // Every warp leaves its part of the tile; the one that arrives last adds them in the order
          // of the splits and finishes.  All arrive, whatever happened, so that the counters return
          // to zero.
          if (splits > 1) {
            const uint32_t w = (uint32_t)warp - 2;
            auto at = [&](uint32_t s) {
              return p.part + ((((size_t)tile * splits + s) * 8 + w) * kCols) * 32 + lane;
            };
            float *to = at(split);
#pragma unroll
            for (uint32_t c = 0; c < kCols; ++c) to[c * 32] = v[c];
            __threadfence();
            __syncwarp();
            uint32_t before = 0;
            if (lane == 0) before = atomicAdd(&p.arrived[tile * 8 + w], 1u);
            mine = __shfl_sync(0xffffffffu, before, 0) + 1 == splits;
            if (mine) {
              if (lane == 0) p.arrived[tile * 8 + w] = 0;
              __threadfence();
#pragma unroll
              for (uint32_t c = 0; c < kCols; ++c) v[c] = 0.f;
              for (uint32_t s = 0; s < splits; ++s) {
                const float *from = at(s);
#pragma unroll
                for (uint32_t c = 0; c < kCols; ++c) v[c] += __ldcg(from + c * 32);
              }
            }
          }
        }
        if (mine) {
#pragma unroll
          for (uint32_t c = 0; c < kCols; c += 32) finish(c, v + c);
        }
      } else {
        const uint32_t b = done & 1, t0 = tmem + b * kBN + half * kCols + lanes;
        ok = __all_sync(0xffffffffu, wait_bar(bar(kBarAcc + b), (done >> 1) & 1, abort_flag,
                                              p.status, kSiteAcc, p.wait_cycles));
        if (!ok) break;
        tc_fence_after();
        ++done;
        // Rolled: unrolled over the columns the epilogue did not stay in the instruction cache (36.5
        // against 32.8 us at 8192 x 1536 x 384 with GELU).
#pragma unroll 1
        for (uint32_t c = 0; c < kCols; c += 32) {
          uint32_t acc[32];
          float v[32];
          tmem_load(t0 + c, acc);
#pragma unroll
          for (int t = 0; t < 32; ++t) v[t] = __uint_as_float(acc[t]);
          finish(c, v);
        }
        tc_fence_before();
        mbar_arrive(bar(kBarFree + b));
      }
    }
    if (mode != kDirect) {
      if (lane == 0) {
        // Residual boxes that an abort left in flight, and every store, end before the CTA does.
        for (; res_used < res_loads; ++res_used)
          drain_bar(bar(res_bar + (res_used & 1)), (res_used >> 1) & 1);
        bulk_wait_all();
      }
      __syncwarp();
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(C::kTmemCols)
                 : "memory");
}

// ---- a few rows -----------------------------------------------------------------------------
// One warp per output column, or the block's four warps with a quarter of K each (kSplit = 4); lane l
// takes columns 8l .. 8l+7 of every 256 of its part.
constexpr uint32_t kGemvWarps = 4;

template <int kM, uint32_t kSplit, int kAct>
__global__ void __launch_bounds__(32 * kGemvWarps) gemv_kernel(const __grid_constant__ LinearFusedProblem p) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t n = (blockIdx.x * kGemvWarps + warp) / kSplit, part = warp % kSplit;
  __shared__ float parts[kSplit][kM];
  const bool live = n < p.n;
  float sum[kM];
#pragma unroll
  for (int i = 0; i < kM; ++i) sum[i] = 0.f;
  if (live) {
    const uint16_t *x = static_cast<const uint16_t *>(p.x);
    const uint16_t *w = static_cast<const uint16_t *>(p.w) + (size_t)n * p.ldw;
#pragma unroll 4
    for (uint32_t c = part * 256 + lane * 8; c < p.k; c += 256 * kSplit) {
      const uint4 wv = __ldg(reinterpret_cast<const uint4 *>(w + c));
      float wf[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t q = u4_at(wv, e / 2);
        wf[e] = c + e < p.k ? (e & 1 ? bf16_hi(q) : bf16_lo(q)) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < kM; ++i) {
        if ((uint32_t)i >= p.m) break;
        const uint4 xv = __ldg(reinterpret_cast<const uint4 *>(x + (size_t)i * p.ldx + c));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t q = u4_at(xv, e / 2);
          const float xf = c + e < p.k ? (e & 1 ? bf16_hi(q) : bf16_lo(q)) : 0.f;
          sum[i] = fmaf(xf, wf[e], sum[i]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kM; ++i) sum[i] = warp_sum(sum[i]);
  if constexpr (kSplit > 1) {
#pragma unroll
    for (int i = 0; i < kM; ++i)
      if (lane == 0) parts[part][i] = sum[i];
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int i = 0; i < kM; ++i) {
      sum[i] = parts[0][i];
#pragma unroll
      for (uint32_t s = 1; s < kSplit; ++s) sum[i] += parts[s][i];
    }
  }
  // Lane i finishes row i.
  float y = 0.f;
#pragma unroll
  for (int i = 0; i < kM; ++i)
    if (lane == (uint32_t)i) y = sum[i];
  if (live && lane < p.m) {
    if (p.bias) y += p.bias[n];
    y = activate<kAct>(y);
    if (p.residual) y += residual_at(p, (size_t)lane * p.ldr + n);
    store_at(p, (size_t)lane * p.ldo + n, y);
  }
}

template <int kM, uint32_t kSplit, int kAct>
cudaError_t launch_columns(const LinearFusedProblem &p, cudaStream_t stream) {
  constexpr uint32_t columns = kGemvWarps / kSplit;
  gemv_kernel<kM, kSplit, kAct><<<(p.n + columns - 1) / columns, 32 * kGemvWarps, 0, stream>>>(p);
  return cudaGetLastError();
}

// Four warps a column against one: 10.1 / 14.3 us for 1 x 1024 x 4096, 10 / 23 us for 2 x 1024 x 4096,
// 10.2 / 10.2 us for 1 x 4096 x 1024, but 18.5 / 14.4 us for 1 x 16384 x 1024.
template <int kAct>
cudaError_t launch_gemv(const LinearFusedProblem &p, cudaStream_t stream) {
  if (p.m == 1)
    return p.n > 8192 ? launch_columns<1, 1, kAct>(p, stream) : launch_columns<1, 4, kAct>(p, stream);
  return p.m <= 2   ? launch_columns<2, 4, kAct>(p, stream)
         : p.m <= 4 ? launch_columns<4, 4, kAct>(p, stream)
                    : launch_columns<8, 4, kAct>(p, stream);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
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
// Row-major [rows, cols] of bf16 or fp32 with a row stride in elements; boxes of 128 bytes of
// columns in the 128-byte swizzle.
bool make_map(CUtensorMap *map, const void *base, uint32_t rows, uint32_t cols, uint64_t ld,
              uint32_t box_rows, bool f32 = false) {
  auto fn = encode_fn();
  if (!fn) return false;
  const uint32_t e = f32 ? 4 : 2;
  cuuint64_t dims[2] = {cols, rows};
  cuuint64_t strides[1] = {ld * e};
  cuuint32_t box[2] = {128 / e, box_rows};
  cuuint32_t elem[2] = {1, 1};
  return fn(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
            const_cast<void *>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int kBN, int kAct, bool kLong>
cudaError_t launch_tiles(const LinearFusedProblem &p, int num_sms, cudaStream_t stream) {
  constexpr uint32_t smem = Cfg<kBN>::kSmemBytes;
  CUtensorMap mx, mw, mr, mo;
  if (!make_map(&mx, p.x, p.m, p.k, p.ldx, kBM) || !make_map(&mw, p.w, p.n, p.k, p.ldw, kBN))
    return cudaErrorInvalidValue;
  mr = mo = mx;
  if (p.epilogue != kDirect && !make_map(&mo, p.out, p.m, p.n, p.ldo, 32, p.out_dtype == TX_F32))
    return cudaErrorInvalidValue;
  if (p.epilogue == kStagedRes &&
      !make_map(&mr, p.residual, p.m, p.n, p.ldr, 32, p.out_dtype == TX_F32))
    return cudaErrorInvalidValue;
  static std::atomic<uint64_t> seen{0};
  cudaError_t e = allow_smem((const void *)linear_kernel<kBN, kAct, kLong>, (int)smem, seen);
  if (e != cudaSuccess) return e;
  const uint64_t tiles = (uint64_t)((p.n + kBN - 1) / kBN) * ((p.m + kBM - 1) / kBM);
  if (tiles > 0x7fffffffull) return cudaErrorInvalidValue;
  const uint32_t grid = p.splits > 1 ? (uint32_t)tiles * p.splits
                                     : (uint32_t)std::min<uint64_t>(tiles, (uint64_t)num_sms);
  linear_kernel<kBN, kAct, kLong><<<grid, kThreads, smem, stream>>>(mx, mw, mr, mo, p);
  return cudaGetLastError();
}

template <int kAct, bool kLong>
cudaError_t launch_wide(const LinearFusedProblem &p, int num_sms, cudaStream_t stream) {
  // Tile width: waves of tiles over the SMs times a tile's cost, and what its first stages and last
  // epilogue add, in microseconds measured at k = 1024 (k = 384 orders the widths alike).  At
  // k = 1024 widths 64 / 128 / 256 take 33 / 29 / 39 us for 33500 x 100, 115 / 71 / 75 us for
  // 33500 x 640, 178 / 107 / 96 us for 33500 x 1024, 21 / 16 / 28 us for 2048 x 1024 and
  // 13 / 15 / 27 us for 777 x 128.
  if (p.splits > 1) return launch_tiles<64, kAct, kLong>(p, num_sms, stream);
  const uint64_t mt = (p.m + kBM - 1) / kBM;
  auto cost = [&](uint64_t bn, uint64_t wave, uint64_t once) {
    return (mt * ((p.n + bn - 1) / bn) + num_sms - 1) / num_sms * wave + once;
  };
  const uint64_t c64 = cost(64, 6, 0), c128 = cost(128, 7, 2), c256 = cost(256, 12, 7);
  if (c256 < c128 && c256 < c64) return launch_tiles<256, kAct, kLong>(p, num_sms, stream);
  if (c128 < c64) return launch_tiles<128, kAct, kLong>(p, num_sms, stream);
  return launch_tiles<64, kAct, kLong>(p, num_sms, stream);
}

// A few rows stream w once; past these sizes the conversions and sums of every row cost more than
// a tile's.  By columns against tiles: 10 / 14 us for 8 x 1024 x 1024, 14 / 18 us for
// 4 x 1024 x 4096, 18 / 22 us for 2 x 4096 x 4096, but 22 / 18 us for 8 x 1024 x 4096, 27 / 22 us
// for 4 x 4096 x 4096 and 22 / 20 us for 2 x 16384 x 1024.
bool by_columns(const LinearFusedProblem &p) {
  return p.m == 1 || (p.m == 2 && p.n <= 8192) ||
         (p.m <= 8 && p.k <= 4096 && (uint64_t)p.m * p.n * p.k <= 1 << 24);
}

template <int kAct>
cudaError_t launch_act(LinearFusedProblem p, int num_sms, cudaStream_t stream) {
  if (by_columns(p)) return launch_gemv<kAct>(p, stream);
  const uint32_t vo = p.out_dtype == TX_BF16 ? 8 : 4, vr = p.residual_dtype == TX_BF16 ? 8 : 4;
  p.out_vec = (uintptr_t)p.out % 16 == 0 && p.ldo % vo == 0;
  p.res_vec = p.residual && (uintptr_t)p.residual % 16 == 0 && p.ldr % vr == 0;
  p.bias_vec = (uintptr_t)p.bias % 16 == 0;
  p.epilogue = !p.out_vec ? kDirect
               : p.residual && p.res_vec && p.residual_dtype == p.out_dtype ? kStagedRes : kStaged;
  return p.k > kPart * kBK ? launch_wide<kAct, true>(p, num_sms, stream)
                           : launch_wide<kAct, false>(p, num_sms, stream);
}

}  // namespace lfused

// k is cut where the 64-column tiles would leave half the SMs without one: as many parts as SMs for
// each tile, of 256 columns at least.  16 x 1024 x 4096 29 -> 18 us, 773 x 117 x 3754 33 -> 22 us,
// 16 x 1024 x 1024 14.3 us either way.
uint32_t linear_fused_splits(const LinearFusedProblem &p, int num_sms, uint32_t *tiles) {
  using namespace lfused;
  const uint64_t t = (uint64_t)((p.m + kBM - 1) / kBM) * ((p.n + 63) / 64);
  *tiles = 0;
  if (by_columns(p) || p.k <= kPart * kBK || 2 * t > (uint64_t)num_sms) return 1;
  *tiles = (uint32_t)t;
  return std::min<uint32_t>((uint32_t)(num_sms / t), (p.k + kBK - 1) / kBK / 4);
}

cudaError_t launch_linear_fused(const LinearFusedProblem &p, int num_sms, cudaStream_t stream) {
  switch (p.act) {
    case TX_ACT_RELU:
      return lfused::launch_act<TX_ACT_RELU>(p, num_sms, stream);
    case TX_ACT_GELU:
      return p.out_dtype == TX_F32 ? lfused::launch_act<lfused::kGeluF32>(p, num_sms, stream)
                                   : lfused::launch_act<TX_ACT_GELU>(p, num_sms, stream);
    case TX_ACT_GELU_TANH:
      return lfused::launch_act<TX_ACT_GELU_TANH>(p, num_sms, stream);
    case TX_ACT_SILU:
      return lfused::launch_act<TX_ACT_SILU>(p, num_sms, stream);
    default:
      return lfused::launch_act<TX_ACT_NONE>(p, num_sms, stream);
  }
}

}  // namespace tx
