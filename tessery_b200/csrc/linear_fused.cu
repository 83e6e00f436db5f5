// Linear layer with bias, activation and residual in its epilogue (tx_linear_fused):
//   out = act(x w^T + bias) + residual,  x [m, k] and w [n, k] bf16, fp32 sums,
// any m, n and k, rows of x and w on 16-byte boundaries.
//
// linear_kernel: 128 x BN tiles on tcgen05 (kind::f16), K through a ring of 64-column stages
// filled by TMA (128-byte swizzle; rows past m or n and columns past k arrive as zeros), two
// accumulators in tensor memory so that four epilogue warps finish one tile while the next is
// multiplied; persistent, one CTA per SM.
// gemv_kernel: a few rows (m <= 8) only stream w once: a warp per output column, w straight from
// global memory into registers, the sums over lanes by shuffles.
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
constexpr int kThreads = 192;  // warp 0 TMA, warp 1 MMA, warps 2-5 epilogue
constexpr int kMaxStages = 8;
constexpr long long kDrainCycles = 2000000000ll;

template <int kBN>
struct Cfg {
  static constexpr uint32_t kABytes = kBM * 128, kBBytes = kBN * 128;
  static constexpr uint32_t kStageBytes = kABytes + kBBytes;
  static constexpr int kFit = (int)((232448 - 1024) / kStageBytes);
  static constexpr int kStages = kFit < kMaxStages ? kFit : kMaxStages;
  static constexpr uint32_t kOffMisc = kStages * kStageBytes;
  static constexpr uint32_t kSmemBytes = kOffMisc + 256;
  static constexpr uint32_t kTmemCols = 2 * kBN;
  static constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) |
                                     ((uint32_t)(kBN >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
};
enum : uint32_t { kBarFull = 0, kBarEmpty = kMaxStages, kBarAcc = 2 * kMaxStages,
                  kBarFree = kBarAcc + 2, kBarDrain = kBarFree + 2, kNumBars = kBarDrain + 1 };
enum : uint32_t { kOffTmem = 8 * kNumBars, kOffAbort = kOffTmem + 4 };
enum : int { kSiteEmpty = 1, kSiteFull = 2, kSiteAcc = 3, kSiteFree = 4 };

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

__device__ __forceinline__ float activate(float y, int act) {
  switch (act) {
    case TX_ACT_RELU:
      return y < 0.f ? 0.f : y;
    case TX_ACT_GELU:
      return 0.5f * y * (1.f + erff(y * 0.70710678118654752f));
    case TX_ACT_GELU_TANH:  // (1 + tanh u) / 2 = 1 / (1 + e^(-2u))
      return __fdividef(y, 1.f + __expf(-1.5957691216057308f * (y + 0.044715f * y * y * y)));
    case TX_ACT_SILU:
      return __fdividef(y, 1.f + __expf(-y));
    default:
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

template <int kBN>
__global__ void __launch_bounds__(kThreads, 1)
    linear_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                  const __grid_constant__ LinearFusedProblem p) {
  using C = Cfg<kBN>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_addr(smem), bars = sbase + C::kOffMisc;
  auto bar = [&](uint32_t i) { return bars + 8u * i; };
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + C::kOffMisc + kOffAbort);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t nt = (p.n + kBN - 1) / kBN, mt = (p.m + kBM - 1) / kBM, tiles = nt * mt;
  const uint32_t nk = (p.k + kBK - 1) / kBK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(bar(kBarFull + s), 1);
      mbar_init(bar(kBarEmpty + s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar(kBarAcc + b), 1);
      mbar_init(bar(kBarFree + b), 128);
    }
    mbar_init(bar(kBarDrain), 1);
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
      for (uint32_t tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
        const int m0 = (int)(tile / nt * kBM), n0 = (int)(tile % nt * kBN);
        for (uint32_t kb = 0; kb < nk; ++kb) {
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
      uint32_t step = 0, done = 0;
      bool ok = true;
      for (uint32_t tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, ++done) {
        const uint32_t b = done & 1, acc = tmem + b * kBN;
        if (done >= 2 && !(ok = wait_bar(bar(kBarFree + b), ((done >> 1) - 1) & 1, abort_flag,
                                         p.status, kSiteFree, p.wait_cycles)))
          break;
        tc_fence_after();
        for (uint32_t kb = 0; kb < nk; ++kb, ++step) {
          const uint32_t s = step % C::kStages;
          if (!(ok = wait_bar(bar(kBarFull + s), (step / C::kStages) & 1, abort_flag, p.status,
                              kSiteFull, p.wait_cycles)))
            break;
          tc_fence_after();
          const uint32_t st = sbase + s * C::kStageBytes;
          const uint64_t ad = sw128_desc(st, 16, 1024), bd = sw128_desc(st + C::kABytes, 16, 1024);
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma(acc, ad + ks * 2, bd + ks * 2, C::kIdesc, kb > 0 || ks > 0);
          umma_commit(bar(kBarEmpty + s));
        }
        if (ok) umma_commit(bar(kBarAcc + b));
      }
      umma_commit(bar(kBarDrain));
      drain_bar(bar(kBarDrain), 0);
    }
    __syncwarp();
  } else {
    const uint32_t quarter = (uint32_t)warp & 3, r = quarter * 32 + lane;
    const bool out16 = p.out_vec, res16 = p.res_vec;
    uint32_t done = 0;
    for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++done) {
      const uint32_t b = done & 1, m = tile / nt * kBM + r, n0 = tile % nt * kBN;
      if (!__all_sync(0xffffffffu, wait_bar(bar(kBarAcc + b), (done >> 1) & 1, abort_flag,
                                            p.status, kSiteAcc, p.wait_cycles)))
        break;
      tc_fence_after();
      const uint32_t t0 = tmem + b * kBN + ((quarter * 32u) << 16);
#pragma unroll 1
      for (uint32_t c = 0; c < kBN; c += 32) {
        if (n0 + c >= p.n) break;
        uint32_t a[32];
        tmem_ld32(t0 + c, a);
        tmem_ld_wait();
        const uint32_t n = n0 + c;
        const bool whole = n + 32 <= p.n;
        if (m < p.m) {
          float v[32];
#pragma unroll
          for (int t = 0; t < 32; ++t) v[t] = __uint_as_float(a[t]);
          if (p.bias) {
#pragma unroll
            for (int t = 0; t < 32; ++t)
              if (whole || n + t < p.n) v[t] += __ldg(p.bias + n + t);
          }
          if (p.act) {
#pragma unroll
            for (int t = 0; t < 32; ++t) v[t] = activate(v[t], p.act);
          }
          if (p.residual) {
            const size_t at = (size_t)m * p.ldr + n;
            if (whole && res16 && p.residual_dtype == 0) {
#pragma unroll
              for (int t = 0; t < 8; ++t) {
                const float4 q = reinterpret_cast<const float4 *>(
                    static_cast<const float *>(p.residual) + at)[t];
                v[4 * t] += q.x; v[4 * t + 1] += q.y; v[4 * t + 2] += q.z; v[4 * t + 3] += q.w;
              }
            } else if (whole && res16) {
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
                if (whole || n + t < p.n) v[t] += residual_at(p, at + t);
            }
          }
          const size_t at = (size_t)m * p.ldo + n;
          if (whole && out16 && p.out_dtype == 0) {
#pragma unroll
            for (int t = 0; t < 8; ++t)
              reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at)[t] =
                  make_float4(v[4 * t], v[4 * t + 1], v[4 * t + 2], v[4 * t + 3]);
          } else if (whole && out16) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
              reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out) + at)[t] = make_uint4(
                  pack_bf16x2(v[8 * t], v[8 * t + 1]), pack_bf16x2(v[8 * t + 2], v[8 * t + 3]),
                  pack_bf16x2(v[8 * t + 4], v[8 * t + 5]), pack_bf16x2(v[8 * t + 6], v[8 * t + 7]));
          } else {
#pragma unroll
            for (int t = 0; t < 32; ++t)
              if (whole || n + t < p.n) store_at(p, at + t, v[t]);
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      mbar_arrive(bar(kBarFree + b));
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
// One warp per output column; lane l takes columns 8l .. 8l+7 of every 256 of K.
constexpr int kGemvWarps = 4;

template <int kM>
__global__ void __launch_bounds__(32 * kGemvWarps) gemv_kernel(const __grid_constant__ LinearFusedProblem p) {
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t n = blockIdx.x * kGemvWarps + (threadIdx.x >> 5);
  if (n >= p.n) return;
  const uint16_t *x = static_cast<const uint16_t *>(p.x);
  const uint16_t *w = static_cast<const uint16_t *>(p.w) + (size_t)n * p.ldw;
  float sum[kM];
#pragma unroll
  for (int i = 0; i < kM; ++i) sum[i] = 0.f;
#pragma unroll 4
  for (uint32_t c = lane * 8; c < p.k; c += 256) {
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
#pragma unroll
  for (int i = 0; i < kM; ++i) sum[i] = warp_sum(sum[i]);
  // Lane i finishes row i.
  float y = 0.f;
#pragma unroll
  for (int i = 0; i < kM; ++i)
    if (lane == (uint32_t)i) y = sum[i];
  if (lane < p.m) {
    if (p.bias) y += p.bias[n];
    y = activate(y, p.act);
    if (p.residual) y += residual_at(p, (size_t)lane * p.ldr + n);
    store_at(p, (size_t)lane * p.ldo + n, y);
  }
}

template <int kM>
cudaError_t launch_gemv(const LinearFusedProblem &p, cudaStream_t stream) {
  gemv_kernel<kM><<<(p.n + kGemvWarps - 1) / kGemvWarps, 32 * kGemvWarps, 0, stream>>>(p);
  return cudaGetLastError();
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
bool make_map(CUtensorMap *map, const void *base, uint32_t rows, uint32_t cols, uint64_t ld,
              uint32_t box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {cols, rows};
  cuuint64_t strides[1] = {ld * 2};
  cuuint32_t box[2] = {kBK, box_rows};
  cuuint32_t elem[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(base), dims, strides, box,
            elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int kBN>
cudaError_t launch_tiles(const LinearFusedProblem &p, int num_sms, cudaStream_t stream) {
  constexpr uint32_t smem = Cfg<kBN>::kSmemBytes;
  CUtensorMap mx, mw;
  if (!make_map(&mx, p.x, p.m, p.k, p.ldx, kBM) || !make_map(&mw, p.w, p.n, p.k, p.ldw, kBN))
    return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(linear_kernel<kBN>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const uint64_t tiles = (uint64_t)((p.n + kBN - 1) / kBN) * ((p.m + kBM - 1) / kBM);
  if (tiles > 0x7fffffffull) return cudaErrorInvalidValue;
  linear_kernel<kBN><<<(uint32_t)std::min<uint64_t>(tiles, (uint64_t)num_sms), kThreads, smem,
                       stream>>>(mx, mw, p);
  return cudaGetLastError();
}

}  // namespace lfused

cudaError_t launch_linear_fused(LinearFusedProblem p, int num_sms, cudaStream_t stream) {
  if (p.m <= 1) return lfused::launch_gemv<1>(p, stream);
  if (p.m <= 2) return lfused::launch_gemv<2>(p, stream);
  if (p.m <= 4) return lfused::launch_gemv<4>(p, stream);
  if (p.m <= 8) return lfused::launch_gemv<8>(p, stream);
  const uint32_t vo = p.out_dtype == TX_BF16 ? 8 : 4, vr = p.residual_dtype == TX_BF16 ? 8 : 4;
  p.out_vec = (uintptr_t)p.out % 16 == 0 && p.ldo % vo == 0;
  p.res_vec = p.residual && (uintptr_t)p.residual % 16 == 0 && p.ldr % vr == 0;
  // The widest tile that still gives every SM one (a wide tile reads x fewer times).
  const uint64_t mt = (p.m + lfused::kBM - 1) / lfused::kBM;
  if (mt * ((p.n + 255) / 256) >= (uint64_t)num_sms) return lfused::launch_tiles<256>(p, num_sms, stream);
  if (mt * ((p.n + 127) / 128) >= (uint64_t)num_sms) return lfused::launch_tiles<128>(p, num_sms, stream);
  return lfused::launch_tiles<64>(p, num_sms, stream);
}

}  // namespace tx
