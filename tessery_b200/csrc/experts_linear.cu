// The experts' products over rows that lie by expert (tx_experts_linear):
//   out[r] = act(x[row(r)] w_e^T + b_e)   or, gated,   act(x g_e^T + bg_e) * (x u_e^T + bu_e),
// e the expert whose range offsets[e] .. offsets[e + 1] - 1 holds r, row(r) = order[r] / top_k or r.
//
// 128 x BN tiles on tcgen05 as in linear_fused.cu: one tile is up to 128 rows of one expert, and with the
// ranges known on the device alone each CTA counts the tiles of every expert first.  The rows of x come by
// TMA gathers of four rows, as many as the tile has, so nothing is sorted into memory first; a gated tile
// holds BN / 2 gate columns and the same up columns side by side in tensor memory.
#include <cuda.h>

#include <algorithm>

#include "../../include/tessattn.h"
#include "common.cuh"
#include "kernels.h"
#include "linear_parts.cuh"
#include "tcgen05.cuh"

namespace tx {
namespace experts {

using namespace ptx;
using namespace lfused;

constexpr int kBM = 128;
constexpr uint32_t kBK = 64;
constexpr int kThreads = 320;  // warp 0 TMA, warp 1 MMA, warps 2-9 epilogue
constexpr int kMaxStages = 8;
constexpr uint32_t kPart = 8;  // K stages (512 columns) of one partial sum
constexpr uint32_t kMaxExperts = 1024;
constexpr uint32_t kFull = 0xffffffffu;

template <int kBN>
struct Cfg {
  static constexpr uint32_t kABytes = kBM * 128, kBBytes = kBN * 128;
  static constexpr uint32_t kStageBytes = kABytes + kBBytes;
  static constexpr uint32_t kTables = 2 * (kMaxExperts + 1) * 4;
  static constexpr int kFit = (int)((232448 - 1024 - 512 - kTables) / kStageBytes);
  static constexpr int kStages = kFit < kMaxStages ? kFit : kMaxStages;
  static constexpr uint32_t kOffMisc = kStages * kStageBytes;
  static constexpr uint32_t kOffTables = kOffMisc + 512;
  static constexpr uint32_t kSmemBytes = kOffTables + kTables;
  static constexpr uint32_t kTmemCols = 2 * kBN;
  static constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) |
                                     ((uint32_t)(kBN >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
};
enum : uint32_t { kBarFull = 0, kBarEmpty = kMaxStages, kBarAcc = 2 * kMaxStages,
                  kBarFree = kBarAcc + 2, kBarDrain = kBarFree + 2, kNumBars = kBarDrain + 1 };
enum : uint32_t { kOffTmem = 8 * kNumBars, kOffAbort = kOffTmem + 4 };
static_assert(kOffAbort + 4 <= 512, "misc area");
enum : int { kSiteEmpty = 1, kSiteFull = 2, kSiteAcc = 3, kSiteFree = 4 };

// Columns x .. x + 63 of four rows, 512 bytes in the 128-byte swizzle.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x,
                                            const int (&r)[4]) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(r[0]), "r"(r[1]), "r"(r[2]),
      "r"(r[3])
      : "memory");
}

// The tables of a launch: start[e] is offsets[e] cut to 0 .. rows and never falling, tiles[e] the row
// tiles of the experts before e.  One warp fills them.
__device__ __forceinline__ void fill_tables(const ExpertsProblem &p, uint32_t *start, uint32_t *tiles) {
  const uint32_t lane = threadIdx.x & 31;
  uint32_t edge = 0, count = 0;
  for (uint32_t e0 = 0; e0 <= p.experts; e0 += 32) {
    const uint32_t e = e0 + lane;
    int32_t raw = e <= p.experts ? __ldg(p.offsets + e) : 0;
    uint32_t v = min((uint32_t)max(raw, 0), p.rows);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {  // the largest so far
      const uint32_t u = __shfl_up_sync(kFull, v, o);
      if ((int)lane >= o) v = max(v, u);
    }
    v = max(v, edge);
    if (e <= p.experts && v != (uint32_t)raw) report_status(p.status, kStatusBadArg);
    uint32_t before = __shfl_up_sync(kFull, v, 1);
    if (lane == 0) before = e0 ? edge : v;
    uint32_t n = e <= p.experts ? (v - before + kBM - 1) / kBM : 0;  // tiles of expert e - 1
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(kFull, n, o);
      if ((int)lane >= o) n += u;
    }
    if (e <= p.experts) {
      start[e] = v;
      tiles[e] = count + n;
    }
    edge = __shfl_sync(kFull, v, 31);
    count += __shfl_sync(kFull, n, 31);
  }
}
// The expert of row tile `mt`, searched by a warp from e on (tiles only grow).
__device__ __forceinline__ uint32_t expert_of(const uint32_t *tiles, uint32_t experts, uint32_t mt,
                                              uint32_t e) {
  const uint32_t lane = threadIdx.x & 31;
  while (true) {
    const uint32_t next = e + 1 + lane;
    const uint32_t hits = __popc(__ballot_sync(kFull, next < experts && tiles[next] <= mt));
    e += hits;
    if (hits < 32) return e;
  }
}

template <int kN>
__device__ __forceinline__ void activate_all(float (&v)[kN], int act) {
  switch (act) {
#define TX_ACT(name)                                      \
  case name:                                              \
    _Pragma("unroll") for (int t = 0; t < kN; ++t) v[t] = activate<name>(v[t]); \
    break;
    TX_ACT(TX_ACT_RELU)
    TX_ACT(TX_ACT_GELU)
    TX_ACT(TX_ACT_GELU_TANH)
    TX_ACT(TX_ACT_SILU)
    TX_ACT(kGeluF32)
#undef TX_ACT
    default:
      break;
  }
}

// kLong: the sum is taken in parts of 512 K that are added in fp32 registers.
template <int kBN, bool kGated, bool kLong>
__global__ void __launch_bounds__(kThreads, 1)
    experts_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                   const __grid_constant__ ExpertsProblem p) {
  using C = Cfg<kBN>;
  constexpr uint32_t kOut = kGated ? kBN / 2 : kBN;  // output columns of a tile
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_addr(smem), bars = sbase + C::kOffMisc;
  auto bar = [&](uint32_t i) { return bars + 8u * i; };
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + C::kOffMisc + kOffAbort);
  uint32_t *start = reinterpret_cast<uint32_t *>(smem + C::kOffTables);
  uint32_t *tiles = start + kMaxExperts + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

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
  if (warp == 2) fill_tables(p, start, tiles);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<uint32_t *>(smem + C::kOffMisc + kOffTmem);
  const uint32_t nt = (p.n + kOut - 1) / kOut, total = tiles[p.experts] * nt;
  const uint32_t nk = (p.k + kBK - 1) / kBK;

  if (warp == 0) {
    uint32_t fills = 0, e = 0;
    bool ok = true;
    for (uint32_t tile = blockIdx.x; ok && tile < total; tile += gridDim.x) {
      const uint32_t mt = tile / nt;
      e = expert_of(tiles, p.experts, mt, e);
      const uint32_t r0 = start[e] + (mt - tiles[e]) * kBM, rows = min(start[e + 1] - r0, (uint32_t)kBM);
      const int n0 = (int)(tile % nt * kOut);
      const uint32_t gathers = (rows + 3) / 4;
      int row[4];  // the rows that this lane gathers; past the tile's last its last again
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t r = r0 + min((uint32_t)lane * 4 + i, rows - 1);
        row[i] = (int)r;
        if (p.order) {
          const uint32_t at = (uint32_t)__ldg(p.order + r) / p.top_k;
          if (at >= p.x_rows) report_status(p.status, kStatusBadArg);
          row[i] = (int)min(at, p.x_rows - 1);
        }
      }
      for (uint32_t kb = 0; kb < nk; ++kb) {
        const uint32_t s = fills % C::kStages, round = fills / C::kStages;
        if (round && !(ok = wait_bar(bar(kBarEmpty + s), (round - 1) & 1, abort_flag, p.status,
                                     kSiteEmpty, p.wait_cycles)))
          break;
        const uint32_t dst = sbase + s * C::kStageBytes;
        if (lane == 0) {
          mbar_expect_tx(bar(kBarFull + s), gathers * 512 + C::kBBytes);
          if constexpr (kGated) {
            tma_load_3d(dst + C::kABytes, &tm_w, bar(kBarFull + s), (int)(kb * kBK), n0, (int)e);
            tma_load_3d(dst + C::kABytes + C::kBBytes / 2, &tm_w, bar(kBarFull + s), (int)(kb * kBK),
                        (int)p.n + n0, (int)e);
          } else {
            tma_load_3d(dst + C::kABytes, &tm_w, bar(kBarFull + s), (int)(kb * kBK), n0, (int)e);
          }
        }
        __syncwarp();
        if ((uint32_t)lane < gathers)
          tma_gather4(dst + (uint32_t)lane * 512, &tm_x, bar(kBarFull + s), (int)(kb * kBK), row);
        ++fills;
      }
      ok = __all_sync(kFull, ok);
    }
    // No copy may land after the CTA has gone.
    if (lane == 0)
      for (uint32_t s = 0; s < (uint32_t)C::kStages && s < fills; ++s)
        drain_bar(bar(kBarFull + s), ((fills - 1 - s) / C::kStages) & 1);
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t step = 0, done = 0;  // K stages, partial sums
      bool ok = true;
      for (uint32_t tile = blockIdx.x; ok && tile < total; tile += gridDim.x) {
        for (uint32_t kb = 0; ok && kb < nk; ++done) {
          const uint32_t b = done & 1, acc = tmem + b * kBN;
          if (done >= 2 && !(ok = wait_bar(bar(kBarFree + b), ((done >> 1) - 1) & 1, abort_flag,
                                           p.status, kSiteFree, p.wait_cycles)))
            break;
          tc_fence_after();
          const uint32_t end = kLong ? min(kb + kPart, nk) : nk;
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
    // Warp w finishes output columns [half * kCols, +kCols) of the 32 rows of its tensor-memory quarter.
    constexpr uint32_t kCols = kOut / 2, kStep = kCols < 32 ? kCols : 32;
    const uint32_t quarter = (uint32_t)warp & 3, half = (uint32_t)(warp - 2) >> 2;
    const uint32_t lanes = (quarter * 32u) << 16;
    const bool f32_out = p.out_dtype == TX_F32;
    uint32_t done = 0, e = 0;
    bool ok = true;
    for (uint32_t tile = blockIdx.x; ok && tile < total; tile += gridDim.x) {
      const uint32_t mt = tile / nt;
      e = expert_of(tiles, p.experts, mt, e);
      const uint32_t r0 = start[e] + (mt - tiles[e]) * kBM, rows = min(start[e + 1] - r0, (uint32_t)kBM);
      const uint32_t n0 = tile % nt * kOut + half * kCols, mine = quarter * 32 + lane;
      const float *bias = p.bias ? p.bias + (size_t)e * (kGated ? 2 : 1) * p.n : nullptr;
      // Bias, activation, gate and store of columns [c, c + kStep); u is the up half.
      auto finish = [&](uint32_t c, float (&v)[kStep], float (&u)[kGated ? kStep : 1]) {
        const uint32_t n = n0 + c;
        if (mine >= rows || n >= p.n) return;
        const bool whole = n + kStep <= p.n;
        if (bias) {
#pragma unroll
          for (uint32_t t = 0; t < kStep; ++t)
            if (whole || n + t < p.n) {
              v[t] += __ldg(bias + n + t);
              if constexpr (kGated) u[t] += __ldg(bias + p.n + n + t);
            }
        }
        activate_all(v, p.act);
        if constexpr (kGated) {
#pragma unroll
          for (uint32_t t = 0; t < kStep; ++t) v[t] *= u[t];
        }
        const size_t at = (size_t)(r0 + mine) * p.ldo + n;
        if (whole && p.out_vec && f32_out) {
#pragma unroll
          for (uint32_t t = 0; t < kStep / 4; ++t)
            reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at)[t] =
                make_float4(v[4 * t], v[4 * t + 1], v[4 * t + 2], v[4 * t + 3]);
        } else if (whole && p.out_vec) {
#pragma unroll
          for (uint32_t t = 0; t < kStep / 8; ++t)
            reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out) + at)[t] =
                make_uint4(pack_bf16x2(v[8 * t], v[8 * t + 1]), pack_bf16x2(v[8 * t + 2], v[8 * t + 3]),
                           pack_bf16x2(v[8 * t + 4], v[8 * t + 5]),
                           pack_bf16x2(v[8 * t + 6], v[8 * t + 7]));
        } else {
#pragma unroll
          for (uint32_t t = 0; t < kStep; ++t)
            if (n + t < p.n) {
              if (f32_out)
                static_cast<float *>(p.out)[at + t] = v[t];
              else
                static_cast<uint16_t *>(p.out)[at + t] = f32_to_bf16_bits(v[t]);
            }
        }
      };
      auto load = [&](uint32_t at, float (&v)[kStep]) {
#pragma unroll
        for (uint32_t c = 0; c < kStep; c += 16) {
          uint32_t a[16];
          tmem_load(at + c, a);
#pragma unroll
          for (int t = 0; t < 16; ++t) v[c + t] = __uint_as_float(a[t]);
        }
      };
      if constexpr (kLong) {
        constexpr uint32_t kHeld = kCols / kStep;
        float v[kHeld][kStep], u[kGated ? kHeld : 1][kGated ? kStep : 1];
        const uint32_t parts = (nk + kPart - 1) / kPart;
        for (uint32_t part = 0; part < parts; ++part, ++done) {
          const uint32_t b = done & 1, t0 = tmem + b * kBN + half * kCols + lanes;
          if (!(ok = __all_sync(kFull, wait_bar(bar(kBarAcc + b), (done >> 1) & 1, abort_flag, p.status,
                                                kSiteAcc, p.wait_cycles))))
            break;
          tc_fence_after();
#pragma unroll
          for (uint32_t c = 0; c < kHeld; ++c) {
            float a[kStep];
            load(t0 + c * kStep, a);
#pragma unroll
            for (uint32_t t = 0; t < kStep; ++t) v[c][t] = part ? v[c][t] + a[t] : a[t];
            if constexpr (kGated) {
              load(t0 + kOut + c * kStep, a);
#pragma unroll
              for (uint32_t t = 0; t < kStep; ++t) u[c][t] = part ? u[c][t] + a[t] : a[t];
            }
          }
          tc_fence_before();
          mbar_arrive(bar(kBarFree + b));
        }
        if (!ok) break;
#pragma unroll
        for (uint32_t c = 0; c < kHeld; ++c) finish(c * kStep, v[c], u[kGated ? c : 0]);
      } else {
        const uint32_t b = done & 1, t0 = tmem + b * kBN + half * kCols + lanes;
        ok = __all_sync(kFull, wait_bar(bar(kBarAcc + b), (done >> 1) & 1, abort_flag, p.status,
                                        kSiteAcc, p.wait_cycles));
        if (!ok) break;
        tc_fence_after();
        ++done;
#pragma unroll 1
        for (uint32_t c = 0; c < kCols; c += kStep) {
          float v[kStep], u[kGated ? kStep : 1];
          load(t0 + c, v);
          if constexpr (kGated) load(t0 + kOut + c, u);
          finish(c, v, u);
          __syncwarp();
        }
        tc_fence_before();
        mbar_arrive(bar(kBarFree + b));
      }
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

// x [rows, k] read one row a box, and w [experts, wide, k] in boxes of box_rows rows; 64 columns of bf16
// in the 128-byte swizzle.
bool make_maps(CUtensorMap *mx, CUtensorMap *mw, const ExpertsProblem &p, uint32_t box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  const uint32_t wide = p.n * (p.gated ? 2 : 1);
  cuuint64_t xd[2] = {p.k, p.x_rows}, xs[1] = {p.ldx * 2};
  cuuint32_t xb[2] = {64, 1}, one[3] = {1, 1, 1};
  cuuint64_t wd[3] = {p.k, wide, p.experts}, ws[2] = {p.ldw * 2, p.expert_stride * 2};
  cuuint32_t wb[3] = {64, box_rows, 1};
  return fn(mx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(p.x), xd, xs, xb, one,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS &&
         fn(mw, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(p.w), wd, ws, wb, one,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int kBN, bool kGated, bool kLong>
cudaError_t launch_tiles(const ExpertsProblem &p, int num_sms, cudaStream_t stream) {
  constexpr uint32_t smem = Cfg<kBN>::kSmemBytes;
  CUtensorMap mx, mw;
  if (!make_maps(&mx, &mw, p, kGated ? kBN / 2 : kBN)) return cudaErrorInvalidValue;
  static std::atomic<uint64_t> seen{0};
  cudaError_t e = allow_smem((const void *)experts_kernel<kBN, kGated, kLong>, (int)smem, seen);
  if (e != cudaSuccess) return e;
  experts_kernel<kBN, kGated, kLong><<<num_sms, kThreads, smem, stream>>>(mx, mw, p);
  return cudaGetLastError();
}

template <bool kGated, bool kLong>
cudaError_t launch_wide(const ExpertsProblem &p, int num_sms, cudaStream_t stream) {
  const uint32_t wide = p.n * (kGated ? 2 : 1);
  if (wide <= 64) return launch_tiles<64, kGated, kLong>(p, num_sms, stream);
  if constexpr (!kLong)
    if (wide > 128 && p.rows > 128 * 64) return launch_tiles<256, kGated, kLong>(p, num_sms, stream);
  return launch_tiles<128, kGated, kLong>(p, num_sms, stream);
}

}  // namespace experts

cudaError_t launch_experts_linear(ExpertsProblem p, int num_sms, cudaStream_t stream) {
  using namespace experts;
  p.out_vec = (uintptr_t)p.out % 16 == 0 && p.ldo % (p.out_dtype == TX_BF16 ? 8 : 4) == 0;
  if (p.act == TX_ACT_GELU && p.out_dtype == TX_F32) p.act = kGeluF32;
  // The accumulator cuts bits off at each of its additions: over 512 K that is far below bf16's rounding,
  // for an fp32 result it is not.
  const bool parts = p.out_dtype == TX_F32 && p.k > kPart * kBK;
  if (p.gated)
    return parts ? launch_wide<true, true>(p, num_sms, stream)
                 : launch_wide<true, false>(p, num_sms, stream);
  return parts ? launch_wide<false, true>(p, num_sms, stream)
               : launch_wide<false, false>(p, num_sms, stream);
}

}  // namespace tx
