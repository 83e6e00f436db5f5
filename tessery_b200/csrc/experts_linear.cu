// The experts' products over rows that lie by expert (tx_experts_linear):
//   out[r] = act(x[row(r)] w_e^T + b_e)   or, gated,   act(x g_e^T + bg_e) * (x u_e^T + bu_e),
// e the expert whose range offsets[e] .. offsets[e + 1] - 1 holds r, row(r) = order[r] / top_k or r.
//
// 128 x BN tiles on tcgen05 as in linear_fused.cu: one tile is up to 128 rows of one expert, and with the
// ranges known on the device alone each CTA counts the tiles of every expert first.  Rows of x that do not
// lie by expert are gathered by two or four warps with 16-byte asynchronous copies into the layout that TMA
// writes, so nothing is sorted into memory first.  (TMA gathers of four rows took 80 cycles each, 2600 a
// stage where the products take 512: 336 against 138 us for the largest case.)  A gated tile holds BN / 2
// gate columns and the same up columns side by side in tensor memory.
// pair_kernel: 256 x 256 tiles by two CTAs, for calls of many rows that lie by expert.  Gathered rows would
// have to be handed from one CTA's threads to the other's products, with an arrival that waits for all copies
// in flight: 244 us where 128 x 256 tiles by one CTA take 117.
//
// Measured: 65536 rows over 64 experts, gated, n 512, k 1024, gathered: 115 us from rest, 1195 TFLOP/s, and
// 139 to 146 us in a loop under the power limit; n 1024, k 512, rows by expert: 61 us, 1120 TFLOP/s, and 83 to
// 85 us in a loop.  Bound: the tensor pipe, 60 % of whose cycles are used, beside L2's way in (12.5 TB/s), and for
// the latter the writes of out; 5.9 and 12.9 % of the rows multiplied, in experts' last tiles, are not there.
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
// warp 0 TMA, warp 1 MMA, warps 2-9 epilogue, and to gather rows those from warp 10 on
constexpr int kThreads = 320;
constexpr int kMaxStages = 8;
constexpr uint32_t kPart = 8;  // K stages (512 columns) of one partial sum
constexpr uint32_t kBufBytes = 32 * 64;  // staging of an epilogue warp: 32 rows of 64 bytes
constexpr uint32_t kBiasBytes = 512;     // of an epilogue warp: its columns' bias
constexpr uint32_t kFull = 0xffffffffu;

template <int kBN>
struct Cfg {
  static constexpr uint32_t kABytes = kBM * 128, kBBytes = kBN * 128;
  static constexpr uint32_t kStageBytes = kABytes + kBBytes;
  static constexpr uint32_t kMaxExperts = 1024;
  static constexpr uint32_t kTables = 2 * (kMaxExperts + 1) * 4;
  static constexpr int kFit =
      (int)((232448 - 512 - kTables - 8 * (kBufBytes + kBiasBytes)) / kStageBytes);
  static constexpr int kStages = kFit < kMaxStages ? kFit : kMaxStages;
  static constexpr uint32_t kOffStaging = kStages * kStageBytes;
  static constexpr uint32_t kOffMisc = kOffStaging + 8 * (kBufBytes + kBiasBytes);
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

__device__ __forceinline__ void pause_cycles(long long n) {
  const long long t0 = clock64();
  while (clock64() - t0 < n) {
  }
}
// wait_bar by a whole warp, with one answer.
template <bool kCluster = false>
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag,
                                          const ExpertsProblem &p, int site) {
  return __all_sync(kFull, wait_bar<kCluster>(bar, parity, abort_flag, p.status, site, p.wait_cycles));
}
// 16 bytes from global to shared memory, of which the first `bytes` are read and the others zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
// Arrives at `bar` when this thread's copies so far have landed.  (The barrier counts every such arrival;
// who waits for it makes the copies visible to the tensor core with fence_proxy_async.)
__device__ __forceinline__ void copies_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// The rows that kWarps warps gather for a tile.  Eight lanes copy a row's 128 bytes of a stage, four warps 32
// rows each in eight steps, into the 128-byte swizzle.  A tile's entries of `order` are fetched while the tile before
// it is copied: waiting for them at its start took 3400 cycles, more than the stages ahead last.
template <uint32_t kWarps>
struct Gather {
  static constexpr uint32_t kEach = 32 / kWarps;  // rows of a thread
  const uint16_t *from[kEach];
  int32_t pair[kEach];
  uint32_t first, chunk, rows, next_rows;
  // warp: 0 .. kWarps - 1
  __device__ __forceinline__ explicit Gather(uint32_t warp) {
    const uint32_t lane = threadIdx.x & 31;
    first = warp * (128 / kWarps) + lane / 8;
    chunk = lane % 8;
    next_rows = 0;
  }
  // The next tile's first row here is r0, and `tile_rows` rows of it exist.
  __device__ __forceinline__ void fetch(const ExpertsProblem &p, uint32_t r0, uint32_t tile_rows) {
    next_rows = tile_rows;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i)
      pair[i] = first + i * 4 < tile_rows ? __ldg(p.order + r0 + first + i * 4) : 0;
  }
  // Turns to the tile fetched last.
  __device__ __forceinline__ void turn(const ExpertsProblem &p) {
    rows = next_rows;
    const uint16_t *x = static_cast<const uint16_t *>(p.x) + chunk * 8;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      // pair / top_k by the reciprocal floor(2^32 / top_k) + 1, which is one too much at most.  (A negative
      // pair is far up among the unsigned ones, where its quotient may yet be a row.)
      uint32_t at = p.top_k > 1 ? __umulhi((uint32_t)pair[i], p.top_k_inv) : (uint32_t)pair[i];
      if (at * p.top_k > (uint32_t)pair[i]) --at;
      if (pair[i] < 0 || at >= p.x_rows) {
        report_status(p.status, kStatusBadArg);
        at = p.x_rows - 1;
      }
      from[i] = x + (size_t)at * p.ldx;
    }
  }
  // Columns kb * kBK .. + kBK - 1, those past k as zeros.
  __device__ __forceinline__ void stage(const ExpertsProblem &p, uint32_t dst, uint32_t kb) const {
    const uint32_t col = kb * kBK + chunk * 8;
    const uint32_t bytes = col < p.k ? min((p.k - col) * 2, 16u) : 0;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      const uint32_t r = first + i * 4;
      if (r < rows)
        copy16(dst + r * 128 + ((chunk ^ (r & 7)) << 4), bytes ? from[i] + kb * kBK : from[i], bytes);
    }
  }
};

// The tables of a launch: start[e] is offsets[e] cut to 0 .. rows and never falling, tiles[e] the tiles
// of kRows rows of the experts before e.  One warp fills them.
template <uint32_t kRows>
__device__ __forceinline__ void fill_tables(const ExpertsProblem &p, uint32_t *start, uint32_t *tiles) {
  const uint32_t lane = threadIdx.x & 31;
  constexpr uint32_t kAhead = 4;  // loads on their way at once
  uint32_t edge = 0, count = 0;
  int32_t ahead[kAhead];
  for (uint32_t e0 = 0; e0 <= p.experts; e0 += 32) {
    const uint32_t e = e0 + lane, turn = e0 / 32 % kAhead;
    if (turn == 0) {
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a)
        ahead[a] = e + a * 32 <= p.experts ? __ldg(p.offsets + e + a * 32) : 0;
    }
    const int32_t raw = turn == 0 ? ahead[0] : turn == 1 ? ahead[1] : turn == 2 ? ahead[2] : ahead[3];
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
    uint32_t n = e <= p.experts ? (v - before + kRows - 1) / kRows : 0;  // tiles of expert e - 1
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

// What an epilogue warp finishes: rows r0 + lane of the output, of which the first `rows` exist.
struct Finish {
  uint32_t r0, rows, staging;
  uint32_t bias;  // in shared memory: its columns', gated the gate's and then the up's
};
// The bias of the warp's kCols columns from n on into shared memory, fetched while the products are made: at
// their end a first look at it took as long as a small tile.
template <bool kGated, uint32_t kCols>
__device__ __forceinline__ void fetch_bias(const ExpertsProblem &p, uint32_t to, uint32_t e, uint32_t n) {
  const uint32_t lane = threadIdx.x & 31;
  const float *bias = p.bias + (size_t)e * (kGated ? 2 : 1) * p.n;
  float v[(kCols + 31) / 32], u[(kCols + 31) / 32];
#pragma unroll
  for (uint32_t c = 0; c < kCols; c += 32) {
    const bool in = c + lane < kCols && n + c + lane < p.n;
    v[c / 32] = in ? __ldg(bias + n + c + lane) : 0.f;
    if constexpr (kGated) u[c / 32] = in ? __ldg(bias + p.n + n + c + lane) : 0.f;
  }
  __syncwarp();
#pragma unroll
  for (uint32_t c = 0; c < kCols; c += 32) {
    if (c + lane >= kCols) continue;
    st_shared(to + (c + lane) * 4, __float_as_uint(v[c / 32]));
    if constexpr (kGated) st_shared(to + (kCols + c + lane) * 4, __float_as_uint(u[c / 32]));
  }
  __syncwarp();
}
// Stores 32 staged rows of kPieces 16-byte pieces (elements of kSize bytes) from column n on, in pieces of 16
// bytes where the rows of out start on such, otherwise of 4, and bf16 rows at odd elements one by one.
template <uint32_t kSize, uint32_t kPieces>
__device__ __forceinline__ void store_staged(const ExpertsProblem &p, const Finish &f, uint32_t n) {
  const uint32_t lane = threadIdx.x & 31;
  auto piece_of = [&](uint32_t r, uint32_t piece) {
    return f.staging + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4);
  };
  uint8_t *to = static_cast<uint8_t *>(p.out) + ((size_t)f.r0 * p.ldo + n) * kSize;
  const size_t pitch = (size_t)p.ldo * kSize;
  if (p.out_step == 16) {
    constexpr uint32_t kEach = 16 / kSize;
    const uint32_t piece = lane & 3, col = n + piece * kEach;
    if (piece >= kPieces || col >= p.n) return;
    const bool whole = col + kEach <= p.n;
#pragma unroll
    for (uint32_t r = lane >> 2; r < 32; r += 8) {
      if (r >= f.rows) break;
      const uint4 o = ld_shared_v4(piece_of(r, piece));
      uint8_t *at = to + r * pitch + piece * 16;
      if (whole) {
        *reinterpret_cast<uint4 *>(at) = o;
      } else {
        for (uint32_t t = 0; col + t < p.n; ++t) {
          if constexpr (kSize == 4)
            reinterpret_cast<uint32_t *>(at)[t] = u4_at(o, t);
          else
            reinterpret_cast<uint16_t *>(at)[t] = (uint16_t)(u4_at(o, t / 2) >> (16 * (t & 1)));
        }
      }
    }
  } else if (p.out_step == 4) {
    // 16 lanes a row: the words of 64 bytes.
    const uint32_t word = lane & 15, col = n + word * (4 / kSize);
    if (word >= 4 * kPieces || col >= p.n) return;
    const bool whole = col + 4 / kSize <= p.n;
#pragma unroll 4
    for (uint32_t r = lane >> 4; r < f.rows; r += 2) {
      const uint32_t o = ld_shared(piece_of(r, word >> 2) + (word & 3) * 4);
      uint8_t *at = to + r * pitch + word * 4;
      if (whole)
        *reinterpret_cast<uint32_t *>(at) = o;
      else
        *reinterpret_cast<uint16_t *>(at) = (uint16_t)o;
    }
  } else if constexpr (kSize == 2) {
    if (lane >= 8 * kPieces || n + lane >= p.n) return;
#pragma unroll 4
    for (uint32_t r = 0; r < f.rows; ++r) {
      const uint32_t o = ld_shared(piece_of(r, lane >> 3) + (lane & 6) * 2);
      *reinterpret_cast<uint16_t *>(to + r * pitch + lane * 2) = (uint16_t)(o >> (16 * (lane & 1)));
    }
  }
}
// Bias, activation, gate and store of columns c .. c + kStep - 1 of the warp's kCols from n0 on, of 32 rows,
// one a lane; u is the up half.  The whole warp calls it.
template <bool kGated, uint32_t kCols, uint32_t kStep>
__device__ __forceinline__ void finish_columns(const ExpertsProblem &p, const Finish &f, uint32_t n0,
                                               uint32_t c, float (&v)[kStep],
                                               float (&u)[kGated ? kStep : 1]) {
  const uint32_t n = n0 + c;
  if (!f.rows || n >= p.n) return;
  const uint32_t lane = threadIdx.x & 31;
  if (p.bias) {
#pragma unroll
    for (uint32_t t = 0; t < kStep; t += 4) {
      const uint4 q = ld_shared_v4(f.bias + (c + t) * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[t + i] += __uint_as_float(u4_at(q, i));
      if constexpr (kGated) {
        const uint4 r = ld_shared_v4(f.bias + (kCols + c + t) * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) u[t + i] += __uint_as_float(u4_at(r, i));
      }
    }
  }
  activate_all(v, p.act);
  if constexpr (kGated) {
#pragma unroll
    for (uint32_t t = 0; t < kStep; ++t) v[t] *= u[t];
  }
  // Through shared memory, so that a warp stores rows of 64 bytes.  The 16-byte pieces of a row are
  // swapped so that neither side meets a bank twice.
  const uint32_t sw = (lane >> 1) & 3, mine = f.staging + lane * 64;
  if (p.out_dtype == TX_F32) {
#pragma unroll
    for (uint32_t h = 0; h < kStep; h += 16) {
      __syncwarp();
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q)
        st_shared_v4(mine + ((q ^ sw) << 4), __float_as_uint(v[h + 4 * q]),
                     __float_as_uint(v[h + 4 * q + 1]), __float_as_uint(v[h + 4 * q + 2]),
                     __float_as_uint(v[h + 4 * q + 3]));
      __syncwarp();
      if (n + h < p.n) store_staged<4, 4>(p, f, n + h);
    }
  } else {
    __syncwarp();
#pragma unroll
    for (uint32_t q = 0; q < kStep / 8; ++q)
      st_shared_v4(mine + ((q ^ sw) << 4), pack_bf16x2(v[8 * q], v[8 * q + 1]),
                   pack_bf16x2(v[8 * q + 2], v[8 * q + 3]), pack_bf16x2(v[8 * q + 4], v[8 * q + 5]),
                   pack_bf16x2(v[8 * q + 6], v[8 * q + 7]));
    __syncwarp();
    store_staged<2, kStep / 8>(p, f, n);
  }
}
template <uint32_t kStep>
__device__ __forceinline__ void load_columns(uint32_t at, float (&v)[kStep]) {
  uint32_t a[kStep];
  tmem_load(at, a);
#pragma unroll
  for (uint32_t t = 0; t < kStep; ++t) v[t] = __uint_as_float(a[t]);
}

template <uint32_t kStep>
__device__ __forceinline__ void zero(float (&v)[kStep]) {
#pragma unroll
  for (uint32_t t = 0; t < kStep; ++t) v[t] = 0.f;
}
// v += the columns, eight at a time: sums hold most registers here.
template <uint32_t kStep>
__device__ __forceinline__ void add_columns(uint32_t at, float (&v)[kStep]) {
#pragma unroll
  for (uint32_t t = 0; t < kStep; t += 8) {
    float a[8];
    load_columns<8>(at + t, a);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) v[t + i] += a[i];
  }
}

// kLong: the sum is taken in parts of 512 K that are added in fp32 registers.  (Added from zero on: with the
// first part taken as it is the compiler held them twice.  Tiles of 256 columns, gated, still pass 24 to 32 bytes
// a thread through local memory.)
// Two warps gather where each epilogue thread holds 128 sums and the others' registers are those that it lacks
// (with four, sums went through local memory), otherwise four.
template <int kBN, bool kLong>
constexpr uint32_t kGathering = kLong && kBN == 256 ? 2 : 4;
template <int kBN, bool kGated, bool kLong, bool kGather>
__global__ void __launch_bounds__(kThreads + (kGather ? 32 * kGathering<kBN, kLong> : 0), 1)
    experts_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                   const __grid_constant__ ExpertsProblem p) {
  using C = Cfg<kBN>;
  constexpr uint32_t kOut = kGated ? kBN / 2 : kBN;  // output columns of a tile
  constexpr uint32_t kGathers = kGathering<kBN, kLong>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_addr(smem), bars = sbase + C::kOffMisc;
  auto bar = [&](uint32_t i) { return bars + 8u * i; };
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + C::kOffMisc + kOffAbort);
  uint32_t *start = reinterpret_cast<uint32_t *>(smem + C::kOffTables);
  uint32_t *tiles = start + C::kMaxExperts + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_w);
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(bar(kBarFull + s), kGather ? 1 + 32 * kGathers : 1);  // the TMA copies, and each gathering thread
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
  if (warp == 2) fill_tables<kBM>(p, start, tiles);
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
      const int r0 = (int)(start[e] + (mt - tiles[e]) * kBM), n0 = (int)(tile % nt * kOut);
      for (uint32_t kb = 0; kb < nk; ++kb) {
        const uint32_t s = fills % C::kStages, round = fills / C::kStages;
        if (round &&
            !(ok = warp_wait(bar(kBarEmpty + s), (round - 1) & 1, abort_flag, p, kSiteEmpty)))
          break;
        const uint32_t dst = sbase + s * C::kStageBytes, x = kb * kBK;
        if (elect_one()) {
          mbar_expect_tx(bar(kBarFull + s), kGather ? C::kBBytes : C::kStageBytes);
          if constexpr (!kGather) tma_load_2d(dst, &tm_x, bar(kBarFull + s), (int)x, r0);
          tma_load_3d(dst + C::kABytes, &tm_w, bar(kBarFull + s), (int)x, n0, (int)e);
          if constexpr (kGated)
            tma_load_3d(dst + C::kABytes + C::kBBytes / 2, &tm_w, bar(kBarFull + s), (int)x,
                        (int)p.n + n0, (int)e);
        }
        __syncwarp();
        ++fills;
      }
    }
    // No copy may land after the CTA has gone.
    if (lane == 0) {
      const long long now = clock64();
      for (uint32_t s = 0; s < (uint32_t)C::kStages && s < fills; ++s)
        drain_bar(bar(kBarFull + s), ((fills - 1 - s) / C::kStages) & 1, now);
    }
    __syncwarp();
  } else if (kGather && warp >= 10) {
    uint32_t fills = 0, e = 0;
    bool ok = true;
    Gather<kGathers> rows((uint32_t)warp - 10);
    auto fetch = [&](uint32_t tile) {
      if (tile >= total) return;
      e = expert_of(tiles, p.experts, tile / nt, e);
      const uint32_t r0 = start[e] + (tile / nt - tiles[e]) * kBM;
      rows.fetch(p, r0, min(start[e + 1] - r0, (uint32_t)kBM));
    };
    fetch(blockIdx.x);
    for (uint32_t tile = blockIdx.x; ok && tile < total; tile += gridDim.x) {
      rows.turn(p);
      fetch(tile + gridDim.x);
      for (uint32_t kb = 0; kb < nk; ++kb) {
        const uint32_t s = fills % C::kStages, round = fills / C::kStages;
        if (round &&
            !(ok = warp_wait(bar(kBarEmpty + s), (round - 1) & 1, abort_flag, p, kSiteEmpty)))
          break;
        rows.stage(p, sbase + s * C::kStageBytes, kb);
        copies_arrive(bar(kBarFull + s));
        ++fills;
      }
    }
    copies_wait();
  } else if (warp == 1) {
    uint32_t step = 0, done = 0;  // K stages, partial sums
    bool ok = true;
    for (uint32_t tile = blockIdx.x; ok && tile < total; tile += gridDim.x) {
      for (uint32_t kb = 0; ok && kb < nk; ++done) {
        const uint32_t b = done & 1, acc = tmem + b * kBN;
        if (done >= 2 &&
            !(ok = warp_wait(bar(kBarFree + b), ((done >> 1) - 1) & 1, abort_flag, p, kSiteFree)))
          break;
        tc_fence_after();
        const uint32_t end = kLong ? min(kb + kPart, nk) : nk;
        for (uint32_t first = kb; kb < end; ++kb, ++step) {
          const uint32_t s = step % C::kStages;
          if (!(ok = warp_wait(bar(kBarFull + s), (step / C::kStages) & 1, abort_flag, p, kSiteFull)))
            break;
          if constexpr (kGather) fence_proxy_async();
          tc_fence_after();
          const uint32_t st = sbase + s * C::kStageBytes;
          const uint64_t ad = sw128_desc(st, 16, 1024), bd = sw128_desc(st + C::kABytes, 16, 1024);
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              umma(acc, ad + ks * 2, bd + ks * 2, C::kIdesc, kb > first || ks > 0);
            umma_commit(bar(kBarEmpty + s));
          }
          __syncwarp();
        }
        if (ok && elect_one()) umma_commit(bar(kBarAcc + b));
        __syncwarp();
      }
    }
    if (elect_one()) umma_commit(bar(kBarDrain));
    __syncwarp();
    drain_bar(bar(kBarDrain), 0);
  } else {
    // Warp w finishes output columns [half * kCols, +kCols) of the 32 rows of its tensor-memory quarter.
    constexpr uint32_t kCols = kOut / 2, kStep = kCols < 32 ? kCols : 32;
    const uint32_t quarter = (uint32_t)warp & 3, half = (uint32_t)(warp - 2) >> 2;
    const uint32_t lanes = (quarter * 32u) << 16;
    const uint32_t staging = sbase + C::kOffStaging + (uint32_t)(warp - 2) * kBufBytes;
    const uint32_t bias = sbase + C::kOffStaging + 8 * kBufBytes + (uint32_t)(warp - 2) * kBiasBytes;
    static_assert(kCols * (kGated ? 8 : 4) <= kBiasBytes, "bias area");
    uint32_t done = 0, e = 0;
    bool ok = true;
    for (uint32_t tile = blockIdx.x; ok && tile < total; tile += gridDim.x) {
      const uint32_t mt = tile / nt;
      e = expert_of(tiles, p.experts, mt, e);
      const uint32_t r0 = start[e] + (mt - tiles[e]) * kBM, rows = min(start[e + 1] - r0, (uint32_t)kBM);
      const uint32_t n0 = tile % nt * kOut + half * kCols;
      const Finish f{r0 + quarter * 32, rows > quarter * 32 ? min(rows - quarter * 32, 32u) : 0, staging,
                     bias};
      if (p.bias && f.rows) fetch_bias<kGated, kCols>(p, bias, e, n0);
      if constexpr (kLong) {
        constexpr uint32_t kHeld = kCols / kStep;
        float v[kHeld][kStep], u[kGated ? kHeld : 1][kGated ? kStep : 1];
#pragma unroll
        for (uint32_t c = 0; c < kHeld; ++c) zero(v[c]);
        if constexpr (kGated) {
#pragma unroll
          for (uint32_t c = 0; c < kHeld; ++c) zero(u[c]);
        }
        const uint32_t parts = (nk + kPart - 1) / kPart;
#pragma unroll 1
        for (uint32_t part = 0; part < parts; ++part, ++done) {
          const uint32_t b = done & 1, t0 = tmem + b * kBN + half * kCols + lanes;
          if (!(ok = __all_sync(kFull, wait_bar(bar(kBarAcc + b), (done >> 1) & 1, abort_flag, p.status,
                                                kSiteAcc, p.wait_cycles))))
            break;
          tc_fence_after();
#pragma unroll
          for (uint32_t c = 0; c < kHeld; ++c) {
            add_columns(t0 + c * kStep, v[c]);
            if constexpr (kGated) add_columns(t0 + kOut + c * kStep, u[c]);
          }
          tc_fence_before();
          mbar_arrive(bar(kBarFree + b));
        }
        if (!ok) break;
#pragma unroll
        for (uint32_t c = 0; c < kHeld; ++c)
          finish_columns<kGated, kCols, kStep>(p, f, n0, c * kStep, v[c], u[kGated ? c : 0]);
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
          load_columns<kStep>(t0 + c, v);
          if constexpr (kGated) load_columns<kStep>(t0 + kOut + c, u);
          finish_columns<kGated, kCols, kStep>(p, f, n0, c, v, u);
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

// ---- two CTAs a tile ------------------------------------------------------------------------
// 256 rows x 256 columns of products a tile, by the two CTAs of a cluster (cta_group::2): each brings and
// holds 128 of the rows and 128 of the columns, so that a stage of 64 K takes 32 KB of shared memory a CTA
// where 128 x 256 tiles take 48 KB.  Between the two CTAs go copies by TMA and products alone, which complete
// at barriers, and tensor memory handed back between its fences.
namespace pair {
constexpr uint32_t kHalfBytes = 128 * 128, kStageBytes = 2 * kHalfBytes;
constexpr uint32_t kRows = 256, kWide = 256, kMaxExperts = 1024;
constexpr int kStages = 6;
constexpr uint32_t kOffStaging = kStages * kStageBytes;
constexpr uint32_t kOffMisc = kOffStaging + 8 * (kBufBytes + kBiasBytes);
constexpr uint32_t kOffTables = kOffMisc + 512;
constexpr uint32_t kSmemBytes = kOffTables + 2 * (kMaxExperts + 1) * 4;
static_assert(kSmemBytes <= 232448, "shared memory");
constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((kWide >> 3) << 17) |
                            ((kRows >> 4) << 24);
// kFullBar: of the even CTA, the copies of both.
enum : uint32_t { kFullBar = 0, kEmpty = kStages, kAcc = 2 * kStages, kFree = kAcc + 2,
                  kDrain = kFree + 2, kBars = kDrain + 1 };
static_assert(8 * kBars + 8 <= 512, "misc area");
constexpr long long kLandCycles = 1 << 20;  // 0.5 ms
}  // namespace pair

template <bool kGated, bool kLong>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                const __grid_constant__ ExpertsProblem p) {
  using namespace pair;
  constexpr uint32_t kOut = kGated ? kWide / 2 : kWide;  // output columns of a tile
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_addr(smem), bars = sbase + kOffMisc;
  auto bar = [&](uint32_t i) { return bars + 8u * i; };
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + kOffMisc + 8 * kBars + 4);
  uint32_t *start = reinterpret_cast<uint32_t *>(smem + kOffTables);
  uint32_t *tiles = start + kMaxExperts + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank(), first_tile = blockIdx.x / 2, tile_step = gridDim.x / 2;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_w);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar(kFullBar + s), 1);
      mbar_init(bar(kEmpty + s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar(kAcc + b), 1);
      mbar_init(bar(kFree + b), 16);  // the epilogue warps of both CTAs
    }
    mbar_init(bar(kDrain), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     bars + 8 * kBars),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == 2) fill_tables<kRows>(p, start, tiles);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<uint32_t *>(smem + kOffMisc + 8 * kBars);
  const uint32_t nt = (p.n + kOut - 1) / kOut, total = tiles[p.experts] * nt;
  const uint32_t nk = (p.k + kBK - 1) / kBK;
  auto full_at_even = [&](uint32_t s) { return cluster_addr(bar(kFullBar + s), 0); };

  if (warp == 0) {
    // This CTA's rows and columns of every stage.
    uint32_t fills = 0, e = 0;
    bool ok = true;
    for (uint32_t tile = first_tile; ok && tile < total; tile += tile_step) {
      const uint32_t mt = tile / nt;
      e = expert_of(tiles, p.experts, mt, e);
      const int r0 = (int)(start[e] + (mt - tiles[e]) * kRows + rank * 128);
      const int n0 = (int)(tile % nt * kOut + rank * (kGated ? p.n : 128));
      for (uint32_t kb = 0; kb < nk; ++kb) {
        const uint32_t s = fills % kStages, round = fills / kStages;
        if (round && !(ok = warp_wait<true>(bar(kEmpty + s), (round - 1) & 1, abort_flag, p, kSiteEmpty)))
          break;
        const uint32_t dst = sbase + s * kStageBytes, full = full_at_even(s);
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(bar(kFullBar + s), 4 * kHalfBytes);
          tma_load_2d_pair(dst, &tm_x, full, (int)(kb * kBK), r0);
          tma_load_3d_pair(dst + kHalfBytes, &tm_w, full, (int)(kb * kBK), n0, (int)e);
        }
        __syncwarp();
        ++fills;
      }
    }
    // No copy may land after the CTAs have gone.
    if (lane == 0 && rank == 0) {
      const long long now = clock64();
      for (uint32_t s = 0; s < (uint32_t)kStages && s < fills; ++s)
        drain_bar<true>(bar(kFullBar + s), ((fills - 1 - s) / kStages) & 1, now);
    }
    // The odd CTA's copies arrive at barriers that it cannot test.  Those in flight when a wait has ended get
    // time to land.
    if (!ok && rank == 1) pause_cycles(kLandCycles);
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      uint32_t step = 0, done = 0;
      bool ok = true;
      for (uint32_t tile = first_tile; ok && tile < total; tile += tile_step) {
        for (uint32_t kb = 0; ok && kb < nk; ++done) {
          const uint32_t b = done & 1, acc = tmem + b * kWide;
          if (done >= 2 &&
              !(ok = warp_wait<true>(bar(kFree + b), ((done >> 1) - 1) & 1, abort_flag, p, kSiteFree)))
            break;
          tc_fence_after();
          const uint32_t end = kLong ? min(kb + kPart, nk) : nk;
          for (uint32_t first = kb; kb < end; ++kb, ++step) {
            const uint32_t s = step % kStages, parity = (step / kStages) & 1;
            if (!(ok = warp_wait<true>(bar(kFullBar + s), parity, abort_flag, p, kSiteFull))) break;
            tc_fence_after();
            const uint32_t st = sbase + s * kStageBytes;
            const uint64_t ad = sw128_desc(st, 16, 1024), bd = sw128_desc(st + kHalfBytes, 16, 1024);
            if (elect_one()) {
#pragma unroll
              for (int ks = 0; ks < 4; ++ks)
                umma_pair(acc, ad + ks * 2, bd + ks * 2, kIdesc, kb > first || ks > 0);
              umma_commit_pair(bar(kEmpty + s));
            }
            __syncwarp();
          }
          if (ok && elect_one()) umma_commit_pair(bar(kAcc + b));
          __syncwarp();
        }
      }
      if (elect_one()) umma_commit_pair(bar(kDrain));
      __syncwarp();
    }
    drain_bar<true>(bar(kDrain), 0);
  } else {
    // Warp w finishes output columns [half * kCols, +kCols) of the 32 rows of its tensor-memory quarter.
    constexpr uint32_t kCols = kOut / 2, kStep = 32;
    const uint32_t quarter = (uint32_t)warp & 3, half = (uint32_t)(warp - 2) >> 2;
    const uint32_t lanes = (quarter * 32u) << 16;
    const uint32_t staging = sbase + kOffStaging + (uint32_t)(warp - 2) * kBufBytes;
    const uint32_t bias = sbase + kOffStaging + 8 * kBufBytes + (uint32_t)(warp - 2) * kBiasBytes;
    static_assert(kCols * (kGated ? 8 : 4) <= kBiasBytes, "bias area");
    uint32_t done = 0, e = 0;
    bool ok = true;
    auto wait_acc = [&] {
      const bool is = __all_sync(kFull, wait_bar<true>(bar(kAcc + (done & 1)), (done >> 1) & 1, abort_flag,
                                                 p.status, kSiteAcc, p.wait_cycles));
      tc_fence_after();
      return is;
    };
    auto give_acc = [&] {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(cluster_addr(bar(kFree + (done & 1)), 0));
      ++done;
    };
    for (uint32_t tile = first_tile; ok && tile < total; tile += tile_step) {
      const uint32_t mt = tile / nt;
      e = expert_of(tiles, p.experts, mt, e);
      const uint32_t r0 = start[e] + (mt - tiles[e]) * kRows + rank * 128 + quarter * 32;
      const uint32_t n0 = tile % nt * kOut + half * kCols;
      const Finish f{r0, start[e + 1] > r0 ? min(start[e + 1] - r0, 32u) : 0, staging, bias};
      if (p.bias && f.rows) fetch_bias<kGated, kCols>(p, bias, e, n0);
      const uint32_t t0 = tmem + half * kCols + lanes;
      if constexpr (kLong) {
        constexpr uint32_t kHeld = kCols / kStep;
        float v[kHeld][kStep], u[kGated ? kHeld : 1][kGated ? kStep : 1];
#pragma unroll
        for (uint32_t c = 0; c < kHeld; ++c) zero(v[c]);
        if constexpr (kGated) {
#pragma unroll
          for (uint32_t c = 0; c < kHeld; ++c) zero(u[c]);
        }
        const uint32_t parts = (nk + kPart - 1) / kPart;
#pragma unroll 1
        for (uint32_t i = 0; i < parts; ++i) {
          if (!(ok = wait_acc())) break;
          const uint32_t at = t0 + (done & 1) * kWide;
#pragma unroll
          for (uint32_t c = 0; c < kHeld; ++c) {
            add_columns(at + c * kStep, v[c]);
            if constexpr (kGated) add_columns(at + kOut + c * kStep, u[c]);
          }
          give_acc();
        }
        if (!ok) break;
#pragma unroll
        for (uint32_t c = 0; c < kHeld; ++c)
          finish_columns<kGated, kCols, kStep>(p, f, n0, c * kStep, v[c], u[kGated ? c : 0]);
      } else {
        if (!(ok = wait_acc())) break;
        const uint32_t at = t0 + (done & 1) * kWide;
        if (f.rows) {
#pragma unroll 1
          for (uint32_t c = 0; c < kCols; c += kStep) {
            float v[kStep], u[kGated ? kStep : 1];
            load_columns<kStep>(at + c, v);
            if constexpr (kGated) load_columns<kStep>(at + kOut + c, u);
            finish_columns<kGated, kCols, kStep>(p, f, n0, c, v, u);
            __syncwarp();
          }
        }
        give_acc();
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  // Neither CTA leaves, nor gives its tensor memory back, while the other may still reach it.
  cluster_sync();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                 : "memory");
}

// x [rows, k] in boxes of a tile's rows, and w [experts, wide, k] in boxes of box_rows rows; 64 columns
// of bf16 in the 128-byte swizzle.
bool make_maps(CUtensorMap *mx, CUtensorMap *mw, const ExpertsProblem &p, uint32_t box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  const uint32_t wide = p.n * (p.gated ? 2 : 1);
  cuuint64_t xd[2] = {p.k, p.x_rows}, xs[1] = {p.ldx * 2};
  cuuint32_t xb[2] = {64, kBM}, one[3] = {1, 1, 1};
  cuuint64_t wd[3] = {p.k, wide, p.experts}, ws[2] = {p.ldw * 2, p.expert_stride * 2};
  cuuint32_t wb[3] = {64, box_rows, 1};
  return fn(mx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(p.x), xd, xs, xb, one,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS &&
         fn(mw, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(p.w), wd, ws, wb, one,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int kBN, bool kGated, bool kLong, bool kGather>
cudaError_t launch_tiles(const ExpertsProblem &p, int num_sms, cudaStream_t stream) {
  constexpr uint32_t smem = Cfg<kBN>::kSmemBytes;
  CUtensorMap mx, mw;
  if (!make_maps(&mx, &mw, p, kGated ? kBN / 2 : kBN)) return cudaErrorInvalidValue;
  static std::atomic<uint64_t> seen{0};
  cudaError_t e =
      allow_smem((const void *)experts_kernel<kBN, kGated, kLong, kGather>, (int)smem, seen);
  if (e != cudaSuccess) return e;
  constexpr uint32_t threads = kThreads + (kGather ? 32 * kGathering<kBN, kLong> : 0);
  experts_kernel<kBN, kGated, kLong, kGather><<<num_sms, threads, smem, stream>>>(mx, mw, p);
  return cudaGetLastError();
}

template <bool kGated, bool kLong>
cudaError_t launch_pairs(const ExpertsProblem &p, int num_sms, cudaStream_t stream) {
  CUtensorMap mx, mw;
  if (!make_maps(&mx, &mw, p, 128)) return cudaErrorInvalidValue;
  static std::atomic<uint64_t> seen{0};
  cudaError_t e = allow_smem((const void *)pair_kernel<kGated, kLong>, (int)pair::kSmemBytes, seen);
  if (e != cudaSuccess) return e;
  pair_kernel<kGated, kLong><<<num_sms / 2 * 2, kThreads, pair::kSmemBytes, stream>>>(mx, mw, p);
  return cudaGetLastError();
}

template <bool kGated, bool kLong, bool kGather>
cudaError_t launch_wide(const ExpertsProblem &p, int num_sms, cudaStream_t stream) {
  const uint32_t wide = p.n * (kGated ? 2 : 1);
  if constexpr (kGather) {
    // 256 columns a tile where tiles of 128 are more than the SMs and an expert has 64 rows or more.  Tiles of
    // 128 against 256 columns, gated, n 512, k 1024: 2048 rows over 8 experts 20 / 18 us, 8192 over 8 34 / 25,
    // 4096 over 64 35 / 33, 65536 over 64 191 / 123, over 512 262 / 222.  n 1024, k 1024: 1024 rows over 8
    // 16 / 17, 2048 21 / 18; n 512, k 2048: 4096 over 8 21 / 24, 6000 31 / 25; n 256, k 768, 16 experts: 8192 rows
    // 14 / 16, 16384 19 / 16; n 264, k 512: 32768 over 64 32 / 29.  In partial sums the tile's own end is longer,
    // and three tiles of 128 for each SM are the border: n 1024, k 1024: 4096 over 8 25 / 29, 6000 31 / 35, 8192
    // 38 / 33, 65536 over 64 218 / 172; k 576 155 / 131; gated, n 512, k 1024: 6000 over 8 29 / 32, 8192 36 / 33,
    // 65536 over 64 212 / 162.
    if (wide > 128 && p.rows >= 64 * p.experts &&
        (p.rows / kBM + (uint64_t)p.experts / 2) * ((wide + 127) / 128) > (kLong ? 3ull : 1ull) * num_sms)
      return launch_tiles<256, kGated, kLong, true>(p, num_sms, stream);
  } else {
    // Tiles of two CTAs where an expert has 128 rows or more and there is work for them.  Tiles of 128 columns
    // against them, gated, n 512, k 1024: 2048 rows over 8 experts 19 / 18 us, 8192 over 8 29 / 23, over 64
    // 40 / 38, 65536 over 64 152 / 100, over 512 228 / 222, 4096 over 64 33 / 37 (but 4096 over 8 19 / 23).
    // n 256, k 768, 16 experts: 8192 rows 13 / 16, 16384 16 / 16, 65536 39 / 30.  In partial sums the tile's own
    // end is longer, n 1024, k 1024: 4096 rows over 8 21 / 31, 8192 31 / 31, 16384 51 / 47; 65536 over 64
    // 164 / 137, k 576 115 / 141 in a loop.
    const uint64_t work = (uint64_t)p.rows * wide * p.k;
    const bool pairs = kLong ? p.k >= 1024 && work >= 1ull << 34 : p.rows > 8192 || work >= 1ull << 32;
    if (wide > 128 && p.rows >= 128 * p.experts && pairs)
      return launch_pairs<kGated, kLong>(p, num_sms, stream);
  }
  // 64 columns a tile where tiles of 128 would leave half the SMs without one (the expert ranges are not
  // known here: at most a tile for each row or expert, and one for every 128 rows): 18 / 12 us for 2 to 32
  // rows over 8 experts, n 768, k 768; but 27 / 35 us for 64 rows over 64 experts, gated, n 512, k 1024.
  const uint64_t tiles = ((uint64_t)std::min(p.rows, p.experts) + p.rows / kBM) * ((wide + 127) / 128);
  if (wide <= 64 || 2 * tiles <= (uint64_t)num_sms)
    return launch_tiles<64, kGated, kLong, kGather>(p, num_sms, stream);
  return launch_tiles<128, kGated, kLong, kGather>(p, num_sms, stream);
}
template <bool kGated, bool kLong>
cudaError_t launch_rows(const ExpertsProblem &p, int num_sms, cudaStream_t stream) {
  return p.order ? launch_wide<kGated, kLong, true>(p, num_sms, stream)
                 : launch_wide<kGated, kLong, false>(p, num_sms, stream);
}

}  // namespace experts

cudaError_t launch_experts_linear(ExpertsProblem p, int num_sms, cudaStream_t stream) {
  using namespace experts;
  const uint32_t size = p.out_dtype == TX_BF16 ? 2 : 4;
  p.out_step = 16;
  while ((uintptr_t)p.out % p.out_step || p.ldo * size % p.out_step) p.out_step = p.out_step == 16 ? 4 : 2;
  p.top_k_inv = p.top_k > 1 ? (uint32_t)((1ull << 32) / p.top_k) + 1 : 0;
  // The short form of GELU is off by 1.4e-6 of the sum, 5 % of the value at -5, which is nothing beside 1 but
  // not where the value is multiplied by the up half.
  if (p.act == TX_ACT_GELU && (p.out_dtype == TX_F32 || p.gated)) p.act = kGeluF32;
  // The accumulator cuts up to 2^-23 off at each of its additions of 16 K: over 32768 that is a sixteenth of
  // half a bf16 step at most, but 1 % of the value over 2^21, and for an fp32 result too much over 512 already.
  const bool parts = p.k > (p.out_dtype == TX_F32 ? kPart * kBK : 32768);
  if (p.gated)
    return parts ? launch_rows<true, true>(p, num_sms, stream)
                 : launch_rows<true, false>(p, num_sms, stream);
  return parts ? launch_rows<false, true>(p, num_sms, stream)
               : launch_rows<false, false>(p, num_sms, stream);
}

}  // namespace tx
