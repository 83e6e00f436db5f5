// Attention under a score rule on the tensor cores: bf16 q, k, v, head_dim a multiple of 8 up
// to 128 (tx_attention_scored).
//
//   z_ij = scale q_i.k_j;  cap: z = c tanh(z / c);  distance bias: z += b_h(j - pos_i)
//   out_i = sum_j softmax_j(z_ij) v_j over the keys the rule leaves open to row i
//
// One CTA takes 128 rows (query tokens x the heads that share a kv head, attn_scored.cuh) and
// walks the 128-key tiles that some row may see.  S = Q K^T and O += P V are tcgen05.mma
// (M = 128) into tensor memory; thread t of the four softmax warps owns row t (tensor-memory
// lane t).  It walks S twice, 32 keys at a time: first the row's maximum (scores with a cap, a
// bias or a mask go back finished), then P = exp2(z - m) as bf16 into tensor memory, the A operand
// of P.V.  Both walks are rolled loops: the same work unrolled over the 128 keys (20 KB of code a
// tile) was bound by instruction fetches.  P is rounded to bf16 (2^-9 of each weight) because the
// product takes bf16; the row sum adds the unrounded weights.  The reference m follows the row's
// running maximum lazily: O and the row sum are rescaled only when a tile's maximum exceeds it by
// more than 2^8, which changes no result (P stays below 2^8 and the sum uses the same reference).
// Two CTAs share an SM, so one's products run beside the other's softmax.
//
// Bound: the softmax warps, by the latency of their chain (two warps per scheduler): 5500 cycles a
// tile and CTA, 7000 with head_dim 128 and a cap.  Two threads a row (eight warps) took 298 against
// 291 us with a long window, 85 against 77 us with a cap, 171 against 181 us with documents (since
// at 164).  Measured: 8192 tokens, window 4096, 16 / 8 heads of 128: 290 us, 710 TFLOP/s of open
// pairs (42 % of the measured bf16 rate); causal with a cap, packed, 16 / 8 heads of 128: 78 us; 8
// texts of 1500 to 2048 in documents with a table, 12 heads of 64: 164 us.
//
// Values that are not finite.  A key that the rule closes to a row has p = 0 there, and the
// product would turn 0 * Inf or 0 * NaN in its value row into NaN.  In tiles that are not wholly
// open to all rows the MMA warp therefore looks the value tile over while the softmax runs; rows
// of v with such a value (rare) are added to O by hand, for the query rows with p > 0 only, and
// zeroed before the product.
#include <cuda.h>
#include <cudaTypedefs.h>

#include "../../include/tessattn.h"
#include "attn_scored.cuh"
#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace tx {
namespace scored_tc {

using namespace ptx;
using namespace scored;

constexpr int kRows = 128;
constexpr int kThreads = 192;  // warps 0-3 softmax, 4 TMA, 5 MMA
constexpr int kTmaWarp = 4, kMmaWarp = 5;
constexpr uint32_t kTmemCols = 256;  // of the 512 of an SM: two CTAs share it
constexpr uint32_t kColO = 128;      // S in columns 0-127, O from here
constexpr float kRescaleThreshold = 8.0f;  // log2 units
constexpr float kLog2e = 1.44269504088896341f;

// Distance biases lie in shared memory in log2 units.  A table small enough lies there once per CTA
// with kKeys copies of its ends on either side, so that a row reads a tile's 128 distances from one
// place; otherwise each warp lays out, tile by tile, the 127 + 32 / pack distances that its rows
// need.  The pack (at most kTablePack) heads' parts lie 32 / pack words apart modulo 32, so that
// the rows of a warp read different banks.
__host__ __device__ constexpr uint32_t bias_pitch(uint32_t n, uint32_t pack) {
  return n + (32 + 32 / pack - n % 32) % 32;
}
__host__ __device__ constexpr uint32_t window_pitch(uint32_t pack) {
  return bias_pitch(127 + 32 / pack, pack);
}
constexpr uint32_t kWindow = kTablePack * window_pitch(kTablePack);  // a warp's
static_assert(window_pitch(1) <= kWindow && 2 * window_pitch(2) <= kWindow, "window area");

template <int kDP>  // head_dim rounded up to whole 64-column (128-byte) blocks
struct Cfg {
  static constexpr uint32_t kTile = 128 * kDP * 2;  // a tile of Q, K or V
  static constexpr uint32_t kAtom = 128 * 128;      // 128 rows x 64 columns, swizzled
  static constexpr int kSlots = kDP == 64 ? 2 : 1;  // K slots, and V slots
  static constexpr uint32_t kOffQ = 0, kOffK = kTile, kOffV = kOffK + kSlots * kTile;
  static constexpr uint32_t kOffMisc = kOffV + kSlots * kTile;
  static constexpr uint32_t kBiases = kDP == 64 ? 7168 : 3200;  // floats for distance biases
  static constexpr uint32_t kMiscBytes = 256 + kDocWords * 4 + 4 * kKeys * 4 + kBiases * 4;
  static_assert(4 * kWindow <= kBiases, "a window for each warp");
  // head_dim up to 64 leaves columns for P beside S: the next tile's Q.K^T is issued as soon as S
  // has been read.  Otherwise P lies over S, and it waits for P.V.
  static constexpr bool kEarly = kDP == 64;
  static constexpr uint32_t kColP = kEarly ? kColO + 64 : 0;
  static constexpr uint32_t kSmemBytes = kOffMisc + kMiscBytes;
  static_assert(2 * (kSmemBytes + 1024) <= 233472, "two CTAs per SM");
};

// Barriers at the start of the misc area.
enum : uint32_t {
  kBarQ = 0, kBarKFull = 1, kBarKEmpty = 3, kBarVFull = 5, kBarVEmpty = 7, kBarS = 9, kBarP = 10,
  kBarO = 11, kBarScan = 12, kBarHand = 13, kBarSRead = 14, kBarPV = 15,
  kNumBars = 16
};
enum : uint32_t { kOffTmem = 128, kOffAbort = 132, kOffFlag = 136, kOffRange = 144, kOffBad = 160,
                  kOffWords = 256,
                  kOffDocs = kOffWords + kDocWords * 4, kOffBias = kOffDocs + 4 * kKeys * 4 };
enum : int { kSiteK = 1, kSiteV = 2, kSiteKFree = 3, kSiteVFree = 4, kSiteS = 5, kSiteP = 6,
             kSiteO = 7, kSiteQ = 8, kSiteVRead = 9, kSiteScan = 10, kSiteHand = 11,
             kSiteSRead = 12, kSitePV = 13 };

struct Gate {  // a bounded wait that gives up once for the whole CTA
  volatile int *abort_flag;
  int *status;
  long long limit;
  __device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, int site) const {
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
  // Waits, up to a fixed limit, for something that completes by itself.
  static __device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) {
    const long long t0 = clock64();
    while (!mbar_test(bar, parity) && clock64() - t0 < 2000000000ll) {
    }
  }
};

// A distance bias in log2 units.  A finite bias too large for them, at either end, stays finite (those
// from 2.36e38 on are one value), and NaN and the infinities stay what they are: only -inf closes a
// key.
__device__ __forceinline__ float bias_log2(float b) {
  const float most = 3.402823466e38f;
  return fabsf(b) <= most ? fminf(fmaxf(b * kLog2e, -most), most) : b;
}

// Looks over `keys` rows of a value tile (one warp).  Returns whether any value is not finite;
// bad[0..3] get the bits of the rows that hold one.
template <uint32_t kTileBytes>
__device__ __forceinline__ bool scan_values(uint32_t tile, int keys, uint32_t *bad, int lane) {
  // x * 0 is NaN exactly where x is not finite, and then the sum stays NaN.
  auto taint = [](uint32_t w, uint32_t acc) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(w), "r"(0u), "r"(acc));
    return d;
  };
  uint32_t acc = 0;
#pragma unroll 8
  for (uint32_t x = lane * 16; x < kTileBytes; x += 512) {
    const uint4 v = ld_shared_v4(tile + x);
    acc = taint(v.x, taint(v.y, taint(v.z, taint(v.w, acc))));
  }
  if (lane < 4) bad[lane] = 0;
  if (!__any_sync(0xffffffffu, acc != 0)) return false;
  __syncwarp();
  uint32_t any = 0;
  for (uint32_t x = lane * 16; x < kTileBytes; x += 512) {
    const uint4 v = ld_shared_v4(tile + x);
    const int row = (int)(x % (128 * 128)) / 128;
    if (row < keys && taint(v.x, taint(v.y, taint(v.z, taint(v.w, 0u))))) {
      atomicOr(&bad[row >> 5], 1u << (row & 31));
      any = 1;
    }
  }
  return __any_sync(0xffffffffu, any) != 0;
}

// The value rows marked in `bad` added to O for the query rows with p > 0 (thread = row, all four
// softmax warps), then zeroed.  `fresh`: O holds nothing yet.  False where a wait gave up.
template <int kDP>
__device__ __noinline__ bool add_by_hand(const volatile uint32_t *bad, uint32_t tile,
                                         uint32_t atom, uint32_t tP, uint32_t tO, bool fresh,
                                         const Gate &gate, uint32_t read, uint32_t turn) {
  for (int j = 0; j < kKeys; ++j) {
    if (!((bad[j >> 5] >> (j & 31)) & 1)) continue;
    uint32_t w[1];
    tmem_load(tP + j / 2, w);
    const float pj = j & 1 ? bf16_hi(w[0]) : bf16_lo(w[0]);
    for (uint32_t c = 0; c < kDP; c += 16) {
      uint32_t o[16];
      tmem_load(tO + c, o);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t chunk = (c & 63) / 8 + q;
        const uint4 v = ld_shared_v4(tile + (c >> 6) * atom + j * 128 +
                                     ((chunk ^ (uint32_t)(j & 7)) * 16));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = e & 1 ? bf16_hi(u4_at(v, e / 2)) : bf16_lo(u4_at(v, e / 2));
          const float old = fresh ? 0.f : __uint_as_float(o[q * 8 + e]);
          o[q * 8 + e] = __float_as_uint(pj == 0.f ? old : fmaf(pj, x, old));
        }
      }
      tmem_st16(tO + c, o);
    }
    tmem_st_wait();
    fresh = false;
  }
  mbar_arrive(read);  // every thread has read the rows
  if (!__all_sync(0xffffffffu, gate.wait(read, turn & 1, kSiteHand))) return false;
  for (int x = (int)threadIdx.x; x < kKeys * (kDP / 8); x += 128) {
    const int row = x / (kDP / 8), ch = x % (kDP / 8);
    if ((bad[row >> 5] >> (row & 31)) & 1)
      st_shared_v4(tile + (ch >> 3) * atom + row * 128 + (ch & 7) * 16, 0, 0, 0, 0);
  }
  fence_proxy_async();
  return true;
}

enum : int { kNoBias = 0, kSlopes = 1, kTable = 2 };

template <int kDP, bool kCap, int kBias>
__global__ void __launch_bounds__(kThreads, 2)
    scored_tc_kernel(const __grid_constant__ CUtensorMap tm_q,
                     const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ ScoredProblem p) {
  using C = Cfg<kDP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_addr(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t *misc = smem + C::kOffMisc;
  const uint32_t bars = sbase + C::kOffMisc;
  auto bar = [&](uint32_t i) { return bars + 8 * i; };
  uint32_t *words = reinterpret_cast<uint32_t *>(misc + kOffWords);
  const Unit u = make_unit<kRows>(p, blockIdx.x);
  if (!u.present) return;  // whole units: every split of one takes the same way
  const Gate gate{reinterpret_cast<volatile int *>(misc + kOffAbort), p.status, p.wait_cycles};
  if (threadIdx.x == 0) {
    mbar_init(bar(kBarQ), 1);
    for (uint32_t i = 0; i < 2; ++i) {
      mbar_init(bar(kBarKFull + i), 1);
      mbar_init(bar(kBarKEmpty + i), 1);
      mbar_init(bar(kBarVFull + i), 1);
      mbar_init(bar(kBarVEmpty + i), 1);
    }
    mbar_init(bar(kBarS), 1);
    mbar_init(bar(kBarP), 128);
    mbar_init(bar(kBarO), 1);
    mbar_init(bar(kBarScan), 1);
    mbar_init(bar(kBarHand), 128);
    mbar_init(bar(kBarSRead), 4);
    mbar_init(bar(kBarPV), 1);
    *gate.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     bars + kOffTmem),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const bool docs = p.q_docs != nullptr;
  if (docs) mark_tiles(p, u, words, reinterpret_cast<int *>(misc + kOffRange));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<uint32_t *>(misc + kOffTmem);
  const uint32_t *marks = docs ? words : nullptr;
  const int first = next_tile(u, marks, u.first);
  const bool work = u.tokens > 0 && first < u.last;

  float m = -INFINITY, l = 0.f;  // softmax threads: the row's reference and sum
  if (work) {
    if (warp == kTmaWarp) {
      if (lane == 0) {
        mbar_expect_tx(bar(kBarQ), C::kTile);
        for (int c = 0; c < kDP / 64; ++c)
          tma_load_3d(sbase + C::kOffQ + c * C::kAtom, &tm_q, bar(kBarQ), c * 64, (int)u.head0,
                      u.s.q_row + u.t0);
        bool ok = true;
        uint32_t n = 0;
        for (int i = first; i < u.last; i = next_tile(u, marks, i + 1), ++n) {
          const uint32_t slot = n % C::kSlots, round = n / C::kSlots;
          const int row = u.s.k_row + key_tile(u, i) * kKeys;
          if (round && !(ok = gate.wait(bar(kBarKEmpty + slot), (round - 1) & 1, kSiteKFree))) break;
          mbar_expect_tx(bar(kBarKFull + slot), C::kTile);
          for (int c = 0; c < kDP / 64; ++c)
            tma_load_3d(sbase + C::kOffK + slot * C::kTile + c * C::kAtom, &tm_k,
                        bar(kBarKFull + slot), c * 64, (int)u.kv, row);
          if (round && !(ok = gate.wait(bar(kBarVEmpty + slot), (round - 1) & 1, kSiteVFree))) {
            Gate::drain(bar(kBarKFull + slot), round & 1);
            break;
          }
          mbar_expect_tx(bar(kBarVFull + slot), C::kTile);
          for (int c = 0; c < kDP / 64; ++c)
            tma_load_3d(sbase + C::kOffV + slot * C::kTile + c * C::kAtom, &tm_v,
                        bar(kBarVFull + slot), c * 64, (int)u.kv, row);
        }
        // Every load issued completes by itself; none may land after the CTA has gone.
        Gate::drain(bar(kBarQ), 0);
        for (uint32_t s = 0; s < (uint32_t)C::kSlots && s < n; ++s) {
          const uint32_t rounds = (n - 1 - s) / C::kSlots;
          Gate::drain(bar(kBarKFull + s), rounds & 1);
          Gate::drain(bar(kBarVFull + s), rounds & 1);
        }
      }
      __syncwarp();
    } else if (warp == kMmaWarp) {
      // D = fp32, A and B bf16; B of P.V is V as stored (MN-major).  N of P.V and the K steps of
      // Q.K^T cover head_dim rounded up to 16 (the columns past it are zeros).
      constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24);
      const uint32_t dsteps = (p.dim + 15) / 16;
      const uint32_t idesc_qk = kIdesc | ((128u >> 3) << 17);
      const uint32_t idesc_pv = kIdesc | (1u << 16) | ((dsteps * 2) << 17);
      const uint64_t qd = sw128_desc(sbase + C::kOffQ, 16, 1024);
      auto wait = [&](uint32_t b, uint32_t parity, int site) {
        return __all_sync(0xffffffffu, gate.wait(b, parity, site)) != 0;
      };
      // Turn n issues Q.K^T of tile n and then P.V of the tile before it (kEarly: as soon as the
      // softmax has read S; else S takes P's place, so P.V goes first).  One place in the code for
      // each product.  A form with two places for Q.K^T, each right by reading, gave NaN or a fault
      // where only the first was reached; the cause is not known, so the loop keeps to one.
      bool ok = wait(bar(kBarQ), 0, kSiteQ);
      bool more = true, odd = false;
      int prev = first;  // the tile whose P.V is due
      uint32_t n = 0;
      for (int i = first; ok && (more || C::kEarly); ++n) {
        const uint32_t slot = n % C::kSlots, par = (n / C::kSlots) & 1;
        // Values of the tile whose P.V is due: looked over while its softmax runs.
        const uint32_t t = C::kEarly ? n - 1 : n, vslot = t % C::kSlots;
        const int k0 = key_tile(u, C::kEarly ? prev : i) * kKeys, keys = min(u.s.nk - k0, kKeys);
        auto look = [&]() {
          if (!wait(bar(kBarVFull + vslot), (t / C::kSlots) & 1, kSiteV)) return false;
          odd = false;
          if (!whole_tile(u, k0)) {
            odd = scan_values<C::kTile>(sbase + C::kOffV + vslot * C::kTile, keys,
                                        reinterpret_cast<uint32_t *>(misc + kOffBad), lane);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kBarScan));
            __syncwarp();
          }
          return true;
        };
        if (C::kEarly && n > 0 && !(ok = look())) break;
        if (more) {
          if (!(ok = wait(bar(kBarKFull + slot), par, kSiteK))) break;
          if (C::kEarly && n > 0 && !(ok = wait(bar(kBarSRead), (n - 1) & 1, kSiteSRead))) break;
          tc_fence_after();
          const uint64_t kd = sw128_desc(sbase + C::kOffK + slot * C::kTile, 16, 1024);
          if (lane == 0) {
#pragma unroll
            for (uint32_t ks = 0; ks < kDP / 16; ++ks)
              if (ks < dsteps) {
                const uint64_t o = (uint64_t)((ks >> 2) * (C::kAtom >> 4) + (ks & 3) * 2);
                umma(tmem, qd + o, kd + o, idesc_qk, ks > 0);
              }
            umma_commit(bar(kBarS));
            umma_commit(bar(kBarKEmpty + slot));
          }
          __syncwarp();
        }
        if (!C::kEarly && !(ok = look())) break;
        if (!C::kEarly || n > 0) {
          if (!(ok = wait(bar(kBarP), t & 1, kSiteP))) break;
          tc_fence_after();
          if (lane == 0) {
            // 16-key steps up to the sequence's end (the probabilities past it are zero).
            const uint32_t steps = (uint32_t)(keys + 15) / 16;
            const uint64_t vd = sw128_desc(sbase + C::kOffV + vslot * C::kTile, C::kAtom, 1024);
#pragma unroll
            for (uint32_t ks = 0; ks < 8; ++ks)
              if (ks < steps)
                umma_ts(tmem + kColO, tmem + C::kColP + ks * 8, vd + (uint64_t)(ks * (2048 >> 4)),
                        idesc_pv, t > 0 || ks > 0 || odd);
            umma_commit(bar(kBarVEmpty + vslot));
            if (C::kEarly) umma_commit(bar(kBarPV));
          }
          __syncwarp();
          if (C::kEarly && !more) break;
        }
        prev = i;
        i = next_tile(u, marks, i + 1);
        more = i < u.last;
      }
      if (lane == 0) {
        umma_commit(bar(kBarO));
        Gate::drain(bar(kBarO), 0);
      }
      __syncwarp();
    } else {
      const int r = (int)threadIdx.x;
      const uint32_t tS = tmem + ((uint32_t)(warp * 32) << 16), tO = tS + kColO, tP = tS + C::kColP;
      const int token = r / (int)p.pack, head = (int)u.head0 + r % (int)p.pack;
      const bool live = token < u.tokens;
      const bool busy = __any_sync(0xffffffffu, live);  // rows past the last token need nothing
      const Row row = make_row(p, u, token, live);
      const float scale2 = p.scale * kLog2e;
      // cap: c tanh(u) in log2 units, u = x cap_u.  Scores up to cap_near: x times a polynomial in x^2 (6
      // instructions, no special function), where its coefficients keep inside of fp32's range.
      // Beyond, for a cap up to 512, the hardware's form for the whole chunk: 2^-21 of the cap is
      // 2^-12 at most, beside P's 2^-9.  A larger cap takes each score by its own size.
      const float cap_u = kCap ? cap_factor(p.scale, p.softcap) : 0.f;
      const float cap2 = kCap ? p.softcap * kLog2e : 0.f;
      const float cap_near = cap_u > 5e-5f && cap_u < 3e4f ? kCapFit / cap_u : -1.f;
      CapPoly cap_x;
      if (kCap) cap_x.set(scale2, cap_u * cap_u);
      const float slope2 = kBias == kSlopes ? bias_log2(-p.slopes[head]) : 0.f;
      // Whether the whole table lies in shared memory, and at which pitch.
      const uint32_t table_pitch = bias_pitch(2 * ((uint32_t)p.reach + kKeys) + 1, p.pack);
      const bool near = kBias == kTable && p.reach <= (int)C::kBiases &&
                        p.pack * table_pitch <= C::kBiases;
      if (near) {  // laid out while the first tiles travel
        float *t = reinterpret_cast<float *>(misc + kOffBias);
        for (uint32_t h = 0; h < p.pack; ++h) {
          const float *from = p.table + (size_t)(u.head0 + h) * (2 * p.reach + 1);
          for (int x = (int)threadIdx.x; x <= 2 * (p.reach + kKeys); x += 128)
            t[h * table_pitch + x] = bias_log2(from[min(max(x - kKeys, 0), 2 * p.reach)]);
        }
        asm volatile("barrier.cta.sync 1, 128;" ::: "memory");  // the softmax warps
      }
      // Table: this warp's window, and this row's place in it (its distance to the tile's key 0).
      const uint32_t pitch = near ? table_pitch : window_pitch(p.pack);
      float *biases = reinterpret_cast<float *>(misc + kOffBias) + (near ? 0 : warp * kWindow);
      const int warp_token = warp * 32 / (int)p.pack, span = 127 + 32 / (int)p.pack;
      const float *bias_row = biases + (r % (int)p.pack) * pitch +
                              (near ? p.reach + kKeys
                                    : (32 / (int)p.pack - 1) - (token - warp_token));
      bool ok = true;
      uint32_t n = 0, scans = 0, hands = 0;
      int32_t *doc_s = reinterpret_cast<int32_t *>(misc + kOffDocs) + warp * kKeys;
      int32_t doc[4];  // documents of the next tile's keys, lane = key
      auto load_docs = [&](int i) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int j = key_tile(u, i) * kKeys + 32 * c + lane;
          doc[c] = i < u.last && j < u.s.nk ? p.k_docs[u.s.k_row + j] : -1;
        }
      };
      if (docs && busy) load_docs(first);
      for (int i = first, next; ok && i < u.last; i = next, ++n) {
        next = next_tile(u, marks, i + 1);
        const int k0 = key_tile(u, i) * kKeys;
        const bool whole = whole_tile(u, k0);
        if (docs && busy) {
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 4; ++c) doc_s[32 * c + lane] = doc[c];
          load_docs(next);
        }
        const float *bias = bias_row;
        if (near) {
          bias += min(max(k0 - row.pos, -(p.reach + kKeys)), p.reach + 1);
        } else if (kBias == kTable && busy) {
          const int d0 = k0 - row.pos + (token - warp_token) - (32 / (int)p.pack - 1);
          __syncwarp();
          for (int h = 0; h < (int)p.pack; ++h) {
            const float *t = p.table + (size_t)((int)u.head0 + h) * (2 * p.reach + 1) + p.reach;
            for (int x = lane; x < span; x += 32)
              biases[h * pitch + x] = bias_log2(__ldg(t + min(max(d0 + x, -p.reach), p.reach)));
          }
        }
        __syncwarp();
        if (!(ok = __all_sync(0xffffffffu, gate.wait(bar(kBarS), n & 1, kSiteS)))) break;
        tc_fence_after();
        // Walks the tile's four chunks of 32 keys.
        auto walk = [&](auto each) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t s[32];
            tmem_load(tS + 32 * c, s);
            each(c, s);
          }
        };
        float top = -INFINITY;
        uint32_t open = 0;  // bit c: a key of chunk c is open to a row of the warp
        if (busy)
          walk([&](int c, uint32_t(&s)[32]) {
            uint32_t mask = ~0u;
            bool full = true;  // every key of the chunk is open to every row of the warp
            if (!whole) {
              mask = row.bits(k0 + 32 * c);
              if (docs) mask &= doc_bits(doc_s[32 * c + lane], row.doc);
              if (!__any_sync(0xffffffffu, mask)) return;
              full = __all_sync(0xffffffffu, mask == ~0u);
            }
            open |= 1u << c;
            if (kCap) {
              float far = 0.f;
#pragma unroll
              for (int t = 0; t < 32; t += 2)
                far = fmaxf(fmaxf(far, fabsf(__uint_as_float(s[t]))),
                            fabsf(__uint_as_float(s[t + 1])));
              if (!__any_sync(0xffffffffu, far > cap_near)) {
#pragma unroll
                for (int t = 0; t < 32; ++t) {
                  const float x = __uint_as_float(s[t]);
                  s[t] = __float_as_uint(x * cap_x(x * x));
                }
              } else if (p.softcap <= 512.f) {
#pragma unroll
                for (int t = 0; t < 32; ++t)
                  s[t] = __float_as_uint(cap_exact(__uint_as_float(s[t]) * cap_u, cap2));
              } else {
#pragma unroll
                for (int t = 0; t < 32; ++t) {
                  const float x = __uint_as_float(s[t]);
                  s[t] = __float_as_uint(cap_scaled(x * scale2, x * cap_u, cap2));
                }
              }
            }
            if (kBias == kSlopes) {
              const float d0 = (float)(k0 + 32 * c - row.pos);
#pragma unroll
              for (int t = 0; t < 32; ++t) {
                const float z = __uint_as_float(s[t]);
                s[t] = __float_as_uint(fmaf(slope2, fabsf(d0 + (float)t), kCap ? z : z * scale2));
              }
            }
            if (kBias == kTable) {
#pragma unroll
              for (int t = 0; t < 32; ++t) {
                const float z = __uint_as_float(s[t]), b = bias[32 * c + t];
                s[t] = __float_as_uint(kCap ? z + b : fmaf(z, scale2, b));
              }
            }
            if (!full) {
#pragma unroll
              for (int t = 0; t < 32; ++t) s[t] = (mask >> t) & 1 ? s[t] : 0xff800000u;
            }
            float other = -INFINITY;
#pragma unroll
            for (int t = 0; t < 32; t += 4) {
              top = fmaxf(fmaxf(top, __uint_as_float(s[t])), __uint_as_float(s[t + 1]));
              other = fmaxf(fmaxf(other, __uint_as_float(s[t + 2])), __uint_as_float(s[t + 3]));
            }
            top = fmaxf(top, other);
            if (kCap || kBias || !whole) tmem_st32(tS + 32 * c, s);
          });
        if (kCap || kBias || !whole) tmem_st_wait();
        if (!kCap && !kBias) top *= scale2;
        if (C::kEarly && n > 0) {  // P and O are P.V's of the previous tile until it has run
          ok = __all_sync(0xffffffffu, gate.wait(bar(kBarPV), (n - 1) & 1, kSitePV));
          tc_fence_after();
        }
        const bool raise = top > m + kRescaleThreshold || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, raise)) {
          const float f = raise ? ex2(m - top) : 1.f;  // 0 where nothing was seen before
          if (raise) m = top;
          l *= f;
          if (n > 0) {
#pragma unroll 1
            for (uint32_t c = 0; c < kDP; c += 32) {
              uint32_t o[32];
              tmem_load(tO + c, o);
#pragma unroll
              for (int t = 0; t < 32; ++t) o[t] = __float_as_uint(__uint_as_float(o[t]) * f);
              tmem_st32(tO + c, o);
            }
          }
        }
        if (busy) {
          const float ref = m == -INFINITY ? 0.f : m;
          const float factor = kCap || kBias ? 1.f : scale2;
          float sum[2] = {0.f, 0.f};
          walk([&](int c, uint32_t(&s)[32]) {
            if (C::kEarly && c == 3) {  // the last of S is in registers
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(bar(kBarSRead));
              __syncwarp();  // together again before the warp-wide store below
            }
            uint32_t w[16];
            if ((open >> c) & 1) {
              // Plain fp32 operations: the packed pairs (f32x2) take 3.3 to 3.9 cycles each against
              // 0.9 to 1.4 of a single one, measured.
#pragma unroll
              for (int t = 0; t < 16; ++t) {
                const float a = ex2(fmaf(__uint_as_float(s[2 * t]), factor, -ref));
                const float b = ex2(fmaf(__uint_as_float(s[2 * t + 1]), factor, -ref));
                sum[0] += a;
                sum[1] += b;
                w[t] = pack_bf16x2(a, b);
              }
            } else {
#pragma unroll
              for (int t = 0; t < 16; ++t) w[t] = 0;
            }
            tmem_st16(tP + 16 * c, w);
          });
          l += sum[0] + sum[1];
        } else if (C::kEarly) {
          if (lane == 0) mbar_arrive(bar(kBarSRead));
          __syncwarp();
        }
        // Rows of V past the sequence's end inside the last 16-key step: zero probabilities, but
        // zero times whatever lies there need not be zero.
        const uint32_t slot = n % C::kSlots, tile_v = sbase + C::kOffV + slot * C::kTile;
        const int keys = min(u.s.nk - k0, kKeys), clear = (keys + 15) / 16 * 16;
        if (keys < clear) {
          ok = __all_sync(0xffffffffu, gate.wait(bar(kBarVFull + slot), (n / C::kSlots) & 1, kSiteVRead)) && ok;
          for (int x = keys * (kDP / 8) + r; x < clear * (kDP / 8); x += 128)
            st_shared_v4(tile_v + ((x % (kDP / 8)) >> 3) * C::kAtom + x / (kDP / 8) * 128 +
                             (x & 7) * 16,
                         0, 0, 0, 0);
          fence_proxy_async();
        }
        tmem_st_wait();
        if (!whole) {
          ok = __all_sync(0xffffffffu, gate.wait(bar(kBarScan), scans++ & 1, kSiteScan)) && ok;
          const volatile uint32_t *odd = reinterpret_cast<uint32_t *>(misc + kOffBad);
          if (ok && (odd[0] | odd[1] | odd[2] | odd[3]))
            ok = add_by_hand<kDP>(odd, tile_v, C::kAtom, tP, tO, n == 0, gate, bar(kBarHand),
                                  hands++);
        }
        tc_fence_before();
        mbar_arrive(bar(kBarP));
      }
      ok = __all_sync(0xffffffffu, gate.wait(bar(kBarO), 0, kSiteO)) && ok;
      tc_fence_after();
      if (ok) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const size_t orow = ((size_t)(u.s.q_row + u.t0 + token) * p.heads + head) * p.dim;
        float *part = p.splits > 1 ? p.part_o + (((size_t)u.slot * p.splits + u.split) * kRows + r) * p.part_dp
                                   : nullptr;
#pragma unroll 1
        for (uint32_t c = 0; c < kDP; c += 32) {
          if (c >= p.dim) break;
          uint32_t o[32];
          tmem_load(tO + c, o);
          const int cols = min(32, (int)(p.dim - c));
          if (!part) {
#pragma unroll
            for (int t = 0; t < 32; ++t)  // a row that saw no key is zeros
              o[t] = l == 0.f ? 0u : __float_as_uint(__uint_as_float(o[t]) * inv);
          }
          if (!live) {
          } else if (part) {
#pragma unroll
            for (int t = 0; t < 8; ++t)
              if (4 * t < cols)
                *reinterpret_cast<uint4 *>(part + c + 4 * t) =
                    make_uint4(o[4 * t], o[4 * t + 1], o[4 * t + 2], o[4 * t + 3]);
          } else if (p.out_dtype == 1) {
            uint16_t *out = static_cast<uint16_t *>(p.out) + orow + c;
#pragma unroll
            for (int t = 0; t < 4; ++t)
              if (8 * t < cols)
                *reinterpret_cast<uint4 *>(out + 8 * t) = make_uint4(
                    pack_bf16x2(__uint_as_float(o[8 * t]), __uint_as_float(o[8 * t + 1])),
                    pack_bf16x2(__uint_as_float(o[8 * t + 2]), __uint_as_float(o[8 * t + 3])),
                    pack_bf16x2(__uint_as_float(o[8 * t + 4]), __uint_as_float(o[8 * t + 5])),
                    pack_bf16x2(__uint_as_float(o[8 * t + 6]), __uint_as_float(o[8 * t + 7])));
          } else {
            float *out = static_cast<float *>(p.out) + orow + c;
#pragma unroll
            for (int t = 0; t < 8; ++t)
              if (4 * t < cols)
                *reinterpret_cast<uint4 *>(out + 4 * t) =
                    make_uint4(o[4 * t], o[4 * t + 1], o[4 * t + 2], o[4 * t + 3]);
          }
          __syncwarp();
        }
      }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  }
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kTmemCols)
                 : "memory");
  if (p.splits > 1) {
    const int r = (int)threadIdx.x;
    if (r < u.tokens * (int)p.pack)
      p.part_ml[((size_t)u.slot * p.splits + u.split) * kRows + r] = make_float2(m, l);
    if (arrive_last(p, u, reinterpret_cast<uint32_t *>(misc + kOffFlag))) {
      join_parts<kRows>(p, u, 1.f);
      zero_padding(p, u);
    }
  } else {
    if (!work) {  // no key is open to any row of the tile
      Unit all = u;
      all.tokens = 0;
      zero_padding(p, all);
    } else {
      zero_padding(p, u);
    }
  }
}

}  // namespace scored_tc

namespace {

PFN_cuTensorMapEncodeTiled_v12000 scored_encode_fn() {
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

// [rows, heads, dim] bf16 with element strides; a box is 64 columns (zeros past dim) of
// `box_heads` heads of `box_rows` rows, in the 128-byte swizzle.
bool scored_map(CUtensorMap *map, const void *base, uint32_t rows, uint32_t heads, uint32_t dim,
                uint64_t row, uint64_t head, uint32_t box_heads, uint32_t box_rows) {
  auto fn = scored_encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {dim, heads, rows};
  cuuint64_t strides[2] = {head * 2, row * 2};
  cuuint32_t box[3] = {64, box_heads, box_rows};
  cuuint32_t elem[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims, strides, box,
            elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int kDP, bool kCap, int kBias>
cudaError_t scored_launch(const ScoredProblem &p, const CUtensorMap (&m)[3], cudaStream_t stream) {
  constexpr uint32_t smem = scored_tc::Cfg<kDP>::kSmemBytes;
  auto kernel = scored_tc::scored_tc_kernel<kDP, kCap, kBias>;
  static std::atomic<uint64_t> seen{0};
  cudaError_t e = allow_smem((const void *)kernel, (int)smem, seen);
  if (e != cudaSuccess) return e;
  const uint32_t grid = p.tiles * p.nseq * (p.heads / p.pack) * p.splits;
  kernel<<<grid, scored_tc::kThreads, smem, stream>>>(m[0], m[1], m[2], p);
  return cudaGetLastError();
}

template <int kDP>
cudaError_t scored_rule(const ScoredProblem &p, const CUtensorMap (&m)[3], cudaStream_t stream) {
  if (p.table)
    return p.softcap > 0.f ? scored_launch<kDP, true, 2>(p, m, stream)
                           : scored_launch<kDP, false, 2>(p, m, stream);
  if (p.slopes)
    return p.softcap > 0.f ? scored_launch<kDP, true, 1>(p, m, stream)
                           : scored_launch<kDP, false, 1>(p, m, stream);
  return p.softcap > 0.f ? scored_launch<kDP, true, 0>(p, m, stream)
                         : scored_launch<kDP, false, 0>(p, m, stream);
}

}  // namespace

bool scored_tc_supported(const ScoredProblem &p) {
  auto ok = [](const void *x, uint64_t row, uint64_t head) {
    return (uintptr_t)x % 16 == 0 && row % 8 == 0 && head % 8 == 0 && row < (1ull << 38) &&
           head < (1ull << 38) && row && head;
  };
  return p.in_dtype == TX_BF16 && p.dim % 8 == 0 && p.dim <= 128 && p.scale > 0.f &&
         ok(p.q, p.q_row, p.q_head) && ok(p.k, p.k_row, p.k_head) && ok(p.v, p.v_row, p.v_head) &&
         (uintptr_t)p.out % 16 == 0;
}

cudaError_t launch_scored_tc(const ScoredProblem &p, cudaStream_t stream) {
  CUtensorMap m[3];
  if (!scored_map(&m[0], p.q, p.rows_q, p.heads, p.dim, p.q_row, p.q_head, p.pack,
                  scored_tc::kRows / p.pack) ||
      !scored_map(&m[1], p.k, p.rows_k, p.kv_heads, p.dim, p.k_row, p.k_head, 1, scored::kKeys) ||
      !scored_map(&m[2], p.v, p.rows_k, p.kv_heads, p.dim, p.v_row, p.v_head, 1, scored::kKeys))
    return cudaErrorInvalidValue;
  return p.dim <= 64 ? scored_rule<64>(p, m, stream) : scored_rule<128>(p, m, stream);
}

// Few rows: up to 8 per kv head for head_dim up to 64 or with a cap, and up to 16 where the
// tensor-memory kernel does not take the call.  Few-rows against tensor-memory kernel, one token of
// 8 texts over 2048 keys: 27 / 28 us at 12 heads of 64, 27 / 34 us with a cap; of 32 texts over 1024
// keys 39 / 46 us.  8 heads of 128, 2 rows each: 29 / 28 us, with a cap 29 / 30 us; 16 rows: 35 / 30
// and 35 / 34 us.  fp32, 16 rows of 128 over 2048 keys: 68 us against 146 in the 64-row kernel.
ScoredRoute scored_route(const ScoredProblem &p) {
  const bool tc = p.rows_k && scored_tc_supported(p), few = p.rows_k && scored_few_supported(p);
  const uint64_t rows = (uint64_t)p.max_q * (p.heads / p.kv_heads);
  if (few && (!tc || (rows <= 8 && (p.dim <= 64 || p.softcap > 0.f)))) return kScoredFew;
  return tc ? kScoredTc : kScoredF32;
}

// The cut of a launch.  Rows: the heads of a pack times tokens (few rows: all heads of a kv head,
// whatever their number).  Splits of the key range: as many as the CTAs that run at once leave
// room for, while a part keeps a few key blocks.
void scored_plan(ScoredProblem *p, ScoredRoute route, int num_sms) {
  const uint32_t group = p->heads / p->kv_heads;
  uint32_t slots = 2 * (uint32_t)num_sms, least = 2 * scored::kKeys;  // CTAs at once, keys a part
  if (route == kScoredFew) {
    p->rows = 16;
    p->pack = group;
    least = 128;
    slots = (uint32_t)(scored_few_resident(*p) * num_sms);
  } else {
    p->rows = route == kScoredTc ? 128 : 64;
    p->pack = group & (0u - group);
    if (p->pack > p->rows) p->pack = p->rows;
    if (route == kScoredTc && p->table && p->pack > scored::kTablePack) p->pack = scored::kTablePack;
  }
  const uint32_t per = p->rows / p->pack;
  p->tiles = (p->max_q + per - 1) / per;
  const uint64_t units = (uint64_t)p->tiles * p->nseq * (p->heads / p->pack);
  const uint64_t fit = slots / units, parts = (p->max_k + least - 1) / least;
  p->splits = (uint32_t)(fit < parts ? fit : parts);
  if (!p->splits) p->splits = 1;
  if (route == kScoredFew) {
    // Where that leaves many CTAs' places empty: waves of CTAs times the keys of one and what its
    // start and the join cost, taken as 512 keys.  11 texts of 1428 to 6289 keys, 32 / 8 heads of
    // 128 in fp32, 88 units on 148 places: 405 us with one part, 249 us with three.
    auto cost = [&](uint64_t n) {
      return (units * n + slots - 1) / slots * (p->max_k / n + 512);
    };
    for (uint64_t n = p->splits + 1; n <= parts && n <= 4 * (fit + 1); ++n)
      if (cost(n) < cost(p->splits)) p->splits = (uint32_t)n;
  }
  p->part_dp = (p->dim + 3) & ~3u;
}

}  // namespace tx
