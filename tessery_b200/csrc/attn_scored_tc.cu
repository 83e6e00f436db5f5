// Attention under a score rule on the tensor cores: bf16 q, k, v, head_dim a multiple of 8 up
// to 128 (tx_attention_scored).
//
//   z_ij = scale q_i.k_j;  cap: z = c tanh(z / c);  distance bias: z += b_h(j - pos_i)
//   out_i = sum_j softmax_j(z_ij) v_j over the keys the rule leaves open to row i
//
// One CTA takes 128 rows (query tokens x the heads that share a kv head, attn_scored.cuh) and
// walks the 128-key tiles that some row may see.  S = Q K^T and O += P V are tcgen05.mma
// (M = 128) into tensor memory; thread t of the four softmax warps owns row t (tensor-memory
// lane t): it reads S, applies cap, bias and mask, and writes P = exp2(z - m) as bf16 over S,
// which is the A operand of P.V.  The reference m follows the row's running maximum lazily: O
// and the row sum are rescaled only when a tile's maximum exceeds it by more than 2^8, which
// changes no result (P stays below 2^8 and the sum uses the same reference).  Two CTAs share an
// SM, so one's products run beside the other's softmax.
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
constexpr uint32_t kTmemCols = 256;  // S (128, P over it), O (head_dim); two CTAs per SM
constexpr uint32_t kColO = 128;
constexpr float kRescaleThreshold = 8.0f;  // log2 units
constexpr float kLog2e = 1.44269504088896341f;

template <int kDP>  // head_dim rounded up to whole 64-column (128-byte) blocks
struct Cfg {
  static constexpr uint32_t kTile = 128 * kDP * 2;  // a tile of Q, K or V
  static constexpr uint32_t kAtom = 128 * 128;      // 128 rows x 64 columns, swizzled
  static constexpr int kSlots = kDP == 64 ? 2 : 1;  // K slots, and V slots
  static constexpr uint32_t kOffQ = 0, kOffK = kTile, kOffV = kOffK + kSlots * kTile;
  static constexpr uint32_t kOffMisc = kOffV + kSlots * kTile;
  static constexpr uint32_t kMiscBytes = 256 + kDocWords * 4 + 4 * kKeys * 4;
  static constexpr uint32_t kSmemBytes = kOffMisc + kMiscBytes;
  static_assert(2 * (kSmemBytes + 1024) <= 233472, "two CTAs per SM");
};

// Barriers at the start of the misc area.
enum : uint32_t {
  kBarQ = 0, kBarKFull = 1, kBarKEmpty = 3, kBarVFull = 5, kBarVEmpty = 7, kBarS = 9, kBarP = 10,
  kBarO = 11, kBarScan = 12, kBarHand = 13, kNumBars = 14
};
enum : uint32_t { kOffTmem = 128, kOffAbort = 132, kOffFlag = 136, kOffRange = 144,
                  kOffBad = 160, kOffWords = 256 };
enum : int { kSiteK = 1, kSiteV = 2, kSiteKFree = 3, kSiteVFree = 4, kSiteS = 5, kSiteP = 6,
             kSiteO = 7, kSiteQ = 8, kSiteVRead = 9, kSiteScan = 10, kSiteHand = 11 };

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

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
// softmax warps), then zeroed.  `fresh`: O holds nothing yet.
template <int kDP>
__device__ __noinline__ void add_by_hand(const volatile uint32_t *bad, uint32_t tile,
                                         uint32_t atom, uint32_t tS, uint32_t tO, bool fresh,
                                         int r, const Gate &gate, uint32_t done, uint32_t turn) {
  for (int j = 0; j < kKeys; ++j) {
    if (!((bad[j >> 5] >> (j & 31)) & 1)) continue;
    uint32_t w;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(w) : "r"(tS + j / 2));
    tmem_ld_wait();
    const float pj = j & 1 ? bf16_hi(w) : bf16_lo(w);
    for (uint32_t c = 0; c < kDP; c += 32) {
      uint32_t o[32];
      tmem_ld32(tO + c, o);
      tmem_ld_wait();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
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
      tmem_st32(tO + c, o);
    }
    tmem_st_wait();
    fresh = false;
  }
  mbar_arrive(done);  // every thread has read the rows
  if (!__all_sync(0xffffffffu, gate.wait(done, turn & 1, kSiteHand))) return;
  for (int x = r; x < kKeys * (kDP / 8); x += 128) {
    const int row = x / (kDP / 8), ch = x % (kDP / 8);
    if ((bad[row >> 5] >> (row & 31)) & 1)
      st_shared_v4(tile + (ch >> 3) * atom + row * 128 + (ch & 7) * 16, 0, 0, 0, 0);
  }
  fence_proxy_async();
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
  int32_t *doc_s = reinterpret_cast<int32_t *>(misc + kOffWords + kDocWords * 4);
  const Unit u = make_unit<kRows>(p, blockIdx.x);
  if (!u.present) return;  // whole units: every split of one takes the same way
  const bool docs = p.q_docs != nullptr;
  if (docs) mark_tiles(p, u, words, reinterpret_cast<int *>(misc + kOffRange));
  const uint32_t *marks = docs ? words : nullptr;
  const int first = next_tile(u, marks, u.first);
  const bool work = u.tokens > 0 && first < u.last;

  float m = -INFINITY, l = 0.f;  // softmax threads: the row's reference and sum
  if (work) {
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
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<uint32_t *>(misc + kOffTmem);

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
      bool ok = wait(bar(kBarQ), 0, kSiteQ);
      uint32_t n = 0;
      for (int i = first; ok && i < u.last; i = next_tile(u, marks, i + 1), ++n) {
        const uint32_t slot = n % C::kSlots, par = (n / C::kSlots) & 1;
        const int k0 = key_tile(u, i) * kKeys, keys = min(u.s.nk - k0, kKeys);
        if (!(ok = wait(bar(kBarKFull + slot), par, kSiteK))) break;
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
        if (!(ok = wait(bar(kBarVFull + slot), par, kSiteV))) break;
        bool odd = false;
        if (!whole_tile(p, u, k0)) {
          odd = scan_values<C::kTile>(sbase + C::kOffV + slot * C::kTile, keys,
                                      reinterpret_cast<uint32_t *>(misc + kOffBad), lane);
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(kBarScan));
        }
        if (!(ok = wait(bar(kBarP), n & 1, kSiteP))) break;
        tc_fence_after();
        if (lane == 0) {
          // 16-key steps up to the sequence's end (the probabilities past it are zero).
          const uint32_t steps = (uint32_t)(keys + 15) / 16;
          const uint64_t vd = sw128_desc(sbase + C::kOffV + slot * C::kTile, C::kAtom, 1024);
#pragma unroll
          for (uint32_t ks = 0; ks < 8; ++ks)
            if (ks < steps)
              umma_ts(tmem + kColO, tmem + ks * 8, vd + (uint64_t)(ks * (2048 >> 4)), idesc_pv,
                      n > 0 || ks > 0 || odd);
          umma_commit(bar(kBarVEmpty + slot));
        }
        __syncwarp();
      }
      if (lane == 0) {
        umma_commit(bar(kBarO));
        Gate::drain(bar(kBarO), 0);
      }
      __syncwarp();
    } else {
      const int r = warp * 32 + lane;
      const uint32_t tS = tmem + ((uint32_t)(warp * 32) << 16), tO = tS + kColO;
      const int token = r / (int)p.pack, head = (int)u.head0 + r % (int)p.pack;
      const bool live = token < u.tokens;
      const Row row = make_row(p, u, token, live);
      const float scale2 = p.scale * kLog2e;
      // cap: c2 tanh(s scale / cap) = c2 - 2 c2 / (1 + 2^(a s))
      const float c2 = kCap ? p.softcap * kLog2e : 0.f;
      const float cap_a = kCap ? 2.f * scale2 / p.softcap : 0.f;
      const float slope2 = kBias == kSlopes ? -p.slopes[head] * kLog2e : 0.f;
      const float *table =
          kBias == kTable ? p.table + (size_t)head * (2 * p.reach + 1) + p.reach : nullptr;
      auto capped = [&](float s) {
        return kCap ? fmaf(-2.f * c2, rcp(1.f + ex2(s * cap_a)), c2) : s * scale2;
      };
      // The score of key j in log2 units.  A finite bias too large for them stays finite.
      auto score = [&](float s, int j) {
        float z = capped(s);
        if (kBias == kSlopes) z = fmaf(slope2, fabsf((float)(j - row.pos)), z);
        if (kBias == kTable) {
          const float b = __ldg(table + min(max(j - row.pos, -p.reach), p.reach));
          z = b == -INFINITY ? b : fmaxf(fmaf(b, kLog2e, z), -3.402823466e38f);
        }
        return z;
      };
      bool ok = true;
      uint32_t n = 0, scans = 0, hands = 0;
      for (int i = first; ok && i < u.last; i = next_tile(u, marks, i + 1), ++n) {
        const int k0 = key_tile(u, i) * kKeys;
        if (docs) {  // this tile's documents, a copy per warp
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int j = k0 + 32 * c + lane;
            doc_s[warp * kKeys + 32 * c + lane] = j < u.s.nk ? p.k_docs[u.s.k_row + j] : -1;
          }
          __syncwarp();
        }
        uint32_t mask[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mask[c] = row.bits(k0 + 32 * c);
          if (docs) {
            uint32_t same = 0;
#pragma unroll
            for (int t = 0; t < 32; ++t)
              same |= (doc_s[warp * kKeys + c * 32 + t] == row.doc ? 1u : 0u) << t;
            mask[c] &= same;
          }
        }
        if (!(ok = __all_sync(0xffffffffu, gate.wait(bar(kBarS), n & 1, kSiteS)))) break;
        tc_fence_after();
        // First pass: the row's maximum; scores with a bias go back finished.
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (!__any_sync(0xffffffffu, mask[c])) continue;
          uint32_t s[32];
          tmem_ld32(tS + 32 * c, s);
          tmem_ld_wait();
#pragma unroll
          for (int t = 0; t < 32; ++t) {
            float z = __uint_as_float(s[t]);
            if (kBias) z = score(z, k0 + 32 * c + t);
            z = (mask[c] >> t) & 1 ? z : -INFINITY;
            top = fmaxf(top, z);
            if (kBias) s[t] = __float_as_uint(z);
          }
          if (kBias) tmem_st32(tS + 32 * c, s);
        }
        if (kBias) tmem_st_wait();
        if (!kBias && top != -INFINITY) top = capped(top);  // increasing in the raw score
        const bool raise = top > m + kRescaleThreshold || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, raise)) {
          const float f = raise ? ex2(m - top) : 1.f;  // 0 where nothing was seen before
          if (raise) m = top;
          l *= f;
          if (n > 0) {
#pragma unroll
            for (int c = 0; c < kDP / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(tO + 32 * c, o);
              tmem_ld_wait();
#pragma unroll
              for (int t = 0; t < 32; ++t) o[t] = __float_as_uint(__uint_as_float(o[t]) * f);
              tmem_st32(tO + 32 * c, o);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t w[16];
          if (!__any_sync(0xffffffffu, mask[c])) {
#pragma unroll
            for (int t = 0; t < 16; ++t) w[t] = 0;
          } else {
            uint32_t s[32];
            tmem_ld32(tS + 32 * c, s);
            tmem_ld_wait();
            float sum = 0.f;
#pragma unroll
            for (int t = 0; t < 32; ++t) {
              float z = __uint_as_float(s[t]);
              float e = kBias ? ex2(z - ref) : kCap ? ex2(capped(z) - ref) : ex2(fmaf(z, scale2, -ref));
              if (!kBias) e = (mask[c] >> t) & 1 ? e : 0.f;
              sum += e;
              s[t] = __float_as_uint(e);
            }
            l += sum;
#pragma unroll
            for (int t = 0; t < 16; ++t)
              w[t] = pack_bf16x2(__uint_as_float(s[2 * t]), __uint_as_float(s[2 * t + 1]));
          }
          tmem_st16(tS + 16 * c, w);
        }
        // Rows of V past the sequence's end inside the last 16-key step: zero probabilities, but
        // zero times whatever lies there need not be zero.
        const int keys = min(u.s.nk - k0, kKeys), clear = (keys + 15) / 16 * 16;
        if (keys < clear) {
          const uint32_t slot = n % C::kSlots;
          ok = __all_sync(0xffffffffu, gate.wait(bar(kBarVFull + slot), (n / C::kSlots) & 1, kSiteVRead));
          for (int x = keys * (kDP / 8) + r; x < clear * (kDP / 8); x += 128) {
            const int vr = x / (kDP / 8), ch = x % (kDP / 8);
            st_shared_v4(sbase + C::kOffV + slot * C::kTile + (ch >> 3) * C::kAtom + vr * 128 +
                             (ch & 7) * 16,
                         0, 0, 0, 0);
          }
          fence_proxy_async();
        }
        tmem_st_wait();
        if (!whole_tile(p, u, k0)) {
          ok = __all_sync(0xffffffffu, gate.wait(bar(kBarScan), scans++ & 1, kSiteScan)) && ok;
          const volatile uint32_t *bad = reinterpret_cast<uint32_t *>(misc + kOffBad);
          if (ok && (bad[0] | bad[1] | bad[2] | bad[3]))
            add_by_hand<kDP>(bad, sbase + C::kOffV + (n % C::kSlots) * C::kTile, C::kAtom, tS, tO,
                             n == 0, r, gate, bar(kBarHand), hands++);
        }
        tc_fence_before();
        mbar_arrive(bar(kBarP));
      }
      ok = __all_sync(0xffffffffu, ok && gate.wait(bar(kBarO), 0, kSiteO));
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
          tmem_ld32(tO + c, o);
          tmem_ld_wait();
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
    if (warp == kMmaWarp)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                   "r"(kTmemCols)
                   : "memory");
  }
  if (p.splits > 1) {
    const int r = (int)threadIdx.x;
    if (r < u.tokens * (int)p.pack)
      p.part_ml[((size_t)u.slot * p.splits + u.split) * kRows + r] = make_float2(m, l);
    if (arrive_last(p, u, reinterpret_cast<uint32_t *>(misc + kOffFlag))) {
      join_parts<kRows>(p, u);
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
  cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
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

// The cut of a launch.  Rows: the heads of a pack times tokens.  Splits of the key range: while
// the units do not fill two CTAs per SM and a part would still hold two key tiles.
void scored_plan(ScoredProblem *p, bool tc, int num_sms) {
  const uint32_t group = p->heads / p->kv_heads;
  p->rows = tc ? 128 : 64;
  p->pack = group & (0u - group);
  if (p->pack > p->rows) p->pack = p->rows;
  const uint32_t per = p->rows / p->pack;
  p->tiles = (p->max_q + per - 1) / per;
  const uint64_t units = (uint64_t)p->tiles * p->nseq * (p->heads / p->pack);
  const uint64_t want = (2ull * (uint64_t)num_sms + units - 1) / units;
  const uint64_t parts = (p->max_k + 2 * scored::kKeys - 1) / (2 * scored::kKeys);
  p->splits = units >= 2ull * (uint64_t)num_sms ? 1u : (uint32_t)(want < parts ? want : parts);
  if (!p->splits) p->splits = 1;
  p->part_dp = (p->dim + 3) & ~3u;
}

}  // namespace tx
