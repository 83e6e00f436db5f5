// Attention under a score rule for few query rows: at most 16 (query tokens x heads) per kv head,
// such as one new token of each text against the keys kept for it (tx_attention_scored; the
// formula is in attn_scored_tc.cu).
//
// Bound: HBM, every key and value row once.  A warp takes 16 keys at a time, in a ring of three
// stages of its own that cp.async fills, so nothing but the ring's arrival holds it up; the four
// warps of a CTA and the CTAs of a split key range are joined at the end (in this order, so the
// result is the same every time).  Both products run on mma.sync with the rows as M: bf16 on
// m16n8k16, the probabilities as two bf16 parts (hi + lo, error 2^-17); fp32 on m16n8k8 TF32 with
// split operands (hi + lo, three products, error 2^-22).  The 64-row fp32 kernel would compute 64
// rows for these (when this one takes which call: scored_route in attn_scored_tc.cu).
//
// Measured: 8 new tokens, 16 query and 8 kv heads of 128, a cap, 64 to 2048 keys each: 22.6 us
// between events; in a graph, from warm caches, 6.9 us with 16 keys each, 14.4 with 256 (start-up,
// split and join) and 24.4 with 2048.  32 texts of 1024 keys, 12 heads of 64 (101 MB): 37 us,
// 2.7 TB/s.  11 texts of 1428 to 6289 keys, 32 / 8 heads of 128 in fp32 (392 MB): 204 us, bound by the
// split operands' products.
#include <cuda_runtime.h>

#include <type_traits>

#include "../../include/tessattn.h"
#include "attn_scored.cuh"
#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace tx {
namespace scored_few {

using namespace scored;
using ptx::ex2;
using ptx::ld_shared_v4;

constexpr int kRows = 16, kBlock = 16, kStages = 3;
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kRescaleThreshold = 5.5f;  // e^5.5 = 2^7.9

template <typename T, int kDP>
struct Cfg {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kRowBytes = kDP * (int)sizeof(T);
  static constexpr int kChunks = kRowBytes / 16;  // 16-byte pieces of a row
  static constexpr int kStageBytes = kBlock * 2 * kRowBytes;
  static constexpr int kWarps = kStageBytes * kStages * 4 <= 224 * 1024 ? 4 : 2;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kQP = kDP + 8;             // query rows, read by 8 bytes
  static constexpr int kOffQ = kWarps * kStages * kStageBytes;
  static constexpr int kSmemBytes = kOffQ + kRows * kQP * (int)sizeof(T) + 64;
  // Where piece c of key or value row r lies.  K is read 16 bytes per lane by 8 rows x 4 lanes, V 4
  // bytes by 4 pairs of rows x 8 lanes; with these exchanges neither meets a bank twice (V rows of
  // 64 bytes: twice).
  static __device__ __forceinline__ int k_at(int r, int c) {
    return r * kRowBytes + (c ^ (kChunks >= 8 ? (r & 1) << 2 : 0)) * 16;
  }
  static __device__ __forceinline__ int v_at(int r, int c) {
    return r * kRowBytes + (c ^ ((((r >> 1) & 3) << 1) & (kChunks - 1))) * 16;
  }
  // CTAs that run at once on an SM, as far as shared memory says.
  static constexpr int kResident = 233472 / (kSmemBytes + 1024) < 4 ? 233472 / (kSmemBytes + 1024) : 4;
  // The ring's memory holds the warps' results at the end.
  static_assert(kWarps * (kRows * kDP * 4 + kRows * 8) <= kOffQ, "join area");
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(real ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t round_tf32(float x) { return __float_as_uint(x) + 0x1000u; }
__device__ __forceinline__ void split(float x, uint32_t &hi, uint32_t &lo) {
  hi = round_tf32(x) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
// c += a b for fp32 operands given as raw bits, through their splits.  Added to c in fp32: the
// tensor core cuts bits off at each of its own additions, always towards zero (8 heads of 128 on one
// kv head, up to 774 keys: off by 9e-7 that way and 1.9e-7 this way, for 18.5 and 20.5 us).
__device__ __forceinline__ void mma_split(float (&c)[4], const uint32_t (&ah)[4],
                                          const uint32_t (&al)[4], float b0, float b1) {
  uint32_t h0, l0, h1, l1;
  split(b0, h0, l0);
  split(b1, h1, l1);
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  mma(sum, al, h0, h1);
  mma(sum, ah, l0, l1);
  mma(sum, ah, h0, h1);
#pragma unroll
  for (int e = 0; e < 4; ++e) c[e] += sum[e];
}
// Whether a word of values is safe in the products: finite, and in fp32 below 2^127, so that the upper
// part of the split is finite too.
__device__ __forceinline__ bool finite_word(uint32_t w, bool f32) {
  if (f32) return (w & 0x7fffffffu) < 0x7f000000u;
  return (w & 0x7f80u) != 0x7f80u && (w & 0x7f800000u) != 0x7f800000u;
}

template <typename T, int kDP>
__global__ void __launch_bounds__(Cfg<T, kDP>::kThreads, Cfg<T, kDP>::kResident)
    scored_few_kernel(const __grid_constant__ ScoredProblem p) {
  using C = Cfg<T, kDP>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = ptx::smem_addr(smem) + warp * kStages * C::kStageBytes;
  T *qs = reinterpret_cast<T *>(smem + C::kOffQ);
  uint32_t *flag = reinterpret_cast<uint32_t *>(smem + C::kOffQ + kRows * C::kQP * (int)sizeof(T));
  const Unit u = make_unit<kRows, kBlock>(p, blockIdx.x);
  if (!u.present) return;
  const int pack = (int)p.pack, rows = u.tokens * pack;

  // Warp w takes blocks first + w, first + w + kWarps, ...
  const T *kp = static_cast<const T *>(p.k) + (size_t)u.kv * p.k_head;
  const T *vp = static_cast<const T *>(p.v) + (size_t)u.kv * p.v_head;
  // Piece x = lane + 32 i of a block: its row and column, the same columns for every i.
  constexpr int kRowsAStep = 32 / C::kChunks > 0 ? 32 / C::kChunks : 1;
  static_assert(C::kChunks <= 32 ? 32 % C::kChunks == 0 : C::kChunks % 32 == 0, "pieces of a row");
  auto fetch = [&](int i, int stage) {
    if (i < u.last) {
      const int k0 = (i < u.a ? i : i - u.a + u.b) * kBlock;
      const uint32_t kd = ring + stage * C::kStageBytes, vd = kd + kBlock * C::kRowBytes;
      if constexpr (C::kChunks <= 32) {
        const int c = lane % C::kChunks, e = c * (16 / (int)sizeof(T)), r0 = lane / C::kChunks;
        const bool in = e < (int)p.dim;
        const size_t at = (size_t)(u.s.k_row + k0 + r0);
        const T *ks = kp + at * p.k_row + e, *vs = vp + at * p.v_row + e;
#pragma unroll
        for (int r = r0, n = 0; n < kBlock / kRowsAStep; ++n, r += kRowsAStep) {
          const bool real = in && k0 + r < u.s.nk;
          cp_async16(kd + C::k_at(r, c), real ? ks : kp, real);
          cp_async16(vd + C::v_at(r, c), real ? vs : vp, real);
          ks += kRowsAStep * p.k_row;
          vs += kRowsAStep * p.v_row;
        }
      } else {
#pragma unroll 4
        for (int x = lane; x < kBlock * C::kChunks; x += 32) {
          const int r = x / C::kChunks, c = x % C::kChunks, e = c * (16 / (int)sizeof(T));
          const bool real = k0 + r < u.s.nk && e < (int)p.dim;
          const size_t at = (size_t)(u.s.k_row + k0 + r);
          cp_async16(kd + C::k_at(r, c), real ? kp + at * p.k_row + e : kp, real);
          cp_async16(vd + C::v_at(r, c), real ? vp + at * p.v_row + e : vp, real);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int ahead = u.first + warp;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s, ahead += C::kWarps) fetch(ahead, s);
  // Query rows, behind the first key blocks; a batch of loads in flight at a time.
  constexpr int kBatch = 16;
  for (int i0 = threadIdx.x; i0 < kRows * kDP; i0 += C::kThreads * kBatch) {
    T v[kBatch];
#pragma unroll
    for (int x = 0; x < kBatch; ++x) {
      const int i = i0 + x * C::kThreads, r = i / kDP, c = i % kDP;
      v[x] = 0;
      if (r < rows && c < (int)p.dim)
        v[x] = static_cast<const T *>(p.q)[(size_t)(u.s.q_row + u.t0 + r / pack) * p.q_row +
                                           (size_t)(u.head0 + r % pack) * p.q_head + c];
    }
#pragma unroll
    for (int x = 0; x < kBatch; ++x) {
      const int i = i0 + x * C::kThreads;
      if (i < kRows * kDP) qs[i / kDP * C::kQP + i % kDP] = v[x];
    }
  }
  __syncthreads();
  // bf16: the query rows as they enter the product, in registers (head_dim 256: read each time).
  constexpr bool kQRegs = !C::kF32 && kDP <= 128;
  uint32_t qa[kQRegs ? C::kChunks / 2 : 1][4];
  auto q_words = [&](int q, int j, uint32_t(&a)[4]) {  // step j of piece group q
    const int c = (4 * q + t) * 8 + 4 * j;
    const uint2 x = *reinterpret_cast<const uint2 *>(qs + g * C::kQP + c);
    const uint2 y = *reinterpret_cast<const uint2 *>(qs + (g + 8) * C::kQP + c);
    a[0] = x.x; a[1] = y.x; a[2] = x.y; a[3] = y.y;
  };
  if constexpr (kQRegs) {
#pragma unroll
    for (int i = 0; i < C::kChunks / 2; ++i) q_words(i / 2, i % 2, qa[i]);
  }

  Row row[2];
  const float *table[2];
  float slope[2], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = g + 8 * h, head = (int)u.head0 + r % pack;
    row[h] = make_row(p, u, r / pack, r < rows);
    table[h] = p.table ? p.table + (size_t)head * (2 * p.reach + 1) + p.reach : nullptr;
    slope[h] = p.slopes ? p.slopes[head] : 0.f;
  }
  const float cap_u = cap_factor(1.f, p.softcap);
  CapPoly cap_fit;
  cap_fit.set(1.f, 1.f);
  float o[kDP / 8][4];

  // Values that are not finite.  A key closed to a row has p = 0 there, and the product would turn
  // 0 * Inf or 0 * NaN into NaN; and a part of an operand times Inf need not be what the whole gives
  // (a lo part is 0 or below it as often as above).  So a warp whose sums come out not finite (rare)
  // walks its keys once more, carefully: with weights of at most 1, with NaN scores taken again
  // whole (fp32), and with the value rows that hold such a value added by hand where p > 0 and
  // zeroed before the product.  The first walk holds nothing of this: with values looked over in
  // every block with a closed key 11 texts in fp32 (above) took 251 us, and with the second walk a
  // flag of one loop 8 new tokens with a cap 24.6.
  auto walk = [&](auto how) {
    constexpr bool careful = decltype(how)::value;
#pragma unroll
    for (int h = 0; h < 2; ++h) m[h] = -INFINITY, l[h] = 0.f;
#pragma unroll
    for (int n = 0; n < kDP / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
    int stage = 0;
    for (int i = u.first + warp; i < u.last; i += C::kWarps) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncwarp();  // every lane's pieces are there, and the stage to fill has been read
      fetch(ahead, (stage + kStages - 1) % kStages);
      ahead += C::kWarps;
      const uint32_t ks = ring + stage * C::kStageBytes, vs = ks + kBlock * C::kRowBytes;
      stage = (stage + 1) % kStages;
      const int k0 = (i < u.a ? i : i - u.a + u.b) * kBlock;

      // S = Q K^T; a 16-byte piece of a key row is lane t's share of two steps (of 16 columns in
      // bf16, 8 in fp32), in the order in which it lies: the query rows are read alike.
      float s[2][4] = {};
#pragma unroll
      for (int q = 0; q < C::kChunks / 4; ++q) {
        uint4 kw[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) kw[n] = ld_shared_v4(ks + C::k_at(8 * n + g, 4 * q + t));
        if constexpr (C::kF32) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int c = (4 * q + t) * 4 + 2 * j;
            const float2 q0 = *reinterpret_cast<const float2 *>(qs + g * C::kQP + c);
            const float2 q1 = *reinterpret_cast<const float2 *>(qs + (g + 8) * C::kQP + c);
            uint32_t ah[4], al[4];
            split(q0.x, ah[0], al[0]);
            split(q1.x, ah[1], al[1]);
            split(q0.y, ah[2], al[2]);
            split(q1.y, ah[3], al[3]);
#pragma unroll
            for (int n = 0; n < 2; ++n)
              mma_split(s[n], ah, al, __uint_as_float(ptx::u4_at(kw[n], 2 * j)),
                        __uint_as_float(ptx::u4_at(kw[n], 2 * j + 1)));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t a[4];
            if constexpr (!kQRegs) q_words(q, j, a);
            const uint32_t(&qw)[4] = kQRegs ? qa[kQRegs ? 2 * q + j : 0] : a;
#pragma unroll
            for (int n = 0; n < 2; ++n)
              mma_bf16(s[n], qw, ptx::u4_at(kw[n], 2 * j), ptx::u4_at(kw[n], 2 * j + 1));
          }
        }
      }

      if constexpr (careful && C::kF32) {
        // An infinite q or k, or one whose upper part rounds up to infinity, makes NaN of its
        // products' parts where the product itself need not be NaN: such scores are taken whole.
        const uint8_t *kb = smem + (ks - ptx::smem_addr(smem));
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (s[n][e] != s[n][e]) {
              const int key = 8 * n + 2 * t + (e & 1);
              const T *a = qs + (g + 8 * (e >> 1)) * C::kQP;
              s[n][e] = 0.f;
#pragma unroll 1
              for (int c = 0; c < kDP; ++c)
                s[n][e] = fmaf(a[c], reinterpret_cast<const float *>(kb + C::k_at(key, c / 4))[c % 4],
                               s[n][e]);
            }
      }

      // Scores, masked.  The step to log2 units comes behind the subtraction of the reference: a
      // large score times log2 e would be rounded before it.
      if constexpr (!C::kF32) {
        if (p.softcap > 0.f) {  // fp32: tanhf below
          float most = 0.f;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[n][e] *= p.scale;
              most = fmaxf(most, fabsf(s[n][e]));
            }
          if (__any_sync(0xffffffffu, most * cap_u > kCapFit)) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[n][e] = cap_scaled(s[n][e], s[n][e] * cap_u, p.softcap);
          } else {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float x = s[n][e] * cap_u;
                s[n][e] *= cap_fit(x * x);
              }
          }
        }
      }
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = e >> 1, j = k0 + 8 * n + 2 * t + (e & 1);
          const Row &w = row[h];
          float z = !C::kF32 && p.softcap > 0.f ? s[n][e] : s[n][e] * p.scale;
          if (C::kF32 && p.softcap > 0.f) z = p.softcap * tanhf(z / p.softcap);
          if (p.slopes) z = fmaf(-slope[h], fabsf((float)(j - w.pos)), z);
          if (p.table) z += __ldg(table[h] + min(max(j - w.pos, -p.reach), p.reach));
          bool open = j < w.prefix || (j >= w.lo && j < w.hi);
          if (p.k_docs) open = open && p.k_docs[u.s.k_row + j] == w.doc;
          s[n][e] = open ? z : -INFINITY;
          top[h] = fmaxf(top[h], s[n][e]);
        }
      bool raise = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        raise = raise || top[h] > m[h] + (careful ? 0.f : kRescaleThreshold) ||
                (m[h] == -INFINITY && top[h] > m[h]);
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float now = fmaxf(m[h], top[h]);
          const float f = m[h] == -INFINITY ? 0.f : exp2f((m[h] - now) * kLog2e);
          m[h] = now;
          l[h] *= f;
#pragma unroll
          for (int n = 0; n < kDP / 8; ++n) {
            o[n][2 * h] *= f;
            o[n][2 * h + 1] *= f;
          }
        }
      }
      const float ref[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] = ex2((s[n][e] - ref[e >> 1]) * kLog2e);
          l[e >> 1] += s[n][e];
        }

      if constexpr (careful) {
        uint32_t bad = 0;
#pragma unroll 4
        for (int x = lane; x < kBlock * C::kChunks; x += 32) {
          const uint4 w = ld_shared_v4(vs + x * 16);
          if (!(finite_word(w.x, C::kF32) && finite_word(w.y, C::kF32) &&
                finite_word(w.z, C::kF32) && finite_word(w.w, C::kF32)))
            bad |= 1u << (x / C::kChunks);
        }
        bad = __reduce_or_sync(0xffffffffu, bad);
        while (bad) {
          const int j = __ffs(bad) - 1;
          bad &= bad - 1;
          float pj[2];  // this row's weight of key j, from the lane that has it
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float mine = 0.f;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (j == 8 * n + (j & 6) + e) mine = s[n][2 * h + e];
            pj[h] = __shfl_sync(0xffffffffu, mine, (lane & ~3) | ((j & 7) >> 1));
          }
#pragma unroll
          for (int n = 0; n < kDP / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              // fp32: column 8n + 2t + (e & 1); bf16: see P.V below
              const int c = C::kF32 ? 8 * n + 2 * t + (e & 1)
                                    : 16 * (n / 2) + 2 * (2 * t + (e & 1)) + (n & 1);
              const int byte = c * (int)sizeof(T);
              const float x = Elem<T>::load(
                  reinterpret_cast<const T *>(smem + (vs - ptx::smem_addr(smem)) +
                                              C::v_at(j, byte / 16) + byte % 16), 0);
              if (!(pj[e >> 1] == 0.f)) o[n][e] = fmaf(pj[e >> 1], x, o[n][e]);
            }
          __syncwarp();
          for (int x = lane; x < C::kChunks; x += 32)
            ptx::st_shared_v4(vs + j * C::kRowBytes + x * 16, 0, 0, 0, 0);
          __syncwarp();
        }
      }

      // O += P V.  S's accumulator holds keys 2t and 2t + 1 of each 8 of a row: how P enters.
      const int sw = (t << 1) & (C::kChunks - 1);  // the rows' exchange of pieces
      const uint32_t vr = vs + 2 * t * C::kRowBytes + (g >> 2) * 16 + (g & 3) * 4;
      auto word = [&](int row, int piece) {
        uint32_t w;
        asm volatile("ld.shared.b32 %0, [%1];"
                     : "=r"(w)
                     : "r"(vr + row * C::kRowBytes + (piece ^ sw) * 16)
                     : "memory");
        return w;
      };
      if constexpr (C::kF32) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          uint32_t ah[4], al[4];
          split(s[kk][0], ah[0], al[0]);
          split(s[kk][2], ah[1], al[1]);
          split(s[kk][1], ah[2], al[2]);
          split(s[kk][3], ah[3], al[3]);
#pragma unroll
          for (int n = 0; n < kDP / 8; ++n)
            mma_split(o[n], ah, al, __uint_as_float(word(8 * kk, 2 * n)),
                      __uint_as_float(word(8 * kk + 1, 2 * n)));
        }
      } else {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float a = s[x >> 1][2 * (x & 1)], b = s[x >> 1][2 * (x & 1) + 1];
          hi[x] = pack_bf16x2(a, b);
          lo[x] = pack_bf16x2(a - ptx::bf16_lo(hi[x]), b - ptx::bf16_hi(hi[x]));
        }
        // A word holds columns 16i + 2g and 16i + 2g + 1 of a key: the even ones go to accumulator
        // 2i, the odd ones to 2i + 1.
#pragma unroll
        for (int i2 = 0; i2 < kDP / 16; ++i2) {
          const uint32_t w0 = word(0, 2 * i2), w1 = word(1, 2 * i2), w2 = word(8, 2 * i2),
                         w3 = word(9, 2 * i2);
          const uint32_t e0 = __byte_perm(w0, w1, 0x5410), e1 = __byte_perm(w2, w3, 0x5410);
          const uint32_t d0 = __byte_perm(w0, w1, 0x7632), d1 = __byte_perm(w2, w3, 0x7632);
          mma_bf16(o[2 * i2], lo, e0, e1);
          mma_bf16(o[2 * i2 + 1], lo, d0, d1);
          mma_bf16(o[2 * i2], hi, e0, e1);
          mma_bf16(o[2 * i2 + 1], hi, d0, d1);
        }
      }
    }
  };
  walk(std::false_type());
  float taint[2] = {0.f, 0.f};  // NaN where a sum is not finite
#pragma unroll
  for (int n = 0; n < kDP / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) taint[e >> 1] = fmaf(o[n][e], 0.f, taint[e >> 1]);
  const bool odd = (g < rows && taint[0] != 0.f) || (g + 8 < rows && taint[1] != 0.f);
  if (__any_sync(0xffffffffu, odd)) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();  // the ring is free
    ahead = u.first + warp;
#pragma unroll 1
    for (int s = 0; s < kStages - 1; ++s, ahead += C::kWarps) fetch(ahead, s);
    walk(std::true_type());
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
  }
  __syncthreads();  // the rings are free: the warps' results go there
  float *wo = reinterpret_cast<float *>(smem) + warp * kRows * kDP;
  float2 *wml = reinterpret_cast<float2 *>(smem + C::kWarps * kRows * kDP * 4) + warp * kRows;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (t == 0) wml[g + 8 * h] = make_float2(m[h], l[h]);
#pragma unroll
    for (int n = 0; n < kDP / 8; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = C::kF32 ? 8 * n + 2 * t + e : 16 * (n / 2) + 2 * (2 * t + e) + (n & 1);
        wo[(g + 8 * h) * kDP + c] = o[n][2 * h + e];
      }
  }
  __syncthreads();
  const float *so = reinterpret_cast<const float *>(smem);
  const float2 *sml = reinterpret_cast<const float2 *>(smem + C::kWarps * kRows * kDP * 4);
  for (int r = warp; r < rows; r += C::kWarps) {
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < C::kWarps; ++w) mm = fmaxf(mm, sml[w * kRows + r].x);
    const float ref = mm == -INFINITY ? 0.f : mm;
    float f[C::kWarps], ll = 0.f;
#pragma unroll
    for (int w = 0; w < C::kWarps; ++w) {
      const float2 v = sml[w * kRows + r];
      f[w] = v.x == -INFINITY ? 0.f : exp2f((v.x - ref) * kLog2e);
      ll += v.x == -INFINITY ? v.y : f[w] * v.y;
    }
    const size_t part = ((size_t)u.slot * p.splits + u.split) * kRows + r;
    const size_t orow = ((size_t)(u.s.q_row + u.t0 + r / pack) * p.heads + u.head0 + r % pack) * p.dim;
    const float inv = p.splits > 1 ? 1.f : ll == 0.f ? 0.f : 1.f / ll;
    if (p.splits > 1 && lane == 0) p.part_ml[part] = make_float2(mm, ll);
    for (int c = lane; c < (int)p.dim; c += 32) {
      float acc = 0.f;
#pragma unroll
      for (int w = 0; w < C::kWarps; ++w)
        if (f[w] != 0.f) acc = fmaf(f[w], so[(w * kRows + r) * kDP + c], acc);
      if (p.splits > 1)
        p.part_o[part * p.part_dp + c] = acc;
      else
        store_out(p, orow + c, ll == 0.f ? 0.f : acc * inv);
    }
  }
  if (p.splits == 1 || arrive_last(p, u, flag)) {
    if (p.splits > 1) join_parts<kRows>(p, u, kLog2e);
    zero_padding(p, u);
  }
}

template <typename T, int kDP>
cudaError_t launch(const ScoredProblem &p, cudaStream_t stream) {
  using C = Cfg<T, kDP>;
  static std::atomic<uint64_t> seen{0};
  cudaError_t e = allow_smem((const void *)scored_few_kernel<T, kDP>, C::kSmemBytes, seen);
  if (e != cudaSuccess) return e;
  const uint32_t grid = p.tiles * p.nseq * (p.heads / p.pack) * p.splits;
  scored_few_kernel<T, kDP><<<grid, C::kThreads, C::kSmemBytes, stream>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_dim(const ScoredProblem &p, cudaStream_t stream) {
  if (p.dim <= 32) return launch<T, 32>(p, stream);
  if (p.dim <= 64) return launch<T, 64>(p, stream);
  if (p.dim <= 128) return launch<T, 128>(p, stream);
  return launch<T, 256>(p, stream);
}

template <typename T>
int resident(uint32_t dim) {
  return dim <= 32    ? Cfg<T, 32>::kResident
         : dim <= 64  ? Cfg<T, 64>::kResident
         : dim <= 128 ? Cfg<T, 128>::kResident
                      : Cfg<T, 256>::kResident;
}

}  // namespace scored_few

int scored_few_resident(const ScoredProblem &p) {
  return p.in_dtype == TX_BF16 ? scored_few::resident<uint16_t>(p.dim)
                               : scored_few::resident<float>(p.dim);
}

// Few rows, and rows of k and v that 16-byte copies can take.
bool scored_few_supported(const ScoredProblem &p) {
  const uint32_t v = p.in_dtype == TX_BF16 ? 8 : 4;
  auto ok = [&](const void *x, uint64_t row, uint64_t head) {
    return (uintptr_t)x % 16 == 0 && row % v == 0 && head % v == 0;
  };
  return (uint64_t)p.max_q * (p.heads / p.kv_heads) <= scored_few::kRows && p.dim % v == 0 &&
         ok(p.k, p.k_row, p.k_head) && ok(p.v, p.v_row, p.v_head);
}

cudaError_t launch_scored_few(const ScoredProblem &p, cudaStream_t stream) {
  return p.in_dtype == TX_BF16 ? scored_few::launch_dim<uint16_t>(p, stream)
                               : scored_few::launch_dim<float>(p, stream);
}

}  // namespace tx
