// Attention under a score rule in fp32 accuracy: fp32 q, k, v of any head_dim up to 256, and
// whatever bf16 shapes or layouts the tensor-memory kernel does not take
// (tx_attention_scored; the formula is in attn_scored_tc.cu).
//
// One CTA takes 64 rows (16 per warp) and walks the visited key tiles in steps of 64 keys staged
// in shared memory as fp32.  Both products run on mma.sync m16n8k8 TF32 with split operands:
// x = hi + lo, hi = x rounded to TF32 (10 mantissa bits), lo = x - hi, and a.b as
// ah.bh + ah.bl + al.bh, which leaves an error of about 2^-22 of each product -- what an fp32
// result needs, and one TF32 product (2^-11) or bf16 does not give.  The register-level
// instruction is used because its operands are split in registers on the way from the staged
// fp32 rows; the tensor-memory instruction would need both parts of K and a transposed V written
// back to shared memory first.  The accumulator of Q.K^T holds keys 2t and 2t + 1 of a row in
// lane t, which is the A operand of P.V once V's rows are taken in that order, so P never leaves
// registers.
//
// Bound: issue slots and latency (the operands' splits are half of the products' instructions).
// Rows arrive by asynchronous copies, K, V and Q at once; warps without rows and blocks of 8 keys
// past the end are skipped.  Measured: 64 texts of 16 to 128 tokens, 12 heads of 32, distance
// slopes: 45.6 us (44 % of issue slots); 32 keys a step with half as many CTAs again: 46.5 us against
// 44.6 when that was measured.
#include <cuda_runtime.h>

#include <type_traits>

#include "../../include/tessattn.h"
#include "attn_scored.cuh"
#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace tx {
namespace scored_f32 {

using namespace scored;
using ptx::ex2;

constexpr int kRows = 64, kThreads = 128, kStep = 64;  // kStep keys staged at a time
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kOdd = 0x1p127f;  // values from here on are added by hand

// Row pitches (floats) that keep the fragment reads free of bank conflicts: Q and K are read as
// pairs (8 words between rows modulo 32), V by single values of every second row (4 words).
template <int kDP>
struct Cfg {
  static constexpr int kQP = kDP + 8, kVP = kDP + 4;
  static constexpr int kKFloats = kStep * kQP > kStep * (kStep + 1) ? kStep * kQP : kStep * (kStep + 1);
  static constexpr uint32_t kOffQ = 0, kOffK = kRows * kQP * 4, kOffV = kOffK + kKFloats * 4;
  static constexpr uint32_t kOffMisc = kOffV + kStep * kVP * 4;
  static constexpr uint32_t kSmemBytes = kOffMisc + 64 + kDocWords * 4 + kStep * 4;
};

__device__ __forceinline__ void split(float x, uint32_t &hi, uint32_t &lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// c += a b from the operands' parts, added to c in fp32: the tensor core cuts bits off at each of its
// own additions, always towards zero (9 heads of 80 over 2183 keys: off by 2.1e-6 that way, 1.9e-7
// this way; 64 short texts 44.6 and 45.4 us).
__device__ __forceinline__ void mma_split(float (&c)[4], const uint32_t (&ah)[4],
                                          const uint32_t (&al)[4], uint32_t bh0, uint32_t bl0,
                                          uint32_t bh1, uint32_t bl1) {
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  mma(sum, al, bh0, bh1);
  mma(sum, ah, bl0, bl1);
  mma(sum, ah, bh0, bh1);
#pragma unroll
  for (int e = 0; e < 4; ++e) c[e] += sum[e];
}

__device__ __forceinline__ float elem(const ScoredProblem &p, const void *x, size_t i) {
  return p.in_dtype == 1 ? bf16_bits_to_f32(static_cast<const uint16_t *>(x)[i])
                         : static_cast<const float *>(x)[i];
}

// kStep rows into `dst` with kPitch, the columns past dim zero.  `at(r)` is row r's first element in
// x, or -1 for a row of zeros.  `vec`: fp32 rows on 16-byte boundaries, copied asynchronously (the
// caller waits for them).
template <int kDP, int kPitch, typename At>
__device__ __forceinline__ void stage(const ScoredProblem &p, float *dst, const void *x, bool vec,
                                      At at) {
  if (vec) {
    const uint32_t to = ptx::smem_addr(dst);
#pragma unroll 4
    for (int i = threadIdx.x; i < kStep * (kDP / 4); i += kThreads) {
      const int r = i / (kDP / 4), c = i % (kDP / 4) * 4;
      const long long from = at(r);
      const bool have = from >= 0 && c < (int)p.dim;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + (r * kPitch + c) * 4),
                   "l"(static_cast<const float *>(x) + (have ? from + c : 0)), "r"(have ? 16 : 0)
                   : "memory");
    }
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < kStep * kDP; i += kThreads) {
      const int r = i / kDP, c = i % kDP;
      const long long from = at(r);
      dst[r * kPitch + c] = from >= 0 && c < (int)p.dim ? elem(p, x, from + c) : 0.f;
    }
  }
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Four CTAs an SM (128 registers a thread) where the accumulators leave room: 66 against 76 us for 64
// short texts with heads of 32 (when that was measured).
template <int kDP>
__global__ void __launch_bounds__(kThreads, kDP <= 64 ? 4 : 1)
    scored_f32_kernel(const __grid_constant__ ScoredProblem p) {
  using C = Cfg<kDP>;
  extern __shared__ __align__(16) uint8_t smem[];
  float *qs = reinterpret_cast<float *>(smem + C::kOffQ);
  float *ks = reinterpret_cast<float *>(smem + C::kOffK);
  float *vs = reinterpret_cast<float *>(smem + C::kOffV);
  int *range = reinterpret_cast<int *>(smem + C::kOffMisc);
  uint32_t *flag = reinterpret_cast<uint32_t *>(smem + C::kOffMisc + 16);
  uint32_t *words = reinterpret_cast<uint32_t *>(smem + C::kOffMisc + 64);
  int32_t *doc_s = reinterpret_cast<int32_t *>(smem + C::kOffMisc + 64 + kDocWords * 4);
  const Unit u = make_unit<kRows>(p, blockIdx.x);
  if (!u.present) return;
  const bool docs = p.q_docs != nullptr;
  if (docs) mark_tiles(p, u, words, range);
  const uint32_t *marks = docs ? words : nullptr;
  const int first = next_tile(u, marks, u.first);
  const int pack = (int)p.pack;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  // This thread's two rows.
  float m[2], l[2];
  Row row[2];
  int head[2];
  const float *table[2];
  float slope[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = warp * 16 + g + 8 * h;
    row[h] = make_row(p, u, r / pack, r / pack < u.tokens);
    head[h] = (int)u.head0 + r % pack;
    table[h] = p.table ? p.table + (size_t)head[h] * (2 * p.reach + 1) + p.reach : nullptr;
    slope[h] = p.slopes ? p.slopes[head[h]] : 0.f;
  }
  float o[kDP / 8][4];

  // 16-byte copies: fp32, and every row of the tensor on a 16-byte boundary.
  auto aligned = [&](const void *x, uint64_t row_stride, uint64_t head_stride) {
    return p.in_dtype == 0 && ((p.dim | row_stride | head_stride) & 3) == 0 && ((uintptr_t)x & 15) == 0;
  };
  const bool vk = aligned(p.k, p.k_row, p.k_head), vv = aligned(p.v, p.v_row, p.v_head);
  const bool busy = warp * 16 / pack < u.tokens;  // this warp has rows
  if (first < u.last)  // query rows; packed heads of a token follow one another
    stage<kDP, C::kQP>(p, qs, p.q, aligned(p.q, p.q_row, p.q_head), [&](int r) -> long long {
      if (r / pack >= u.tokens) return -1;
      return (long long)((size_t)(u.s.q_row + u.t0 + r / pack) * p.q_row +
                         (size_t)(u.head0 + r % pack) * p.q_head);
    });

  // Values that are not finite.  A key closed to a row has p = 0 there, and the product would turn
  // 0 * Inf or 0 * NaN into NaN; and the parts of an infinite operand make NaN where the whole need
  // not.  So a CTA whose sums come out not finite (rare) walks its keys once more, carefully: with
  // NaN scores taken again whole, and with the value rows that hold such a value added by hand where
  // p > 0 and zeroed before the product.
  auto walk = [&](auto how) {
    constexpr bool careful = decltype(how)::value;
#pragma unroll
    for (int h = 0; h < 2; ++h) m[h] = -INFINITY, l[h] = 0.f;
#pragma unroll
    for (int i = 0; i < kDP / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    for (int i = first; i < u.last; i = next_tile(u, marks, i + 1)) {
      const int tile0 = key_tile(u, i) * kKeys;
      for (int k0 = tile0; k0 < min(tile0 + kKeys, u.s.nk); k0 += kStep) {
        const int live = min(kStep, u.s.nk - k0);
        __syncthreads();  // the previous step's rows have been read
        const size_t kr = (size_t)(u.s.k_row + k0);
        stage<kDP, C::kQP>(p, ks, p.k, vk, [&](int r) -> long long {
          return r < live ? (long long)((kr + r) * p.k_row + (size_t)u.kv * p.k_head) : -1;
        });
        stage<kDP, C::kVP>(p, vs, p.v, vv, [&](int r) -> long long {
          return r < live ? (long long)((kr + r) * p.v_row + (size_t)u.kv * p.v_head) : -1;
        });
        if (docs)
          for (int j = threadIdx.x; j < kStep; j += kThreads)
            doc_s[j] = j < live ? p.k_docs[kr + j] : -1;
        copies_done();
        bool any_odd = false;
        if constexpr (careful) {
          // Whether a value is not finite, or as good as that to the split below (2^127 or more):
          // each thread looks over the ones that it copied.  x * 2 * 0 is NaN exactly there, and
          // then the sum stays NaN.
          float taint = 0.f;
          auto look = [&](float x) { taint = fmaf(x * 2.f, 0.f, taint); };
          if (vv) {
#pragma unroll 4
            for (int x = threadIdx.x; x < kStep * (kDP / 4); x += kThreads) {
              const float4 v = *reinterpret_cast<const float4 *>(vs + x / (kDP / 4) * C::kVP +
                                                                 x % (kDP / 4) * 4);
              look(v.x), look(v.y), look(v.z), look(v.w);
            }
          } else {
#pragma unroll 4
            for (int x = threadIdx.x; x < kStep * kDP; x += kThreads)
              look(vs[x / kDP * C::kVP + x % kDP]);
          }
          any_odd = __syncthreads_or(taint != 0.f);
        } else {
          __syncthreads();
        }
        if (!busy && !any_odd) continue;  // the hand sums below keep the CTA in step

        // S = Q K^T
        float s[kStep / 8][4];
#pragma unroll
        for (int n = 0; n < kStep / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll 2
        for (int kk = 0; kk < kDP / 8; ++kk) {
          uint32_t ah[4], al[4];
          const float *qr = qs + (warp * 16 + g) * C::kQP + kk * 8 + 2 * t;
          const float2 q0 = *reinterpret_cast<const float2 *>(qr);
          const float2 q1 = *reinterpret_cast<const float2 *>(qr + 8 * C::kQP);
          split(q0.x, ah[0], al[0]);
          split(q1.x, ah[1], al[1]);
          split(q0.y, ah[2], al[2]);
          split(q1.y, ah[3], al[3]);
#pragma unroll
          for (int n = 0; n < kStep / 8; ++n) {
            if (n * 8 >= live) break;
            const float2 b =
                *reinterpret_cast<const float2 *>(ks + (n * 8 + g) * C::kQP + kk * 8 + 2 * t);
            uint32_t bh0, bl0, bh1, bl1;
            split(b.x, bh0, bl0);
            split(b.y, bh1, bl1);
            mma_split(s[n], ah, al, bh0, bl0, bh1, bl1);
          }
        }

        if constexpr (careful) {
          // An infinite q or k, or one whose upper part rounds up to infinity, makes NaN of its
          // products' parts where the product itself need not be NaN: such scores are taken whole.
#pragma unroll
          for (int n = 0; n < kStep / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (s[n][e] != s[n][e]) {
                const float *a = qs + (warp * 16 + g + 8 * (e >> 1)) * C::kQP;
                const float *b = ks + (n * 8 + 2 * t + (e & 1)) * C::kQP;
                s[n][e] = 0.f;
#pragma unroll 1
                for (int c = 0; c < kDP; ++c) s[n][e] = fmaf(a[c], b[c], s[n][e]);
              }
        }

        // Scores, masked; then the running maximum and the probabilities.  One branch per part of the
        // rule around the loop over the scores.  The step to log2 units comes behind the subtraction
        // of the reference: a large score times log2 e would be rounded before it.
        auto each = [&](auto change) {
#pragma unroll
          for (int n = 0; n < kStep / 8; ++n) {
            if (n * 8 >= live) break;
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = change(s[n][e], e >> 1, n * 8 + 2 * t + (e & 1));
          }
        };
        if (p.softcap > 0.f) {
          each([&](float z, int, int) { return p.softcap * tanhf(z * p.scale / p.softcap); });
        } else {
          each([&](float z, int, int) { return z * p.scale; });
        }
        if (p.slopes)
          each([&](float z, int h, int j) {
            return fmaf(-slope[h], fabsf((float)(k0 + j - row[h].pos)), z);
          });
        if (p.table)
          each([&](float z, int h, int j) {
            return z + __ldg(table[h] + min(max(k0 + j - row[h].pos, -p.reach), p.reach));
          });
        const int end = k0 + kStep;
        if (!(end <= u.whole_prefix || (k0 >= u.whole_lo && end <= u.whole_hi)))
          each([&](float z, int h, int jj) {
            const Row &w = row[h];
            const int j = k0 + jj;
            bool open = j < w.prefix || (j >= w.lo && j < w.hi);
            if (docs) open = open && doc_s[jj] == w.doc;
            return open ? z : -INFINITY;
          });
        float top[2] = {-INFINITY, -INFINITY};
        each([&](float z, int h, int) {
          top[h] = fmaxf(top[h], z);
          return z;
        });
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        }
        float ref[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float now = fmaxf(m[h], top[h]);
          ref[h] = now == -INFINITY ? 0.f : now;
          const float f = m[h] == -INFINITY ? 0.f : exp2f((m[h] - now) * kLog2e);
          m[h] = now;
          l[h] *= f;
#pragma unroll
          for (int n = 0; n < kDP / 8; ++n) {
            o[n][2 * h] *= f;
            o[n][2 * h + 1] *= f;
          }
        }
        each([&](float z, int h, int) {
          const float pj = ex2((z - ref[h]) * kLog2e);  // 0 below 2^-126: nothing beside the row's largest, 1
          l[h] += pj;
          return pj;
        });

        if (careful && any_odd) {
          // A value of v in this step is not finite (or near that): its key counts for the rows that
          // see it and for no other, and zero times it would not be zero.  Such keys (rare) are added by
          // hand where p > 0 and taken out of the product.
          __syncthreads();  // the K rows are free: P goes there
          constexpr int kPP = kStep + 1;
#pragma unroll
          for (int n = 0; n < kStep / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              ks[(warp * 16 + g + 8 * (e >> 1)) * kPP + n * 8 + 2 * t + (e & 1)] = s[n][e];
          __syncwarp();
          uint32_t bad[kStep / 32];
          for (int x = 0; x < kStep / 32; ++x) {
            bool odd = false;
            for (int c = 0; c < kDP; ++c) odd |= !(fabsf(vs[(x * 32 + lane) * C::kVP + c]) < kOdd);
            bad[x] = __ballot_sync(0xffffffffu, odd);
          }
          for (int jj = 0; jj < kStep; ++jj) {
            if (!((bad[jj >> 5] >> (jj & 31)) & 1)) continue;
#pragma unroll
            for (int n = 0; n < kDP / 8; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float pj = ks[(warp * 16 + g + 8 * (e >> 1)) * kPP + jj];
                if (!(pj == 0.f)) o[n][e] = fmaf(pj, vs[jj * C::kVP + n * 8 + 2 * t + (e & 1)], o[n][e]);
              }
          }
          __syncthreads();  // every warp has read the rows
          for (int jj = warp; jj < kStep; jj += kThreads / 32)
            if ((bad[jj >> 5] >> (jj & 31)) & 1)
              for (int c = lane; c < kDP; c += 32) vs[jj * C::kVP + c] = 0.f;
          __syncthreads();
        }

        // O += P V
#pragma unroll
        for (int kk = 0; kk < kStep / 8; ++kk) {
          if (kk * 8 >= live) break;
          uint32_t ah[4], al[4];
          split(s[kk][0], ah[0], al[0]);
          split(s[kk][2], ah[1], al[1]);
          split(s[kk][1], ah[2], al[2]);
          split(s[kk][3], ah[3], al[3]);
#pragma unroll
          for (int n = 0; n < kDP / 8; ++n) {
            const float *v0 = vs + (kk * 8 + 2 * t) * C::kVP + n * 8 + g;
            uint32_t bh0, bl0, bh1, bl1;
            split(v0[0], bh0, bl0);
            split(v0[C::kVP], bh1, bl1);
            mma_split(o[n], ah, al, bh0, bl0, bh1, bl1);
          }
        }
      }
    }
  };
  walk(std::false_type());
  float taint = 0.f;  // NaN where a sum is not finite
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if ((warp * 16 + g + 8 * h) / pack < u.tokens)
#pragma unroll
      for (int n = 0; n < kDP / 8; ++n)
        taint = fmaf(o[n][2 * h], 0.f, fmaf(o[n][2 * h + 1], 0.f, taint));
  if (__syncthreads_or(taint != 0.f)) walk(std::true_type());

#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    const int r = warp * 16 + g + 8 * h;
    if (r / pack >= u.tokens) continue;
    const float inv = p.splits > 1 ? 1.f : l[h] == 0.f ? 0.f : 1.f / l[h];
    const size_t part = ((size_t)u.slot * p.splits + u.split) * kRows + r;
    const size_t orow = ((size_t)(u.s.q_row + u.t0 + r / pack) * p.heads + head[h]) * p.dim;
    if (p.splits > 1 && t == 0) p.part_ml[part] = make_float2(m[h], l[h]);
#pragma unroll
    for (int n = 0; n < kDP / 8; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t c = n * 8 + 2 * t + e;
        if (c >= p.dim) continue;
        if (p.splits > 1)
          p.part_o[part * p.part_dp + c] = o[n][2 * h + e];
        else
          store_out(p, orow + c, o[n][2 * h + e] * inv);
      }
  }
  if (p.splits == 1 || arrive_last(p, u, flag)) {
    if (p.splits > 1) join_parts<kRows>(p, u, kLog2e);
    zero_padding(p, u);
  }
}

template <int kDP>
cudaError_t launch(const ScoredProblem &p, cudaStream_t stream) {
  constexpr uint32_t smem = Cfg<kDP>::kSmemBytes;
  static std::atomic<uint64_t> seen{0};
  cudaError_t e = allow_smem((const void *)scored_f32_kernel<kDP>, (int)smem, seen);
  if (e != cudaSuccess) return e;
  const uint32_t grid = p.tiles * p.nseq * (p.heads / p.pack) * p.splits;
  scored_f32_kernel<kDP><<<grid, kThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace scored_f32

cudaError_t launch_scored_f32(const ScoredProblem &p, cudaStream_t stream) {
  if (p.dim <= 32) return scored_f32::launch<32>(p, stream);
  if (p.dim <= 64) return scored_f32::launch<64>(p, stream);
  if (p.dim <= 128) return scored_f32::launch<128>(p, stream);
  return scored_f32::launch<256>(p, stream);
}

}  // namespace tx
