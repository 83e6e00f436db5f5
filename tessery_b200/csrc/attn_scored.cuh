// What the kernels of attention under a score rule share: how a launch is cut into CTAs, which
// key tiles a CTA visits, which keys a query row may see, and how partial results over a split
// key range are joined.
//
// Rows.  A CTA's kRows rows are kRows / pack query tokens of `pack` heads that read the same
// kv head (row r: token r / pack, head r % pack), so those heads share every key and value
// tile; pack is the largest power of two that divides the heads per kv head (at most kRows).
// Query token i of a sequence with nq queries and nk keys stands at position i + nk - nq.
#pragma once

#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace tx {
namespace scored {

constexpr int kKeys = 128;        // keys per tile
constexpr uint32_t kTablePack = 4;  // most heads of a pack with a distance table (tensor-memory route)
constexpr uint32_t kDocWords = 512;  // bits for the key tiles of a document mask: 16384 tiles

struct Seq {
  int q_row, k_row;  // first row of the sequence in q and k
  int nq, nk;
};

// Rows of sequence s.  Offsets and lengths come from device arrays: they are held to the
// tensors' rows, and a length above the stated maximum is reported.
__device__ __forceinline__ Seq load_seq(const ScoredProblem &p, uint32_t s) {
  Seq o;
  auto side = [&](const int32_t *cu, const int32_t *len, uint32_t most, uint32_t rows, int *row,
                  int *n) {
    long long r0 = cu ? cu[s] : (long long)s * most;
    long long c = cu ? (long long)cu[s + 1] - cu[s] : len ? (long long)len[s] : (long long)most;
    if (c > (long long)most || r0 < 0 || c < 0 || r0 + c > (long long)rows) {
      if (threadIdx.x == 0) report_status(p.status, kStatusBadArg);
      r0 = min(max(r0, 0ll), (long long)rows);
      c = min(min(max(c, 0ll), (long long)most), (long long)rows - r0);
    }
    *row = (int)r0;
    *n = (int)c;
  };
  side(p.cu_q, p.q_lengths, p.max_q, p.rows_q, &o.q_row, &o.nq);
  side(p.cu_k, p.k_lengths, p.max_k, p.rows_k, &o.k_row, &o.nk);
  return o;
}

// One CTA's work.
struct Unit {
  Seq s;
  uint32_t head0, kv;      // first query head of the pack, kv head
  uint32_t split;          // which part of the key range
  uint32_t slot;           // index of the unit without its split
  int t0;                  // first query token
  int tokens;              // query tokens of the sequence in this tile
  int present;             // rows' tokens the layout has here: those past `tokens` get zeros
  int prefix;              // keys [0, prefix) are open to every row
  // key tiles in order: [0, a) then [b, ...), `count` in all; this CTA visits [first, last)
  int a, b, first, last;
  // keys that all rows see: [whole_lo, whole_hi) and [0, whole_prefix) (none with documents)
  int whole_lo, whole_hi, whole_prefix;
};

// Key range of a query position without the prefix: [lo, hi).
__device__ __forceinline__ void row_range(const ScoredProblem &p, int pos, int nk, int *lo,
                                          int *hi) {
  // Neither end may pass 32 bits: a position is negative where there are more queries than keys, and
  // a reach may be any int.
  int l = 0, h = nk;
  if (p.left >= 0 && pos > p.left) l = pos - p.left;
  if (p.causal) h = min(h, pos + 1);
  if (p.right >= 0 && pos < 0x7fffffff - p.right) h = min(h, pos + p.right + 1);
  *lo = l;
  *hi = h;
}

// Blocks run the last token tiles first: under a causal rule they see the most keys.
// kTile: keys of a visited tile.
template <int kRows, int kTile = kKeys>
__device__ __forceinline__ Unit make_unit(const ScoredProblem &p, uint32_t block) {
  Unit u;
  const uint32_t groups = p.heads / p.pack;
  u.split = block % p.splits;
  uint32_t rest = block / p.splits;
  u.slot = rest;
  const uint32_t hg = rest % groups;
  rest /= groups;
  const uint32_t s = rest % p.nseq, tile = p.tiles - 1 - rest / p.nseq;
  u.s = load_seq(p, s);
  u.head0 = hg * p.pack;
  u.kv = u.head0 / (p.heads / p.kv_heads);
  const int per = kRows / (int)p.pack;
  u.t0 = (int)tile * per;
  u.tokens = max(0, min(per, u.s.nq - u.t0));
  u.present = p.cu_q ? u.tokens
                     : max(0, min(per, min((int)p.max_q, (int)p.rows_q - u.s.q_row) - u.t0));
  u.prefix = p.prefix ? min(max(p.prefix[s], 0), u.s.nk) : 0;
  u.a = u.b = u.first = u.last = u.whole_lo = u.whole_hi = u.whole_prefix = 0;
  if (!u.tokens) return u;
  const int p0 = u.t0 + u.s.nk - u.s.nq;
  int lo, hi, last_lo, first_hi;
  row_range(p, p0, u.s.nk, &lo, &first_hi);           // both ends grow with the position
  row_range(p, p0 + u.tokens - 1, u.s.nk, &last_lo, &hi);
  if (!p.q_docs) {
    u.whole_lo = last_lo;
    u.whole_hi = first_hi;
    u.whole_prefix = u.prefix;
  }
  u.a = (u.prefix + kTile - 1) / kTile;
  u.b = max(u.a, lo / kTile);
  const int end = hi > lo ? (hi + kTile - 1) / kTile : 0;
  const int count = u.a + max(0, end - u.b);
  u.first = (int)((long long)count * u.split / p.splits);
  u.last = (int)((long long)count * (u.split + 1) / p.splits);
  return u;
}
__device__ __forceinline__ int key_tile(const Unit &u, int i) { return i < u.a ? i : i - u.a + u.b; }

// With documents: the bits of the visited tiles that hold a key of a document that the unit's
// rows may hold (their ids between the rows' least and greatest), by all threads of the CTA.
// `words` holds (last - first + 31) / 32 words.  Ends with the threads in step.
__device__ __forceinline__ void mark_tiles(const ScoredProblem &p, const Unit &u, uint32_t *words,
                                           int *range) {
  const int lane = (int)(threadIdx.x & 31), warp = (int)(threadIdx.x >> 5),
            warps = (int)(blockDim.x >> 5);
  // Documents of kAhead tiles a warp, the first of them on their way while the rows' range is found.
  constexpr int kAhead = 4;
  const int32_t *kd = p.k_docs + u.s.k_row;
  int d[kAhead][kKeys / 32];
  auto load = [&](int i0) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int i = i0 + a * warps;
#pragma unroll
      for (int c = 0; c < kKeys / 32; ++c) {
        const int j = key_tile(u, i) * kKeys + c * 32 + lane;
        d[a][c] = i < u.last && j < u.s.nk ? kd[j] : -1;
      }
    }
  };
  load(u.first + warp);
  if (threadIdx.x == 0) {
    range[0] = 0x7fffffff;
    range[1] = -1;
  }
  for (int i = threadIdx.x; i < (u.last - u.first + 31) / 32; i += blockDim.x) words[i] = 0;
  __syncthreads();
  const int32_t *qd = p.q_docs + u.s.q_row + u.t0;
  for (int i = warp * 32; i < u.tokens; i += warps * 32) {
    const int id = i + lane < u.tokens ? qd[i + lane] : -1;
    const int least = __reduce_min_sync(0xffffffffu, id < 0 ? 0x7fffffff : id);
    const int most = __reduce_max_sync(0xffffffffu, id);
    if (lane == 0 && most >= 0) {
      atomicMin(&range[0], least);
      atomicMax(&range[1], most);
    }
  }
  __syncthreads();
  const int lo = range[0], hi = range[1];
  for (int i0 = u.first + warp; i0 < u.last; i0 += warps * kAhead) {
    if (i0 != u.first + warp) load(i0);
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      bool hit = false;
#pragma unroll
      for (int c = 0; c < kKeys / 32; ++c) hit |= d[a][c] >= lo && d[a][c] <= hi;
      const int at = i0 + a * warps - u.first;
      if (__any_sync(0xffffffffu, hit) && lane == 0)
        atomicOr(&words[at >> 5], 1u << (at & 31));
    }
  }
  __syncthreads();
}
// Whether the tile from k0 holds kKeys keys and all are open to every row of the unit, as far as
// ranges tell.
__device__ __forceinline__ bool whole_tile(const Unit &u, int k0) {
  const int end = k0 + kKeys;
  return end <= u.whole_prefix || (k0 >= u.whole_lo && end <= u.whole_hi);
}
// The first visited tile at or after i (u.last when there is none).
__device__ __forceinline__ int next_tile(const Unit &u, const uint32_t *words, int i) {
  if (!words) return i;
  while (i < u.last) {
    const int at = i - u.first;
    const uint32_t w = words[at >> 5] >> (at & 31);
    if (w) return min(i + __ffs(w) - 1, u.last);
    i = u.first + ((at >> 5) + 1) * 32;
  }
  return u.last;
}

// Bits t of [c0, c0 + 32) that lie in [lo, hi).
__device__ __forceinline__ uint32_t interval_bits(int c0, int lo, int hi) {
  const int l = min(max(lo - c0, 0), 32), h = min(max(hi - c0, 0), 32);
  const uint32_t below_h = (uint32_t)((1ull << h) - 1), below_l = (uint32_t)((1ull << l) - 1);
  return below_h & ~below_l;
}

// Bits of 32 keys, whose documents the lanes hold (lane = key), that lie in this lane's own
// document: a pair of votes for each document that the warp's rows are in, most often one or two.
__device__ __forceinline__ uint32_t doc_bits(int32_t key_doc, int32_t row_doc) {
  uint32_t bits = 0, todo = __ballot_sync(0xffffffffu, row_doc >= 0);
  while (todo) {
    const int32_t d = __shfl_sync(0xffffffffu, row_doc, __ffs(todo) - 1);
    const uint32_t same = __ballot_sync(0xffffffffu, key_doc == d);
    if (row_doc == d) bits = same;
    todo &= ~__ballot_sync(0xffffffffu, row_doc == d);
  }
  return bits;
}

// One row's view of the keys.
struct Row {
  int pos, lo, hi, prefix, doc;
  __device__ __forceinline__ uint32_t bits(int c0) const {
    return interval_bits(c0, lo, hi) | interval_bits(c0, 0, prefix);
  }
};
__device__ __forceinline__ Row make_row(const ScoredProblem &p, const Unit &u, int token,
                                        bool live) {
  Row r;
  r.pos = u.t0 + token + u.s.nk - u.s.nq;
  row_range(p, r.pos, u.s.nk, &r.lo, &r.hi);
  r.prefix = u.prefix;
  r.doc = -1;
  if (p.q_docs && live) r.doc = p.q_docs[u.s.q_row + u.t0 + token];
  if (!live || (p.q_docs && r.doc < 0)) r.lo = r.hi = r.prefix = 0;
  return r;
}

// c tanh(z / c) for a cap c.  For arguments u = z / c up to kCapFit by a fit of degree 4 to tanh(u) / u
// in u^2 (weighted least squares refined to equal ripples, relative error 6e-7), beyond as
// 1 - 2 / (1 + e^(2u)) by hardware, 2^-21 of the cap: either is off relative to the result, whatever
// the cap (the second form alone is off by 1.2e-3 for scores below 8 under a cap of 1e4).
constexpr float kCapFit = 0.75f;
struct CapPoly {  // a tanh(u) / u with u^2 = q w
  float a0, a1, a2, a3, a4;
  __device__ __forceinline__ void set(float a, float q) {
    a0 = a * 0.999999435f;
    a1 = a * -0.333282516f * q;
    a2 = a * 0.132589833f * q * q;
    a3 = a * -0.0500563042f * q * q * q;
    a4 = a * 0.0129296325f * q * q * q * q;
  }
  __device__ __forceinline__ float operator()(float w) const {
    return fmaf(fmaf(fmaf(fmaf(a4, w, a3), w, a2), w, a1), w, a0);
  }
};
__device__ __forceinline__ float cap_exact(float u, float c) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ptx::ex2(u * (2.f * 1.44269504088896341f))));
  return fmaf(-2.f * c, r, c);
}
__device__ __forceinline__ float cap_scaled(float z, float u, float c) {
  CapPoly fit;
  fit.set(1.f, 1.f);
  return fabsf(u) <= kCapFit ? z * fit(u * u) : cap_exact(u, c);
}
// The factor from x to u where z = scale x; finite, so that a score of zero stays zero under the
// smallest of caps.
__device__ __forceinline__ float cap_factor(float scale, float c) {
  return c > 0.f ? fminf(scale / c, 3.402823466e38f) : 0.f;
}

// Zeros for the query rows of a padded layout past the sequence's length.
__device__ __forceinline__ void zero_padding(const ScoredProblem &p, const Unit &u) {
  for (int t = u.tokens; t < u.present; ++t) {
    const size_t at = ((size_t)(u.s.q_row + u.t0 + t) * p.heads + u.head0) * p.dim;
    const uint32_t n = p.pack * p.dim;
    for (uint32_t c = threadIdx.x; c < n; c += blockDim.x) {
      if (p.out_dtype == 1)
        static_cast<uint16_t *>(p.out)[at + c] = 0;
      else
        static_cast<float *>(p.out)[at + c] = 0.f;
    }
  }
}

// Joining a split key range.  Each CTA of a unit leaves, per row, its unnormalised sum O (fp32),
// its reference m (in the kernel's units of the score; -inf when it saw no key) and row sum l; the CTA that arrives last
// adds the parts in the order of the splits, so the result does not depend on which it was.
//
// Called by every thread of the CTA once its partials are written; true in the CTA that has to
// join.  Every CTA arrives, whatever happened to it, so the counters always return to zero.
__device__ __forceinline__ bool arrive_last(const ScoredProblem &p, const Unit &u,
                                            uint32_t *flag) {
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t n = atomicAdd(&p.part_arrived[u.slot], 1u);
    *flag = n + 1 == p.splits;
    if (*flag) p.part_arrived[u.slot] = 0;
  }
  __syncthreads();
  const bool last = *flag != 0;
  if (last) __threadfence();
  return last;
}

__device__ __forceinline__ void store_out(const ScoredProblem &p, size_t at, float v) {
  if (p.out_dtype == 1)
    static_cast<uint16_t *>(p.out)[at] = f32_to_bf16_bits(v);
  else
    static_cast<float *>(p.out)[at] = v;
}

// One warp per row.  The splits' weights first, lane = split; then 16 bytes of the row per lane, the
// lanes that a row leaves over (dim below 128) taking every second, fourth or eighth split, with
// eight loads in flight each.  (Walked split by split with one load in flight, 37 parts of 16 rows
// took 90 us of the 145 us at 16384 keys.)
// `log2e`: the factor of m's units to log2 units.
template <int kRows>
__device__ __forceinline__ void join_parts(const ScoredProblem &p, const Unit &u, float log2e) {
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const size_t base = (size_t)u.slot * p.splits * kRows;
  const uint32_t need = (p.part_dp + 3) / 4;  // lanes for a row
  const uint32_t width = need > 16 ? 32 : need > 8 ? 16 : need > 4 ? 8 : 4, sets = 32 / width;
  const uint32_t set = lane / width;
  for (int r = (int)warp; r < u.tokens * (int)p.pack; r += (int)warps) {
    auto part = [&](uint32_t s) { return base + (size_t)s * kRows + r; };
    const float2 none = make_float2(-INFINITY, 0.f);
    const float2 ml = lane < p.splits ? p.part_ml[part(lane)] : none;
    float m = ml.x;
    for (uint32_t s = lane + 32; s < p.splits; s += 32) m = fmaxf(m, p.part_ml[part(s)].x);
    m = warp_max(m);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = exp2f((ml.x - ref) * log2e) * ml.y;
    for (uint32_t s = lane + 32; s < p.splits; s += 32) {
      const float2 v = p.part_ml[part(s)];
      l += exp2f((v.x - ref) * log2e) * v.y;
    }
    l = warp_sum(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const size_t orow = ((size_t)(u.s.q_row + u.t0 + r / (int)p.pack) * p.heads + u.head0 +
                         r % (int)p.pack) * p.dim;
    for (uint32_t c0 = 0; c0 < p.dim; c0 += 4 * width) {
      const uint32_t c = c0 + 4 * (lane % width);
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (uint32_t s0 = 0; s0 < p.splits; s0 += 32) {
        // Of split s0 + lane; 0 for one that saw no key.
        const float at = s0 == 0 ? ml.x : s0 + lane < p.splits ? p.part_ml[part(s0 + lane)].x : none.x;
        const float weight = exp2f((at - ref) * log2e);
        const uint32_t end = min(32u, p.splits - s0);
        for (uint32_t x0 = 0; x0 < end; x0 += 8 * sets) {
          float4 v[8];
#pragma unroll
          for (uint32_t x = 0; x < 8; ++x) {
            const uint32_t s = x0 + x * sets + set;
            v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (s < end && c < p.part_dp)
              v[x] = *reinterpret_cast<const float4 *>(p.part_o + part(s0 + s) * p.part_dp + c);
          }
#pragma unroll
          for (uint32_t x = 0; x < 8; ++x) {
            const float f = __shfl_sync(0xffffffffu, weight, (x0 + x * sets + set) & 31);
            if (f != 0.f && x0 + x * sets + set < end) {
              acc[0] = fmaf(f, v[x].x, acc[0]);
              acc[1] = fmaf(f, v[x].y, acc[1]);
              acc[2] = fmaf(f, v[x].z, acc[2]);
              acc[3] = fmaf(f, v[x].w, acc[3]);
            }
          }
        }
      }
      for (uint32_t o = width; o < 32; o <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], o);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (set == 0 && c + e < p.dim) store_out(p, orow + c + e, acc[e] * inv);
    }
  }
}

}  // namespace scored
}  // namespace tx
