// Position rotation of the query and key heads of a batch of tokens, optionally behind a
// per-head RMSNorm, in one pass over both tensors (tx_rotary).
//
// A head x of `dim` columns is normalised (y = x * rsqrt(mean(x^2) + eps) * w, or y = x) and
// its first `rot` columns turned in pairs by the angle pos * f[c], f a table of rot / 2
// inverse frequencies: (a, b) -> (a C - b S, b C + a S), C and S the cosine and sine times
// `amplitude` (S negated for the inverse).  Pair c is columns (c, c + rot/2) in the half
// layout and (2c, 2c + 1) in the interleaved one; columns past `rot` pass through.  The angle
// is the fp32 product, as everywhere in this library; everything is computed in fp32 and
// rounded once on the way out.
//
// Bound: HBM, one read and one write of every element; ~6 flops per element.  A warp per token, so
// that the sines and cosines serve every head, and no shared memory.  Measured: 65536 packed tokens,
// 16 + 8 heads of 128 in bf16 with both norms (805 MB): 151 us, 5.3 TB/s; 8192 tokens, 12 + 12
// heads of 32 in fp32 (50 MB): 12.6 us, 4.0 TB/s; 8 tokens: 9.2 us from cold caches and 5.1 us from
// warm ones, a warp's 12 steps through its token's 24 heads (queueing the call takes the host 6.7 us).
#include <cuda_runtime.h>

#include "../../include/tessattn.h"
#include "common.cuh"
#include "kernels.h"

namespace tx {
namespace {

// V consecutive elements, moved as one access where V elements are 4, 8 or 16 bytes.
template <int V, typename T>
struct Raw {
  static constexpr int kBytes = V * (int)sizeof(T);
  uint32_t w[(kBytes + 3) / 4];
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (kBytes == 16) {
      const uint4 v = *reinterpret_cast<const uint4 *>(p);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (kBytes == 8) {
      const uint2 v = *reinterpret_cast<const uint2 *>(p);
      w[0] = v.x; w[1] = v.y;
    } else if constexpr (kBytes == 4) {
      w[0] = *reinterpret_cast<const uint32_t *>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t *>(p);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < (kBytes + 3) / 4; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void floats(float (&f)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (sizeof(T) == 4)
        f[i] = __uint_as_float(w[i]);
      else
        f[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
  }
};
template <int V, typename T>
__device__ __forceinline__ void load_vec(const T *p, float (&f)[V]) {
  Raw<V, T> r;
  r.load(p);
  r.floats(f);
}
template <int V>
__device__ __forceinline__ void store_vec(float *p, const float (&f)[V]) {
  if constexpr (V == 8) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else if constexpr (V == 4) {
    *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    p[0] = f[0];
  }
}
template <int V>
__device__ __forceinline__ void store_vec(uint16_t *p, const float (&f)[V]) {
  if constexpr (V == 8)
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                               pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  else if constexpr (V == 4)
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
  else
    p[0] = f32_to_bf16_bits(f[0]);
}

// The sequence of packed row `tok`: the last s in [0, nseq) with cu[s] <= tok, by a search
// whose 32 lanes probe at once (two dependent loads for up to 1024 sequences).
__device__ __forceinline__ uint32_t warp_find_seq(const int32_t *cu, uint32_t nseq, uint32_t tok,
                                                  uint32_t lane) {
  uint32_t lo = 0, n = nseq;  // the answer is in [lo, lo + n)
  while (n > 1) {
    const uint32_t step = (n + 31) / 32;
    const uint32_t at = lane * step;
    const bool le = at < n && (uint32_t)cu[lo + at] <= tok;
    const uint32_t hits = __popc(__ballot_sync(0xffffffffu, le));  // le is monotone in lane
    const uint32_t skip = (hits ? hits - 1 : 0) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  return lo;
}

// A head is cut into slots of 2V columns, held by one lane as two vectors of V: in a rotated
// slot the second vector holds the partners (half layout) or the slot is V adjacent pairs
// (interleaved).  kLanes lanes cover a head with kSlots slots each, so a warp takes
// 32 / kLanes heads at a time; one warp per token, so the sines and cosines of a lane's slots
// serve every head of the token.
template <typename TI, typename TO, int V, int kLanes, int kSlots>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryProblem p) {
  constexpr uint32_t kHeads = 32 / kLanes;  // heads per step of a warp
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t tok = blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
  if (tok >= p.tokens) return;
  const uint32_t sub = lane % kLanes;
  const uint32_t half = p.rot / 2, rslots = half / V;

  // Columns of this lane's slots.
  uint32_t ca[kSlots], cb[kSlots];
  bool turned[kSlots], has_a[kSlots], has_b[kSlots];
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    const uint32_t slot = sub + s * kLanes;
    turned[s] = slot < rslots;
    if (turned[s]) {
      ca[s] = p.interleaved ? slot * 2 * V : slot * V;
      cb[s] = p.interleaved ? ca[s] + V : ca[s] + half;
      has_a[s] = has_b[s] = true;
    } else {
      ca[s] = p.rot + (slot - rslots) * 2 * V;
      cb[s] = ca[s] + V;
      has_a[s] = ca[s] < p.dim;
      has_b[s] = cb[s] < p.dim;
    }
  }
  const uint32_t total = p.q.heads + p.k.heads;
  // A step's heads are on their way while those before them are worked on, the first ones while the
  // position is looked up and its sines and cosines are taken.
  Raw<V, TI> ra[kSlots], rb[kSlots];
  auto fetch = [&](uint32_t h0) {
    const uint32_t hh = h0 + lane / kLanes;
    const bool is_k = hh >= p.q.heads;
    const RotaryTensor &t = is_k ? p.k : p.q;
    const TI *in = static_cast<const TI *>(t.x) + (size_t)tok * t.x_token +
                   (size_t)(is_k ? hh - p.q.heads : hh) * t.x_head;
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      ra[s].clear();
      rb[s].clear();
      if (hh < total && has_a[s]) ra[s].load(in + ca[s]);
      if (hh < total && has_b[s]) rb[s].load(in + cb[s]);
    }
  };
  fetch(0);

  uint32_t pos;
  if (p.positions)
    pos = (uint32_t)p.positions[tok];
  else if (p.cu)
    pos = tok - (uint32_t)p.cu[warp_find_seq(p.cu, p.nseq, tok, lane)];
  else
    pos = tok % p.seq;
  float co[kSlots][V], si[kSlots][V];
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    const uint32_t slot = sub + s * kLanes;
    if (turned[s]) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float sn, cs;
        rope_sincos(__fmul_rn((float)pos, __ldg(p.inv_freq + slot * V + i)), &sn, &cs);
        co[s][i] = cs * p.amplitude;
        si[s][i] = sn * p.amplitude_sin;
      }
    }
  }

  // 2-byte elements fill the registers with one step in flight: 148 us rolled, 158 us by twos; fp32
  // 13.2 us rolled, 12.6 us by twos (the sizes above).
  constexpr int kSteps = sizeof(TI) == 2 ? 1 : 2;
#pragma unroll kSteps
  for (uint32_t h0 = 0; h0 < total; h0 += kHeads) {
    const uint32_t hh = h0 + lane / kLanes;
    const bool live = hh < total, is_k = hh >= p.q.heads;
    const RotaryTensor &t = is_k ? p.k : p.q;
    const uint32_t h = is_k ? hh - p.q.heads : hh;
    TO *out = static_cast<TO *>(t.out) + (size_t)tok * t.out_token + (size_t)h * t.out_head;
    float a[kSlots][V], b[kSlots][V];
    float ss = 0.f;
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      ra[s].floats(a[s]);
      rb[s].floats(b[s]);
#pragma unroll
      for (int i = 0; i < V; ++i) ss += a[s][i] * a[s][i] + b[s][i] * b[s][i];
    }
    fetch(h0 + kHeads);
    if (p.norm) {
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (live && t.norm_w) {
        const float inv = rsqrtf(ss / (float)p.dim + p.eps);
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
          float w[V];
          if (has_a[s]) {
            load_vec<V>(t.norm_w + ca[s], w);
#pragma unroll
            for (int i = 0; i < V; ++i) a[s][i] *= inv * w[i];
          }
          if (has_b[s]) {
            load_vec<V>(t.norm_w + cb[s], w);
#pragma unroll
            for (int i = 0; i < V; ++i) b[s][i] *= inv * w[i];
          }
        }
      }
    }
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      if (turned[s]) {
        if (p.interleaved) {
          // Pairs (2i, 2i + 1) of the slot's 2V columns, the first V of them in a.
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float &u = 2 * i < V ? a[s][(2 * i) % V] : b[s][(2 * i) % V];
            float &v = 2 * i + 1 < V ? a[s][(2 * i + 1) % V] : b[s][(2 * i + 1) % V];
            const float x = u, y = v;
            u = x * co[s][i] - y * si[s][i];
            v = y * co[s][i] + x * si[s][i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float x = a[s][i], y = b[s][i];
            a[s][i] = x * co[s][i] - y * si[s][i];
            b[s][i] = y * co[s][i] + x * si[s][i];
          }
        }
      }
      if (live && has_a[s]) store_vec<V>(out + ca[s], a[s]);
      if (live && has_b[s]) store_vec<V>(out + cb[s], b[s]);
    }
  }
}

template <typename TI, typename TO, int V, int kLanes, int kSlots>
cudaError_t run(const RotaryProblem &p, cudaStream_t stream) {
  // Few tokens: a warp per block, so that they spread over the SMs.
  const uint32_t warps = p.tokens >= 8 * 148 ? 8 : 1;
  rotary_kernel<TI, TO, V, kLanes, kSlots>
      <<<(p.tokens + warps - 1) / warps, 32 * warps, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename TI, typename TO, int V>
cudaError_t run_lanes(const RotaryProblem &p, cudaStream_t stream) {
  const uint32_t half = p.rot / 2;
  const uint32_t slots = half / V + (p.dim - p.rot + 2 * V - 1) / (2 * V);
  if constexpr (V > 1) {
    if (slots <= 4) return run<TI, TO, V, 4, 1>(p, stream);
    if (slots <= 8) return run<TI, TO, V, 8, 1>(p, stream);
    if (slots <= 16) return run<TI, TO, V, 16, 1>(p, stream);
    return run<TI, TO, V, 32, 1>(p, stream);
  } else {
    if (slots <= 32) return run<TI, TO, 1, 32, 1>(p, stream);
    return run<TI, TO, 1, 32, 4>(p, stream);
  }
}

template <typename TI, typename TO>
cudaError_t run_types(const RotaryProblem &p, uint32_t v, cudaStream_t stream) {
  if constexpr (sizeof(TI) == 2)
    if (v == 8) return run_lanes<TI, TO, 8>(p, stream);
  if (v >= 4) return run_lanes<TI, TO, 4>(p, stream);
  return run_lanes<TI, TO, 1>(p, stream);
}

bool aligned(const RotaryTensor &t, size_t v, size_t esz_in, size_t esz_out) {
  if (!t.heads) return true;
  // An output vector of 8 fp32 is stored as two accesses of 16 bytes.
  const size_t out_bytes = v * esz_out < 16 ? v * esz_out : 16;
  return (uintptr_t)t.x % (v * esz_in) == 0 && (uintptr_t)t.out % out_bytes == 0 &&
         t.x_token % v == 0 && t.x_head % v == 0 && t.out_token % v == 0 && t.out_head % v == 0 &&
         (uintptr_t)t.norm_w % (v * 2) == 0;
}

}  // namespace

// Vector width: the widest of 8 (bf16 in), 4 and 1 elements for which the rotated and the
// remaining columns are whole slots of 2V and every row starts on a vector.
uint32_t rotary_vector(const RotaryProblem &p) {
  const size_t ei = p.in_dtype == TX_BF16 ? 2 : 4, eo = p.out_dtype == TX_BF16 ? 2 : 4;
  for (uint32_t v = p.in_dtype == TX_BF16 ? 8 : 4; v > 1; v /= 2) {
    if (v == 2) break;
    if (p.rot % (2 * v) == 0 && p.dim % (2 * v) == 0 && aligned(p.q, v, ei, eo) &&
        aligned(p.k, v, ei, eo))
      return v;
  }
  return 1;
}

cudaError_t launch_rotary(const RotaryProblem &p, cudaStream_t stream) {
  if (!p.tokens) return cudaSuccess;
  const uint32_t v = rotary_vector(p);
  if (p.in_dtype == TX_F32 && p.out_dtype == TX_F32) return run_types<float, float>(p, v, stream);
  if (p.in_dtype == TX_F32) return run_types<float, uint16_t>(p, v, stream);
  if (p.out_dtype == TX_F32) return run_types<uint16_t, float>(p, v, stream);
  return run_types<uint16_t, uint16_t>(p, v, stream);
}

}  // namespace tx
