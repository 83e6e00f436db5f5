// The rows between two blocks of a layer in one pass (tx_block_norm):
//   z = y, or the experts' rows joined: z[t] = sum_j weights[t, j] y[places[t, j]]
//   r = x_scale x + y_scale gate * norm_after(z),   h = norm_before(r),
// a norm being RMS (v rsqrt(mean(v^2) + eps) (w + offset) + b), LayerNorm (the same of v - mean(v)) or
// none.  Everything is fp32 from the loads to the one rounding of each output; h is the norm of r as it
// is before r is rounded.  The joined sum runs in the order of j, and a row whose place is negative is not read.
//
// Bound: HBM, each row read once and written once.  A row lives in the registers of the threads that take
// it, so that the mean and the deviations of a LayerNorm are two passes over registers.
#include <cuda_runtime.h>

#include "../../include/tessattn.h"
#include "common.cuh"
#include "kernels.h"

namespace tx {
namespace {

// V elements of fp32 or bf16 as they lie in memory.
template <int V, typename T>
struct Words {
  static constexpr int kWords = V * (int)sizeof(T) / 4;
  uint32_t w[kWords ? kWords : 1];
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (V == 1) {
      if constexpr (sizeof(T) == 4)
        w[0] = __float_as_uint(*p);
      else
        w[0] = (uint32_t)*p << 16;
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 v = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint32_t *>(p) + i);
        w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
      }
    }
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (V == 1 || sizeof(T) == 4)
      return __uint_as_float(w[i]);
    else
      return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
};

template <int V>
__device__ __forceinline__ void store_as(void *base, int dtype, size_t at, const float *f) {
  if constexpr (V == 1) {
    if (dtype == TX_BF16)
      static_cast<uint16_t *>(base)[at] = f32_to_bf16_bits(f[0]);
    else
      static_cast<float *>(base)[at] = f[0];
  } else if (dtype == TX_BF16) {
    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(base) + at) =
        make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                   pack_bf16x2(f[6], f[7]));
  } else {
    float4 *p = reinterpret_cast<float4 *>(static_cast<float *>(base) + at);
    p[0] = make_float4(f[0], f[1], f[2], f[3]);
    p[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
}
template <int V>
__device__ __forceinline__ void load_as(const void *base, int dtype, size_t at, float *f) {
  if (dtype == TX_BF16) {
    Words<V, uint16_t> r;
    r.load(static_cast<const uint16_t *>(base) + at);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = r.at(i);
  } else {
    Words<V, float> r;
    r.load(static_cast<const float *>(base) + at);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = r.at(i);
  }
}

// The sum of v over the kThreads threads of a row; `turn` numbers the row's sums, so that two sums in turn
// use buffers of their own.
template <int kThreads>
__device__ __forceinline__ float row_sum(float v, float (*buf)[32], int &turn) {
  v = warp_sum(v);
  if constexpr (kThreads > 32) {
    float *b = buf[turn++ & 1];
    if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = v;
    __syncthreads();
    v = b[0];
#pragma unroll
    for (int i = 1; i < kThreads / 32; ++i) v += b[i];
  }
  return v;
}

// A row's elements: thread t holds vectors t, t + kThreads, ... of V elements.
template <int kThreads, int V, int C>
__device__ __forceinline__ void apply_norm(const BlockNorm &n, float (&v)[C][V], uint32_t cols,
                                           uint32_t t, float (*buf)[32], int &turn) {
  if (n.kind == TX_NORM_NONE) return;
  auto in = [&](int c) { return (t + c * kThreads) * V < cols; };
  if (n.kind == TX_NORM_LAYER) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[c][i];
    const float mean = row_sum<kThreads>(s, buf, turn) / (float)cols;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < V; ++i) v[c][i] = in(c) ? v[c][i] - mean : 0.f;
  }
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) ss = fmaf(v[c][i], v[c][i], ss);
  const float inv = rsqrtf(row_sum<kThreads>(ss, buf, turn) / (float)cols + n.eps);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (!in(c)) continue;
    const size_t at = (size_t)(t + c * kThreads) * V;
    float w[V];
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = 1.f;
    if (n.weight) {
      load_as<V>(n.weight, n.dtype, at, w);
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] += n.offset;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[c][i] = v[c][i] * inv * w[i];
    if (n.bias) {
      load_as<V>(n.bias, n.dtype, at, w);
#pragma unroll
      for (int i = 0; i < V; ++i) v[c][i] += w[i];
    }
  }
}

template <typename XT, typename YT, int kThreads, int V, int C>
__global__ void __launch_bounds__(kThreads > 32 ? kThreads : 256)
    block_norm_kernel(const __grid_constant__ BlockNormProblem p) {
  __shared__ float buf[2][32];
  int turn = 0;
  const uint32_t t = kThreads > 32 ? threadIdx.x : threadIdx.x & 31;
  const uint32_t row = kThreads > 32 ? blockIdx.x : blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  auto in = [&](int c) { return (t + c * kThreads) * V < p.cols; };
  Words<V, XT> x[C];
  if (p.x) {
    const XT *from = static_cast<const XT *>(p.x) + (size_t)row * p.ldx;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (in(c)) x[c].load(from + (size_t)(t + c * kThreads) * V);
  }
  float v[C][V];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) v[c][i] = 0.f;
  if (p.places) {
#pragma unroll 2
    for (uint32_t j = 0; j < p.top_k; ++j) {
      const int32_t place = __ldg(p.places + (size_t)row * p.top_k + j);
      if (place < 0) continue;
      if ((uint32_t)place >= p.y_rows) {
        report_status(p.status, kStatusBadArg);
        continue;
      }
      const float w = __ldg(p.weights + (size_t)row * p.top_k + j);
      const YT *from = static_cast<const YT *>(p.y) + (size_t)place * p.ldy;
      Words<V, YT> y[C];
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (in(c)) y[c].load(from + (size_t)(t + c * kThreads) * V);
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (in(c))
#pragma unroll
          for (int i = 0; i < V; ++i) v[c][i] = fmaf(w, y[c].at(i), v[c][i]);
    }
  } else if (p.y) {
    const YT *from = static_cast<const YT *>(p.y) + (size_t)row * p.ldy;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (in(c)) {
        Words<V, YT> y;
        y.load(from + (size_t)(t + c * kThreads) * V);
#pragma unroll
        for (int i = 0; i < V; ++i) v[c][i] = y.at(i);
      }
  }
  if (p.y) apply_norm<kThreads, V, C>(p.after, v, p.cols, t, buf, turn);
  if (p.gate) {
    uint32_t g = 0;
    if (p.cu)
      g = warp_find_seq(p.cu, p.gate_rows, row, threadIdx.x & 31);
    else if (p.seq)
      g = row / p.seq;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (!in(c)) continue;
      float f[V];
      load_as<V>(p.gate, p.gate_dtype, (size_t)g * p.ldg + (size_t)(t + c * kThreads) * V, f);
#pragma unroll
      for (int i = 0; i < V; ++i) v[c][i] *= f[i];
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (!in(c)) continue;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[c][i] = p.y ? v[c][i] * p.y_scale : 0.f;
      if (p.x) v[c][i] = fmaf(p.x_scale, x[c].at(i), v[c][i]);
    }
    if (p.out)
      store_as<V>(p.out, p.out_dtype, (size_t)row * p.ldo + (size_t)(t + c * kThreads) * V, v[c]);
  }
  if (!p.h) return;
  apply_norm<kThreads, V, C>(p.before, v, p.cols, t, buf, turn);
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (in(c))
      store_as<V>(p.h, p.h_dtype, (size_t)row * p.ldh + (size_t)(t + c * kThreads) * V, v[c]);
}

template <typename XT, typename YT, int kThreads, int V, int C>
cudaError_t run(const BlockNormProblem &p, cudaStream_t stream) {
  const uint32_t blocks = kThreads > 32 ? p.rows : (p.rows + 7) / 8;
  block_norm_kernel<XT, YT, kThreads, V, C>
      <<<blocks, kThreads > 32 ? kThreads : 256, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename XT, typename YT>
cudaError_t run_types(const BlockNormProblem &p, cudaStream_t stream) {
  if (!p.vec) {
    if (p.cols <= 32 * 8) return run<XT, YT, 32, 1, 8>(p, stream);
    if (p.cols <= 128 * 16) return run<XT, YT, 128, 1, 16>(p, stream);
    return run<XT, YT, 512, 1, 32>(p, stream);
  }
  if (p.cols <= 32 * 8) return run<XT, YT, 32, 8, 1>(p, stream);
  if (p.cols <= 32 * 16) return run<XT, YT, 32, 8, 2>(p, stream);
  if (p.cols <= 32 * 32) return run<XT, YT, 32, 8, 4>(p, stream);
  if (p.cols <= 128 * 16) return run<XT, YT, 128, 8, 2>(p, stream);
  if (p.cols <= 128 * 32) return run<XT, YT, 128, 8, 4>(p, stream);
  return run<XT, YT, 512, 8, 4>(p, stream);
}

}  // namespace

cudaError_t launch_block_norm(BlockNormProblem p, cudaStream_t stream) {
  p.vec = p.cols % 8 == 0;
  auto row = [&](const void *base, uint64_t ld) {
    if (base && ((uintptr_t)base % 16 || ld % 8)) p.vec = false;
  };
  row(p.x, p.ldx); row(p.y, p.ldy); row(p.out, p.ldo); row(p.h, p.ldh); row(p.gate, p.ldg);
  for (const BlockNorm *n : {&p.after, &p.before}) {
    row(n->weight, 0);
    row(n->bias, 0);
  }
  if (p.x_dtype == TX_F32)
    return p.y_dtype == TX_F32 ? run_types<float, float>(p, stream)
                               : run_types<float, uint16_t>(p, stream);
  return p.y_dtype == TX_F32 ? run_types<uint16_t, float>(p, stream)
                             : run_types<uint16_t, uint16_t>(p, stream);
}

}  // namespace tx
