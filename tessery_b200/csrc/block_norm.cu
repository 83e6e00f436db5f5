// The rows between two blocks of a layer in one pass (tx_block_norm):
//   z = y, or the experts' rows joined: z[t] = sum_j weights[t, j] y[places[t, j]]
//   r = x_scale x + y_scale gate * norm_after(z),   h = norm_before(r),
// a norm being RMS (v rsqrt(mean(v^2) + eps) (w + offset) + b), LayerNorm (the same of v - mean(v)) or
// none.  Everything is fp32 from the loads to the one rounding of each output; h is the norm of r as it
// is before r is rounded.  The joined sum runs in the order of j, and a row whose place is negative is not read.
//
// Bound: HBM, each row read once and written once.  A row is W warps with C vectors of V elements a thread in
// registers, so that the mean and the deviations of a LayerNorm are two passes over registers, and its words
// are loaded a row ahead.  Measured: 33500 rows of 1024, normed on both sides (412 MB): 71 us, 5.8 TB/s; 8192
// rows of 1024 joined from 8 experts' with a gate by sequence (219 MB): 48 us, 4.5 TB/s; 8 rows: 8 us.  A warp
// a row without loads ahead (100 registers, 16 warps an SM) took 79 and 66 us; rows through a ring in shared
// memory filled by bulk copies 112 and 60 us; half as many warps with twice the vectors 76 and 68 us.
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/tessattn.h"
#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace tx {
namespace {

// V elements of fp32 or bf16 as they lie in memory.
template <int V, typename T>
struct Words {
  static constexpr int kWords = V * (int)sizeof(T) / 4;
  uint32_t w[kWords ? kWords : 1];
  __device__ __forceinline__ void load(const void *base, int, size_t at) {
    const T *p = static_cast<const T *>(base) + at;
    if constexpr (V == 1) {
      if constexpr (sizeof(T) == 4)
        w[0] = __float_as_uint(*p);
      else
        w[0] = (uint32_t)*p << 16;
    } else if constexpr (kWords == 2) {
      const uint2 v = *reinterpret_cast<const uint2 *>(p);
      w[0] = v.x; w[1] = v.y;
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
// The same with the type looked up as they are loaded.
struct Any {};
template <int V>
struct Words<V, Any> {
  float f[V];
  __device__ __forceinline__ void load(const void *base, int dtype, size_t at) {
    if (dtype == TX_BF16) {
      Words<V, uint16_t> r;
      r.load(base, dtype, at);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = r.at(i);
    } else {
      Words<V, float> r;
      r.load(base, dtype, at);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = r.at(i);
    }
  }
  __device__ __forceinline__ float at(int i) const { return f[i]; }
};

// V values in fp32, in pairs that one instruction works on (one value: alone).
template <int V>
struct Row {
  uint64_t p[V / 2];
  __device__ __forceinline__ void fill(float x) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) p[i] = ptx::f2(x, x);
  }
  template <typename W>
  __device__ __forceinline__ void from(const W &w) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) p[i] = ptx::f2(w.at(2 * i), w.at(2 * i + 1));
  }
  __device__ __forceinline__ void add(float x) {
    const uint64_t y = ptx::f2(x, x);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) p[i] = ptx::add2(p[i], y);
  }
  __device__ __forceinline__ void add(const Row &b) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) p[i] = ptx::add2(p[i], b.p[i]);
  }
  __device__ __forceinline__ void mul(float x) {
    const uint64_t y = ptx::f2(x, x);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) p[i] = ptx::mul2(p[i], y);
  }
  __device__ __forceinline__ void mul(const Row &b) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) p[i] = ptx::mul2(p[i], b.p[i]);
  }
  // this + x b
  __device__ __forceinline__ void fma(float x, const Row &b) {
    const uint64_t y = ptx::f2(x, x);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) p[i] = ptx::fma2(y, b.p[i], p[i]);
  }
  __device__ __forceinline__ float sum() const {
    uint64_t s = p[0];
#pragma unroll
    for (int i = 1; i < V / 2; ++i) s = ptx::add2(s, p[i]);
    const float2 f = ptx::f2_unpack(s);
    return f.x + f.y;
  }
  __device__ __forceinline__ float squares() const {
    uint64_t s = ptx::mul2(p[0], p[0]);
#pragma unroll
    for (int i = 1; i < V / 2; ++i) s = ptx::fma2(p[i], p[i], s);
    const float2 f = ptx::f2_unpack(s);
    return f.x + f.y;
  }
  __device__ __forceinline__ void store(void *base, int dtype, size_t at) const {
    float2 f[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) f[i] = ptx::f2_unpack(p[i]);
    if (dtype == TX_BF16) {
      uint16_t *to = static_cast<uint16_t *>(base) + at;
      if constexpr (V == 4)
        *reinterpret_cast<uint2 *>(to) =
            make_uint2(pack_bf16x2(f[0].x, f[0].y), pack_bf16x2(f[1].x, f[1].y));
      else
        *reinterpret_cast<uint4 *>(to) =
            make_uint4(pack_bf16x2(f[0].x, f[0].y), pack_bf16x2(f[1].x, f[1].y),
                       pack_bf16x2(f[2].x, f[2].y), pack_bf16x2(f[3].x, f[3].y));
    } else {
      float4 *to = reinterpret_cast<float4 *>(static_cast<float *>(base) + at);
#pragma unroll
      for (int i = 0; i < V / 4; ++i)
        to[i] = make_float4(f[2 * i].x, f[2 * i].y, f[2 * i + 1].x, f[2 * i + 1].y);
    }
  }
};
template <>
struct Row<1> {
  float s;
  __device__ __forceinline__ void fill(float x) { s = x; }
  template <typename W>
  __device__ __forceinline__ void from(const W &w) {
    s = w.at(0);
  }
  __device__ __forceinline__ void add(float x) { s += x; }
  __device__ __forceinline__ void add(const Row &b) { s += b.s; }
  __device__ __forceinline__ void mul(float x) { s *= x; }
  __device__ __forceinline__ void mul(const Row &b) { s *= b.s; }
  __device__ __forceinline__ void fma(float x, const Row &b) { s = fmaf(x, b.s, s); }
  __device__ __forceinline__ float sum() const { return s; }
  __device__ __forceinline__ float squares() const { return s * s; }
  __device__ __forceinline__ void store(void *base, int dtype, size_t at) const {
    if (dtype == TX_BF16)
      static_cast<uint16_t *>(base)[at] = f32_to_bf16_bits(s);
    else
      static_cast<float *>(base)[at] = s;
  }
};
template <int V>
__device__ __forceinline__ Row<V> load_row(const void *base, int dtype, size_t at) {
  Row<V> r;
  if (dtype == TX_BF16) {
    Words<V, uint16_t> w;
    w.load(base, dtype, at);
    r.from(w);
  } else {
    Words<V, float> w;
    w.load(base, dtype, at);
    r.from(w);
  }
  return r;
}

// The W warps of a row: their sums meet in shared memory, in two buffers by turns (who writes one again has
// passed the barrier of the other, before which all had read it).
template <int W>
struct RowTeam {
  float (*buf)[W];  // [2][W]
  uint32_t barrier;  // 1 or 2
  int turn;
  __device__ __forceinline__ float sum(float v) {
    v = warp_sum(v);
    if constexpr (W > 1) {
      float *b = buf[turn++ & 1];
      if ((threadIdx.x & 31) == 0) b[threadIdx.x / 32 % W] = v;
      // (Barriers by a number that the compiler knows: otherwise a block holds all 16 of them, and four
      // blocks an SM's.)
      if (barrier == 1)
        asm volatile("bar.sync 1, %0;" ::"n"(32 * W) : "memory");
      else
        asm volatile("bar.sync 2, %0;" ::"n"(32 * W) : "memory");
      v = b[0];
#pragma unroll
      for (int i = 1; i < W; ++i) v += b[i];
    }
    return v;
  }
};

// scale: a factor of all that comes out.
template <int W, int V, int C>
__device__ __forceinline__ void apply_norm(const BlockNorm &n, Row<V> (&v)[C], uint32_t cols,
                                           float inv_cols, uint32_t t, RowTeam<W> &team, float scale) {
  auto in = [&](int c) { return (t + c * 32 * W) * V < cols; };
  if (n.kind == TX_NORM_NONE) {
    if (scale != 1.f) {
#pragma unroll
      for (int c = 0; c < C; ++c) v[c].mul(scale);
    }
    return;
  }
  if (n.kind == TX_NORM_LAYER) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) s += v[c].sum();
    const float mean = team.sum(s) * inv_cols;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (in(c))
        v[c].add(-mean);
      else
        v[c].fill(0.f);
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) ss += v[c].squares();
  const float inv = rsqrtf(fmaf(team.sum(ss), inv_cols, n.eps)) * scale;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    v[c].mul(inv);
    if (!in(c)) continue;
    const size_t at = (size_t)(t + c * 32 * W) * V;
    if (n.weight) {
      Row<V> w = load_row<V>(n.weight, n.dtype, at);
      if (n.offset != 0.f) w.add(n.offset);
      v[c].mul(w);
    }
    if (n.bias) v[c].fma(scale, load_row<V>(n.bias, n.dtype, at));
  }
}

// Rows of a block, and blocks of an SM as registers allow.
template <int W, int C, int V>
struct Shape {
  static constexpr int kRows = W >= 4 ? 1 : W == 1 ? 4 : 2;
  static constexpr int kThreads = 32 * W * kRows;
  static constexpr int kWide = C * V >= 32 ? 512 : C * V >= 16 ? 768 : 1024;
  static constexpr int kResident = kWide / kThreads > 0 ? kWide / kThreads : 1;
};

template <typename XT, typename YT, int W, int V, int C, bool kJoin>
__global__ void __launch_bounds__(Shape<W, C, V>::kThreads, Shape<W, C, V>::kResident)
    block_norm_kernel(const __grid_constant__ BlockNormProblem p) {
  constexpr int kRows = Shape<W, C, V>::kRows;
  constexpr int kFit = (W < 4 ? 64 : 128) / (C * (int)sizeof(Words<V, YT>));
  constexpr int kAhead = kFit < 1 ? 1 : kFit > 8 ? 8 : kFit;  // joined rows on their way at once
  __shared__ float buf[kRows][2][W];
  const uint32_t own = threadIdx.x / (32 * W), t = threadIdx.x % (32 * W), lane = threadIdx.x & 31;
  RowTeam<W> team{buf[own], 1 + own, 0};
  const uint32_t step = gridDim.x * kRows;
  const float inv_cols = 1.f / (float)p.cols;
  auto in = [&](int c) { return (t + c * 32 * W) * V < p.cols; };
  Words<V, XT> x[C];
  Words<V, YT> y[C];
  int32_t place = -1;
  float weight = 0.f;
  auto fetch = [&](uint32_t row) {
    if (row >= p.rows) return;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (!in(c)) continue;
      const size_t at = (size_t)(t + c * 32 * W) * V;
      if (p.x) x[c].load(p.x, p.x_dtype, (size_t)row * p.ldx + at);
      if (!kJoin && p.y) y[c].load(p.y, p.y_dtype, (size_t)row * p.ldy + at);
    }
    if (kJoin && lane < p.top_k) {
      place = __ldg(p.places + (size_t)row * p.top_k + lane);
      weight = __ldg(p.weights + (size_t)row * p.top_k + lane);
    }
  };
  uint32_t row = blockIdx.x * kRows + own;
  fetch(row);
  for (; row < p.rows; row += step) {
    Row<V> v[C], r[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      v[c].fill(0.f);
      r[c].fill(0.f);
      if (in(c)) {
        if (!kJoin && p.y) v[c].from(y[c]);
        if (p.x) r[c].from(x[c]);
      }
      r[c].mul(p.x_scale);
    }
    const int32_t here = place;
    const float here_weight = weight;
    fetch(row + step);
    if constexpr (kJoin) {
      if (lane < p.top_k && here >= 0 && (uint32_t)here >= p.y_rows)
        report_status(p.status, kStatusBadArg);
      for (uint32_t j0 = 0; j0 < p.top_k; j0 += kAhead) {
        Words<V, YT> z[kAhead][C];
        float w[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const uint32_t j = j0 + a;
          const uint32_t at = (uint32_t)__shfl_sync(0xffffffffu, here, j & 31);
          w[a] = __shfl_sync(0xffffffffu, here_weight, j & 31);
          const bool is = j < p.top_k && at < p.y_rows;  // a negative place is beyond all rows
          if (!is) w[a] = 0.f;
#pragma unroll
          for (int c = 0; c < C; ++c) {
            if (is && in(c)) {
              z[a][c].load(p.y, p.y_dtype, (size_t)at * p.ldy + (size_t)(t + c * 32 * W) * V);
            } else {
              z[a][c] = {};
            }
          }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
#pragma unroll
          for (int c = 0; c < C; ++c) {
            Row<V> f;
            f.from(z[a][c]);
            v[c].fma(w[a], f);
          }
      }
    }
    if (p.y) {
      apply_norm<W, V, C>(p.after, v, p.cols, inv_cols, t, team, p.y_scale);
      if (p.gate) {
        const uint32_t g = p.cu ? warp_find_seq(p.cu, p.gate_rows, row, lane) : p.seq ? row / p.seq : 0;
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (in(c))
            v[c].mul(load_row<V>(p.gate, p.gate_dtype, (size_t)g * p.ldg + (size_t)(t + c * 32 * W) * V));
      }
#pragma unroll
      for (int c = 0; c < C; ++c) r[c].add(v[c]);
    }
    if (p.out) {
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (in(c))
          r[c].store(p.out, p.out_dtype, (size_t)row * p.ldo + (size_t)(t + c * 32 * W) * V);
    }
    if (!p.h) continue;
    apply_norm<W, V, C>(p.before, r, p.cols, inv_cols, t, team, 1.f);
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (in(c)) r[c].store(p.h, p.h_dtype, (size_t)row * p.ldh + (size_t)(t + c * 32 * W) * V);
  }
}

template <typename XT, typename YT, int W, int V, int C>
cudaError_t run(const BlockNormProblem &p, int num_sms, cudaStream_t stream) {
  using S = Shape<W, C, V>;
  const uint32_t blocks = std::min<uint32_t>((p.rows + S::kRows - 1) / S::kRows,
                                             (uint32_t)(num_sms * S::kResident));
  if (p.places)
    block_norm_kernel<XT, YT, W, V, C, true><<<blocks, S::kThreads, 0, stream>>>(p);
  else
    block_norm_kernel<XT, YT, W, V, C, false><<<blocks, S::kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

// As many warps as the row has vectors for, up to 16.  (Above 8192 columns of fp32 in and out the 16-warp shape
// keeps 432 bytes a thread in local memory.  512 rows of 16384, fp32 and bf16 in: 41 us, the floor being 15.)
template <typename XT, typename YT>
cudaError_t run_vectors(const BlockNormProblem &p, int num_sms, cudaStream_t stream) {
  const uint32_t warps = (p.cols + 255) / 256;
  if (warps <= 1) return run<XT, YT, 1, 8, 1>(p, num_sms, stream);
  if (warps <= 2) return run<XT, YT, 2, 8, 1>(p, num_sms, stream);
  if (warps <= 3) return run<XT, YT, 3, 8, 1>(p, num_sms, stream);
  if (warps <= 4) return run<XT, YT, 4, 8, 1>(p, num_sms, stream);
  if (warps <= 8) return run<XT, YT, 8, 8, 1>(p, num_sms, stream);
  if (warps <= 16) return run<XT, YT, 8, 8, 2>(p, num_sms, stream);
  if (warps <= 32) return run<XT, YT, 16, 8, 2>(p, num_sms, stream);
  return run<XT, YT, 16, 8, 4>(p, num_sms, stream);
}
// Widths of whole fours: a warp for every 128 columns, then two and eight vectors a thread.  Both arguments' types
// are looked up as they are loaded, which costs: 8192 rows of 1020 take 43 us, of 1024 21.  Against shapes of as
// many warps as the row has vectors (16 at most), 8.4 million elements normed on both sides: 180 columns 84 / 49
// us, 252 64 / 38, 508 37 / 37, 516 72 / 65, 1020 43 / 39, 1500 43 / 53, 2044 35 / 43, 2052 129 / 47, 4092 87 / 33,
// 4100 89 / 70, 8188 67 / 57: few shapes serve all widths, at up to 2.7 times the time just above 128 and 2048.
// The widest shape and the widest of run_ones keep up to 368 bytes a thread in local memory.
cudaError_t run_fours(const BlockNormProblem &p, int num_sms, cudaStream_t stream) {
  const uint32_t warps = (p.cols + 127) / 128;
  if (warps <= 1) return run<Any, Any, 1, 4, 1>(p, num_sms, stream);
  if (warps <= 4) return run<Any, Any, 4, 4, 1>(p, num_sms, stream);
  if (warps <= 16) return run<Any, Any, 8, 4, 2>(p, num_sms, stream);
  return run<Any, Any, 16, 4, 8>(p, num_sms, stream);
}
// Rows that start anywhere, element by element, eight a thread where 16 warps hold them: bound by instructions
// and waits (8192 rows of 1023 take 70 us, of 1024 21).  Half as many warps as the next width wants: 33500 rows
// of 383 110 us with two warps, 144 with four; 2000 rows of 5001 with 16 elements a thread 174, with 32 312.
cudaError_t run_ones(const BlockNormProblem &p, int num_sms, cudaStream_t stream) {
  if (p.cols <= 32 * 8) return run<Any, Any, 1, 1, 8>(p, num_sms, stream);
  if (p.cols <= 64 * 8) return run<Any, Any, 2, 1, 8>(p, num_sms, stream);
  if (p.cols <= 128 * 8) return run<Any, Any, 4, 1, 8>(p, num_sms, stream);
  if (p.cols <= 256 * 8) return run<Any, Any, 8, 1, 8>(p, num_sms, stream);
  if (p.cols <= 512 * 8) return run<Any, Any, 16, 1, 8>(p, num_sms, stream);
  if (p.cols <= 512 * 16) return run<Any, Any, 16, 1, 16>(p, num_sms, stream);
  return run<Any, Any, 16, 1, 32>(p, num_sms, stream);
}

}  // namespace

cudaError_t launch_block_norm(const BlockNormProblem &p, int num_sms, cudaStream_t stream) {
  // The widest of 8, 4 and 1 elements in which every row is whole vectors on their boundaries.
  uint32_t v = p.cols % 8 == 0 ? 8 : p.cols % 4 == 0 ? 4 : 1;
  auto row = [&](const void *base, uint64_t ld, int dtype) {
    if (!base) return;
    while (v > 1 && (ld % v || (uintptr_t)base % std::min<uint64_t>(16, v * (dtype == TX_BF16 ? 2 : 4))))
      v = v == 8 ? 4 : 1;
  };
  row(p.x, p.ldx, p.x_dtype);
  row(p.y, p.ldy, p.y_dtype);
  row(p.out, p.ldo, p.out_dtype);
  row(p.h, p.ldh, p.h_dtype);
  row(p.gate, p.ldg, p.gate_dtype);
  for (const BlockNorm *n : {&p.after, &p.before}) {
    row(n->weight, 0, n->dtype);
    row(n->bias, 0, n->dtype);
  }
  if (v == 1) return run_ones(p, num_sms, stream);
  if (v == 4) return run_fours(p, num_sms, stream);
  if (p.x_dtype == TX_F32)
    return p.y_dtype == TX_F32 ? run_vectors<float, float>(p, num_sms, stream)
                               : run_vectors<float, uint16_t>(p, num_sms, stream);
  return p.y_dtype == TX_F32 ? run_vectors<uint16_t, float>(p, num_sms, stream)
                             : run_vectors<uint16_t, uint16_t>(p, num_sms, stream);
}

}  // namespace tx
