// npu_gated_add_rms_norm: the norm after a block, the block's gate and residual scale, and the norm before the next
// block in one pass, with its gradient and a form that quantises the rows for the next int8 matmul.
//
//   z = x * r1 * w1          r1 = 1 / sqrt(mean(x^2) + eps)      (without post_gamma: z = x)
//   h = a * residual + g * z                                     (without gate: g = 1)
//   y = h * r2 * w2          r2 = 1 / sqrt(mean(h^2) + eps)
//
// gradient, for dy and dh' (the gradient that reaches h directly), xn = x r1, hn = h r2:
//   u  = dy * w2             dh = dh' + r2 * (u - hn * mean(u * hn))      dw2 = sum over rows of dy * hn
//   dresidual = a * dh       dg = dh * z (summed to g's shape)            dz = dh * g
//   dw1 = sum over rows of dz * xn      v = dz * w1      dx = r1 * (v - xn * mean(v * xn))
//
// Bound by HBM: the forward pass reads x and the residual and writes y and h, the gradient reads x, the residual and both
// gradients and writes two, each once; a row stays in its CTA's registers between the reductions.  Everything between
// loading and storing is fp32: h is not rounded before its norm, and the gradient computes it again from x and the
// residual instead of reading the rounded one.  Sums over rows (dw1, dw2, a shared gate) are kept in registers by CTAs
// that take contiguous rows, written once per CTA as fp32 and added by a second kernel in a fixed order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"

namespace b200q {
namespace {

// A thread's place among the threads that share a row, and its columns: eight values i, VEC: eight neighbours
// (columns (i * threads + tid) * 8 ..), one or two 16-byte accesses; else columns (i * 8 + j) * threads + tid, one by one,
// for any width and alignment.
struct Place {
  int tid, threads;
  template <bool VEC>
  __device__ __forceinline__ int col(int i, int j) const {
    return VEC ? (i * threads + tid) * 8 + j : (i * 8 + j) * threads + tid;
  }
};

// Eight values as they lie in memory, and pairs of them as floats.
template <typename T>
struct Pack8 {
  uint4 v[sizeof(T) / 2];
};
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ row, int i, int width, const Place& at, Pack8<T>& raw) {
  const int c = at.col<VEC>(i, 0);
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < (int)sizeof(T) / 2; ++q)
      raw.v[q] = c < width ? ld_stream(reinterpret_cast<const uint4*>(row + c) + q) : make_uint4(0, 0, 0, 0);
  } else if constexpr (sizeof(T) == 4) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = c + j * at.threads < width ? __ldg(reinterpret_cast<const uint32_t*>(row) + c + j * at.threads) : 0u;
    raw.v[0] = make_uint4(w[0], w[1], w[2], w[3]);
    raw.v[1] = make_uint4(w[4], w[5], w[6], w[7]);
  } else {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = c + j * at.threads < width ? (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(row) + c + j * at.threads) : 0u;
    raw.v[0] = make_uint4(w[0] | (w[1] << 16), w[2] | (w[3] << 16), w[4] | (w[5] << 16), w[6] | (w[7] << 16));
  }
}
template <typename T>
__device__ __forceinline__ float2 pair_of(const Pack8<T>& raw, int j) {   // values 2j, 2j+1
  const uint4& q = raw.v[sizeof(T) == 4 ? j >> 1 : 0];
  if constexpr (sizeof(T) == 4) return (j & 1) ? make_float2(__uint_as_float(q.z), __uint_as_float(q.w)) : make_float2(__uint_as_float(q.x), __uint_as_float(q.y));
  else return unpack2<T>(j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w);
}
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float2 v) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __float22half2_rn(v);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __float22bfloat162_rn(v);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ T narrow(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* __restrict__ row, int i, int width, const Place& at, const float2 (&f)[4]) {
  const int c = at.col<VEC>(i, 0);
  if constexpr (VEC) {
    if (c >= width) return;
    if constexpr (sizeof(T) == 4) {
      __stcs(reinterpret_cast<float4*>(row + c), make_float4(f[0].x, f[0].y, f[1].x, f[1].y));
      __stcs(reinterpret_cast<float4*>(row + c) + 1, make_float4(f[2].x, f[2].y, f[3].x, f[3].y));
    } else {
      __stcs(reinterpret_cast<uint4*>(row + c), make_uint4(pack_pair<T>(f[0]), pack_pair<T>(f[1]), pack_pair<T>(f[2]), pack_pair<T>(f[3])));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j * at.threads < width) row[c + j * at.threads] = narrow<T>((j & 1) ? f[j >> 1].y : f[j >> 1].x);
  }
}

// Eight parameter values.  Past the width the last column's are read: they only ever meet zeros there.
template <typename P, bool VEC>
__device__ __forceinline__ void param8(const P* __restrict__ p, int i, int width, const Place& at, float2 (&f)[4]) {
  const int c = at.col<VEC>(i, 0);
  if constexpr (VEC) {
    load_smooth8(p + min(c, width - 8), f);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      f[j] = make_float2(to_f32<P>(p[min(c + 2 * j * at.threads, width - 1)]), to_f32<P>(p[min(c + (2 * j + 1) * at.threads, width - 1)]));
  }
}

// The gate of a row: rows_per consecutive rows share row `row / rows_per` of p, which is one value (per_row) or `width`.
struct Gate {
  const void* p;
  int per_row;
  int64_t rows_per;
};
template <typename P, bool VEC>
__device__ __forceinline__ void gate8(const Gate& g, int64_t gate_row, int i, int width, const Place& at, float2 (&f)[4]) {
  if (g.p == nullptr || g.per_row) {
    const float v = g.p == nullptr ? 1.0f : to_f32<P>(static_cast<const P*>(g.p)[gate_row]);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = make_float2(v, v);
  } else {
    param8<P, VEC>(static_cast<const P*>(g.p) + gate_row * width, i, width, at, f);
  }
}

__device__ __forceinline__ float2 splat(float v) { return make_float2(v, v); }

// Sums of N values over the threads of a row; `red` must not be in use by an earlier call (two buffers, used in turn).
// `barrier`: named barrier of the row's threads (a single warp needs none).
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*red)[32], const Place& at, int barrier) {
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if (at.threads == 32) return;
  const int warp = at.tid >> 5, lane = at.tid & 31, nwarps = at.threads >> 5;
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (lane == 0) red[k][warp] = v[k];
  named_barrier_sync(barrier, at.threads);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    v[k] = lane < nwarps ? red[k][lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
}

__device__ __forceinline__ float rstd_of(float sum, float inv_width, float eps) {
  return __frsqrt_rn(__fadd_rn(__fmul_rn(sum, inv_width), eps));
}

struct NormArgs {
  const void* x;
  const void* residual;
  void* y;
  void* h;
  float* rstd;
  float* post_rstd;
  float* scale;              // quantised form: y is int8 with this scale a row
  const void* gamma;
  const void* post;
  const void* smooth;
  int smooth_f32;
  Gate gate;
  float alpha, eps, inv_width;
  int64_t rows;
  int width;
};

// One CTA a row at a time.  The next row's x and residual are in flight from the moment this row's have become h.  With
// ITERS 1 (rows spread over many threads: few rows, where latency counts) the parameters are loaded with the row, not behind
// the reductions.
template <typename T, typename P, bool VEC, int ITERS, bool QUANT, int MAX_THREADS>
__global__ void __launch_bounds__(MAX_THREADS)
gated_norm_kernel(const NormArgs a) {
  constexpr bool EARLY = ITERS == 1;
  __shared__ float red[3][1][32];
  const Place at{(int)threadIdx.x, (int)blockDim.x};
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.residual);
  const P* gamma = static_cast<const P*>(a.gamma);
  const P* post = static_cast<const P*>(a.post);
  auto smooth8 = [&](int i, float2(&f)[4]) {
    if (a.smooth_f32) param8<float, VEC>(static_cast<const float*>(a.smooth), i, a.width, at, f);
    else param8<T, VEC>(static_cast<const T*>(a.smooth), i, a.width, at, f);
  };
  Pack8<T> xr[ITERS], rr[ITERS];
  auto load_row = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      load8<T, VEC>(x + row * a.width, i, a.width, at, xr[i]);
      load8<T, VEC>(res + row * a.width, i, a.width, at, rr[i]);
    }
  };
  if ((int64_t)blockIdx.x < a.rows) load_row(blockIdx.x);
  float2 early_post[4], early_gamma[4], early_smooth[4];
  if constexpr (EARLY) {
    if (post != nullptr) param8<P, VEC>(post, 0, a.width, at, early_post);
    param8<P, VEC>(gamma, 0, a.width, at, early_gamma);
    if (QUANT && a.smooth != nullptr) smooth8(0, early_smooth);
  }
  const float2 alpha = splat(a.alpha);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t gate_row = a.gate.rows_per == 1 ? row : row / a.gate.rows_per;
    float2 early_gate[4];
    if constexpr (EARLY) gate8<P, VEC>(a.gate, gate_row, 0, a.width, at, early_gate);
    float r1 = 1.0f;
    if (post != nullptr) {
      float2 s2 = splat(0.0f);
#pragma unroll
      for (int i = 0; i < ITERS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 v = pair_of<T>(xr[i], j);
          s2 = __ffma2_rn(v, v, s2);
        }
      float s[1] = {s2.x + s2.y};
      row_sum<1>(s, red[0], at, 1);
      r1 = rstd_of(s[0], a.inv_width, a.eps);
      if (threadIdx.x == 0 && a.post_rstd != nullptr) a.post_rstd[row] = r1;
    }
    float2 h[ITERS][4];
    float2 s2 = splat(0.0f);
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      float2 g[4], w[4];
      if constexpr (!EARLY) {
        gate8<P, VEC>(a.gate, gate_row, i, a.width, at, g);
        if (post != nullptr) param8<P, VEC>(post, i, a.width, at, w);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 z = pair_of<T>(xr[i], j);
        if (post != nullptr) z = __fmul2_rn(__fmul2_rn(z, splat(r1)), EARLY ? early_post[j] : w[j]);
        h[i][j] = __ffma2_rn(EARLY ? early_gate[j] : g[j], z, __fmul2_rn(alpha, pair_of<T>(rr[i], j)));
        s2 = __ffma2_rn(h[i][j], h[i][j], s2);
      }
      store8<T, VEC>(static_cast<T*>(a.h) + row * a.width, i, a.width, at, h[i]);
    }
    if (row + gridDim.x < a.rows) load_row(row + gridDim.x);
    float s[1] = {s2.x + s2.y};
    row_sum<1>(s, red[1], at, 1);
    const float r2 = rstd_of(s[0], a.inv_width, a.eps);
    if (threadIdx.x == 0 && a.rstd != nullptr) a.rstd[row] = r2;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      float2 w[4], sm[4];
      if constexpr (!EARLY) {
        param8<P, VEC>(gamma, i, a.width, at, w);
        if (QUANT && a.smooth != nullptr) smooth8(i, sm);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 y = __fmul2_rn(__fmul2_rn(h[i][j], splat(r2)), EARLY ? early_gamma[j] : w[j]);
        if (QUANT) {
          if (a.smooth != nullptr) y = __fmul2_rn(y, EARLY ? early_smooth[j] : sm[j]);
          amax = fmaxf(amax, fmaxf(fabsf(y.x), fabsf(y.y)));
        }
        h[i][j] = y;
      }
      if (!QUANT) store8<T, VEC>(static_cast<T*>(a.y) + row * a.width, i, a.width, at, h[i]);
    }
    if constexpr (QUANT) {
      amax = block_max(amax, red[2][0]);
      const float scale = scale_of_amax(amax);
      if (threadIdx.x == 0) a.scale[row] = scale;
      const float inv = quant_inverse(scale);
      int8_t* q = static_cast<int8_t*>(a.y) + row * a.width;
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
        const uint2 o = inv == inv ? quantize8<false>(h[i], scale, inv) : quantize8<true>(h[i], scale, inv);
        const int c = at.col<VEC>(i, 0);
        if constexpr (VEC) {
          if (c < a.width) st_stream(reinterpret_cast<uint2*>(q + c), o);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (c + j * at.threads < a.width) q[c + j * at.threads] = (int8_t)(((j < 4 ? o.x : o.y) >> (8 * (j & 3))) & 0xff);
        }
      }
    }
    // The buffers of one row are written again for the next one only behind another buffer's barrier, except when a row
    // has a single reduction.
    if (post == nullptr && !QUANT) __syncthreads();
  }
}

struct NormGradArgs {
  const void* dy;
  const void* dh;            // or NULL
  const void* x;
  const void* residual;
  const float* rstd;
  const float* post_rstd;
  const void* gamma;
  const void* post;
  Gate gate;
  void* dx;
  void* dres;
  void* dgate;               // written here when every element of the gate has its own row (or is one value a row)
  float* part_gamma;         // [CTAs, width] sums of the CTA's rows
  float* part_post;          // the same
  float* part_gate;          // [CTAs + gates - 1, width]: CTA c's rows of gate g at c + g
  float alpha, inv_width;
  int64_t rows;
  int width;
};

constexpr int kNormGradThreads = 512;     // at most: the sums over rows need up to 128 registers a thread

// A CTA takes the rows [rows * c / CTAs, rows * (c + 1) / CTAs), `threads_per_row` threads a row and as many rows at a time as
// fit into the CTA.  Its threads keep the same columns throughout, so the sums over its rows stay with them: in registers
// while a row is one vector a thread (ITERS 1), else in shared memory, in two planes of four columns a vector, so that a
// warp's 16-byte accesses touch every bank once.  At the end (for a gate: at the end of the gate's rows) the CTA's row groups
// add theirs in shared memory in a fixed order and one partial row goes out.  SUM_GATE: the gate's gradient is a sum over the
// rows that share a gate; without it there is no gate, or one value a row, or one gate a row.
template <typename T, typename P, bool VEC, int ITERS, bool SUM_GATE>
__global__ void __launch_bounds__(kNormGradThreads, 1)
gated_norm_grad_kernel(const NormGradArgs a, int threads_per_row) {
  constexpr bool SHARED = ITERS > 1;
  extern __shared__ float4 column_sums[];                  // SHARED: gamma's, post gamma's and the gate's sums; else [width] floats
  __shared__ float red[2][kNormGradThreads / 32][2][32];
  const int group = threadIdx.x / threads_per_row, groups = blockDim.x / threads_per_row;
  const Place at{(int)threadIdx.x - group * threads_per_row, threads_per_row};
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.residual);
  const T* dy = static_cast<const T*>(a.dy);
  const T* dhp = static_cast<const T*>(a.dh);
  const P* gamma = static_cast<const P*>(a.gamma);
  const P* post = static_cast<const P*>(a.post);
  const float2 alpha = splat(a.alpha);
  float2 sums[3][4];                                       // gamma, post gamma, gate; of the vector at hand when SHARED
#pragma unroll
  for (int w = 0; w < 3; ++w)
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[w][j] = splat(0.0f);
  auto place = [&](int w, int half, int i) -> float4& { return column_sums[((2 * w + half) * ITERS + i) * threads_per_row + at.tid]; };
  auto fetch = [&](int w, int i) {
    if constexpr (SHARED) {
      const float4 p = place(w, 0, i), q = place(w, 1, i);
      sums[w][0] = make_float2(p.x, p.y), sums[w][1] = make_float2(p.z, p.w), sums[w][2] = make_float2(q.x, q.y), sums[w][3] = make_float2(q.z, q.w);
    }
  };
  auto put = [&](int w, int i) {
    if constexpr (SHARED) {
      place(w, 0, i) = make_float4(sums[w][0].x, sums[w][0].y, sums[w][1].x, sums[w][1].y);
      place(w, 1, i) = make_float4(sums[w][2].x, sums[w][2].y, sums[w][3].x, sums[w][3].y);
    }
  };
  auto clear = [&](int w) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[w][j] = splat(0.0f);
#pragma unroll
    for (int i = 0; i < ITERS; ++i) put(w, i);
  };
  clear(0), clear(1), clear(2);
  // Adds the groups' sums and stores them as one row; called by the whole CTA.
  auto flush = [&](int w, float* to) {
    if (!SHARED && groups > 1) {
      float* joined = reinterpret_cast<float*>(column_sums);
      for (int g = 0; g < groups; ++g) {
        if (g == group) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int c = at.col<VEC>(0, j);
            const float v = (j & 1) ? sums[w][j >> 1].y : sums[w][j >> 1].x;
            if (c < a.width) joined[c] = g == 0 ? v : joined[c] + v;
          }
        }
        __syncthreads();
      }
      for (int c = threadIdx.x; c < a.width; c += blockDim.x) to[c] = joined[c];
      __syncthreads();
    } else {
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
        fetch(w, i);
        store8<float, VEC>(to, i, a.width, at, sums[w]);
      }
    }
  };
  const int64_t r0 = a.rows * blockIdx.x / gridDim.x, r1 = a.rows * (blockIdx.x + 1) / gridDim.x;
  int64_t seg = r0;
  while (seg < r1) {
    const int64_t gate = SUM_GATE ? seg / a.gate.rows_per : 0;
    const int64_t seg_end = SUM_GATE ? min(r1, (gate + 1) * a.gate.rows_per) : r1;
    Pack8<T> xr[ITERS], rr[ITERS], yr[ITERS], hr[ITERS];
    float rs2 = 0.0f, rs1 = 1.0f;
    auto load_x = [&](int64_t row) {
#pragma unroll
      for (int i = 0; i < ITERS; ++i) load8<T, VEC>(x + row * a.width, i, a.width, at, xr[i]);
      rs2 = a.rstd[row];
      if (post != nullptr) rs1 = a.post_rstd[row];
    };
    auto load_rest = [&](int64_t row) {
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
        load8<T, VEC>(res + row * a.width, i, a.width, at, rr[i]);
        load8<T, VEC>(dy + row * a.width, i, a.width, at, yr[i]);
        if (dhp != nullptr) load8<T, VEC>(dhp + row * a.width, i, a.width, at, hr[i]);
      }
    };
    if (seg + group < seg_end) {
      load_x(seg + group);
      load_rest(seg + group);
    }
#pragma unroll 1
    for (int64_t row = seg + group; row < seg_end; row += groups) {
      const int64_t gate_row = SUM_GATE ? gate : row;
      const bool more = row + groups < seg_end;
      const float2 s1 = splat(rs1), s2 = splat(rs2);
      // xn, z and hn of one pair of columns
      auto normed = [&](int i, int j, const float2(&g)[4], const float2(&w1)[4], float2& xn, float2& z) {
        const float2 v = pair_of<T>(xr[i], j);
        xn = __fmul2_rn(v, s1);
        z = post != nullptr ? __fmul2_rn(xn, w1[j]) : v;
        return __fmul2_rn(__ffma2_rn(g[j], z, __fmul2_rn(alpha, pair_of<T>(rr[i], j))), s2);
      };
      float2 dot2 = splat(0.0f);
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
        float2 g[4], w1[4], w2[4];
        gate8<P, VEC>(a.gate, gate_row, i, a.width, at, g);
        if (post != nullptr) param8<P, VEC>(post, i, a.width, at, w1);
        param8<P, VEC>(gamma, i, a.width, at, w2);
        fetch(0, i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float2 xn, z;
          const float2 hn = normed(i, j, g, w1, xn, z);
          const float2 d = __fmul2_rn(pair_of<T>(yr[i], j), hn);
          dot2 = __ffma2_rn(d, w2[j], dot2);
          sums[0][j] = __fadd2_rn(sums[0][j], d);
        }
        put(0, i);
      }
      float dot[1] = {dot2.x + dot2.y};
      row_sum<1>(dot, red[0][group], at, 1 + group);
      const float2 nc2 = splat(-dot[0] * a.inv_width);
      float2 dots_v = splat(0.0f), dots_g = splat(0.0f);   // v . xn, dh . z
      float2 keep[ITERS][4];                               // v
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
        float2 g[4], w1[4], w2[4], out[4], dg[4];
        gate8<P, VEC>(a.gate, gate_row, i, a.width, at, g);
        if (post != nullptr) param8<P, VEC>(post, i, a.width, at, w1);
        param8<P, VEC>(gamma, i, a.width, at, w2);
        if (post != nullptr) fetch(1, i);
        if (SUM_GATE) fetch(2, i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float2 xn, z;
          const float2 hn = normed(i, j, g, w1, xn, z);
          const float2 u = __fmul2_rn(pair_of<T>(yr[i], j), w2[j]);
          float2 dh = __fmul2_rn(s2, __ffma2_rn(hn, nc2, u));
          if (dhp != nullptr) dh = __fadd2_rn(dh, pair_of<T>(hr[i], j));
          out[j] = __fmul2_rn(alpha, dh);
          if (SUM_GATE) {
            sums[2][j] = __ffma2_rn(dh, z, sums[2][j]);
          } else {
            dg[j] = __fmul2_rn(dh, z);
            dots_g = __fadd2_rn(dots_g, dg[j]);
          }
          float2 dz = __fmul2_rn(dh, g[j]);
          if (post != nullptr) {
            const float2 t = __fmul2_rn(dz, xn);
            sums[1][j] = __fadd2_rn(sums[1][j], t);
            dots_v = __ffma2_rn(t, w1[j], dots_v);
            dz = __fmul2_rn(dz, w1[j]);
          }
          keep[i][j] = dz;
        }
        if (post != nullptr) put(1, i);
        if (SUM_GATE) put(2, i);
        store8<T, VEC>(static_cast<T*>(a.dres) + row * a.width, i, a.width, at, out);
        // one gate a row: its gradient is dh * z itself
        if (!SUM_GATE && a.dgate != nullptr && !a.gate.per_row) store8<P, VEC>(static_cast<P*>(a.dgate) + row * a.width, i, a.width, at, dg);
      }
      if (more) load_rest(row + groups);                   // in flight from here on
      float dots[2] = {dots_v.x + dots_v.y, dots_g.x + dots_g.y};
      row_sum<2>(dots, red[1][group], at, 1 + group);
      const float2 nc1 = splat(-dots[0] * a.inv_width);
      if (!SUM_GATE && a.dgate != nullptr && a.gate.per_row && at.tid == 0) static_cast<P*>(a.dgate)[row] = narrow<P>(dots[1]);
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
        if (post != nullptr) {
#pragma unroll
          for (int j = 0; j < 4; ++j) keep[i][j] = __fmul2_rn(s1, __ffma2_rn(__fmul2_rn(pair_of<T>(xr[i], j), s1), nc1, keep[i][j]));
        }
        store8<T, VEC>(static_cast<T*>(a.dx) + row * a.width, i, a.width, at, keep[i]);
      }
      if (more) load_x(row + groups);
    }
    if constexpr (SUM_GATE) {
      flush(2, a.part_gate + (blockIdx.x + gate) * a.width);
      clear(2);
    }
    seg = seg_end;
  }
  flush(0, a.part_gamma + (int64_t)blockIdx.x * a.width);
  if (post != nullptr) flush(1, a.part_post + (int64_t)blockIdx.x * a.width);
}

// Adds the CTAs' partial sums: blockIdx.y 0 = gamma, 1 = post gamma, 2 + g = gate g.  A block owns 32 columns; its 32
// warps' lanes walk the partial rows in a fixed order.
struct NormSumArgs {
  const float* part_gamma;
  const float* part_post;
  const float* part_gate;
  void* dgamma;
  void* dpost;
  void* dgate;
  int dtype;                 // of the parameters
  int64_t rows, rows_per, width;
  int ctas;
};

__global__ void __launch_bounds__(1024)
gated_norm_sum_kernel(const NormSumArgs a) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  const float* part = blockIdx.y == 0 ? a.part_gamma : blockIdx.y == 1 ? a.part_post : a.part_gate;
  if (part == nullptr) return;
  int64_t p0 = 0, p1 = a.ctas, g = 0;
  if (blockIdx.y >= 2) {
    // the CTAs whose rows [rows c / ctas, rows (c + 1) / ctas) meet the gate's rows [g rows_per, (g + 1) rows_per)
    g = blockIdx.y - 2;
    const int64_t first = g * a.rows_per, last = min(a.rows, first + a.rows_per) - 1;
    // floor(rows c / ctas) <= r  <=>  c < (r + 1) ctas / rows: the CTA of row `first`, and one past that of row `last`
    p0 = ((first + 1) * a.ctas + a.rows - 1) / a.rows - 1;
    p1 = ((last + 1) * a.ctas + a.rows - 1) / a.rows;
    if (p1 > a.ctas) p1 = a.ctas;
    p0 += g;
    p1 += g;
  }
  float s = 0.0f;
  if (c < a.width)
    for (int64_t p = p0 + warp; p < p1; p += 32) s += part[p * a.width + c];
  red[warp][lane] = s;
  __syncthreads();
  s = red[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int64_t col = (int64_t)blockIdx.x * 32 + warp;
  if (lane == 0 && col < a.width) {
    if (blockIdx.y == 0) store_from_f32(a.dgamma, a.dtype, col, s);
    else if (blockIdx.y == 1) store_from_f32(a.dpost, a.dtype, col, s);
    else store_from_f32(a.dgate, a.dtype, g * a.width + col, s);
  }
}

constexpr int kNormMaxWidth = 16384;

// Vectors of eight need a width that they divide and 16-byte aligned rows and parameters.
inline bool norm_vec(int64_t width, std::initializer_list<const void*> ptrs) {
  if (width % 8 != 0) return false;
  for (const void* p : ptrs)
    if (!aligned(p, 16)) return false;
  return true;
}

// Few rows (no more than SMs): as many threads a row as it has vectors, for the shortest way through a row.  Otherwise
// 256 threads or fewer with up to four vectors each, so that several rows are in flight on an SM.
template <typename T, typename P, bool VEC, bool QUANT>
int launch_norm(const NormArgs& a, cudaStream_t st) {
  const int64_t vecs = ceil_div(a.width, 8);
  int iters = vecs > 1024 ? 4 : 1;
  if (a.rows > sm_count())
    while (iters < 4 && vecs > iters * 256) iters *= 2;
  const int threads = (int)ceil_div(ceil_div(vecs, iters), 32) * 32;
#define B200Q_NORM(I, MAX)                                                                       \
  {                                                                                              \
    constexpr auto kern = gated_norm_kernel<T, P, VEC, I, QUANT, MAX>;                           \
    const int64_t cap = (int64_t)sm_count() * resident_ctas<kern>(threads);                      \
    kern<<<(unsigned)(a.rows < cap ? a.rows : cap), threads, 0, st>>>(a);                        \
  }
  if (iters == 1) B200Q_NORM(1, 1024) else if (iters == 2) B200Q_NORM(2, 256) else B200Q_NORM(4, 512)
#undef B200Q_NORM
  return check_launch("gated_add_rms_norm");
}

// CTAs of the gradient kernel: one an SM, each of which writes one row of partial sums per parameter.
inline int grad_ctas(int64_t rows) {
  const int64_t cap = sm_count();
  return (int)(rows < cap ? rows : cap);
}

template <typename T, typename P, bool VEC>
int launch_norm_grad(const NormGradArgs& a, const NormSumArgs& s, bool sum_gate, cudaStream_t st) {
  // One vector a thread up to 4096 columns; the CTA's other threads take more rows at the same time.
  const int64_t vecs = ceil_div(a.width, 8);
  const int iters = vecs > 2 * kNormGradThreads ? 4 : vecs > kNormGradThreads ? 2 : 1;
  const int threads = (int)ceil_div(ceil_div(vecs, iters), 32) * 32;
  const int64_t most_rows = ceil_div(a.rows, s.ctas);
  int groups = kNormGradThreads / threads;
  if (groups > 15 && threads > 32) groups = 15;             // named barriers 1 .. 15
  if (groups > most_rows) groups = (int)most_rows;
  // Sums of every column (three, two planes of 16 bytes a vector: at most 192 KB), or one row for joining the groups.
  const int smem = iters > 1 ? 3 * 2 * 16 * iters * threads : groups > 1 ? (int)a.width * 4 : 0;
#define B200Q_NORM_GRAD_CASE(I)                                                                                                  \
  {                                                                                                                              \
    if (I > 1) {                                                                                                                 \
      constexpr int most = 3 * 2 * 16 * I * kNormGradThreads;                                                                    \
      if (int rc = ensure_dynamic_smem<gated_norm_grad_kernel<T, P, VEC, I, true>>(most, "gated_add_rms_norm_grad")) return rc;  \
      if (int rc = ensure_dynamic_smem<gated_norm_grad_kernel<T, P, VEC, I, false>>(most, "gated_add_rms_norm_grad")) return rc; \
    }                                                                                                                            \
    if (sum_gate) gated_norm_grad_kernel<T, P, VEC, I, true><<<s.ctas, groups * threads, smem, st>>>(a, threads);                \
    else gated_norm_grad_kernel<T, P, VEC, I, false><<<s.ctas, groups * threads, smem, st>>>(a, threads);                        \
  }
  if (iters == 1) B200Q_NORM_GRAD_CASE(1) else if (iters == 2) B200Q_NORM_GRAD_CASE(2) else B200Q_NORM_GRAD_CASE(4)
#undef B200Q_NORM_GRAD_CASE
  if (int rc = check_launch("gated_add_rms_norm_grad")) return rc;
  const int64_t gates = sum_gate ? ceil_div(a.rows, s.rows_per) : 0;
  dim3 grid((unsigned)ceil_div(a.width, 32), (unsigned)(2 + gates));
  gated_norm_sum_kernel<<<grid, 1024, 0, st>>>(s);
  return check_launch("gated_add_rms_norm_grad (sums)");
}

template <typename T, typename P>
int norm_forward(const NormArgs& a, bool quant, cudaStream_t st) {
  const bool vec = norm_vec(a.width, {a.x, a.residual, a.y, a.h, a.gamma, a.post, a.smooth, a.gate.per_row ? nullptr : a.gate.p});
  if (quant) return vec ? launch_norm<T, P, true, true>(a, st) : launch_norm<T, P, false, true>(a, st);
  return vec ? launch_norm<T, P, true, false>(a, st) : launch_norm<T, P, false, false>(a, st);
}

inline bool norm_dtype(int d) { return d == B200Q_BF16 || d == B200Q_F16 || d == B200Q_F32; }

// Does the gate's gradient add over rows?
inline bool gate_is_shared(const b200q_gated_norm_args& a) { return a.gate != nullptr && a.gate_rows > 1; }

int norm_checks(const b200q_gated_norm_args& a, const char* op) {
  B200Q_REQUIRE(a.rows >= 0 && a.width >= 0, B200Q_ERR_BAD_ARG, "%s: negative size", op);
  B200Q_REQUIRE(norm_dtype(a.dtype), B200Q_ERR_UNSUPPORTED, "%s: x must be bf16, f16 or f32 (dtype enum %d)", op, a.dtype);
  B200Q_REQUIRE(a.width <= kNormMaxWidth && a.rows <= 0x7fffffffLL, B200Q_ERR_UNSUPPORTED, "%s: rows of %lld elements (at most %d)", op,
                (long long)a.width, kNormMaxWidth);
  B200Q_REQUIRE(a.param_dtype == a.dtype || a.param_dtype == B200Q_F32, B200Q_ERR_UNSUPPORTED,
                "%s: gamma, post_gamma and gate must all be f32 or all have x's dtype", op);
  B200Q_REQUIRE(a.gate == nullptr || a.gate_rows >= 1, B200Q_ERR_BAD_ARG, "%s: gate_rows must be at least 1", op);
  B200Q_REQUIRE(a.gate == nullptr || !a.gate_per_row || a.gate_rows == 1, B200Q_ERR_UNSUPPORTED, "%s: a gate of one value belongs to one row", op);
  return B200Q_OK;
}

bool norm_aligned(int dtype, std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (!aligned(p, dtype == B200Q_F32 ? 4 : 2)) return false;
  return true;
}

}  // namespace
}  // namespace b200q

#define B200Q_NORM_TYPES(dtype, param_dtype, CALL)                                          \
  if ((dtype) == B200Q_F32) return CALL(float, float);                                      \
  if ((dtype) == B200Q_BF16) {                                                              \
    if ((param_dtype) == B200Q_F32) return CALL(__nv_bfloat16, float);                      \
    return CALL(__nv_bfloat16, __nv_bfloat16);                                              \
  }                                                                                         \
  if ((param_dtype) == B200Q_F32) return CALL(__half, float);                               \
  return CALL(__half, __half);

extern "C" int b200q_gated_norm(const b200q_gated_norm_args* a, void* stream) {
  using namespace b200q;
  clear_error();
  constexpr const char* op = "gated_add_rms_norm";
  B200Q_REQUIRE(a != nullptr, B200Q_ERR_BAD_ARG, "%s: args is NULL", op);
  if (int rc = norm_checks(*a, op)) return rc;
  const bool quant = a->scale != nullptr;
  B200Q_REQUIRE(!quant || a->smooth == nullptr || a->smooth_dtype == B200Q_F32 || a->smooth_dtype == a->dtype, B200Q_ERR_UNSUPPORTED,
                "%s: smooth scales must be f32 or have x's dtype", op);
  B200Q_REQUIRE(quant || a->smooth == nullptr, B200Q_ERR_BAD_ARG, "%s: smooth scales belong to the quantised form (scale is NULL)", op);
  if (a->rows == 0) return B200Q_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->width == 0) {
    cudaError_t e = cudaSuccess;
    if (quant) e = cudaMemsetAsync(a->scale, 0, (size_t)a->rows * 4, st);
    return e == cudaSuccess ? B200Q_OK : fail(B200Q_ERR_LAUNCH, "%s: %s", op, cudaGetErrorString(e));
  }
  B200Q_REQUIRE(a->x != nullptr && a->residual != nullptr && a->y != nullptr && a->h != nullptr && a->gamma != nullptr, B200Q_ERR_BAD_ARG,
                "%s: NULL buffer", op);
  B200Q_REQUIRE(norm_aligned(a->dtype, {a->x, a->residual, a->h, quant ? nullptr : a->y}) && norm_aligned(a->param_dtype, {a->gamma, a->post_gamma, a->gate}) &&
                    norm_aligned(a->smooth_dtype, {a->smooth}) && norm_aligned(B200Q_F32, {a->rstd, a->post_rstd, a->scale}),
                B200Q_ERR_BAD_ARG, "%s: misaligned buffer", op);
  NormArgs n{};
  n.x = a->x; n.residual = a->residual; n.y = a->y; n.h = a->h; n.rstd = a->rstd; n.post_rstd = a->post_rstd; n.scale = a->scale;
  n.gamma = a->gamma; n.post = a->post_gamma;
  n.smooth = a->smooth; n.smooth_f32 = a->smooth_dtype == B200Q_F32;
  n.gate = {a->gate, a->gate_per_row, a->gate != nullptr ? a->gate_rows : 1};
  n.alpha = a->residual_scale; n.eps = a->epsilon; n.inv_width = 1.0f / (float)a->width;
  n.rows = a->rows; n.width = (int)a->width;
#define B200Q_CALL(T, P) norm_forward<T, P>(n, quant, st)
  B200Q_NORM_TYPES(a->dtype, a->param_dtype, B200Q_CALL)
#undef B200Q_CALL
}

extern "C" size_t b200q_gated_norm_grad_workspace_bytes(const b200q_gated_norm_args* a) {
  using namespace b200q;
  if (a == nullptr || a->rows <= 0 || a->width <= 0) return 0;
  const int64_t ctas = grad_ctas(a->rows);
  const int64_t gates = gate_is_shared(*a) ? ctas + ceil_div(a->rows, a->gate_rows) : 0;
  return (size_t)(2 * ctas + gates) * (size_t)a->width * 4;
}

extern "C" int b200q_gated_norm_grad(const b200q_gated_norm_args* a, const b200q_gated_norm_grads* g, void* stream) {
  using namespace b200q;
  clear_error();
  constexpr const char* op = "gated_add_rms_norm_grad";
  B200Q_REQUIRE(a != nullptr && g != nullptr, B200Q_ERR_BAD_ARG, "%s: args is NULL", op);
  if (int rc = norm_checks(*a, op)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool shared = gate_is_shared(*a);
  if (a->width == 0) return B200Q_OK;
  if (a->rows == 0) {
    const size_t bytes = (size_t)a->width * (a->param_dtype == B200Q_F32 ? 4 : 2);
    cudaError_t e = g->dgamma != nullptr ? cudaMemsetAsync(g->dgamma, 0, bytes, st) : cudaSuccess;
    if (e == cudaSuccess && a->post_gamma != nullptr && g->dpost_gamma != nullptr) e = cudaMemsetAsync(g->dpost_gamma, 0, bytes, st);
    return e == cudaSuccess ? B200Q_OK : fail(B200Q_ERR_LAUNCH, "%s: %s", op, cudaGetErrorString(e));
  }
  B200Q_REQUIRE(a->x != nullptr && a->residual != nullptr && a->gamma != nullptr && a->rstd != nullptr && g->dy != nullptr && g->dx != nullptr &&
                    g->dresidual != nullptr && g->dgamma != nullptr && (a->post_gamma == nullptr || (a->post_rstd != nullptr && g->dpost_gamma != nullptr)) &&
                    (a->gate == nullptr || g->dgate != nullptr),
                B200Q_ERR_BAD_ARG, "%s: NULL buffer", op);
  B200Q_REQUIRE(norm_aligned(a->dtype, {a->x, a->residual, g->dy, g->dh, g->dx, g->dresidual}) &&
                    norm_aligned(a->param_dtype, {a->gamma, a->post_gamma, a->gate, g->dgamma, g->dpost_gamma, g->dgate}) &&
                    norm_aligned(B200Q_F32, {a->rstd, a->post_rstd}),
                B200Q_ERR_BAD_ARG, "%s: misaligned buffer", op);
  const int64_t gates = shared ? ceil_div(a->rows, a->gate_rows) : 0;
  B200Q_REQUIRE(gates <= 65533, B200Q_ERR_UNSUPPORTED, "%s: more than 65533 gates that are shared by several rows", op);
  const size_t need = b200q_gated_norm_grad_workspace_bytes(a);
  B200Q_REQUIRE(g->workspace != nullptr && g->workspace_bytes >= need && aligned(g->workspace, 256), B200Q_ERR_WORKSPACE,
                "%s: needs %zu bytes of 256-byte aligned workspace, got %zu", op, need, g->workspace_bytes);
  const int ctas = grad_ctas(a->rows);
  // Partial rows lie `width` apart, so vectors of them are aligned exactly when the width allows vectors at all.
  float* part = static_cast<float*>(g->workspace);
  NormGradArgs n{};
  n.dy = g->dy; n.dh = g->dh; n.x = a->x; n.residual = a->residual; n.rstd = a->rstd; n.post_rstd = a->post_rstd;
  n.gamma = a->gamma; n.post = a->post_gamma;
  n.gate = {a->gate, a->gate_per_row, a->gate != nullptr ? a->gate_rows : 1};
  n.dx = g->dx; n.dres = g->dresidual; n.dgate = shared ? nullptr : (a->gate != nullptr ? g->dgate : nullptr);
  n.part_gamma = part; n.part_post = part + (int64_t)ctas * a->width; n.part_gate = shared ? part + 2 * (int64_t)ctas * a->width : nullptr;
  n.alpha = a->residual_scale; n.inv_width = 1.0f / (float)a->width;
  n.rows = a->rows; n.width = (int)a->width;
  NormSumArgs s{};
  s.part_gamma = n.part_gamma; s.part_post = a->post_gamma != nullptr ? n.part_post : nullptr; s.part_gate = n.part_gate;
  s.dgamma = g->dgamma; s.dpost = g->dpost_gamma; s.dgate = g->dgate; s.dtype = a->param_dtype;
  s.rows = a->rows; s.rows_per = shared ? a->gate_rows : 1; s.width = a->width; s.ctas = ctas;
  const bool vec = norm_vec(a->width, {a->x, a->residual, g->dy, g->dh, g->dx, g->dresidual, a->gamma, a->post_gamma,
                                       a->gate_per_row ? nullptr : a->gate, a->gate_per_row || shared ? nullptr : g->dgate});
#define B200Q_CALL(T, P) (vec ? launch_norm_grad<T, P, true>(n, s, shared, st) : launch_norm_grad<T, P, false>(n, s, shared, st))
  B200Q_NORM_TYPES(a->dtype, a->param_dtype, B200Q_CALL)
#undef B200Q_CALL
}
#undef B200Q_NORM_TYPES
