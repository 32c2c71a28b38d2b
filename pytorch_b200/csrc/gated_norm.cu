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

// A parameter vector (gamma, post gamma) or the gate: f32, bf16 or f16.
struct Param {
  const void* p;
  int dtype;
};
// Gate of row r, column c: p[(r / rows_per) * row_stride + (per_row ? 0 : c)].
struct Gate {
  const void* p;
  int dtype;
  int per_row;               // one value a row
  int64_t rows_per;          // consecutive rows that share a gate
  int64_t row_stride;        // elements between the gates
};

// Eight values of a thread.  VEC: eight neighbours (columns (i * threads + t) * 8 ..), one or two 16-byte accesses;
// else columns (i * 8 + j) * threads + t, one by one, for any width and alignment.
template <bool VEC>
__device__ __forceinline__ int col_of(int i, int j) {
  return VEC ? (i * (int)blockDim.x + (int)threadIdx.x) * 8 + j : (i * 8 + j) * (int)blockDim.x + (int)threadIdx.x;
}

template <typename T>
struct Pack8 {
  uint4 v[sizeof(T) / 2];
};

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ row, int i, int width, Pack8<T>& raw) {
  if constexpr (VEC) {
    const int c = col_of<true>(i, 0);
#pragma unroll
    for (int q = 0; q < (int)sizeof(T) / 2; ++q)
      raw.v[q] = c < width ? ld_stream(reinterpret_cast<const uint4*>(row + c) + q) : make_uint4(0, 0, 0, 0);
  } else {
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = col_of<false>(i, j);
      if (c < width) e[j] = row[c];
      else if constexpr (sizeof(T) == 4) e[j] = 0.0f;
      else reinterpret_cast<uint16_t*>(e)[j] = 0;
    }
  }
}
template <typename T>
__device__ __forceinline__ float2 pair_of(const Pack8<T>& raw, int j) {   // values 2j, 2j+1
  if constexpr (sizeof(T) == 4) {
    const float* f = reinterpret_cast<const float*>(&raw);
    return make_float2(f[2 * j], f[2 * j + 1]);
  } else {
    return unpack2<T>(reinterpret_cast<const uint32_t*>(&raw)[j]);
  }
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
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* __restrict__ row, int i, int width, const float2 (&f)[4]) {
  if constexpr (VEC) {
    const int c = col_of<true>(i, 0);
    if (c >= width) return;
    if constexpr (sizeof(T) == 4) {
      __stcs(reinterpret_cast<float4*>(row + c), make_float4(f[0].x, f[0].y, f[1].x, f[1].y));
      __stcs(reinterpret_cast<float4*>(row + c) + 1, make_float4(f[2].x, f[2].y, f[3].x, f[3].y));
    } else {
      __stcs(reinterpret_cast<uint4*>(row + c), make_uint4(pack_pair<T>(f[0]), pack_pair<T>(f[1]), pack_pair<T>(f[2]), pack_pair<T>(f[3])));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = col_of<false>(i, j);
      const float v = (j & 1) ? f[j >> 1].y : f[j >> 1].x;
      if (c >= width) continue;
      if constexpr (sizeof(T) == 4) row[c] = v;
      else if constexpr (std::is_same<T, __half>::value) row[c] = __float2half_rn(v);
      else row[c] = __float2bfloat16_rn(v);
    }
  }
}

// Eight parameter values (zero past the width).  The dtype is the same for all threads.
template <bool VEC>
__device__ __forceinline__ void param8(const void* p, int dtype, int64_t base, int i, int width, float2 (&f)[4]) {
  if constexpr (VEC) {
    const int c = col_of<true>(i, 0);
    if (c >= width) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = make_float2(0.0f, 0.0f);
    } else if (dtype == B200Q_F32) {
      load_smooth8(static_cast<const float*>(p) + base + c, f);
    } else if (dtype == B200Q_BF16) {
      load_smooth8(static_cast<const __nv_bfloat16*>(p) + base + c, f);
    } else {
      load_smooth8(static_cast<const __half*>(p) + base + c, f);
    }
  } else {
    float* e = reinterpret_cast<float*>(f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = col_of<false>(i, j);
      e[j] = c < width ? load_as_f32(p, dtype, base + c) : 0.0f;
    }
  }
}

template <bool VEC>
__device__ __forceinline__ void gate8(const Gate& g, int64_t row, int i, int width, float2 (&f)[4]) {
  if (g.p == nullptr) {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = make_float2(1.0f, 1.0f);
  } else if (g.per_row) {
    const float v = load_as_f32(g.p, g.dtype, (row / g.rows_per) * g.row_stride);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = make_float2(v, v);
  } else {
    param8<VEC>(g.p, g.dtype, (row / g.rows_per) * g.row_stride, i, width, f);
  }
}

// Sums of N values over the CTA; `red` must not be in use by an earlier call (two buffers, used in turn).
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float (*red)[32]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nwarps = blockDim.x >> 5;
#pragma unroll
  for (int k = 0; k < N; ++k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if (lane == 0) red[k][warp] = v[k];
  }
  __syncthreads();
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
  Param gamma, post, smooth;
  Gate gate;
  float alpha, eps, inv_width;
  int64_t rows;
  int width;
};

template <typename T, bool VEC, int ITERS, bool QUANT>
__global__ void __launch_bounds__(1024)
gated_norm_kernel(const NormArgs a) {
  __shared__ float red[3][1][32];
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.residual);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    Pack8<T> xr[ITERS], rr[ITERS];
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      load8<T, VEC>(x + row * a.width, i, a.width, xr[i]);
      load8<T, VEC>(res + row * a.width, i, a.width, rr[i]);
    }
    float r1 = 1.0f;
    if (a.post.p != nullptr) {
      float s[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < ITERS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 v = pair_of<T>(xr[i], j);
          s[0] = fmaf(v.x, v.x, fmaf(v.y, v.y, s[0]));
        }
      block_sum<1>(s, red[0]);
      r1 = rstd_of(s[0], a.inv_width, a.eps);
      if (threadIdx.x == 0 && a.post_rstd != nullptr) a.post_rstd[row] = r1;
    }
    float2 h[ITERS][4];
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      float2 g[4], w[4];
      gate8<VEC>(a.gate, row, i, a.width, g);
      if (a.post.p != nullptr) param8<VEC>(a.post.p, a.post.dtype, 0, i, a.width, w);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 z = pair_of<T>(xr[i], j);
        if (a.post.p != nullptr) z = make_float2(z.x * r1 * w[j].x, z.y * r1 * w[j].y);
        const float2 r = pair_of<T>(rr[i], j);
        h[i][j] = make_float2(fmaf(g[j].x, z.x, a.alpha * r.x), fmaf(g[j].y, z.y, a.alpha * r.y));
        s[0] = fmaf(h[i][j].x, h[i][j].x, fmaf(h[i][j].y, h[i][j].y, s[0]));
      }
      store8<T, VEC>(static_cast<T*>(a.h) + row * a.width, i, a.width, h[i]);
    }
    block_sum<1>(s, red[1]);
    const float r2 = rstd_of(s[0], a.inv_width, a.eps);
    if (threadIdx.x == 0 && a.rstd != nullptr) a.rstd[row] = r2;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      float2 w[4], sm[4];
      param8<VEC>(a.gamma.p, a.gamma.dtype, 0, i, a.width, w);
      if (QUANT && a.smooth.p != nullptr) param8<VEC>(a.smooth.p, a.smooth.dtype, 0, i, a.width, sm);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 y = make_float2(h[i][j].x * r2 * w[j].x, h[i][j].y * r2 * w[j].y);
        if (QUANT) {
          if (a.smooth.p != nullptr) y = make_float2(y.x * sm[j].x, y.y * sm[j].y);
          amax = fmaxf(amax, fmaxf(fabsf(y.x), fabsf(y.y)));
        }
        h[i][j] = y;
      }
      if (!QUANT) store8<T, VEC>(static_cast<T*>(a.y) + row * a.width, i, a.width, h[i]);
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
        if constexpr (VEC) {
          const int c = col_of<true>(i, 0);
          if (c < a.width) st_stream(reinterpret_cast<uint2*>(q + c), o);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int c = col_of<false>(i, j);
            if (c < a.width) q[c] = (int8_t)(((j < 4 ? o.x : o.y) >> (8 * (j & 3))) & 0xff);
          }
        }
      }
    }
    // The buffers of one row are written again for the next one only behind another buffer's barrier, except when a row
    // has a single reduction.
    if (a.post.p == nullptr && !QUANT) __syncthreads();
  }
}

struct NormGradArgs {
  const void* dy;
  const void* dh;            // or NULL
  const void* x;
  const void* residual;
  const float* rstd;
  const float* post_rstd;
  Param gamma, post;
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

// CTA c takes the rows [rows * c / CTAs, rows * (c + 1) / CTAs).  SUM_GATE: the gate's gradient
// is a sum over the rows that share a gate; without it there is no gate, or one value a row, or one gate a row.
template <typename T, bool VEC, int ITERS, bool SUM_GATE>
__global__ void __launch_bounds__(kNormGradThreads)
gated_norm_grad_kernel(const NormGradArgs a) {
  __shared__ float red[2][2][32];
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.residual);
  const T* dy = static_cast<const T*>(a.dy);
  const T* dhp = static_cast<const T*>(a.dh);
  const bool post = a.post.p != nullptr;
  float2 sum2[ITERS][4], sum1[ITERS][4], sumg[SUM_GATE ? ITERS : 1][4];
#pragma unroll
  for (int i = 0; i < ITERS; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sum2[i][j] = sum1[i][j] = make_float2(0.0f, 0.0f);
      if (SUM_GATE) sumg[SUM_GATE ? i : 0][j] = make_float2(0.0f, 0.0f);
    }
  const int64_t r0 = a.rows * blockIdx.x / gridDim.x, r1 = a.rows * (blockIdx.x + 1) / gridDim.x;
  for (int64_t row = r0; row < r1; ++row) {
    Pack8<T> xr[ITERS], rr[ITERS], yr[ITERS], hr[ITERS];
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      load8<T, VEC>(x + row * a.width, i, a.width, xr[i]);
      load8<T, VEC>(res + row * a.width, i, a.width, rr[i]);
      load8<T, VEC>(dy + row * a.width, i, a.width, yr[i]);
      if (dhp != nullptr) load8<T, VEC>(dhp + row * a.width, i, a.width, hr[i]);
    }
    const float rs2 = a.rstd[row], rs1 = post ? a.post_rstd[row] : 1.0f;
    float dot[1] = {0.0f};
    auto hn_of = [&](int i, int j, const float2 (&g)[4], const float2 (&w1)[4], float2& xn, float2& z) {
      const float2 v = pair_of<T>(xr[i], j), r = pair_of<T>(rr[i], j);
      xn = make_float2(v.x * rs1, v.y * rs1);
      z = post ? make_float2(xn.x * w1[j].x, xn.y * w1[j].y) : v;
      return make_float2(fmaf(g[j].x, z.x, a.alpha * r.x) * rs2, fmaf(g[j].y, z.y, a.alpha * r.y) * rs2);
    };
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      float2 g[4], w1[4], w2[4];
      gate8<VEC>(a.gate, row, i, a.width, g);
      if (post) param8<VEC>(a.post.p, a.post.dtype, 0, i, a.width, w1);
      param8<VEC>(a.gamma.p, a.gamma.dtype, 0, i, a.width, w2);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 xn, z;
        const float2 hn = hn_of(i, j, g, w1, xn, z);
        const float2 d = pair_of<T>(yr[i], j);
        dot[0] = fmaf(d.x * w2[j].x, hn.x, fmaf(d.y * w2[j].y, hn.y, dot[0]));
        sum2[i][j].x = fmaf(d.x, hn.x, sum2[i][j].x);
        sum2[i][j].y = fmaf(d.y, hn.y, sum2[i][j].y);
      }
    }
    block_sum<1>(dot, red[0]);
    const float c2 = dot[0] * a.inv_width;
    float dots[2] = {0.0f, 0.0f};                          // v . xn, dh . z
    float2 keep[ITERS][4];                                 // v
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      float2 g[4], w1[4], w2[4], out[4], dg[4];
      gate8<VEC>(a.gate, row, i, a.width, g);
      if (post) param8<VEC>(a.post.p, a.post.dtype, 0, i, a.width, w1);
      param8<VEC>(a.gamma.p, a.gamma.dtype, 0, i, a.width, w2);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 xn, z;
        const float2 hn = hn_of(i, j, g, w1, xn, z);
        const float2 d = pair_of<T>(yr[i], j);
        float2 dh = make_float2(rs2 * fmaf(-hn.x, c2, d.x * w2[j].x), rs2 * fmaf(-hn.y, c2, d.y * w2[j].y));
        if (dhp != nullptr) {
          const float2 e = pair_of<T>(hr[i], j);
          dh = make_float2(dh.x + e.x, dh.y + e.y);
        }
        out[j] = make_float2(a.alpha * dh.x, a.alpha * dh.y);
        dg[j] = make_float2(dh.x * z.x, dh.y * z.y);
        if (SUM_GATE) {
          sumg[SUM_GATE ? i : 0][j].x += dg[j].x;
          sumg[SUM_GATE ? i : 0][j].y += dg[j].y;
        }
        dots[1] += dg[j].x + dg[j].y;
        float2 dz = make_float2(dh.x * g[j].x, dh.y * g[j].y);
        if (post) {
          sum1[i][j].x = fmaf(dz.x, xn.x, sum1[i][j].x);
          sum1[i][j].y = fmaf(dz.y, xn.y, sum1[i][j].y);
          dz = make_float2(dz.x * w1[j].x, dz.y * w1[j].y);
          dots[0] = fmaf(dz.x, xn.x, fmaf(dz.y, xn.y, dots[0]));
        }
        keep[i][j] = dz;
      }
      store8<T, VEC>(static_cast<T*>(a.dres) + row * a.width, i, a.width, out);
      if (!SUM_GATE && a.dgate != nullptr && !a.gate.per_row) {
        // one gate a row: its gradient is dh * z itself
        const int64_t base = row * a.width;
        if (a.gate.dtype == B200Q_F32) store8<float, VEC>(static_cast<float*>(a.dgate) + base, i, a.width, dg);
        else if (a.gate.dtype == B200Q_BF16) store8<__nv_bfloat16, VEC>(static_cast<__nv_bfloat16*>(a.dgate) + base, i, a.width, dg);
        else store8<__half, VEC>(static_cast<__half*>(a.dgate) + base, i, a.width, dg);
      }
    }
    block_sum<2>(dots, red[1]);
    const float c1 = dots[0] * a.inv_width;
    if (!SUM_GATE && a.dgate != nullptr && a.gate.per_row && threadIdx.x == 0) store_from_f32(a.dgate, a.gate.dtype, row, dots[1]);
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      if (post) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 v = pair_of<T>(xr[i], j);
          keep[i][j] = make_float2(rs1 * fmaf(-v.x * rs1, c1, keep[i][j].x), rs1 * fmaf(-v.y * rs1, c1, keep[i][j].y));
        }
      }
      store8<T, VEC>(static_cast<T*>(a.dx) + row * a.width, i, a.width, keep[i]);
    }
    if (SUM_GATE) {
      const int64_t gate = row / a.gate.rows_per;
      if (row + 1 == r1 || (row + 1) / a.gate.rows_per != gate) {
        float* part = a.part_gate + (blockIdx.x + gate) * a.width;
#pragma unroll
        for (int i = 0; i < ITERS; ++i) {
          store8<float, VEC>(part, i, a.width, sumg[SUM_GATE ? i : 0]);
#pragma unroll
          for (int j = 0; j < 4; ++j) sumg[SUM_GATE ? i : 0][j] = make_float2(0.0f, 0.0f);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    store8<float, VEC>(a.part_gamma + (int64_t)blockIdx.x * a.width, i, a.width, sum2[i]);
    if (post) store8<float, VEC>(a.part_post + (int64_t)blockIdx.x * a.width, i, a.width, sum1[i]);
  }
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
  int gamma_dtype, post_dtype, gate_dtype;
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
    p0 = (first + 1) * a.ctas / a.rows;
    while (p0 > 0 && a.rows * p0 / a.ctas > first) --p0;
    while (a.rows * (p0 + 1) / a.ctas <= first) ++p0;
    p1 = p0;
    while (p1 < a.ctas && a.rows * p1 / a.ctas <= last) ++p1;
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
    if (blockIdx.y == 0) store_from_f32(a.dgamma, a.gamma_dtype, col, s);
    else if (blockIdx.y == 1) store_from_f32(a.dpost, a.post_dtype, col, s);
    else store_from_f32(a.dgate, a.gate_dtype, g * a.width + col, s);
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

template <typename T, bool VEC, bool QUANT>
int launch_norm(const NormArgs& a, cudaStream_t st) {
  const int64_t vecs = ceil_div(a.width, 8);
  const int iters = vecs > 1024 ? 2 : 1;
  const int threads = (int)ceil_div(ceil_div(vecs, iters), 32) * 32;
  int per_sm = 1;
#define B200Q_NORM(I)                                                                            \
  {                                                                                              \
    auto kern = gated_norm_kernel<T, VEC, I, QUANT>;                                             \
    cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, 0);                    \
    const int64_t cap = (int64_t)sm_count() * (per_sm > 0 ? per_sm : 1);                         \
    kern<<<(unsigned)(a.rows < cap ? a.rows : cap), threads, 0, st>>>(a);                        \
  }
  if (iters == 1) B200Q_NORM(1) else B200Q_NORM(2)
#undef B200Q_NORM
  return check_launch("gated_add_rms_norm");
}

// CTAs of the gradient kernel: the partial sums cost a row of fp32 each, so no more than two on an SM.
inline int grad_ctas(int64_t rows) {
  const int64_t cap = 2 * (int64_t)sm_count();
  return (int)(rows < cap ? rows : cap);
}

template <typename T, bool VEC>
int launch_norm_grad(const NormGradArgs& a, const NormSumArgs& s, bool sum_gate, cudaStream_t st) {
  const int64_t vecs = ceil_div(a.width, 8);
  const int iters = vecs > 2 * kNormGradThreads ? 4 : vecs > kNormGradThreads ? 2 : 1;
  const int threads = (int)ceil_div(ceil_div(vecs, iters), 32) * 32;
#define B200Q_NORM_GRAD_CASE(I)                                                                          \
  {                                                                                                      \
    if (sum_gate) gated_norm_grad_kernel<T, VEC, I, true><<<s.ctas, threads, 0, st>>>(a);                \
    else gated_norm_grad_kernel<T, VEC, I, false><<<s.ctas, threads, 0, st>>>(a);                        \
  }
  if (iters == 1) B200Q_NORM_GRAD_CASE(1) else if (iters == 2) B200Q_NORM_GRAD_CASE(2) else B200Q_NORM_GRAD_CASE(4)
#undef B200Q_NORM_GRAD_CASE
  if (int rc = check_launch("gated_add_rms_norm_grad")) return rc;
  const int64_t gates = sum_gate ? ceil_div(a.rows, s.rows_per) : 0;
  dim3 grid((unsigned)ceil_div(a.width, 32), (unsigned)(2 + gates));
  gated_norm_sum_kernel<<<grid, 1024, 0, st>>>(s);
  return check_launch("gated_add_rms_norm_grad (sums)");
}

template <typename T>
int norm_forward(const NormArgs& a, bool quant, cudaStream_t st) {
  const bool vec = norm_vec(a.width, {a.x, a.residual, a.y, a.h, a.gamma.p, a.post.p, a.smooth.p, a.gate.per_row ? nullptr : a.gate.p});
  if (quant) return vec ? launch_norm<T, true, true>(a, st) : launch_norm<T, false, true>(a, st);
  return vec ? launch_norm<T, true, false>(a, st) : launch_norm<T, false, false>(a, st);
}

inline bool norm_dtype(int d) { return d == B200Q_BF16 || d == B200Q_F16 || d == B200Q_F32; }

// Gates of `kind` share rows (their gradient is a sum over rows)?
inline bool gate_is_shared(const b200q_gated_norm_args& a) {
  return a.gate != nullptr && !(a.gate_per_row && a.gate_rows == 1) && a.gate_rows > 1;
}

int norm_checks(const b200q_gated_norm_args& a, const char* op) {
  B200Q_REQUIRE(a.rows >= 0 && a.width >= 0, B200Q_ERR_BAD_ARG, "%s: negative size", op);
  B200Q_REQUIRE(norm_dtype(a.dtype), B200Q_ERR_UNSUPPORTED, "%s: x must be bf16, f16 or f32 (dtype enum %d)", op, a.dtype);
  B200Q_REQUIRE(a.width <= kNormMaxWidth && a.rows <= 0x7fffffffLL, B200Q_ERR_UNSUPPORTED, "%s: rows of %lld elements (at most %d)", op,
                (long long)a.width, kNormMaxWidth);
  B200Q_REQUIRE(norm_dtype(a.gamma_dtype) && (a.post_gamma == nullptr || norm_dtype(a.post_gamma_dtype)) &&
                    (a.gate == nullptr || norm_dtype(a.gate_dtype)),
                B200Q_ERR_UNSUPPORTED, "%s: gamma, post_gamma and gate must be bf16, f16 or f32", op);
  B200Q_REQUIRE(a.gate == nullptr || a.gate_rows >= 1, B200Q_ERR_BAD_ARG, "%s: gate_rows must be at least 1", op);
  B200Q_REQUIRE(a.gate == nullptr || !a.gate_per_row || a.gate_rows == 1, B200Q_ERR_UNSUPPORTED, "%s: a gate of one value belongs to one row", op);
  return B200Q_OK;
}

bool norm_aligned(const void* p, int dtype) { return p == nullptr || aligned(p, dtype == B200Q_F32 ? 4 : 2); }

}  // namespace
}  // namespace b200q

extern "C" int b200q_gated_norm(const b200q_gated_norm_args* a, void* stream) {
  using namespace b200q;
  clear_error();
  constexpr const char* op = "gated_add_rms_norm";
  B200Q_REQUIRE(a != nullptr, B200Q_ERR_BAD_ARG, "%s: args is NULL", op);
  if (int rc = norm_checks(*a, op)) return rc;
  const bool quant = a->scale != nullptr;
  B200Q_REQUIRE(!quant || a->smooth == nullptr || norm_dtype(a->smooth_dtype), B200Q_ERR_UNSUPPORTED, "%s: smooth scales must be bf16, f16 or f32", op);
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
  B200Q_REQUIRE(norm_aligned(a->x, a->dtype) && norm_aligned(a->residual, a->dtype) && norm_aligned(a->h, a->dtype) &&
                    (quant || norm_aligned(a->y, a->dtype)) && norm_aligned(a->gamma, a->gamma_dtype) && norm_aligned(a->post_gamma, a->post_gamma_dtype) &&
                    norm_aligned(a->gate, a->gate_dtype) && norm_aligned(a->smooth, a->smooth_dtype) && aligned(a->rstd, 4) &&
                    aligned(a->post_rstd, 4) && aligned(a->scale, 4),
                B200Q_ERR_BAD_ARG, "%s: misaligned buffer", op);
  NormArgs n{};
  n.x = a->x; n.residual = a->residual; n.y = a->y; n.h = a->h; n.rstd = a->rstd; n.post_rstd = a->post_rstd; n.scale = a->scale;
  n.gamma = {a->gamma, a->gamma_dtype};
  n.post = {a->post_gamma, a->post_gamma_dtype};
  n.smooth = {a->smooth, a->smooth_dtype};
  n.gate = {a->gate, a->gate_dtype, a->gate_per_row, a->gate != nullptr ? a->gate_rows : 1, a->gate_per_row ? 1 : a->width};
  n.alpha = a->residual_scale; n.eps = a->epsilon; n.inv_width = 1.0f / (float)a->width;
  n.rows = a->rows; n.width = (int)a->width;
  if (a->dtype == B200Q_BF16) return norm_forward<__nv_bfloat16>(n, quant, st);
  if (a->dtype == B200Q_F16) return norm_forward<__half>(n, quant, st);
  return norm_forward<float>(n, quant, st);
}

extern "C" size_t b200q_gated_norm_grad_workspace_bytes(const b200q_gated_norm_args* a) {
  using namespace b200q;
  if (a == nullptr || a->rows <= 0 || a->width <= 0) return 0;
  const int64_t ctas = grad_ctas(a->rows);
  const int64_t gates = gate_is_shared(*a) ? ctas + ceil_div(a->rows, a->gate_rows) : 0;
  return (size_t)(2 * ctas + gates) * (size_t)((a->width + 3) & ~int64_t(3)) * 4;
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
    cudaError_t e = g->dgamma != nullptr ? cudaMemsetAsync(g->dgamma, 0, (size_t)a->width * (a->gamma_dtype == B200Q_F32 ? 4 : 2), st) : cudaSuccess;
    if (e == cudaSuccess && a->post_gamma != nullptr && g->dpost_gamma != nullptr)
      e = cudaMemsetAsync(g->dpost_gamma, 0, (size_t)a->width * (a->post_gamma_dtype == B200Q_F32 ? 4 : 2), st);
    return e == cudaSuccess ? B200Q_OK : fail(B200Q_ERR_LAUNCH, "%s: %s", op, cudaGetErrorString(e));
  }
  B200Q_REQUIRE(a->x != nullptr && a->residual != nullptr && a->gamma != nullptr && a->rstd != nullptr && g->dy != nullptr && g->dx != nullptr &&
                    g->dresidual != nullptr && g->dgamma != nullptr && (a->post_gamma == nullptr || (a->post_rstd != nullptr && g->dpost_gamma != nullptr)) &&
                    (a->gate == nullptr || g->dgate != nullptr),
                B200Q_ERR_BAD_ARG, "%s: NULL buffer", op);
  B200Q_REQUIRE(norm_aligned(a->x, a->dtype) && norm_aligned(a->residual, a->dtype) && norm_aligned(g->dy, a->dtype) && norm_aligned(g->dh, a->dtype) &&
                    norm_aligned(g->dx, a->dtype) && norm_aligned(g->dresidual, a->dtype) && norm_aligned(a->gamma, a->gamma_dtype) &&
                    norm_aligned(g->dgamma, a->gamma_dtype) && norm_aligned(a->post_gamma, a->post_gamma_dtype) &&
                    norm_aligned(g->dpost_gamma, a->post_gamma_dtype) && norm_aligned(a->gate, a->gate_dtype) && norm_aligned(g->dgate, a->gate_dtype) &&
                    aligned(a->rstd, 4) && aligned(a->post_rstd, 4),
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
  n.gamma = {a->gamma, a->gamma_dtype};
  n.post = {a->post_gamma, a->post_gamma_dtype};
  n.gate = {a->gate, a->gate_dtype, a->gate_per_row, a->gate != nullptr ? a->gate_rows : 1, a->gate_per_row ? 1 : a->width};
  n.dx = g->dx; n.dres = g->dresidual; n.dgate = shared ? nullptr : (a->gate != nullptr ? g->dgate : nullptr);
  n.part_gamma = part; n.part_post = part + (int64_t)ctas * a->width; n.part_gate = shared ? part + 2 * (int64_t)ctas * a->width : nullptr;
  n.alpha = a->residual_scale; n.inv_width = 1.0f / (float)a->width;
  n.rows = a->rows; n.width = (int)a->width;
  NormSumArgs s{};
  s.part_gamma = n.part_gamma; s.part_post = a->post_gamma != nullptr ? n.part_post : nullptr; s.part_gate = n.part_gate;
  s.dgamma = g->dgamma; s.dpost = g->dpost_gamma; s.dgate = g->dgate;
  s.gamma_dtype = a->gamma_dtype; s.post_dtype = a->post_gamma_dtype; s.gate_dtype = a->gate_dtype;
  s.rows = a->rows; s.rows_per = shared ? a->gate_rows : 1; s.width = a->width; s.ctas = ctas;
  const bool vec = norm_vec(a->width, {a->x, a->residual, g->dy, g->dh, g->dx, g->dresidual, a->gamma, a->post_gamma,
                                       a->gate_per_row ? nullptr : a->gate, a->gate_per_row || shared ? nullptr : g->dgate});
#define B200Q_NORM_GRAD(T) (vec ? launch_norm_grad<T, true>(n, s, shared, st) : launch_norm_grad<T, false>(n, s, shared, st))
  if (a->dtype == B200Q_BF16) return B200Q_NORM_GRAD(__nv_bfloat16);
  if (a->dtype == B200Q_F16) return B200Q_NORM_GRAD(__half);
  return B200Q_NORM_GRAD(float);
#undef B200Q_NORM_GRAD
}
