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
// The forward pass reads x and the residual and writes y and h, the gradient reads x, the residual and both gradients and writes
// two; a row stays in its CTA's registers between the reductions.  For rows of full vectors the forward pass is bound by HBM (0.86 of it)
// and the gradient by the latency of its two reductions a row (0.66).  Rows of other widths pass value by value (0.2 to 0.36), and from
// 4097 columns on their gradient reads each operand three times.  Everything between loading and storing is fp32: h is not rounded
// before its norm, and the gradient computes it again from x and the residual instead of reading the rounded one.  Sums over rows (dw1,
// dw2, a shared gate) are kept in shared memory or registers by CTAs that take contiguous rows, written once per CTA as fp32 and added
// by a second kernel in a fixed order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"

namespace b200q {
namespace {

// A thread's place among the threads that share a row, and its columns: eight values i, VEC: eight neighbours
// (columns (i * threads + tid) * 8 ..), one or two 16-byte accesses, every one of them inside the row (the launch sees to that:
// predicates cost these kernels more than memory does); else columns (i * 8 + j) * threads + tid, one by one, for any width
// and alignment.
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
// ONCE: the row is read once and need not stay in L1 (where the parameters are).
template <typename T, bool VEC, bool ONCE = true>
__device__ __forceinline__ void load8(const T* __restrict__ row, int i, int width, const Place& at, Pack8<T>& raw) {
  const int c = at.col<VEC>(i, 0);
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < (int)sizeof(T) / 2; ++q)
      raw.v[q] = ONCE ? ld_stream(reinterpret_cast<const uint4*>(row + c) + q) : __ldg(reinterpret_cast<const uint4*>(row + c) + q);
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

// Eight parameter values.  Past the width the last column's are read, and the row's values are zero there.  CLEAR: the parameter is
// taken as zero too, so that an infinite one makes nothing there that reaches the other columns through a row's sum or maximum (in the
// gradient the column itself does: every column of such a row is NaN by the formulas).  The value is loaded first and then chosen: loads
// that wait for a predicate took up to 1.6 times as long for rows above 8192 columns.
template <typename P, bool VEC, bool CLEAR>
__device__ __forceinline__ void param8(const P* __restrict__ p, int i, int width, const Place& at, float2 (&f)[4]) {
  const int c = at.col<VEC>(i, 0);
  if constexpr (VEC) {
    load_smooth8(p + c, f);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = make_float2(to_f32<P>(p[min(c + 2 * j * at.threads, width - 1)]), to_f32<P>(p[min(c + (2 * j + 1) * at.threads, width - 1)]));
      if constexpr (CLEAR) f[j] = make_float2(c + 2 * j * at.threads < width ? f[j].x : 0.0f, c + (2 * j + 1) * at.threads < width ? f[j].y : 0.0f);
    }
  }
}

// The gate of a row: rows_per consecutive rows share row `row / rows_per` of p, which is one value (per_row) or `width`.
struct Gate {
  const void* p;
  int per_row;
  int64_t rows_per;
};
template <typename P, bool VEC, bool CLEAR>
__device__ __forceinline__ void gate8(const Gate& g, int64_t gate_row, int i, int width, const Place& at, float2 (&f)[4]) {
  if (g.p == nullptr || g.per_row) {
    const float v = g.p == nullptr ? 1.0f : to_f32<P>(static_cast<const P*>(g.p)[gate_row]);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = make_float2(v, v);
  } else {
    param8<P, VEC, CLEAR>(static_cast<const P*>(g.p) + gate_row * width, i, width, at, f);
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

// The same for up to 16 warps, with one round of 16-byte loads in place of the second round of shuffles; `red` holds zeros behind the
// row's warps.
template <int N>
__device__ __forceinline__ void row_sum16(float (&v)[N], float (*red)[32], const Place& at, int barrier) {
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if (at.threads == 32) return;
#pragma unroll
  for (int k = 0; k < N; ++k)
    if ((at.tid & 31) == 0) red[k][at.tid >> 5] = v[k];
  named_barrier_sync(barrier, at.threads);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float4* p = reinterpret_cast<const float4*>(red[k]);
    const float4 a = p[0], b = p[1], c = p[2], d = p[3];
    v[k] = (((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w))) + (((c.x + c.y) + (c.z + c.w)) + ((d.x + d.y) + (d.z + d.w)));
  }
}

// The larger magnitude, NaN if either is NaN (fmaxf would pass over it, and a row that is all NaN would leave quantised as zeros with
// scale 0).  Behind it NaN stays the largest: its bits are above infinity's.
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(fabsf(b)));
  return m;
}

// Maxima of N non-negative values over the threads of a row.
template <int N>
__device__ __forceinline__ void row_max(float (&v)[N], float (*red)[32], const Place& at, int barrier) {
  unsigned m[N];
#pragma unroll
  for (int k = 0; k < N; ++k) m[k] = __reduce_max_sync(0xffffffffu, __float_as_uint(v[k]));
  if (at.threads > 32) {
    const int warp = at.tid >> 5, lane = at.tid & 31, nwarps = at.threads >> 5;
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (lane == 0) red[k][warp] = __uint_as_float(m[k]);
    named_barrier_sync(barrier, at.threads);
#pragma unroll
    for (int k = 0; k < N; ++k) m[k] = __reduce_max_sync(0xffffffffu, __float_as_uint(lane < nwarps ? red[k][lane] : 0.0f));
  }
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = __uint_as_float(m[k]);
}

template <bool VEC>
__device__ __forceinline__ void store8_int8(int8_t* __restrict__ row, int i, int width, const Place& at, uint2 v) {
  const int c = at.col<VEC>(i, 0);
  if constexpr (VEC) {
    st_stream(reinterpret_cast<uint2*>(row + c), v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j * at.threads < width) row[c + j * at.threads] = (int8_t)(((j < 4 ? v.x : v.y) >> (8 * (j & 3))) & 0xff);
  }
}

__device__ __forceinline__ float rstd_of(float sum, float inv_width, float eps) {
  return __frsqrt_rn(__fadd_rn(__fmul_rn(sum, inv_width), eps));
}

// ------------------------------------------------------------------------------------------------ rows through shared memory
// For more than a handful of rows, the CTA's first warp brings its rows into a ring in shared memory with bulk copies, a chunk
// of `groups` consecutive rows of every operand a stage, so that the loads of several rows are always under way and no
// registers hold rows.  It refills a chunk's stage while it works on the next chunk (a warp of its own would cost the others a
// quarter of their registers: 17 warps get 96 each, 16 get 128).  A chunk is one contiguous piece of each operand; a piece that
// does not start or end on a 16-byte boundary (rows of odd width) is copied from the boundary before to the one behind, except
// at the operand's end, whose last bytes the warp copies by itself.  Operands start on a 16-byte boundary.
// The ring leaves part of the SM's 228 KB to L1, which holds the parameters.
constexpr int kRowPipeSmem = 150 * 1024;
constexpr int kRowPipeMaxStages = 4;

// Where the filling of the ring stands: next row, stage, and whether every wait was met.
struct RowPipeFeed {
  int row;
  int stage;
  uint32_t phase;
  bool ok;
  __device__ __forceinline__ void next(int to, int stages) {
    row = to;
    if (++stage == stages) { stage = 0; phase ^= 1; }
  }
};

struct RowPipe {
  uint8_t* data;             // [stages][arrays][array_bytes]
  uint64_t* full;
  uint64_t* empty;
  volatile int* abort_flag;
  int stages, arrays, array_bytes;
  int64_t row_bytes, total_bytes;
  __device__ __forceinline__ uint8_t* slot(int stage, int array) const { return data + (int64_t)(stage * arrays + array) * array_bytes; }
};

// Host and device: bytes of one operand's place in a stage.
inline __host__ __device__ int row_pipe_array_bytes(int groups, int64_t row_bytes) { return (int)((groups * row_bytes + 16 + 15) & ~int64_t(15)); }

__device__ __forceinline__ RowPipe row_pipe_init(uint8_t* smem, int stages, int arrays, int groups, int64_t row_bytes, int64_t rows, int readers) {
  __shared__ uint64_t bars[2 * kRowPipeMaxStages];
  __shared__ int abort_word;
  RowPipe p{smem, bars, bars + kRowPipeMaxStages, &abort_word, stages, arrays, row_pipe_array_bytes(groups, row_bytes), row_bytes, rows * row_bytes};
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&p.full[i], 1);
      mbar_init(&p.empty[i], readers);
    }
    abort_word = 0;
    fence_mbar_init();
  }
  __syncthreads();
  return p;
}

// One chunk, rows [row, row + count), by a whole warp: waits for the stage and starts its copies.
template <int ARRAYS>
__device__ __forceinline__ bool row_pipe_fill(const RowPipe& p, const void* const (&src)[ARRAYS], int stage, uint32_t phase, int64_t row, int count,
                                              int lane) {
  if (!__all_sync(0xffffffffu, mbar_wait(&p.empty[stage], phase ^ 1, p.abort_flag, kDevTimeoutProducer))) return false;
  const int64_t lo = row * p.row_bytes, hi = lo + count * p.row_bytes, first = lo & ~int64_t(15);
  int64_t last = (hi + 15) & ~int64_t(15);
  if (last > p.total_bytes) {                              // the operand's end: its last bytes one by one
    last = p.total_bytes & ~int64_t(15);
    for (int q = 0; q < ARRAYS; ++q)
      if (src[q] != nullptr && last + lane < hi) p.slot(stage, q)[last - first + lane] = static_cast<const uint8_t*>(src[q])[last + lane];
    __syncwarp();
  }
  const uint32_t bytes = (uint32_t)(last - first);
  int copies = 0;
#pragma unroll
  for (int q = 0; q < ARRAYS; ++q) copies += src[q] != nullptr;
  if (lane == 0) mbar_arrive_expect_tx(&p.full[stage], bytes * copies);
  __syncwarp();
#pragma unroll
  for (int q = 0; q < ARRAYS; ++q)
    if (lane == q && src[q] != nullptr && bytes != 0) bulk_load(p.slot(stage, q), static_cast<const uint8_t*>(src[q]) + first, bytes, &p.full[stage]);
  return true;
}

// Eight values of a row in shared memory.
template <typename T, bool VEC>
__device__ __forceinline__ Pack8<T> smem8(const uint8_t* row, int i, int width, const Place& at) {
  Pack8<T> raw;
  const int c = at.col<VEC>(i, 0);
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < (int)sizeof(T) / 2; ++q)
      raw.v[q] = reinterpret_cast<const uint4*>(row + c * (int)sizeof(T))[q];
  } else {
    using Word = typename Chunk<sizeof(T)>::type;
    const Word* p = reinterpret_cast<const Word*>(row);
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = c + j * at.threads < width ? (uint32_t)p[c + j * at.threads] : 0u;
    if constexpr (sizeof(T) == 4) {
      raw.v[0] = make_uint4(w[0], w[1], w[2], w[3]);
      raw.v[1] = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
      raw.v[0] = make_uint4(w[0] | (w[1] << 16), w[2] | (w[3] << 16), w[4] | (w[5] << 16), w[6] | (w[7] << 16));
    }
  }
  return raw;
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

// Bound by HBM for many rows (8192 of 4096 bf16: 47 us, 5.7 TB/s; int8 rows 54), by the latency of its reductions for few (16 of 8192,
// int8: 4.4 us).  One CTA a row at a time.  The next row's x and residual are in flight from the moment this row's have become h.  With
// ITERS 1 (rows spread over many threads: few rows, where latency counts) the parameters are loaded with the row, not behind
// the reductions.
template <typename T, typename P, bool VEC, int ITERS, bool QUANT, int MAX_THREADS, int MIN_CTAS>
__global__ void __launch_bounds__(MAX_THREADS, MIN_CTAS)
gated_norm_kernel(const NormArgs a) {
  constexpr bool EARLY = ITERS == 1;
  __shared__ float red[3][1][32];
  const Place at{(int)threadIdx.x, (int)blockDim.x};
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.residual);
  const P* gamma = static_cast<const P*>(a.gamma);
  const P* post = static_cast<const P*>(a.post);
  auto smooth8 = [&](int i, float2(&f)[4]) {
    if (a.smooth_f32) param8<float, VEC, true>(static_cast<const float*>(a.smooth), i, a.width, at, f);
    else param8<T, VEC, true>(static_cast<const T*>(a.smooth), i, a.width, at, f);
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
    if (post != nullptr) param8<P, VEC, true>(post, 0, a.width, at, early_post);
    param8<P, VEC, true>(gamma, 0, a.width, at, early_gamma);
    if (QUANT && a.smooth != nullptr) smooth8(0, early_smooth);
  }
  const float2 alpha = splat(a.alpha);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t gate_row = a.gate.rows_per == 1 ? row : a.gate.rows_per >= a.rows ? 0 : row / a.gate.rows_per;
    float2 early_gate[4];
    if constexpr (EARLY) gate8<P, VEC, true>(a.gate, gate_row, 0, a.width, at, early_gate);
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
        gate8<P, VEC, true>(a.gate, gate_row, i, a.width, at, g);
        if (post != nullptr) param8<P, VEC, true>(post, i, a.width, at, w);
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
        param8<P, VEC, true>(gamma, i, a.width, at, w);
        if (QUANT && a.smooth != nullptr) smooth8(i, sm);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 y = __fmul2_rn(__fmul2_rn(h[i][j], splat(r2)), EARLY ? early_gamma[j] : w[j]);
        if (QUANT) {
          if (a.smooth != nullptr) y = __fmul2_rn(y, EARLY ? early_smooth[j] : sm[j]);
          amax = max_or_nan(max_or_nan(amax, y.x), y.y);
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
        store8_int8<VEC>(q, i, a.width, at, inv == inv ? quantize8<false>(h[i], scale, inv) : quantize8<true>(h[i], scale, inv));
      }
    }
    // The buffers of one row are written again for the next one only behind another buffer's barrier, except when a row
    // has a single reduction.
    if (post == nullptr && !QUANT) __syncthreads();
  }
}

// The same for rows that do not come as full vectors, through shared memory (6124 rows of 1111 f16: 27 us, 2.0 TB/s; values come and go
// one by one, which takes several times the instructions): `threads_per_row` threads work on two rows at once
// (the reductions' latencies and the parameters are then shared by two rows), as many such groups as fit into the CTA.
constexpr int kRowPipeThreads = 512;      // at most

template <typename T, typename P, bool QUANT>
__global__ void __launch_bounds__(kRowPipeThreads, 1)
gated_norm_pipe_kernel(const NormArgs a, int threads_per_row, int stages) {
  constexpr bool VEC = false;
  constexpr int ITERS = 1, ROWS = 2;
  extern __shared__ __align__(16) uint8_t pipe_smem[];
  __shared__ float red[3][kRowPipeThreads / 32][ROWS][32];
  const int groups = blockDim.x / threads_per_row, chunk_rows = groups * ROWS;
  const RowPipe pipe = row_pipe_init(pipe_smem, stages, 2, chunk_rows, (int64_t)a.width * sizeof(T), a.rows, blockDim.x / 32);
  const int r0 = (int)(a.rows * blockIdx.x / gridDim.x), r1 = (int)(a.rows * (blockIdx.x + 1) / gridDim.x);   // fewer than 2^30 rows
  const void* const src[2] = {a.x, a.residual};
  RowPipeFeed feed{r0, 0, 0, true};
  auto fill = [&]() {                                      // by the first warp
    if (feed.row >= r1 || !feed.ok) return;
    feed.ok = row_pipe_fill(pipe, src, feed.stage, feed.phase, feed.row, min(chunk_rows, r1 - feed.row), threadIdx.x & 31);
    feed.next(feed.row + chunk_rows, stages);
  };
  if (threadIdx.x < 32)
    for (int i = 0; i < stages; ++i) fill();
  int stage = 0;
  uint32_t phase = 0;
  const int group = threadIdx.x / threads_per_row;
  const Place at{(int)threadIdx.x - group * threads_per_row, threads_per_row};
  const P* post = static_cast<const P*>(a.post);
  const float2 alpha = splat(a.alpha);
  // A thread's columns stay the same: so do its parameters, but for the gate.
  float2 w_post[4], w_gamma[4], w_smooth[4], g[4];
  if (post != nullptr) param8<P, VEC, true>(post, 0, a.width, at, w_post);
  param8<P, VEC, true>(static_cast<const P*>(a.gamma), 0, a.width, at, w_gamma);
  if (QUANT && a.smooth != nullptr) {
    if (a.smooth_f32) param8<float, VEC, true>(static_cast<const float*>(a.smooth), 0, a.width, at, w_smooth);
    else param8<T, VEC, true>(static_cast<const T*>(a.smooth), 0, a.width, at, w_smooth);
  }
  // The gate of the group's rows, walked along; rows_per 1: the row itself.
  const int rows_per = (int)min(a.gate.rows_per, a.rows);
  int have_gate = -1, gate_at = (r0 + group * ROWS) / rows_per, gate_end = (gate_at + 1) * rows_per;
  bool ok = true;
  for (int chunk = r0; chunk < r1; chunk += chunk_rows) {
    ok = mbar_wait(&pipe.full[stage], phase, pipe.abort_flag, kDevTimeoutEpilogue) && ok;
    if (threadIdx.x < 32 && chunk > r0) fill();
    const int row = chunk + group * ROWS;
    if (row < r1) {                                        // the same for all threads of the row
      // Past the CTA's last row the row before is worked on again and not stored.
      const int live = min(ROWS, r1 - row);
      const uint8_t *xs[ROWS], *rs[ROWS];
      int gate_row[ROWS];
      const int off = (int)((chunk * pipe.row_bytes) & 15) + group * ROWS * (int)pipe.row_bytes;
#pragma unroll
      for (int k = 0; k < ROWS; ++k) {
        const int kk = min(k, live - 1);
        xs[k] = pipe.slot(stage, 0) + off + kk * (int)pipe.row_bytes;
        rs[k] = pipe.slot(stage, 1) + off + kk * (int)pipe.row_bytes;
        if (rows_per == 1) {
          gate_row[k] = row + kk;
        } else {
          while (row + kk >= gate_end) ++gate_at, gate_end += rows_per;
          gate_row[k] = gate_at;
        }
      }
      float r1s[ROWS];
#pragma unroll
      for (int k = 0; k < ROWS; ++k) r1s[k] = 1.0f;
      Pack8<T> xr[ROWS];
#pragma unroll
      for (int k = 0; k < ROWS; ++k) xr[k] = smem8<T, VEC>(xs[k], 0, a.width, at);
      if (post != nullptr) {
        float2 s2[ROWS];
        float s[ROWS];
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
          s2[k] = splat(0.0f);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 v = pair_of<T>(xr[k], j);
            s2[k] = __ffma2_rn(v, v, s2[k]);
          }
          s[k] = s2[k].x + s2[k].y;
        }
        row_sum<ROWS>(s, red[0][group], at, 1 + group);
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
          r1s[k] = rstd_of(s[k], a.inv_width, a.eps);
          if (at.tid == 0 && a.post_rstd != nullptr && ok && k < live) a.post_rstd[row + k] = r1s[k];
        }
      }
      float2 h[ROWS][ITERS][4], s2[ROWS];
#pragma unroll
      for (int k = 0; k < ROWS; ++k) s2[k] = splat(0.0f);
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
          if (gate_row[k] != have_gate) gate8<P, VEC, true>(a.gate, gate_row[k], i, a.width, at, g);
          have_gate = gate_row[k];
          const Pack8<T> rr = smem8<T, VEC>(rs[k], i, a.width, at);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float2 z = pair_of<T>(xr[k], j);
            if (post != nullptr) z = __fmul2_rn(__fmul2_rn(z, splat(r1s[k])), w_post[j]);
            h[k][i][j] = __ffma2_rn(g[j], z, __fmul2_rn(alpha, pair_of<T>(rr, j)));
            s2[k] = __ffma2_rn(h[k][i][j], h[k][i][j], s2[k]);
          }
          if (ok && k < live) store8<T, VEC>(static_cast<T*>(a.h) + (int64_t)(row + k) * a.width, i, a.width, at, h[k][i]);
        }
      }
      float s[ROWS], r2[ROWS], amax[ROWS];
#pragma unroll
      for (int k = 0; k < ROWS; ++k) s[k] = s2[k].x + s2[k].y;
      row_sum<ROWS>(s, red[1][group], at, 1 + group);
#pragma unroll
      for (int k = 0; k < ROWS; ++k) {
        r2[k] = rstd_of(s[k], a.inv_width, a.eps);
        amax[k] = 0.0f;
        if (at.tid == 0 && a.rstd != nullptr && ok && k < live) a.rstd[row + k] = r2[k];
      }
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float2 y = __fmul2_rn(__fmul2_rn(h[k][i][j], splat(r2[k])), w_gamma[j]);
            if (QUANT) {
              if (a.smooth != nullptr) y = __fmul2_rn(y, w_smooth[j]);
              amax[k] = max_or_nan(max_or_nan(amax[k], y.x), y.y);
            }
            h[k][i][j] = y;
          }
          if (!QUANT && ok && k < live) store8<T, VEC>(static_cast<T*>(a.y) + (int64_t)(row + k) * a.width, i, a.width, at, h[k][i]);
        }
      }
      if constexpr (QUANT) {
        row_max<ROWS>(amax, red[2][group], at, 1 + group);
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
          if (!ok || k >= live) continue;
          const float scale = scale_of_amax(amax[k]);
          if (at.tid == 0) a.scale[row + k] = scale;
          const float inv = quant_inverse(scale);
#pragma unroll
          for (int i = 0; i < ITERS; ++i)
            store8_int8<VEC>(static_cast<int8_t*>(a.y) + (int64_t)(row + k) * a.width, i, a.width, at,
                             inv == inv ? quantize8<false>(h[k][i], scale, inv) : quantize8<true>(h[k][i], scale, inv));
        }
      } else if (post == nullptr) {
        // a single reduction a row: its buffer is written again only behind this barrier
        if (at.threads > 32) named_barrier_sync(1 + group, at.threads);
      }
    }
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&pipe.empty[stage]);
    if (++stage == stages) { stage = 0; phase ^= 1; }
  }
  // Give copies that are still in flight time to land before shared memory is released.
  if (!feed.ok || *pipe.abort_flag)
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  __syncthreads();
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

constexpr int kNormGradThreads = 512;

// The arithmetic of one row of the gradient for ITERS vectors of a thread (with one, hn stays in registers between the passes).
// `load` gives operand q (0 x, 1 residual, 2 dy, 3 dh) of vector i, `params` gamma, post gamma and the row's gate, `sums` keeps the sums
// over rows (0 gamma, 1 post gamma, 2 a shared gate).  Operands and parameters are asked for again in each of the three passes, between
// which the two reductions lie.
template <typename T, typename P, bool VEC, int ITERS, bool SUM_GATE, typename Load, typename Params, typename Sums>
__device__ __forceinline__ void norm_grad_row(const NormGradArgs& a, const Place& at, int64_t row, float rs1, float rs2, const Load& load,
                                              const Params& params, Sums& sums, float (*red0)[32], float (*red1)[32], int barrier, bool ok) {
  const bool post = a.post != nullptr;
  const float2 alpha = splat(a.alpha), s1 = splat(rs1), s2 = splat(rs2);
  constexpr bool KEEP_HN = ITERS == 1;
  float2 hn_kept[KEEP_HN ? 4 : 1];
  float2 dot2 = splat(0.0f);
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    float2 g[4], w1[4], w2[4];
    params.gate(i, g);
    if (post) params.post(i, w1);
    params.gamma(i, w2);
    const Pack8<T> xr = load(0, i), rr = load(1, i), yr = load(2, i);
    float2(&acc)[4] = sums.open(0, i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float2 z = pair_of<T>(xr, j);
      if (post) z = __fmul2_rn(__fmul2_rn(z, s1), w1[j]);
      const float2 hn = __fmul2_rn(__ffma2_rn(g[j], z, __fmul2_rn(alpha, pair_of<T>(rr, j))), s2);
      if constexpr (KEEP_HN) hn_kept[j] = hn;
      const float2 d = __fmul2_rn(pair_of<T>(yr, j), hn);
      dot2 = __ffma2_rn(d, w2[j], dot2);
      acc[j] = __fadd2_rn(acc[j], d);
    }
    sums.close(0, i);
  }
  float dot[1] = {dot2.x + dot2.y};
  row_sum16<1>(dot, red0, at, barrier);
  const float2 nc2 = splat(-dot[0] * a.inv_width);
  float2 dots_v = splat(0.0f), dots_g = splat(0.0f);       // v . xn, dh . z
  float2 keep[ITERS][4];                                   // v
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    float2 g[4], w1[4], w2[4], out[4], dg[4];
    params.gate(i, g);
    if (post) params.post(i, w1);
    params.gamma(i, w2);
    const Pack8<T> xr = load(0, i), rr = load(1, i), yr = load(2, i);
    Pack8<T> hr;
    if (a.dh != nullptr) hr = load(3, i);
    float2(&acc1)[4] = sums.open(1, i);
    float2(&accg)[4] = sums.open(2, i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 xn = __fmul2_rn(pair_of<T>(xr, j), s1);
      const float2 z = post ? __fmul2_rn(xn, w1[j]) : xn;   // without post gamma s1 is 1
      const float2 hn = KEEP_HN ? hn_kept[KEEP_HN ? j : 0] : __fmul2_rn(__ffma2_rn(g[j], z, __fmul2_rn(alpha, pair_of<T>(rr, j))), s2);
      float2 dh = __fmul2_rn(s2, __ffma2_rn(hn, nc2, __fmul2_rn(pair_of<T>(yr, j), w2[j])));
      if (a.dh != nullptr) dh = __fadd2_rn(dh, pair_of<T>(hr, j));
      out[j] = __fmul2_rn(alpha, dh);
      if (SUM_GATE) {
        accg[j] = __ffma2_rn(dh, z, accg[j]);
      } else {
        dg[j] = __fmul2_rn(dh, z);
        dots_g = __fadd2_rn(dots_g, dg[j]);
      }
      float2 dz = __fmul2_rn(dh, g[j]);
      if (post) {
        const float2 t = __fmul2_rn(dz, xn);
        acc1[j] = __fadd2_rn(acc1[j], t);
        dots_v = __ffma2_rn(t, w1[j], dots_v);
        dz = __fmul2_rn(dz, w1[j]);
      }
      keep[i][j] = dz;
    }
    if (post) sums.close(1, i);
    if (SUM_GATE) sums.close(2, i);
    if (ok) {
      store8<T, VEC>(static_cast<T*>(a.dres) + row * a.width, i, a.width, at, out);
      // one gate a row: its gradient is dh * z itself
      if (!SUM_GATE && a.dgate != nullptr && !a.gate.per_row) store8<P, VEC>(static_cast<P*>(a.dgate) + row * a.width, i, a.width, at, dg);
    }
  }
  float dots[2] = {dots_v.x + dots_v.y, dots_g.x + dots_g.y};
  if constexpr (SUM_GATE) {
    float only[1] = {dots[0]};
    row_sum16<1>(only, red1, at, barrier);
    dots[0] = only[0];
  } else {
    row_sum16<2>(dots, red1, at, barrier);
  }
  const float2 nc1 = splat(-dots[0] * a.inv_width);
  if (!ok) return;
  if (!SUM_GATE && a.dgate != nullptr && a.gate.per_row && at.tid == 0) static_cast<P*>(a.dgate)[row] = narrow<P>(dots[1]);
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    if (post) {
      const Pack8<T> xr = load(0, i);
#pragma unroll
      for (int j = 0; j < 4; ++j) keep[i][j] = __fmul2_rn(s1, __ffma2_rn(__fmul2_rn(pair_of<T>(xr, j), s1), nc1, keep[i][j]));
    }
    store8<T, VEC>(static_cast<T*>(a.dx) + row * a.width, i, a.width, at, keep[i]);
  }
}

// Parameters read where they are wanted (from L1), and parameters that stay in registers.
template <typename P, bool VEC>
struct GlobalParams {
  const NormGradArgs& a;
  const Place& at;
  int64_t gate_row;
  __device__ __forceinline__ void gate(int i, float2 (&f)[4]) const { gate8<P, VEC, false>(a.gate, gate_row, i, a.width, at, f); }
  __device__ __forceinline__ void post(int i, float2 (&f)[4]) const { param8<P, VEC, false>(static_cast<const P*>(a.post), i, a.width, at, f); }
  __device__ __forceinline__ void gamma(int i, float2 (&f)[4]) const { param8<P, VEC, false>(static_cast<const P*>(a.gamma), i, a.width, at, f); }
};
struct RegisterParams {
  float2 g[4], w1[4], w2[4];
  static __device__ __forceinline__ void copy(const float2 (&from)[4], float2 (&f)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = from[j];
  }
  __device__ __forceinline__ void gate(int, float2 (&f)[4]) const { copy(g, f); }
  __device__ __forceinline__ void post(int, float2 (&f)[4]) const { copy(w1, f); }
  __device__ __forceinline__ void gamma(int, float2 (&f)[4]) const { copy(w2, f); }
};

// Sums over rows in registers.
template <int ITERS>
struct RegisterSums {
  float2 v[3][ITERS][4];
  __device__ __forceinline__ float2 (&open(int w, int i))[4] { return v[w][i]; }
  __device__ __forceinline__ void close(int, int) {}
  __device__ __forceinline__ void clear(int w) {
#pragma unroll
    for (int i = 0; i < ITERS; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[w][i][j] = make_float2(0.0f, 0.0f);
  }
};
// Sums over rows in shared memory, in two planes of four columns a vector, so that a warp's 16-byte accesses touch every bank
// once.
template <int ITERS>
struct SharedSums {
  float4* base;
  int threads, tid;
  float2 v[3][4];
  __device__ __forceinline__ float4& place(int w, int half, int i) { return base[((2 * w + half) * ITERS + i) * threads + tid]; }
  __device__ __forceinline__ float4 peek(int w, int half, int i, int further) const { return base[((2 * w + half) * ITERS + i) * threads + tid + further]; }
  __device__ __forceinline__ float2 (&open(int w, int i))[4] {
    const float4 p = place(w, 0, i), q = place(w, 1, i);
    v[w][0] = make_float2(p.x, p.y), v[w][1] = make_float2(p.z, p.w), v[w][2] = make_float2(q.x, q.y), v[w][3] = make_float2(q.z, q.w);
    return v[w];
  }
  __device__ __forceinline__ void close(int w, int i) {
    place(w, 0, i) = make_float4(v[w][0].x, v[w][0].y, v[w][1].x, v[w][1].y);
    place(w, 1, i) = make_float4(v[w][2].x, v[w][2].y, v[w][3].x, v[w][3].y);
  }
  __device__ __forceinline__ void clear(int w) {
#pragma unroll
    for (int i = 0; i < ITERS; ++i) place(w, 0, i) = place(w, 1, i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
};

// A CTA takes the rows [rows * c / CTAs, rows * (c + 1) / CTAs), `threads_per_row` threads a row and as many rows at a time as
// fit into the CTA.  Its threads keep the same columns throughout, so the sums over its rows stay with them; at the end (for a
// gate: at the end of the gate's rows) the CTA's row groups are joined in a fixed order and one partial row goes out.  SUM_GATE:
// the gate's gradient is a sum over the rows that share a gate; without it there is no gate, or one value a row, or one gate a
// row.  This form reads the rows straight from global memory, any width and alignment; the next row is on its way into L2.
template <typename T, typename P, bool VEC, int ITERS, bool SUM_GATE, int MAX_THREADS, int MIN_CTAS>
__global__ void __launch_bounds__(MAX_THREADS, MIN_CTAS)
gated_norm_grad_kernel(const NormGradArgs a, int threads_per_row) {
  constexpr bool KEEP = ITERS <= 2;
  extern __shared__ float4 column_sums[];
  __shared__ __align__(16) float red[2][MAX_THREADS / 32][2][32];
  for (int i = threadIdx.x; i < 2 * (MAX_THREADS / 32) * 64; i += blockDim.x) (&red[0][0][0][0])[i] = 0.0f;
  __syncthreads();
  const int group = threadIdx.x / threads_per_row, groups = blockDim.x / threads_per_row;
  const Place at{(int)threadIdx.x - group * threads_per_row, threads_per_row};
  SharedSums<ITERS> sums{column_sums, (int)blockDim.x, (int)threadIdx.x};
  sums.clear(0), sums.clear(1), sums.clear(2);
  auto flush = [&](int w, float* to) {                     // by the whole CTA
    if (groups > 1) __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
        float2(&v)[4] = sums.open(w, i);
        for (int g = 1; g < groups; ++g) {
          const float4 p = sums.peek(w, 0, i, g * threads_per_row), q = sums.peek(w, 1, i, g * threads_per_row);
          v[0] = make_float2(v[0].x + p.x, v[0].y + p.y), v[1] = make_float2(v[1].x + p.z, v[1].y + p.w);
          v[2] = make_float2(v[2].x + q.x, v[2].y + q.y), v[3] = make_float2(v[3].x + q.z, v[3].y + q.w);
        }
        store8<float, VEC>(to, i, a.width, at, v);
      }
    }
    if (groups > 1) __syncthreads();
  };
  const int64_t r0 = a.rows * blockIdx.x / gridDim.x, r1 = a.rows * (blockIdx.x + 1) / gridDim.x;
  for (int64_t seg = r0; seg < r1;) {
    const int64_t gate = SUM_GATE ? seg / a.gate.rows_per : 0;
    const int64_t seg_end = SUM_GATE ? min(r1, (gate + 1) * a.gate.rows_per) : r1;
    for (int64_t row = seg + group; row < seg_end; row += groups) {
      if (row + groups < r1) {
        const int64_t next = (row + groups) * a.width;
        for (int c = at.tid * (128 / (int)sizeof(T)); c < a.width; c += at.threads * (128 / (int)sizeof(T))) {
          prefetch_l2(static_cast<const T*>(a.x) + next + c);
          prefetch_l2(static_cast<const T*>(a.residual) + next + c);
          prefetch_l2(static_cast<const T*>(a.dy) + next + c);
          if (a.dh != nullptr) prefetch_l2(static_cast<const T*>(a.dh) + next + c);
        }
      }
      // The row's operands stay in registers where there is room, else they are read again for each pass (from L1).
      Pack8<T> kept[4][KEEP ? ITERS : 1];
      auto fetch = [&](int q, int i) {
        Pack8<T> raw;
        load8<T, VEC, KEEP>(static_cast<const T*>(q == 0 ? a.x : q == 1 ? a.residual : q == 2 ? a.dy : a.dh) + row * a.width, i, a.width, at, raw);
        return raw;
      };
      if constexpr (KEEP) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int i = 0; i < ITERS; ++i)
            if (q < 3 || a.dh != nullptr) kept[q][i] = fetch(q, i);
      }
      auto load = [&](int q, int i) {
        if constexpr (KEEP) return kept[q][i];
        else return fetch(q, i);
      };
      const GlobalParams<P, VEC> params{a, at, SUM_GATE ? gate : row};
      norm_grad_row<T, P, VEC, ITERS, SUM_GATE>(a, at, row, a.post != nullptr ? a.post_rstd[row] : 1.0f, a.rstd[row], load, params, sums,
                                                red[0][group], red[1][group], 1 + group, true);
    }
    if (SUM_GATE) {
      flush(2, a.part_gate + (blockIdx.x + gate) * a.width);
      sums.clear(2);
    }
    seg = seg_end;
  }
  flush(0, a.part_gamma + (int64_t)blockIdx.x * a.width);
  if (a.post != nullptr) flush(1, a.part_post + (int64_t)blockIdx.x * a.width);
}

// Full vectors, one a thread, so that everything fits into registers: the row's operands, those of the next row on their way, the
// parameters and the sums.
template <typename T, typename P, bool SUM_GATE>
__global__ void __launch_bounds__(kNormGradThreads, 1)
gated_norm_grad_vector_kernel(const NormGradArgs a, int threads_per_row) {
  constexpr bool VEC = true;
  constexpr bool AHEAD = sizeof(T) == 2;                   // fp32 rows have no registers to wait in: they wait in L2
  extern __shared__ float4 joined[];                       // [2][threads]
  __shared__ __align__(16) float red[2][kNormGradThreads / 32][2][32];
  for (int i = threadIdx.x; i < 2 * (kNormGradThreads / 32) * 64; i += blockDim.x) (&red[0][0][0][0])[i] = 0.0f;
  __syncthreads();
  const int group = threadIdx.x / threads_per_row, groups = blockDim.x / threads_per_row;
  const Place at{(int)threadIdx.x - group * threads_per_row, threads_per_row};
  RegisterSums<1> sums;
  sums.clear(0), sums.clear(1), sums.clear(2);
  auto flush = [&](int w, float* to) {                     // by the whole CTA
    float2(&v)[4] = sums.open(w, 0);
    if (groups > 1) {
      __syncthreads();
      if (group > 0) {
        joined[threadIdx.x] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        joined[blockDim.x + threadIdx.x] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
      }
      __syncthreads();
    }
    if (group == 0) {
      for (int g = 1; g < groups; ++g) {
        const float4 p = joined[threadIdx.x + g * threads_per_row], q = joined[blockDim.x + threadIdx.x + g * threads_per_row];
        v[0] = make_float2(v[0].x + p.x, v[0].y + p.y), v[1] = make_float2(v[1].x + p.z, v[1].y + p.w);
        v[2] = make_float2(v[2].x + q.x, v[2].y + q.y), v[3] = make_float2(v[3].x + q.z, v[3].y + q.w);
      }
      store8<float, VEC>(to, 0, a.width, at, v);
    }
  };
  auto fetch = [&](int64_t row, Pack8<T>(&to)[4], float& rs1, float& rs2) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q < 3 || a.dh != nullptr)
        load8<T, VEC>(static_cast<const T*>(q == 0 ? a.x : q == 1 ? a.residual : q == 2 ? a.dy : a.dh) + row * a.width, 0, a.width, at, to[q]);
    rs2 = a.rstd[row];
    rs1 = a.post != nullptr ? a.post_rstd[row] : 1.0f;
  };
  RegisterParams params;
  if (a.post != nullptr) param8<P, VEC, false>(static_cast<const P*>(a.post), 0, a.width, at, params.w1);
  param8<P, VEC, false>(static_cast<const P*>(a.gamma), 0, a.width, at, params.w2);
  const int64_t r0 = a.rows * blockIdx.x / gridDim.x, r1 = a.rows * (blockIdx.x + 1) / gridDim.x;
  for (int64_t seg = r0; seg < r1;) {
    const int64_t gate = SUM_GATE ? seg / a.gate.rows_per : 0;
    const int64_t seg_end = SUM_GATE ? min(r1, (gate + 1) * a.gate.rows_per) : r1;
    if (SUM_GATE) gate8<P, VEC, false>(a.gate, gate, 0, a.width, at, params.g);
    Pack8<T> kept[4], next[4];
    float rs1 = 1.0f, rs2 = 0.0f, next1 = 1.0f, next2 = 0.0f;
    if (AHEAD && seg + group < seg_end) fetch(seg + group, next, next1, next2);
    for (int64_t row = seg + group; row < seg_end; row += groups) {
      if constexpr (AHEAD) {
#pragma unroll
        for (int q = 0; q < 4; ++q) kept[q] = next[q];
        rs1 = next1, rs2 = next2;
        if (row + groups < seg_end) fetch(row + groups, next, next1, next2);
      } else {
        if (row + groups < r1) {
          const int64_t ahead = (row + groups) * a.width + at.tid * 8;
          if (at.tid % 4 == 0) {                           // one of the four threads of a 128-byte line
            prefetch_l2(static_cast<const T*>(a.x) + ahead);
            prefetch_l2(static_cast<const T*>(a.residual) + ahead);
            prefetch_l2(static_cast<const T*>(a.dy) + ahead);
            if (a.dh != nullptr) prefetch_l2(static_cast<const T*>(a.dh) + ahead);
          }
        }
        fetch(row, kept, rs1, rs2);
      }
      if (!SUM_GATE) gate8<P, VEC, false>(a.gate, row, 0, a.width, at, params.g);
      auto load = [&](int q, int) { return kept[q]; };
      norm_grad_row<T, P, VEC, 1, SUM_GATE>(a, at, row, rs1, rs2, load, params, sums, red[0][group], red[1][group], 1 + group, true);
    }
    if (SUM_GATE) {
      flush(2, a.part_gate + (blockIdx.x + gate) * a.width);
      sums.clear(2);
    }
    seg = seg_end;
  }
  flush(0, a.part_gamma + (int64_t)blockIdx.x * a.width);
  if (a.post != nullptr) flush(1, a.part_post + (int64_t)blockIdx.x * a.width);
}

// The same for rows that do not come as full vectors, through shared memory (6124 rows of 1111 f16 with a gate for every 1531: 55 us);
// sums in registers, joined by the CTA's row groups in
// shared memory in a fixed order.
template <typename T, typename P, bool SUM_GATE>
__global__ void __launch_bounds__(kRowPipeThreads, 1)
gated_norm_grad_pipe_kernel(const NormGradArgs a, int threads_per_row, int stages) {
  extern __shared__ __align__(16) uint8_t pipe_smem[];
  constexpr bool VEC = false;
  constexpr int ITERS = 1;
  __shared__ __align__(16) float red[2][kRowPipeThreads / 32][2][32];
  for (int i = threadIdx.x; i < 2 * (kRowPipeThreads / 32) * 64; i += blockDim.x) (&red[0][0][0][0])[i] = 0.0f;   // behind the next barrier
  const int readers = blockDim.x, groups = readers / threads_per_row;
  const RowPipe pipe = row_pipe_init(pipe_smem, stages, 4, groups, (int64_t)a.width * sizeof(T), a.rows, readers / 32);
  float* joined = reinterpret_cast<float*>(pipe.slot(stages, 0));   // [width] behind the ring
  const int r0 = (int)(a.rows * blockIdx.x / gridDim.x), r1 = (int)(a.rows * (blockIdx.x + 1) / gridDim.x);   // fewer than 2^30 rows
  // Chunks do not cross the end of a gate's rows, which the feed and the rows walk along (a division for every chunk cost more).
  const int rows_per = (int)min(a.gate.rows_per, a.rows);
  const int gate0 = SUM_GATE ? r0 / rows_per : 0, gate0_end = SUM_GATE ? (gate0 + 1) * rows_per : 0;
  auto chunk_end = [&](int row, int& gate_end) {
    int end = min(row + groups, r1);
    if (SUM_GATE) {
      if (row == gate_end) gate_end += rows_per;
      end = min(end, gate_end);
    }
    return end;
  };
  const void* const src[4] = {a.x, a.residual, a.dy, a.dh};
  RowPipeFeed feed{r0, 0, 0, true};
  int feed_gate_end = gate0_end;
  auto fill = [&]() {                                      // by the first warp
    if (feed.row >= r1 || !feed.ok) return;
    const int end = chunk_end(feed.row, feed_gate_end);
    feed.ok = row_pipe_fill(pipe, src, feed.stage, feed.phase, feed.row, end - feed.row, threadIdx.x & 31);
    feed.next(end, stages);
  };
  if (threadIdx.x < 32)
    for (int i = 0; i < stages; ++i) fill();
  int stage = 0;
  uint32_t phase = 0;
  {
    const int group = threadIdx.x / threads_per_row;
    const Place at{(int)threadIdx.x - group * threads_per_row, threads_per_row};
    RegisterSums<ITERS> sums;
    sums.clear(0), sums.clear(1), sums.clear(2);
    auto flush = [&](int w, float* to) {                   // by the whole CTA
      if (groups > 1) {
        for (int g = 0; g < groups; ++g) {
          if (g == group) {
#pragma unroll
            for (int i = 0; i < ITERS; ++i)
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const int c = at.col<VEC>(i, j);
                const float v = (j & 1) ? sums.v[w][i][j >> 1].y : sums.v[w][i][j >> 1].x;
                if (c < a.width) joined[c] = g == 0 ? v : joined[c] + v;
              }
          }
          __syncthreads();
        }
        for (int c = threadIdx.x; c < a.width; c += readers) to[c] = joined[c];
        __syncthreads();
      } else {
#pragma unroll
        for (int i = 0; i < ITERS; ++i) store8<float, VEC>(to, i, a.width, at, sums.v[w][i]);
      }
    };
    // The statistics of this group's next row are loaded a chunk ahead.
    float next1 = 1.0f, next2 = 0.0f;
    auto look = [&](int chunk, int end) {
      if (chunk + group < end) {
        next2 = a.rstd[chunk + group];
        if (a.post != nullptr) next1 = a.post_rstd[chunk + group];
      }
    };
    int gate = gate0, gate_end = gate0_end, end = r0 < r1 ? chunk_end(r0, gate_end) : r0;
    look(r0, end);
    // A thread's columns stay the same: so do its parameters, but for the gate.
    RegisterParams params;
    if (a.post != nullptr) param8<P, VEC, false>(static_cast<const P*>(a.post), 0, a.width, at, params.w1);
    param8<P, VEC, false>(static_cast<const P*>(a.gamma), 0, a.width, at, params.w2);
    int have_gate = -1;
    bool ok = true;
    for (int chunk = r0; chunk < r1;) {
      const int row = chunk + group;
      const float rs1 = next1, rs2 = next2;
      const bool last_of_gate = SUM_GATE && (end == r1 || end == gate_end);
      const int next_end = end < r1 ? chunk_end(end, gate_end) : end;
      look(end, next_end);
      ok = mbar_wait(&pipe.full[stage], phase, pipe.abort_flag, kDevTimeoutEpilogue) && ok;
      if (threadIdx.x < 32 && chunk > r0) fill();
      const int row_gate = SUM_GATE ? gate : row;
      if (row < end) {                                     // the same for all threads of the row
        const int off = (int)((chunk * pipe.row_bytes) & 15) + group * (int)pipe.row_bytes;
        Pack8<T> kept[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (q < 3 || a.dh != nullptr) kept[q] = smem8<T, VEC>(pipe.slot(stage, q) + off, 0, a.width, at);
        auto load = [&](int q, int) { return kept[q]; };
        if (row_gate != have_gate) gate8<P, VEC, false>(a.gate, row_gate, 0, a.width, at, params.g);
        have_gate = row_gate;
        norm_grad_row<T, P, VEC, ITERS, SUM_GATE>(a, at, row, rs1, rs2, load, params, sums, red[0][group], red[1][group], 1 + group, ok);
      }
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(&pipe.empty[stage]);
      if (++stage == stages) { stage = 0; phase ^= 1; }
      if (last_of_gate) {
        flush(2, a.part_gate + (int64_t)(blockIdx.x + gate) * a.width);
        sums.clear(2);
        ++gate;
      }
      chunk = end;
      end = next_end;
    }
    flush(0, a.part_gamma + (int64_t)blockIdx.x * a.width);
    if (a.post != nullptr) flush(1, a.part_post + (int64_t)blockIdx.x * a.width);
  }
  // Give copies that are still in flight time to land before shared memory is released.
  if (!feed.ok || *pipe.abort_flag)
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  __syncthreads();
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

// Vectors a thread takes of a row in the kernels that read rows straight into registers.
inline int norm_iters(int64_t width, bool many) {
  if (width > 8192) return 4;
  if (!many || width % 512 != 0) return 1;
  return width <= 4096 ? 2 : width % 1024 == 0 ? 4 : 1;
}

// Full vectors: a width that whole warps of vectors make up, however many vectors a thread takes, and 16-byte aligned rows and
// parameters.
inline bool norm_vec(int64_t width, std::initializer_list<const void*> ptrs) {
  const int64_t step = width > 8192 ? 1024 : width > 4096 ? 512 : 256;
  if (width % step != 0) return false;
  for (const void* p : ptrs)
    if (!aligned(p, 16)) return false;
  return true;
}

// Shape of a launch with rows through shared memory: threads a row (one vector each), groups of `rows` rows at a time, stages.
struct RowPipePlan {
  int threads, groups, stages, smem;
  bool fits;
};
inline RowPipePlan row_pipe_plan(int64_t width, int element, int arrays, int rows, int64_t all_rows, int64_t ctas, int extra) {
  RowPipePlan p{};
  if (all_rows >= (1LL << 30)) return p;                   // rows are counted in 32 bits
  const int64_t rows_per_cta = ceil_div(all_rows, ctas);
  p.threads = (int)ceil_div(ceil_div(width, 8), 32) * 32;
  if (p.threads > kRowPipeThreads) return p;
  p.groups = kRowPipeThreads / p.threads;
  if (p.groups > 14) p.groups = 14;                         // named barriers 1 .. 14
  if (p.groups * rows > rows_per_cta) p.groups = (int)ceil_div(rows_per_cta, rows);
  const int stage = arrays * row_pipe_array_bytes(p.groups * rows, width * element);
  p.stages = (kRowPipeSmem - extra) / stage;
  if (p.stages > kRowPipeMaxStages) p.stages = kRowPipeMaxStages;
  p.smem = p.stages * stage + extra;
  p.fits = p.stages >= 2;
  return p;
}

// Full vectors: a handful of rows (no more than two an SM) get as many threads a row as it has vectors, for the shortest way
// through a row; more rows 256 threads (512 above 8192 columns) with two or four vectors each, four CTAs an SM (4096 bf16 columns,
// one vector a thread against two: 16 rows 6.1 / 8.2 us, 296 8.2 / 10.2, 600 10.2 / 10.2, 4096 32.8 / 30.7).  Many rows that are not
// made of full vectors go through shared memory from a few hundred columns up to 4096 and from a 16-byte boundary on (f16, straight
// from global memory against through shared memory: 600 rows of 1111 8.2 / 10.2 us, 6124 32.8 / 30.7, 3000 of 4000 51.2 / 45.1;
// 6124 of 264 16.4 / 16.4, 20000 of 96 18.4 / 20.5).  What a width off the grid of full vectors costs, bf16, forward: 16384 rows of 1152
// 64 us and 6144 of 2880 68 (where 8192 of 4096 take 47), 2048 of 12296 266 (of 12288 47).
template <typename T, typename P, bool VEC, bool QUANT>
int launch_norm(const NormArgs& a, cudaStream_t st) {
  const bool many = a.rows > 2 * sm_count();
  if constexpr (!VEC) {
    const int64_t ctas = a.rows < sm_count() ? a.rows : sm_count();
    const RowPipePlan p = row_pipe_plan(a.width, sizeof(T), 2, 2, a.rows, ctas, 0);
    if (a.rows > 8 * sm_count() && a.width >= 512 && p.fits && aligned(a.x, 16) && aligned(a.residual, 16)) {
      constexpr auto kern = gated_norm_pipe_kernel<T, P, QUANT>;
      if (int rc = ensure_dynamic_smem<kern>(kRowPipeSmem, "gated_add_rms_norm")) return rc;
      kern<<<(unsigned)ctas, p.groups * p.threads, p.smem, st>>>(a, p.threads, p.stages);
      return check_launch("gated_add_rms_norm");
    }
  }
  const int iters = norm_iters(a.width, many && VEC);
  const int threads = (int)ceil_div(ceil_div(a.width, 8 * iters), 32) * 32;
#define B200Q_NORM(I, MAX, MIN)                                                                  \
  {                                                                                              \
    constexpr auto kern = gated_norm_kernel<T, P, VEC, I, QUANT, MAX, MIN>;                      \
    const int64_t cap = (int64_t)sm_count() * resident_ctas<kern>(threads);                      \
    kern<<<(unsigned)(a.rows < cap ? a.rows : cap), threads, 0, st>>>(a);                        \
  }
  if (iters == 1) {
    B200Q_NORM(1, 1024, 1)
  } else if (iters == 2) {
    if constexpr (VEC) B200Q_NORM(2, 256, 4)
  } else {
    B200Q_NORM(4, 512, 1)
  }
#undef B200Q_NORM
  return check_launch("gated_add_rms_norm");
}

// CTAs of the gradient kernels, each of which writes one row of partial sums per parameter: one an SM.
inline int grad_ctas(int64_t rows) { return (int)(rows < sm_count() ? rows : sm_count()); }

// Full vectors: one CTA of 512 threads an SM.  Up to 4096 columns a thread has one vector of a row, and everything fits into its
// registers (8192 rows of 4096 bf16 with all three sums: 93 us, 4.3 TB/s, half of the issue slots, the packed fp32 pipe and the
// row sums' shuffles; two vectors a thread with the sums in shared memory took 121, rows through shared memory 176 to 203; 16384 rows of 1024
// 45 against 61); above two (4096 rows of 8192: 125 us) or four vectors a thread.
// Else through shared memory, up to 4096 columns and from a 16-byte boundary on (f16, read three times from global memory against
// that: 100 rows of 1111 65 / 16 us, 6124 309 / 59, 3000 of 4000 342 / 84, 20000 of 96 364 / 47), and straight for what is left, with
// spills of 1 to 1.4 KB a thread (bf16: 4096 rows of 5376 620 us, 2048 of 12296 687, where 2048 of 12288 take 172).
template <typename T, typename P, bool VEC>
int launch_norm_grad(const NormGradArgs& a, const NormSumArgs& s, bool sum_gate, cudaStream_t st) {
#define B200Q_NORM_GRAD(I, MAX, MIN, SUM)                                                                                \
  {                                                                                                                      \
    constexpr auto kern = gated_norm_grad_kernel<T, P, VEC, I, SUM, MAX, MIN>;                                           \
    if (int rc = ensure_dynamic_smem<kern>(3 * 2 * 16 * I * MAX, "gated_add_rms_norm_grad")) return rc;                  \
    int groups = MAX / threads;                                                                                          \
    if (groups > 15) groups = 15;                          /* named barriers */                                          \
    if (groups > ceil_div(a.rows, s.ctas)) groups = (int)ceil_div(a.rows, s.ctas);                                       \
    /* three sums of every column: at most 192 KB */                                                                     \
    kern<<<s.ctas, groups * threads, 3 * 2 * 16 * I * groups * threads, st>>>(a, threads);                               \
  }
#define B200Q_NORM_GRAD_BOTH(I, MAX, MIN)                                                                                \
  if (sum_gate) B200Q_NORM_GRAD(I, MAX, MIN, true) else B200Q_NORM_GRAD(I, MAX, MIN, false)
  if constexpr (VEC) {
    if (a.width <= 8 * kNormGradThreads) {
      const int threads = (int)(a.width / 8);
      int groups = kNormGradThreads / threads;
      if (groups > 15) groups = 15;                        // named barriers
      if (groups > ceil_div(a.rows, s.ctas)) groups = (int)ceil_div(a.rows, s.ctas);
      const int smem = 2 * 16 * groups * threads;
      if (sum_gate) gated_norm_grad_vector_kernel<T, P, true><<<s.ctas, groups * threads, smem, st>>>(a, threads);
      else gated_norm_grad_vector_kernel<T, P, false><<<s.ctas, groups * threads, smem, st>>>(a, threads);
    } else {
      const int iters = a.width > 8192 ? 4 : 2;
      const int threads = (int)(a.width / (8 * iters));
      if (iters == 4) {
        B200Q_NORM_GRAD_BOTH(4, 512, 1)
      } else {
        B200Q_NORM_GRAD_BOTH(2, 512, 1)
      }
    }
  } else {
    const RowPipePlan p = row_pipe_plan(a.width, sizeof(T), 4, 1, a.rows, s.ctas, (int)((a.width * 4 + 15) & ~15));
    if (p.fits && aligned(a.x, 16) && aligned(a.residual, 16) && aligned(a.dy, 16) && aligned(a.dh, 16)) {
#define B200Q_NORM_GRAD_PIPE(SUM)                                                                                        \
  {                                                                                                                      \
    constexpr auto kern = gated_norm_grad_pipe_kernel<T, P, SUM>;                                                        \
    if (int rc = ensure_dynamic_smem<kern>(kRowPipeSmem, "gated_add_rms_norm_grad")) return rc;                          \
    kern<<<s.ctas, p.groups * p.threads, p.smem, st>>>(a, p.threads, p.stages);                                          \
  }
      if (sum_gate) B200Q_NORM_GRAD_PIPE(true) else B200Q_NORM_GRAD_PIPE(false)
#undef B200Q_NORM_GRAD_PIPE
    } else {
      const int threads = (int)ceil_div(ceil_div(a.width, 32), 32) * 32;
      B200Q_NORM_GRAD_BOTH(4, 512, 1)
    }
  }
#undef B200Q_NORM_GRAD_BOTH
#undef B200Q_NORM_GRAD
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
  if (a->width == 0) {                                       // the mean over nothing is NaN (all bits set): the statistics are defined here too
    cudaError_t e = cudaSuccess;
    if (quant) e = cudaMemsetAsync(a->scale, 0, (size_t)a->rows * 4, st);
    for (float* stat : {a->rstd, a->post_rstd})
      if (e == cudaSuccess && stat != nullptr) e = cudaMemsetAsync(stat, 0xFF, (size_t)a->rows * 4, st);
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
