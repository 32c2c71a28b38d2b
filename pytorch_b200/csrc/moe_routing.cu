// Tokens to experts and back: the data movement of a mixture-of-experts layer.
//
//   n = tokens * topk assignments, assignment i = (token i / topk, slot i % topk), expert e_i
//   row of i      #{j : e_j < e_i, or e_j = e_i and j < i}        (a stable sort by expert)
//   route         out[row_i] = x[i / topk], optionally times the expert's smooth scales and quantised to int8
//   combine       y[t] = sum_k w[t,k] * rows[row of (t,k)]        (fp32 sum in the order of k, rounded once)
//   combine grad  drows[row of (t,k)] = w[t,k] * dy[t],  dw[t,k] = <rows[row of (t,k)], dy[t]>
//
// An expert outside the layer's range (-1 for a padded token) has no row: its row index is -1, its place in
// `combine` adds nothing and is not read, and the rows past the last expert's are zero.
//
// Everything here is bound by HBM (or, for a decode step, by the latency of a launch), so each op touches its big
// operands once and uses few launches: up to kDirectIds assignments every CTA finds its own rows by comparing
// with all indices (one launch); more are sorted first by one cluster of CTAs in shared memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"

namespace b200q {
namespace {

constexpr int kMaxExperts = 1024;
// Assignments up to which every CTA counts for itself instead of a sort in front.  With 4096 columns and 64 experts, one launch
// against two: copied 128 rows 8.2 / 10.2 us, 1024 10.2 / 12.3, 4096 18.4 / 18.4; quantised 128 6.1 / 12.3, 2048 16.4 / 18.4,
// 4096 34.8 / 22.5.
constexpr int kDirectIds = 2048;
constexpr int kKeyShift = 12;             // (expert, assignment) in one word on that path: 1025 keys x 4096 places
static_assert(kDirectIds <= (1 << kKeyShift), "an assignment's number fits below the expert");
constexpr int kNoExpert = -1;

// Expert relative to the range [begin, begin + experts), or kNoExpert.  begin is not negative, so as an unsigned number the
// difference of an index before it, or of a negative one, is past any range.
__device__ __forceinline__ int expert_in_range(int64_t id, int64_t begin, int experts) {
  const uint64_t e = static_cast<uint64_t>(id) - static_cast<uint64_t>(begin);
  return e < static_cast<uint64_t>(experts) ? static_cast<int>(e) : kNoExpert;
}
template <typename IdT>
__device__ __forceinline__ int expert_of(const IdT* __restrict__ ids, int64_t i, int64_t begin, int experts) {
  return expert_in_range(static_cast<int64_t>(ids[i]), begin, experts);
}

// ------------------------------------------------------------------------------------------------ sorting
// Stable counting sort of up to 2^31 indices by one cluster of CTAs.  Warp w of CTA c owns a contiguous piece of
// the indices, so (c, w, position) is the order of the assignments.  Pass 1 counts every warp's experts in shared
// memory; a prefix over warps, over the CTAs of the cluster (through distributed shared memory) and over the experts
// turns the counts into first rows; pass 2 walks the indices again, 32 a step, and hands the rows out: the lanes with the
// same expert find one another by a ballot for each bit of the expert's number, and one of them moves the expert's next
// row on.  row_info, when wanted, gets the token and the expert of every row that has an owner.  No global scratch, no atomics
// outside shared memory, no waiting but the cluster's barrier.
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortBatch = 8;             // index loads in flight per lane
constexpr int kExpertBits = 11;           // hold the numbers 0 .. kMaxExperts (fewer ballots for fewer experts gained nothing: 18.4 us with 6 and 11)
static_assert(kMaxExperts < (1 << kExpertBits), "an expert's number and the one for none");

template <typename IdT>
__global__ void __launch_bounds__(kSortThreads, 1)
moe_sort_kernel(const IdT* __restrict__ ids, int64_t n, int64_t begin, int experts, int64_t strict_limit,
                int32_t* __restrict__ row_idx, int32_t* __restrict__ row_src, int64_t* __restrict__ expert_tokens,
                int cumulative, int32_t* __restrict__ valid_rows, int2* __restrict__ row_info, int topk) {
  extern __shared__ int sort_smem[];
  int* hist = sort_smem;                                   // [kSortWarps][experts]
  int* total = hist + kSortWarps * experts;                // [experts] this CTA's counts
  __shared__ int warp_sums[32];
  launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank(), ctas = (int)cluster_nctarank();
  const int64_t steps = (n + 31) >> 5;                     // groups of 32 indices, dealt out in contiguous pieces
  const int64_t piece = rank * (int64_t)kSortWarps + warp, pieces = (int64_t)ctas * kSortWarps;
  const int64_t s0 = steps * piece / pieces, s1 = steps * (piece + 1) / pieces;
  int* mine = hist + warp * experts;
  // The experts of one batch of steps (kNoExpert past the end or outside the range).
  auto load = [&](int64_t s, int (&e)[kSortBatch]) {
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b) {
      const int64_t i = (s + b) * 32 + lane;
      e[b] = kNoExpert;
      if (s + b < s1 && i < n) {
        const int64_t id = static_cast<int64_t>(ids[i]);
        e[b] = expert_in_range(id, begin, experts);
        if (strict_limit && e[b] < 0 && id >= strict_limit) record_device_error(kDevExpertRange);
      }
    }
  };
  int e[kSortBatch];
  load(s0, e);
  for (int i = lane; i < experts; i += 32) mine[i] = 0;
  __syncwarp();
  for (int64_t s = s0;;) {
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b)
      if (e[b] >= 0) atomicAdd(mine + e[b], 1);
    s += kSortBatch;
    if (s >= s1) break;
    load(s, e);
  }
  __syncthreads();

  // One expert a thread: its rows in this CTA's warps, in the lower CTAs and in all, then a scan over the experts.
  const int x = threadIdx.x;
  int count[kSortWarps];
  int here = 0;
  if (x < experts) {
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) count[w] = hist[w * experts + x];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) here += count[w];
    total[x] = here;
  }
  int lower = 0, all = here;
  if (ctas > 1) {
    cluster_sync_all();
    all = 0;
    if (x < experts) {
      for (int c = 0; c < ctas; ++c) {
        const int v = (int)ld_shared_cluster_u32(map_to_cta(smem_u32(total + x), c));
        if (c < rank) lower += v;
        all += v;
      }
    }
  }
  int incl = all;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int v = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    warp_sums[lane] = v;
  }
  __syncthreads();
  if (warp > 0) incl += warp_sums[warp - 1];
  const int valid = warp_sums[31];
  if (x < experts) {
    int next = incl - all + lower;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      hist[w * experts + x] = next;
      next += count[w];
    }
    if (rank == 0 && expert_tokens != nullptr) expert_tokens[x] = cumulative ? incl : all;
  }
  if (rank == 0 && threadIdx.x == 0 && valid_rows != nullptr) *valid_rows = valid;
  if (row_src != nullptr)                                  // rows that no assignment owns
    for (int64_t r = valid + (int64_t)rank * kSortThreads + threadIdx.x; r < n; r += (int64_t)ctas * kSortThreads) row_src[r] = -1;
  __syncthreads();

  if (s1 - s0 > kSortBatch) load(s0, e);                   // else they are still there
  for (int64_t s = s0; s < s1;) {
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b) {
      if (s + b >= s1) break;
      const int key = e[b] < 0 ? experts : e[b];
      unsigned same = 0xffffffffu;
#pragma unroll
      for (int q = 0; q < kExpertBits; ++q) {
        const bool one = (key >> q) & 1;
        const unsigned ballot = __ballot_sync(0xffffffffu, one);
        same &= one ? ballot : ~ballot;
      }
      const int leader = __ffs(same) - 1;
      int base = 0;
      if (e[b] >= 0 && lane == leader) {
        base = mine[key];
        mine[key] = base + __popc(same);
      }
      base = __shfl_sync(0xffffffffu, base, leader);
      const int64_t i = (s + b) * 32 + lane;
      const int row = e[b] >= 0 ? base + __popc(same & ((1u << lane) - 1)) : -1;
      if (i < n) row_idx[i] = row;
      if (row >= 0 && row_src != nullptr) row_src[row] = (int32_t)i;
      if (row >= 0 && row_info != nullptr) row_info[row] = make_int2((int)i / topk, key);
      __syncwarp();
    }
    s += kSortBatch;
    if (s < s1) load(s, e);
  }
  if (ctas > 1) cluster_sync_all();                        // nobody leaves while its counts may still be read
}

// ------------------------------------------------------------------------------------------------ direct counting
// The word that orders the assignments: expert, then number; padded ones behind every expert.
template <typename IdT>
__device__ __forceinline__ int direct_key(const IdT* __restrict__ ids, int i, int64_t begin, int experts) {
  const int e = expert_of(ids, i, begin, experts);
  return ((e < 0 ? experts : e) << kKeyShift) | i;
}

// Rows of the COUNT assignments first, first + 1, ... (those below n), by the whole CTA: how many keys are smaller.
template <int COUNT, typename IdT>
__device__ __forceinline__ void direct_rows(const IdT* __restrict__ ids, int n, int64_t begin, int experts, int first,
                                            int (&red)[COUNT][32], int (&rows)[COUNT]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nwarps = blockDim.x >> 5;
  int key[COUNT], cnt[COUNT];
#pragma unroll
  for (int k = 0; k < COUNT; ++k) {
    key[k] = direct_key(ids, min(first + k, n - 1), begin, experts);
    cnt[k] = 0;
  }
  for (int j = threadIdx.x; j < n; j += blockDim.x) {
    const int other = direct_key(ids, j, begin, experts);
#pragma unroll
    for (int k = 0; k < COUNT; ++k) cnt[k] += other < key[k];
  }
  __syncthreads();                                         // `red` may still be read from an earlier round
#pragma unroll
  for (int k = 0; k < COUNT; ++k) {
    const int c = __reduce_add_sync(0xffffffffu, cnt[k]);
    if (lane == 0) red[k][warp] = c;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < COUNT; ++k) rows[k] = __reduce_add_sync(0xffffffffu, lane < nwarps ? red[k][lane] : 0);
}

// Rows of every expert (cumulative or not), by one CTA, for the direct path.
template <typename IdT>
__device__ __forceinline__ void direct_expert_tokens(const IdT* __restrict__ ids, int n, int64_t begin, int experts, int64_t strict_limit,
                                                     int64_t* __restrict__ expert_tokens, int cumulative) {
  __shared__ int count[kMaxExperts];
  for (int e = threadIdx.x; e < experts; e += blockDim.x) count[e] = 0;
  __syncthreads();
  for (int j = threadIdx.x; j < n; j += blockDim.x) {
    const int e = expert_of(ids, j, begin, experts);
    if (e >= 0) atomicAdd(&count[e], 1);                   // integers: the same sum in any order
    if (strict_limit && static_cast<int64_t>(ids[j]) >= strict_limit) record_device_error(kDevExpertRange);
  }
  __syncthreads();
  if (expert_tokens == nullptr || threadIdx.x >= 32) return;
  int run = 0;
  for (int e0 = 0; e0 < experts; e0 += 32) {
    const int e = e0 + threadIdx.x;
    const int c = e < experts ? count[e] : 0;
    int incl = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if ((int)threadIdx.x >= o) incl += v;
    }
    if (e < experts) expert_tokens[e] = cumulative ? run + incl : c;
    run += __shfl_sync(0xffffffffu, incl, 31);
  }
}

// ------------------------------------------------------------------------------------------------ rows as bytes
template <int BYTES> struct Chunk;
template <> struct Chunk<16> { using type = uint4; };
template <> struct Chunk<8> { using type = uint2; };
template <> struct Chunk<4> { using type = uint32_t; };
template <> struct Chunk<2> { using type = uint16_t; };
template <> struct Chunk<1> { using type = uint8_t; };

struct RouteIds {
  const void* ids;
  int64_t n;                 // tokens * topk
  int64_t begin;
  int experts, topk;
  int64_t strict_limit;      // indices from here on are an error (0: they are merely outside the range)
};

// Copy, few assignments: one CTA a token finds the rows of its topk slots and copies the token there; one more CTA
// counts the experts' rows.
template <typename IdT, typename VT>
__global__ void __launch_bounds__(256)
moe_copy_direct_kernel(const RouteIds r, const VT* __restrict__ x, VT* __restrict__ out, int nvec, int64_t out_rows,
                       const float* __restrict__ token_scale, float* __restrict__ out_scale, int32_t* __restrict__ row_idx,
                       int32_t* __restrict__ row_src, int64_t* __restrict__ expert_tokens, int cumulative) {
  const IdT* ids = static_cast<const IdT*>(r.ids);
  const int n = (int)r.n, tokens = n / r.topk;
  if ((int)blockIdx.x == tokens) {
    direct_expert_tokens(ids, n, r.begin, r.experts, r.strict_limit, expert_tokens, cumulative);
    return;
  }
  constexpr int KC = 8;
  __shared__ int red[KC][32];
  const int t = blockIdx.x;
  for (int k0 = 0; k0 < r.topk; k0 += KC) {
    int rows[KC];
    direct_rows(ids, n, r.begin, r.experts, t * r.topk + k0, red, rows);
    const int kc = min(KC, r.topk - k0);
    bool live[KC];
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      const int i = t * r.topk + k0 + k;
      live[k] = k < kc && expert_of(ids, min(i, n - 1), r.begin, r.experts) >= 0;
      if (k < kc && threadIdx.x == 0) {
        row_idx[i] = live[k] ? rows[k] : -1;
        if (row_src != nullptr) row_src[rows[k]] = live[k] ? i : -1;
        if (out_scale != nullptr && rows[k] < out_rows) out_scale[rows[k]] = live[k] ? token_scale[t] : 0.0f;
      }
    }
    for (int v = threadIdx.x; v < nvec; v += blockDim.x) {
      const VT val = x[(int64_t)t * nvec + v];
#pragma unroll
      for (int k = 0; k < KC; ++k)
        if (k < kc && rows[k] < out_rows) out[(int64_t)rows[k] * nvec + v] = live[k] ? val : VT{};
    }
  }
}

// Copy, many assignments: a warp takes 32 * U vectors of one token, reads them once and writes them to the token's
// rows.  The blocks past the last token clear the rows that no assignment owns.  Bound by HBM: 8192 tokens of 4096 bf16 to eight rows
// each (604 MB) in 98 us behind a sort of 14.
template <typename VT, int U>
__global__ void __launch_bounds__(256)
moe_copy_kernel(const VT* __restrict__ x, VT* __restrict__ out, int64_t tokens, int topk, int64_t nvec, int segs, int64_t out_rows,
                const float* __restrict__ token_scale, float* __restrict__ out_scale, const int32_t* row_idx,
                const int32_t* valid_rows, int64_t move_blocks) {
  const int lane = threadIdx.x & 31;
  if ((int64_t)blockIdx.x >= move_blocks) {
    wait_for_primary();
    const int64_t zb = blockIdx.x - move_blocks, zn = gridDim.x - move_blocks;
    for (int64_t row = ld_of_primary(valid_rows) + zb; row < out_rows; row += zn) {
      for (int64_t v = threadIdx.x; v < nvec; v += blockDim.x) out[row * nvec + v] = VT{};
      if (out_scale != nullptr && threadIdx.x == 0) out_scale[row] = 0.0f;
    }
    return;
  }
  const int64_t unit = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t t = unit / segs;
  if (t >= tokens) return;
  const int seg = (int)(unit - t * segs);
  const int64_t v0 = (int64_t)seg * (32 * U) + lane;
  VT val[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (v0 + 32 * u < nvec) val[u] = x[t * nvec + v0 + 32 * u];
  wait_for_primary();                                      // the sort's rows; x does not depend on it
  for (int k0 = 0; k0 < topk; k0 += 32) {
    const int mine = k0 + lane < topk ? ld_of_primary(row_idx + t * topk + k0 + lane) : -1;
    const int kc = min(32, topk - k0);
    for (int k = 0; k < kc; ++k) {
      const int64_t row = __shfl_sync(0xffffffffu, mine, k);
      if (row < 0 || row >= out_rows) continue;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v0 + 32 * u < nvec) out[row * nvec + v0 + 32 * u] = val[u];
      if (out_scale != nullptr && seg == 0 && lane == 0) out_scale[row] = token_scale[t];
    }
  }
}

// ------------------------------------------------------------------------------------------------ routing + int8
// One row: smooth multiply, row maximum, scale, quantised values, all with the helpers (and bits) of
// npu_dynamic_quant.  The CTA owns the row; each thread holds ITERS vectors of eight values.
// FULL: every thread's every vector is inside the row (no predicates; this kernel is bound by instruction issue).
template <typename ST, int ITERS, bool FULL>
__device__ __forceinline__ void load_smooth_row(const ST* __restrict__ smooth, int nvec, float2 (&sm)[ITERS][4]) {
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) sm[i][j] = make_float2(1.0f, 1.0f);
    if (smooth != nullptr && (FULL || v < nvec)) load_smooth8(smooth + (int64_t)v * 8, sm[i]);
  }
}
template <typename T, int ITERS, bool FULL>
__device__ __forceinline__ void load_row(const T* __restrict__ x, int nvec, uint4 (&to)[ITERS]) {
#pragma unroll
  for (int q = 0; q < ITERS; ++q) {
    const int v = threadIdx.x + q * blockDim.x;
    to[q] = FULL || v < nvec ? __ldg(reinterpret_cast<const uint4*>(x) + v) : make_uint4(0, 0, 0, 0);
  }
}

// `meanwhile` runs when the row's values have become products and its registers are free.
template <typename T, int ITERS, bool FULL, typename F>
__device__ __forceinline__ void quant_row_store(const uint4 (&raw)[ITERS], const float2 (&sm)[ITERS][4], int nvec,
                                                int8_t* __restrict__ y, float* __restrict__ scale_out, float* red, const F& meanwhile) {
  float2 f[ITERS][4];
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < ITERS; ++i) products8<T, true>(raw[i], sm[i], f[i], amax);
  meanwhile();
  amax = block_max(amax, red);
  const float scale = scale_of_amax(amax);
  if (threadIdx.x == 0) *scale_out = scale;
  const float inv = quant_inverse(scale);
  uint2* yr = reinterpret_cast<uint2*>(y) + threadIdx.x;
  if (inv == inv) {
#pragma unroll
    for (int i = 0; i < ITERS; ++i)
      if (FULL || threadIdx.x + i * blockDim.x < nvec) st_stream(yr + i * blockDim.x, quantize8<false>(f[i], scale, inv));
  } else {
#pragma unroll
    for (int i = 0; i < ITERS; ++i)
      if (FULL || threadIdx.x + i * blockDim.x < nvec) st_stream(yr + i * blockDim.x, quantize8<true>(f[i], scale, inv));
  }
}

// The same for any width and alignment: two passes over the row.
template <typename T, typename ST>
__device__ __forceinline__ void quant_row_generic(const T* __restrict__ x, const ST* __restrict__ smooth, int64_t width,
                                                  int8_t* __restrict__ y, float* __restrict__ scale_out, float* red) {
  float amax = 0.0f;
  for (int64_t c = threadIdx.x; c < width; c += blockDim.x) {
    float f = to_f32<T>(x[c]);
    if (smooth != nullptr) f = __fmul_rn(f, to_f32<ST>(smooth[c]));
    amax = fmaxf(amax, fabsf(f));
  }
  amax = block_max(amax, red);
  const float scale = __fdiv_rn(amax, 127.0f);
  if (threadIdx.x == 0) *scale_out = scale;
  for (int64_t c = threadIdx.x; c < width; c += blockDim.x) {
    float f = to_f32<T>(x[c]);
    if (smooth != nullptr) f = __fmul_rn(f, to_f32<ST>(smooth[c]));
    int q = 0;
    if (scale != 0.0f) q = max(-128, min(127, __float2int_rn(__fdiv_rn(f, scale))));
    y[c] = static_cast<int8_t>(q);
  }
}

__device__ __forceinline__ void zero_quant_row(int8_t* __restrict__ y, float* __restrict__ scale_out, int64_t width) {
  for (int64_t c = threadIdx.x; c < width; c += blockDim.x) y[c] = 0;
  if (threadIdx.x == 0) *scale_out = 0.0f;
}

// Few assignments: one CTA an assignment.  ITERS 0: any width and alignment.
template <typename IdT, typename T, typename ST, int ITERS>
__global__ void __launch_bounds__(512)
moe_quant_direct_kernel(const RouteIds r, const T* __restrict__ x, int64_t width, const ST* __restrict__ smooth, int smooth_rows,
                        int8_t* __restrict__ out, float* __restrict__ out_scale, int32_t* __restrict__ row_idx,
                        int32_t* __restrict__ row_src, int64_t* __restrict__ expert_tokens, int cumulative) {
  const IdT* ids = static_cast<const IdT*>(r.ids);
  const int n = (int)r.n;
  if ((int)blockIdx.x == n) {
    direct_expert_tokens(ids, n, r.begin, r.experts, r.strict_limit, expert_tokens, cumulative);
    return;
  }
  __shared__ int red_i[1][32];
  __shared__ float red[32];
  const int i = blockIdx.x;
  const T* xr = x + (int64_t)(i / r.topk) * width;
  const int nvec = (int)(width >> 3);
  uint4 raw[ITERS ? ITERS : 1];
  float2 sm_row[ITERS ? ITERS : 1][4];
  const int e = expert_of(ids, i, r.begin, r.experts);
  const ST* sm = smooth == nullptr ? nullptr : smooth + (smooth_rows > 1 ? (int64_t)max(e, 0) * width : 0);
  if constexpr (ITERS > 0) {                               // in flight while the row is being found
    load_smooth_row<ST, ITERS, false>(sm, nvec, sm_row);
    load_row<T, ITERS, false>(xr, nvec, raw);
  }
  int rows[1];
  direct_rows(ids, n, r.begin, r.experts, i, red_i, rows);
  const int64_t row = rows[0];
  if (threadIdx.x == 0) {
    row_idx[i] = e >= 0 ? (int)row : -1;
    if (row_src != nullptr) row_src[row] = e >= 0 ? i : -1;
  }
  if (e < 0) {
    zero_quant_row(out + row * width, out_scale + row, width);
    return;
  }
  if constexpr (ITERS > 0) quant_row_store<T, ITERS, false>(raw, sm_row, nvec, out + row * width, out_scale + row, red, [] {});
  else quant_row_generic<T, ST>(xr, sm, width, out + row * width, out_scale + row, red);
}

// Many assignments: persistent CTAs take contiguous pieces of the sorted rows, so a piece mostly stays with one expert,
// whose smooth scales stay in registers.  The next row is on its way from the moment this one has become products (with FULL; with
// predicates on every vector it sets out before them, into registers of its own).  4099 tokens of 5120 f16 to six rows each, with
// the sort: 68 us so, 75 with the load before the products; of 5112 columns 88 and 80.  Half of the issue slots are used, the rest waits
// for gathered rows with the 14 warps an SM that the registers leave.
template <typename T, typename ST, int ITERS, bool FULL>
__global__ void __launch_bounds__(512)
moe_quant_kernel(int64_t n, const T* __restrict__ x, int64_t width, const ST* __restrict__ smooth, int smooth_rows, int8_t* __restrict__ out,
                 float* __restrict__ out_scale, const int2* row_info, const int32_t* valid_rows) {
  __shared__ float red[2][32];
  wait_for_primary();
  const int nvec = (int)(width >> 3);
  const int64_t valid = ld_of_primary(valid_rows);
  const int64_t r0 = valid * blockIdx.x / gridDim.x, r1 = valid * (blockIdx.x + 1) / gridDim.x;
  constexpr int N = ITERS ? ITERS : 1;
  uint4 raw[N], nxt[FULL ? 1 : N];
  float2 sm_row[N][4];
  int sm_expert = -1;
  auto load = [&](int token) {
    if constexpr (ITERS > 0 && FULL) load_row<T, ITERS, FULL>(x + token * width, nvec, raw);
    if constexpr (ITERS > 0 && !FULL) load_row<T, ITERS, FULL>(x + token * width, nvec, nxt);
  };
  // A row's token and expert are read two rows ahead, its x one row ahead.
  int2 here = make_int2(0, 0), after = make_int2(0, 0);
  if (r0 < r1) {
    after = ld_of_primary_cached(row_info + r0);
    load(after.x);
  }
  int2 later = r0 + 1 < r1 ? ld_of_primary_cached(row_info + r0 + 1) : make_int2(0, 0);
  // This CTA's share of the rows that no assignment owns.
  const int64_t idle = n - valid;
  for (int64_t row = valid + idle * blockIdx.x / gridDim.x; row < valid + idle * (blockIdx.x + 1) / gridDim.x; ++row) {
    if constexpr (ITERS > 0) {
      for (int v = threadIdx.x; v < nvec; v += blockDim.x) st_stream(reinterpret_cast<uint2*>(out + row * width) + v, make_uint2(0, 0));
      if (threadIdx.x == 0) out_scale[row] = 0.0f;
    } else {
      zero_quant_row(out + row * width, out_scale + row, width);
    }
  }
  int par = 0;
  for (int64_t row = r0; row < r1; ++row) {
    here = after;
    after = later;
    if constexpr (ITERS > 0 && !FULL) {
#pragma unroll
      for (int q = 0; q < ITERS; ++q) raw[q] = nxt[q];
      if (row + 1 < r1) load(after.x);
    }
    if (row + 2 < r1) later = ld_of_primary_cached(row_info + row + 2);
    par ^= 1;                                              // a buffer is written again only behind the other one's barrier
    const ST* sm = smooth == nullptr ? nullptr : smooth + (smooth_rows > 1 ? here.y * width : 0);
    if constexpr (ITERS > 0) {
      if (sm_expert < 0 || (smooth_rows > 1 && here.y != sm_expert)) {
        load_smooth_row<ST, ITERS, FULL>(sm, nvec, sm_row);
        sm_expert = here.y;
      }
      quant_row_store<T, ITERS, FULL>(raw, sm_row, nvec, out + row * width, out_scale + row, red[par], [&] {
        if (FULL && row + 1 < r1) load(after.x);
      });
    } else {
      quant_row_generic<T, ST>(x + here.x * width, sm, width, out + row * width, out_scale + row, red[par]);
    }
  }
}

// ------------------------------------------------------------------------------------------------ combine
// Values of one 16-byte vector (or one element) as floats and back.
template <typename T, bool VEC>
struct Lanes {
  static constexpr int N = VEC ? 16 / (int)sizeof(T) : 1;
  using Raw = typename Chunk<VEC ? 16 : (int)sizeof(T)>::type;
  static __device__ __forceinline__ void unpack(const Raw& raw, float (&f)[N]) {
    const T* p = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = to_f32<T>(p[j]);
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[N]) {
    Raw raw;
    T* p = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if constexpr (sizeof(T) == 4) p[j] = f[j];
      else if constexpr (std::is_same<T, __half>::value) p[j] = __float2half_rn(f[j]);
      else p[j] = __float2bfloat16_rn(f[j]);
    }
    return raw;
  }
};

__device__ __forceinline__ float load_as_f32(const void* p, int dtype, int64_t i) {
  if (dtype == B200Q_F32) return static_cast<const float*>(p)[i];
  if (dtype == B200Q_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_from_f32(void* p, int dtype, int64_t i, float v) {
  if (dtype == B200Q_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == B200Q_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// Few tokens, short rows, any width (2.8 us for 16 tokens with eight rows of 4096 bf16: the latency of a launch and two dependent
// loads).  A thread owns one vector of one token: the loads of up to KC rows are issued before the first is used, the sum
// runs in fp32 in the order of the slots.
template <typename T, bool VEC, int KC>
__global__ void __launch_bounds__(256)
moe_combine_kernel(const T* __restrict__ rows, int64_t num_rows, const int32_t* __restrict__ row_idx, const void* __restrict__ weights,
                   int weight_dtype, T* __restrict__ out, int64_t tokens, int topk, int64_t nvec) {
  using L = Lanes<T, VEC>;
  using Raw = typename L::Raw;
  const int64_t unit = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t t = unit / nvec, v = unit - t * nvec;
  if (t >= tokens) return;
  float acc[L::N];
#pragma unroll
  for (int j = 0; j < L::N; ++j) acc[j] = 0.0f;
  for (int k0 = 0; k0 < topk; k0 += KC) {
    int64_t row[KC];
    Raw raw[KC];
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      row[k] = k0 + k < topk ? row_idx[t * topk + k0 + k] : -1;
      if (row[k] >= num_rows) row[k] = -1;
    }
#pragma unroll
    for (int k = 0; k < KC; ++k)
      if (row[k] >= 0) raw[k] = reinterpret_cast<const Raw*>(rows)[row[k] * nvec + v];
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      if (row[k] < 0) continue;
      float f[L::N];
      L::unpack(raw[k], f);
      const float w = weights != nullptr ? load_as_f32(weights, weight_dtype, t * topk + k0 + k) : 1.0f;
#pragma unroll
      for (int j = 0; j < L::N; ++j) acc[j] = fmaf(w, f[j], acc[j]);
    }
  }
  reinterpret_cast<Raw*>(out)[t * nvec + v] = L::pack(acc);
}

// Gradient of combine: one CTA a token; dy's vector stays in registers while the topk rows pass by, so dy and the
// rows are read once and drows written once.  `marks` gets a bit for every row that has an owner: a second owner
// (whose gradient would have to be added) is recorded as an error, and moe_clear_rows_kernel clears the rows
// without one.
template <typename T, bool VEC, int KC>
__global__ void __launch_bounds__(256)
moe_combine_grad_kernel(const T* __restrict__ dy, const T* __restrict__ rows, int64_t num_rows, const int32_t* __restrict__ row_idx,
                        const void* __restrict__ weights, int weight_dtype, T* __restrict__ drows, void* __restrict__ dweights,
                        uint32_t* __restrict__ marks, int topk, int64_t nvec) {
  using L = Lanes<T, VEC>;
  using Raw = typename L::Raw;
  __shared__ float red[KC][8];
  const int64_t t = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nwarps = blockDim.x >> 5;
  for (int k0 = 0; k0 < topk; k0 += KC) {
    int64_t row[KC];
    float w[KC], dot[KC];
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      row[k] = k0 + k < topk ? row_idx[t * topk + k0 + k] : -1;
      if (row[k] >= num_rows) row[k] = -1;
      w[k] = row[k] >= 0 && weights != nullptr ? load_as_f32(weights, weight_dtype, t * topk + k0 + k) : 1.0f;
      dot[k] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < KC; ++k)
      if ((int)threadIdx.x == k && row[k] >= 0) {
        const uint32_t bit = 1u << (row[k] & 31);
        if (atomicOr(marks + (row[k] >> 5), bit) & bit) record_device_error(kDevRowTwice);
      }
    for (int64_t v = threadIdx.x; v < nvec; v += blockDim.x) {
      float g[L::N];
      L::unpack(reinterpret_cast<const Raw*>(dy)[t * nvec + v], g);
      Raw raw[KC];
      if (dweights != nullptr) {
#pragma unroll
        for (int k = 0; k < KC; ++k)
          if (row[k] >= 0) raw[k] = reinterpret_cast<const Raw*>(rows)[row[k] * nvec + v];
      }
#pragma unroll
      for (int k = 0; k < KC; ++k) {
        if (row[k] < 0) continue;
        float f[L::N];
        if (dweights != nullptr) {
          L::unpack(raw[k], f);
#pragma unroll
          for (int j = 0; j < L::N; ++j) dot[k] = fmaf(f[j], g[j], dot[k]);
        }
#pragma unroll
        for (int j = 0; j < L::N; ++j) f[j] = w[k] * g[j];
        reinterpret_cast<Raw*>(drows)[row[k] * nvec + v] = L::pack(f);
      }
    }
    if (dweights == nullptr) continue;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KC; ++k) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot[k] += __shfl_xor_sync(0xffffffffu, dot[k], o);
      if (lane == 0) red[k][warp] = dot[k];
    }
    __syncthreads();
    if ((int)threadIdx.x < KC && k0 + (int)threadIdx.x < topk) {
      float s = 0.0f;
      for (int i = 0; i < nwarps; ++i) s += red[threadIdx.x][i];
      store_from_f32(dweights, weight_dtype, t * topk + k0 + threadIdx.x, s);   // no row: nothing was added
    }
  }
}

// Values of a 16-byte vector as pairs of floats, for the packed two-wide arithmetic, and back.
template <typename T>
__device__ __forceinline__ void unpack_pairs(const uint4& raw, float2 (&f)[16 / (2 * (int)sizeof(T))]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = make_float2(__uint_as_float(raw.x), __uint_as_float(raw.y));
    f[1] = make_float2(__uint_as_float(raw.z), __uint_as_float(raw.w));
  } else {
    f[0] = unpack2<T>(raw.x), f[1] = unpack2<T>(raw.y), f[2] = unpack2<T>(raw.z), f[3] = unpack2<T>(raw.w);
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack_pairs(const float2 (&f)[16 / (2 * (int)sizeof(T))]) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
  } else if constexpr (std::is_same<T, __half>::value) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 h = __float22half2_rn(f[j]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_bfloat162 h = __float22bfloat162_rn(f[j]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Both directions for many tokens, as a pipeline: a producer warp brings the rows of a token (lane k the row of slot k) and,
// for the gradient, dy into shared memory with bulk copies, kGatherBytes of every row a stage; eight warps work on them,
// a 16-byte vector of every row a thread.  The rows lie all over HBM and their indices have to be read first; the ring of
// copies keeps about 200 KB an SM in flight whatever the registers allow, and the indices of the next token are read a
// token ahead.  Bound by HBM: 8192 tokens with eight rows of 4096 bf16 each take 103 us forward (604 MB, 5.9 TB/s) and 181 for the
// gradients (1.14 GB, 6.3 TB/s).  Waits are bounded; a thread that gives one up goes on without loading or storing, so that the barriers
// still meet.
constexpr int kGatherBytes = 4096;        // of a row, per stage
constexpr int kGatherWarps = 8;
constexpr int kGatherThreads = 32 * (kGatherWarps + 1);
constexpr int kGatherSmem = 112 * 1024;   // two CTAs an SM

template <int KC, bool GRAD>
struct GatherLayout {
  static constexpr int kRows = KC + (GRAD ? 1 : 0);
  static constexpr int kStageBytes = kRows * kGatherBytes;
  static constexpr int kFit = (kGatherSmem - 1024) / kStageBytes;
  static constexpr int kStages = kFit < 16 ? kFit : 16;
  static constexpr int kBarOff = kStages * kStageBytes;        // full[S], empty[S]
  static constexpr int kMetaOff = kBarOff + 2 * kStages * 8;   // per stage and slot: row, weight; then whether all slots have rows
  static constexpr int kDynamic = kMetaOff + kStages * (KC + 1) * 8 + 128;
};

template <typename T, int KC, bool GRAD>
__global__ void __launch_bounds__(kGatherThreads, 2)
moe_gather_kernel(const T* __restrict__ dy, const T* __restrict__ rows, int64_t num_rows, const int32_t* __restrict__ row_idx,
                  const void* __restrict__ weights, int weight_dtype, T* __restrict__ out, void* __restrict__ dweights,
                  uint32_t* __restrict__ marks, int64_t tokens, int topk, int64_t row_bytes) {
  using L = GatherLayout<KC, GRAD>;
  using E = Lanes<T, true>;
  extern __shared__ uint8_t gather_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(gather_raw) + 127) & ~uintptr_t(127));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* empty = full + L::kStages;
  int2* meta = reinterpret_cast<int2*>(smem + L::kMetaOff);
  __shared__ int abort_word;
  __shared__ float red[2][KC][kGatherWarps];
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kGatherWarps);
    }
    abort_word = 0;
    fence_mbar_init();
  }
  __syncthreads();
  const int segs = (int)((row_bytes + kGatherBytes - 1) / kGatherBytes);
  int stage = 0;
  uint32_t phase = 0;

  if (warp == kGatherWarps) {
    // ------------------------------------------------------------ producer: lane k copies slot k, lane KC copies dy
    int next = -1;
    float next_w = 1.0f;
    auto look = [&](int64_t t) {
      next = lane < topk && t < tokens ? row_idx[t * topk + lane] : -1;
      if (weights != nullptr && lane < topk && t < tokens) next_w = load_as_f32(weights, weight_dtype, t * topk + lane);
    };
    look(blockIdx.x);
    bool ok = true;
    for (int64_t t = blockIdx.x; t < tokens && ok; t += gridDim.x) {
      const int64_t row = next < num_rows ? next : -1;
      const float w = next_w;
      look(t + gridDim.x);
      const uint8_t* src = nullptr;
      if (row >= 0) {
        src = reinterpret_cast<const uint8_t*>(rows) + row * row_bytes;
        if (GRAD) {
          const uint32_t bit = 1u << (row & 31);
          if (atomicOr(marks + (row >> 5), bit) & bit) record_device_error(kDevRowTwice);
        }
      }
      if (GRAD && lane == KC) src = reinterpret_cast<const uint8_t*>(dy) + t * row_bytes;
      const int copies = __popc(__ballot_sync(0xffffffffu, src != nullptr));
      const int all = copies == KC + (GRAD ? 1 : 0);
      for (int sg = 0; sg < segs; ++sg) {
        const uint32_t bytes = (uint32_t)min((int64_t)kGatherBytes, row_bytes - (int64_t)sg * kGatherBytes);
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1, abort_flag, kDevTimeoutProducer));
        if (!ok) break;
        if (lane < KC) meta[stage * (KC + 1) + lane] = make_int2((int)row, __float_as_int(w));
        if (lane == KC) meta[stage * (KC + 1) + KC] = make_int2(all, 0);
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(&full[stage], bytes * copies);
        __syncwarp();
        if (src != nullptr)
          bulk_load(smem + stage * L::kStageBytes + lane * kGatherBytes, src + (int64_t)sg * kGatherBytes, bytes, &full[stage]);
        if (++stage == L::kStages) { stage = 0; phase ^= 1; }
      }
    }
    // Give copies that are still in flight time to land before shared memory is released.
    if (!ok)
      for (int i = 0; i < 200; ++i) __nanosleep(1000);
  } else {
    // ------------------------------------------------------------ eight warps: one vector of every row a thread
    bool ok = true;
    int par = 0;
    for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x, par ^= 1) {
      float2 dot[KC];
#pragma unroll
      for (int k = 0; k < KC; ++k) dot[k] = make_float2(0.0f, 0.0f);
      for (int sg = 0; sg < segs; ++sg) {
        ok = mbar_wait(&full[stage], phase, abort_flag, kDevTimeoutEpilogue) && ok;
        const int64_t at = (int64_t)sg * kGatherBytes + threadIdx.x * 16;
        if (ok && at < row_bytes) {
          const uint8_t* in = smem + stage * L::kStageBytes + threadIdx.x * 16;
          const int2* slots = meta + stage * (KC + 1);
          if constexpr (GRAD) {
            float2 g[E::N / 2];
            unpack_pairs<T>(*reinterpret_cast<const uint4*>(in + KC * kGatherBytes), g);
            auto slot = [&](int k, int2 m) {
              float2 f[E::N / 2];
              unpack_pairs<T>(*reinterpret_cast<const uint4*>(in + k * kGatherBytes), f);
              const float2 w = make_float2(__int_as_float(m.y), __int_as_float(m.y));
#pragma unroll
              for (int j = 0; j < E::N / 2; ++j) {
                dot[k] = __ffma2_rn(f[j], g[j], dot[k]);
                f[j] = __fmul2_rn(w, g[j]);
              }
              __stcs(reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(out) + m.x * row_bytes + at), pack_pairs<T>(f));
            };
            if (slots[KC].x) {                             // the same for all threads
#pragma unroll
              for (int k = 0; k < KC; ++k) slot(k, slots[k]);
            } else {
#pragma unroll
              for (int k = 0; k < KC; ++k)
                if (slots[k].x >= 0) slot(k, slots[k]);
            }
          } else {
            float2 acc[E::N / 2];
#pragma unroll
            for (int j = 0; j < E::N / 2; ++j) acc[j] = make_float2(0.0f, 0.0f);
            auto slot = [&](int k) {
              float2 f[E::N / 2];
              unpack_pairs<T>(*reinterpret_cast<const uint4*>(in + k * kGatherBytes), f);
              const float w = __int_as_float(slots[k].y);
#pragma unroll
              for (int j = 0; j < E::N / 2; ++j) acc[j] = __ffma2_rn(make_float2(w, w), f[j], acc[j]);
            };
            if (slots[KC].x) {                             // the same for all threads: no branch between the loads
#pragma unroll
              for (int k = 0; k < KC; ++k) slot(k);
            } else {
#pragma unroll
              for (int k = 0; k < KC; ++k)
                if (slots[k].x >= 0) slot(k);
            }
            __stcs(reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(out) + t * row_bytes + at), pack_pairs<T>(acc));
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
        if (++stage == L::kStages) { stage = 0; phase ^= 1; }
      }
      if constexpr (GRAD) {
#pragma unroll
        for (int k = 0; k < KC; ++k) {
          float d = dot[k].x + dot[k].y;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
          if (lane == 0) red[par][k][warp] = d;
        }
        named_barrier_sync(1, 32 * kGatherWarps);
        if (ok && (int)threadIdx.x < topk) {
          float s = 0.0f;
#pragma unroll
          for (int i = 0; i < kGatherWarps; ++i) s += red[par][threadIdx.x][i];
          store_from_f32(dweights, weight_dtype, t * topk + threadIdx.x, s);   // no row: nothing was added
        }
      }
    }
  }
  __syncthreads();
}

template <typename VT>
__global__ void __launch_bounds__(256)
moe_clear_rows_kernel(const uint32_t* __restrict__ marks, VT* __restrict__ drows, int64_t num_rows, int64_t nvec) {
  const int lane = threadIdx.x & 31;
  const int64_t warp = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5, nwarps = ((int64_t)gridDim.x * blockDim.x) >> 5;
  for (int64_t row = warp; row < num_rows; row += nwarps) {
    if ((marks[row >> 5] >> (row & 31)) & 1u) continue;
    for (int64_t v = lane; v < nvec; v += 32) drows[row * nvec + v] = VT{};
  }
}

// Widest power of two up to 16 that divides a row of `bytes` bytes and all the addresses.
inline int chunk_bytes(int64_t bytes, std::initializer_list<const void*> ptrs) {
  for (int c = 16; c > 1; c >>= 1) {
    bool ok = bytes % c == 0;
    for (const void* p : ptrs) ok = ok && aligned(p, c);
    if (ok) return c;
  }
  return 1;
}

inline int element_bytes(int dtype) {
  switch (dtype) {
    case B200Q_BF16: case B200Q_F16: return 2;
    case B200Q_F32: case B200Q_I32: return 4;
    case B200Q_I8: return 1;
    default: return 0;
  }
}

// Launches the sort: one cluster of a CTA for every 2048 indices, up to sixteen (sort and a copy of 16-byte rows with 1 / 4 / 16
// CTAs: 8192 indices of 64 experts 18.4 / 12.3 / 12.3 us, 32768 51.2 / 20.4 / 14.3, 65536 94.2 / 36.9 / 18.4, of 1000 experts
// 108.5 / 38.9 / 22.5).
constexpr int kSortClusterMax = 16;

template <typename IdT>
int launch_sort(const RouteIds& r, int32_t* row_idx, int32_t* row_src, int64_t* expert_tokens, int cumulative, int32_t* valid_rows,
                     int2* row_info, cudaStream_t st) {
  constexpr auto kern = moe_sort_kernel<IdT>;
  const int smem = (kSortWarps + 1) * r.experts * (int)sizeof(int);
  if (int rc = ensure_dynamic_smem<kern>((kSortWarps + 1) * kMaxExperts * (int)sizeof(int), "moe_route (sort)")) return rc;
  if (int rc = ensure_wide_clusters<kern>("moe_route (sort)")) return rc;
  int ctas = 1;
  while (ctas < kSortClusterMax && (int64_t)ctas * 2048 < r.n) ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t err = cudaLaunchKernelEx(&cfg, kern, static_cast<const IdT*>(r.ids), r.n, r.begin, r.experts, r.strict_limit,
                                       row_idx, row_src, expert_tokens, cumulative, valid_rows, row_info, r.topk);
  if (err != cudaSuccess) return fail(B200Q_ERR_LAUNCH, "moe_route (sort): %s", cudaGetErrorString(err));
  return check_launch("moe_route (sort)");
}

template <typename IdT, int BYTES>
int launch_copy(const b200q_moe_route_args& a, const RouteIds& r, int64_t row_bytes, int32_t* valid_rows, cudaStream_t st) {
  using VT = typename Chunk<BYTES>::type;
  const VT* x = static_cast<const VT*>(a.x);
  VT* out = static_cast<VT*>(a.out);
  const float* scale = a.out_scale != nullptr ? static_cast<const float*>(a.scale) : nullptr;
  const int64_t nvec = row_bytes / BYTES;
  if (r.n <= kDirectIds) {
    moe_copy_direct_kernel<IdT, VT><<<(unsigned)(a.tokens + 1), 256, 0, st>>>(r, x, out, (int)nvec, a.out_rows, scale, a.out_scale, a.row_idx,
                                                                              a.row_src, a.expert_tokens, a.cumulative);
    return check_launch("moe_route (copy, few tokens)");
  }
  if (int rc = launch_sort<IdT>(r, a.row_idx, a.row_src, a.expert_tokens, a.cumulative, valid_rows, nullptr, st)) return rc;
  constexpr int U = 4;
  const int64_t segs = nvec == 0 ? 1 : ceil_div(nvec, 32 * U);
  const int64_t move_blocks = ceil_div(a.tokens * segs, 8), blocks = move_blocks + 2 * sm_count();
  B200Q_REQUIRE(blocks <= 0x7fffffffLL, B200Q_ERR_UNSUPPORTED, "moe_route: too many rows");
  return launch_dependent(moe_copy_kernel<VT, U>, (unsigned)blocks, 256, st, "moe_route (copy)", x, out, a.tokens, r.topk, nvec, (int)segs, a.out_rows,
                          scale, a.out_scale, static_cast<const int32_t*>(a.row_idx), static_cast<const int32_t*>(valid_rows), move_blocks);
}

template <typename IdT, typename T, typename ST, int ITERS>
int launch_route_quant_direct(const b200q_moe_route_args& a, const RouteIds& r, int threads, cudaStream_t st) {
  moe_quant_direct_kernel<IdT, T, ST, ITERS><<<(unsigned)(r.n + 1), threads, 0, st>>>(
      r, static_cast<const T*>(a.x), a.hidden, static_cast<const ST*>(a.scale), (int)a.scale_rows, static_cast<int8_t*>(a.out), a.out_scale, a.row_idx,
      a.row_src, a.expert_tokens, a.cumulative);
  return check_launch("moe_route (quantised, few tokens)");
}

template <typename T, typename ST, int ITERS, bool FULL>
int launch_route_quant_sorted(const b200q_moe_route_args& a, int64_t n, int threads, const int2* row_info, const int32_t* valid_rows, cudaStream_t st) {
  constexpr auto kern = moe_quant_kernel<T, ST, ITERS, FULL>;
  const int64_t cap = (int64_t)sm_count() * resident_ctas<kern>(threads);
  return launch_dependent(kern, (unsigned)(n < cap ? n : cap), threads, st, "moe_route (quantised)", n, static_cast<const T*>(a.x), a.hidden,
                          static_cast<const ST*>(a.scale), (int)a.scale_rows, static_cast<int8_t*>(a.out), a.out_scale, row_info, valid_rows);
}

template <typename IdT, typename T, typename ST>
int launch_route_quant(const b200q_moe_route_args& a, const RouteIds& r, int2* row_info, int32_t* valid_rows, cudaStream_t st) {
  const bool vec = a.hidden % 8 == 0 && a.hidden > 0 && a.hidden <= 8 * 512 * 4 && aligned(a.x, 16) && aligned(a.out, 8) &&
                   (a.scale == nullptr || aligned(a.scale, 16));
  const int nvec = vec ? (int)(a.hidden / 8) : 0;
  auto threads_for = [&](int iters) { return (int)ceil_div(ceil_div(nvec, iters), 32) * 32; };
  if (r.n <= kDirectIds) {
    // Latency counts: few vectors a thread.
    if (!vec) return launch_route_quant_direct<IdT, T, ST, 0>(a, r, 256, st);
    if (nvec <= 128) return launch_route_quant_direct<IdT, T, ST, 1>(a, r, threads_for(1), st);
    if (nvec <= 1024) return launch_route_quant_direct<IdT, T, ST, 2>(a, r, threads_for(2), st);
    return launch_route_quant_direct<IdT, T, ST, 4>(a, r, threads_for(4), st);
  }
  if (int rc = launch_sort<IdT>(r, a.row_idx, a.row_src, a.expert_tokens, a.cumulative, valid_rows, row_info, st)) return rc;
  // What a row costs besides its vectors (the maximum's way through the warps, the scale) is shared by fewer warps with four vectors
  // a thread.  4096 tokens to six rows each, with 1 / 2 / 4: 512 columns 24.6 / 22.5 / 24.6 us, 1024 34.8 / 28.7 / 26.6, 2048 55.3 /
  // 41.0 / 38.9, 4096 102.4 / 69.6 / 63.5, 8192 - / 139.2 / 133.1.
  if (!vec) return launch_route_quant_sorted<T, ST, 0, false>(a, r.n, 256, row_info, valid_rows, st);
  const int iters = nvec < 128 ? 2 : 4, threads = threads_for(iters);
  const bool full = nvec == threads * iters;
  if (iters == 2)
    return full ? launch_route_quant_sorted<T, ST, 2, true>(a, r.n, threads, row_info, valid_rows, st)
                : launch_route_quant_sorted<T, ST, 2, false>(a, r.n, threads, row_info, valid_rows, st);
  return full ? launch_route_quant_sorted<T, ST, 4, true>(a, r.n, threads, row_info, valid_rows, st)
              : launch_route_quant_sorted<T, ST, 4, false>(a, r.n, threads, row_info, valid_rows, st);
}

template <typename IdT>
int route(const b200q_moe_route_args& a, const RouteIds& r, int2* row_info, int32_t* valid_rows, cudaStream_t st) {
  if (!a.quantise) {
    const int64_t bytes = a.hidden * element_bytes(a.x_dtype);
    switch (chunk_bytes(bytes, {a.x, a.out})) {
      case 16: return launch_copy<IdT, 16>(a, r, bytes, valid_rows, st);
      case 8: return launch_copy<IdT, 8>(a, r, bytes, valid_rows, st);
      case 4: return launch_copy<IdT, 4>(a, r, bytes, valid_rows, st);
      case 2: return launch_copy<IdT, 2>(a, r, bytes, valid_rows, st);
      default: return launch_copy<IdT, 1>(a, r, bytes, valid_rows, st);
    }
  }
  const bool f32 = a.scale == nullptr || a.scale_dtype == B200Q_F32;
  if (a.x_dtype == B200Q_BF16)
    return f32 ? launch_route_quant<IdT, __nv_bfloat16, float>(a, r, row_info, valid_rows, st)
               : launch_route_quant<IdT, __nv_bfloat16, __nv_bfloat16>(a, r, row_info, valid_rows, st);
  return f32 ? launch_route_quant<IdT, __half, float>(a, r, row_info, valid_rows, st)
             : launch_route_quant<IdT, __half, __half>(a, r, row_info, valid_rows, st);
}

// [valid rows: 1 word, padded to 256 bytes][row -> token and expert: 2 n words, quantised form only]
size_t route_workspace(int64_t n, int quantise) {
  if (n <= kDirectIds) return 0;
  return 256 + (quantise ? (size_t)n * 8 : 0);
}

template <typename T, bool VEC>
int launch_combine(const void* rows, int64_t num_rows, const int32_t* row_idx, const void* w, int w_dtype, void* out, int64_t tokens, int topk,
                   int64_t hidden, cudaStream_t st) {
  const int64_t nvec = hidden / Lanes<T, VEC>::N, blocks = ceil_div(tokens * nvec, 256);
  B200Q_REQUIRE(blocks <= 0x7fffffffLL, B200Q_ERR_UNSUPPORTED, "moe_combine: too many tokens");
  const T* r = static_cast<const T*>(rows);
  T* o = static_cast<T*>(out);
#define B200Q_COMBINE(KC) moe_combine_kernel<T, VEC, KC><<<(unsigned)blocks, 256, 0, st>>>(r, num_rows, row_idx, w, w_dtype, o, tokens, topk, nvec)
  if (topk == 1) B200Q_COMBINE(1);
  else if (topk == 2) B200Q_COMBINE(2);
  else if (topk <= 4) B200Q_COMBINE(4);
  else B200Q_COMBINE(8);
#undef B200Q_COMBINE
  return check_launch("moe_combine");
}

// The pipeline pays from one token a CTA on and for rows that fill a quarter of a stage; it has up to eight slots.  A thread a
// vector against the pipeline, eight bf16 rows a token, forward and gradient: 148 tokens of 4096 columns 8.2 / 8.2 and 18.4 /
// 16.4 us, 300 14.3 / 12.3 and 24.6 / 20.5, 2048 57.3 / 32.8 and 79.9 / 59.4, 8192 190.5 / 108.5 and 278.5 / 200.7; 8192 tokens
// of 256 columns 20.5 / 24.6 and 43.0 / 55.3, of 512 32.7 / 28.7 and 63.5 / 59.4.  What more than eight slots cost without it: 4096 tokens
// of 4096 bf16, 8 / 9 / 16 slots: forward 51 / 133 / 166 us, gradient 109 / 191 / 257.
inline bool use_gather(int64_t tokens, int64_t topk, int64_t row_bytes) {
  return topk <= 8 && tokens >= 2 * sm_count() && row_bytes >= 1024;
}

template <typename T, int KC, bool GRAD>
int launch_gather(const void* dy, const void* rows, int64_t num_rows, const int32_t* row_idx, const void* w, int w_dtype, void* out, void* dw,
                  uint32_t* marks, int64_t tokens, int topk, int64_t row_bytes, cudaStream_t st) {
  using L = GatherLayout<KC, GRAD>;
  constexpr auto kern = moe_gather_kernel<T, KC, GRAD>;
  if (int rc = ensure_dynamic_smem<kern>(L::kDynamic, "moe_combine")) return rc;
  const int64_t cap = 2 * (int64_t)sm_count();
  kern<<<(unsigned)(tokens < cap ? tokens : cap), kGatherThreads, L::kDynamic, st>>>(
      static_cast<const T*>(dy), static_cast<const T*>(rows), num_rows, row_idx, w, w_dtype, static_cast<T*>(out), dw, marks, tokens, topk, row_bytes);
  return check_launch(GRAD ? "moe_combine_grad" : "moe_combine");
}

template <typename T, bool GRAD>
int gather(const void* dy, const void* rows, int64_t num_rows, const int32_t* row_idx, const void* w, int w_dtype, void* out, void* dw,
           uint32_t* marks, int64_t tokens, int topk, int64_t row_bytes, cudaStream_t st) {
#define B200Q_GATHER(KC) return launch_gather<T, KC, GRAD>(dy, rows, num_rows, row_idx, w, w_dtype, out, dw, marks, tokens, topk, row_bytes, st)
  if (topk == 1) B200Q_GATHER(1);
  if (topk == 2) B200Q_GATHER(2);
  if (topk <= 4) B200Q_GATHER(4);
  if (topk <= 6) B200Q_GATHER(6);
  B200Q_GATHER(8);
#undef B200Q_GATHER
}

template <typename T>
int combine(const void* rows, int64_t num_rows, const int32_t* row_idx, const void* w, int w_dtype, void* out, int64_t tokens, int topk,
            int64_t hidden, cudaStream_t st) {
  if (chunk_bytes(hidden * (int)sizeof(T), {rows, out}) == 16 && use_gather(tokens, topk, hidden * (int)sizeof(T)))
    return gather<T, false>(nullptr, rows, num_rows, row_idx, w, w_dtype, out, nullptr, nullptr, tokens, topk, hidden * (int)sizeof(T), st);
  if (chunk_bytes(hidden * (int)sizeof(T), {rows, out}) == 16)
    return launch_combine<T, true>(rows, num_rows, row_idx, w, w_dtype, out, tokens, topk, hidden, st);
  return launch_combine<T, false>(rows, num_rows, row_idx, w, w_dtype, out, tokens, topk, hidden, st);
}

template <typename T, bool VEC>
int launch_combine_grad(const b200q_moe_combine_grad_args& a, cudaStream_t st) {
  using L = Lanes<T, VEC>;
  const int64_t nvec = a.hidden / L::N;
  const T* dy = static_cast<const T*>(a.dy);
  const T* rows = static_cast<const T*>(a.rows);
  T* drows = static_cast<T*>(a.drows);
  uint32_t* marks = static_cast<uint32_t*>(a.workspace);
  cudaError_t err = cudaMemsetAsync(marks, 0, (size_t)ceil_div(a.num_rows, 32) * 4, st);
  if (err != cudaSuccess) return fail(B200Q_ERR_LAUNCH, "moe_combine_grad: memset: %s", cudaGetErrorString(err));
  if (VEC && a.dweights != nullptr && use_gather(a.tokens, a.topk, a.hidden * (int)sizeof(T))) {
    if (int rc = gather<T, true>(dy, rows, a.num_rows, a.row_idx, a.weights, a.weight_dtype, drows, a.dweights, marks, a.tokens, (int)a.topk,
                                 a.hidden * (int)sizeof(T), st))
      return rc;
  } else if (a.tokens > 0) {
    const int threads = nvec >= 256 ? 256 : (int)(nvec <= 32 ? 32 : ceil_div(nvec, 32) * 32);
#define B200Q_COMBINE_GRAD(KC)                                                                                                       \
  moe_combine_grad_kernel<T, VEC, KC><<<(unsigned)a.tokens, threads, 0, st>>>(dy, rows, a.num_rows, a.row_idx, a.weights, a.weight_dtype, \
                                                                              drows, a.dweights, marks, (int)a.topk, nvec)
    if (a.topk == 1) B200Q_COMBINE_GRAD(1);
    else if (a.topk == 2) B200Q_COMBINE_GRAD(2);
    else if (a.topk <= 4) B200Q_COMBINE_GRAD(4);
    else B200Q_COMBINE_GRAD(8);
#undef B200Q_COMBINE_GRAD
    if (int rc = check_launch("moe_combine_grad")) return rc;
  }
  using VT = typename L::Raw;
  const int64_t want = ceil_div(a.num_rows, 8), cap = (int64_t)sm_count() * 4;
  moe_clear_rows_kernel<VT><<<(unsigned)(want < cap ? want : cap), 256, 0, st>>>(marks, static_cast<VT*>(a.drows), a.num_rows, nvec);
  return check_launch("moe_combine_grad (rows without an owner)");
}

template <typename T>
int combine_grad(const b200q_moe_combine_grad_args& a, cudaStream_t st) {
  const bool rows_ok = a.rows == nullptr || aligned(a.rows, 16);
  if (rows_ok && chunk_bytes(a.hidden * (int)sizeof(T), {a.dy, a.drows}) == 16) return launch_combine_grad<T, true>(a, st);
  return launch_combine_grad<T, false>(a, st);
}

bool float_dtype(int d) { return d == B200Q_BF16 || d == B200Q_F16 || d == B200Q_F32; }

}  // namespace
}  // namespace b200q

extern "C" size_t b200q_moe_route_workspace_bytes(int64_t assignments, int quantise) {
  return assignments > 0 ? b200q::route_workspace(assignments, quantise) : 0;
}

extern "C" int b200q_moe_route(const b200q_moe_route_args* a, void* stream) {
  using namespace b200q;
  clear_error();
  B200Q_REQUIRE(a != nullptr, B200Q_ERR_BAD_ARG, "moe_route: args is NULL");
  B200Q_REQUIRE(a->tokens >= 0 && a->topk >= 0 && a->hidden >= 0 && a->out_rows >= 0, B200Q_ERR_BAD_ARG, "moe_route: negative size");
  B200Q_REQUIRE(a->topk <= 1024 && a->tokens <= 0x7fffffffLL && a->tokens * a->topk < 0x7fffffffLL && a->hidden <= (1LL << 28),
                B200Q_ERR_UNSUPPORTED, "moe_route: more than 2^31-2 assignments, 1024 slots or 2^28 columns");
  B200Q_REQUIRE(a->idx_dtype == B200Q_I32 || a->idx_dtype == B200Q_I64, B200Q_ERR_UNSUPPORTED, "moe_route: expert indices must be i32 or i64");
  B200Q_REQUIRE(a->expert_begin >= 0, B200Q_ERR_BAD_ARG, "moe_route: negative expert_begin (a negative index is a padded token's)");
  B200Q_REQUIRE(a->expert_end > a->expert_begin && a->expert_end - a->expert_begin <= kMaxExperts, B200Q_ERR_UNSUPPORTED,
                "moe_route: the expert range must hold 1 to %d experts", kMaxExperts);
  const int64_t n = a->tokens * a->topk;
  if (a->quantise) {
    B200Q_REQUIRE(a->x_dtype == B200Q_BF16 || a->x_dtype == B200Q_F16, B200Q_ERR_UNSUPPORTED, "moe_route: quantised rows need a bf16 or f16 x");
    B200Q_REQUIRE(a->scale == nullptr || a->scale_dtype == B200Q_F32 || a->scale_dtype == a->x_dtype, B200Q_ERR_UNSUPPORTED,
                  "moe_route: smooth scales must be f32 or x's dtype");
    B200Q_REQUIRE(a->scale == nullptr || a->scale_rows == 1 || a->scale_rows == a->expert_end - a->expert_begin, B200Q_ERR_BAD_ARG,
                  "moe_route: smooth scales need one row, or one for each expert of the range");
    B200Q_REQUIRE(a->out_rows == n, B200Q_ERR_BAD_ARG, "moe_route: the quantised form writes every row (out_rows = tokens * topk)");
  } else {
    B200Q_REQUIRE(element_bytes(a->x_dtype) != 0, B200Q_ERR_UNSUPPORTED, "moe_route: unsupported dtype of x");
    B200Q_REQUIRE(a->out_rows <= n, B200Q_ERR_BAD_ARG, "moe_route: out_rows is larger than tokens * topk");
    B200Q_REQUIRE((a->scale == nullptr) == (a->out_scale == nullptr) && (a->scale == nullptr || a->scale_dtype == B200Q_F32), B200Q_ERR_BAD_ARG,
                  "moe_route: a token's scale (f32) needs out_scale, and the other way round");
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (n == 0) {
    if (a->expert_tokens != nullptr) {
      cudaError_t e = cudaMemsetAsync(a->expert_tokens, 0, (size_t)(a->expert_end - a->expert_begin) * 8, st);
      if (e != cudaSuccess) return fail(B200Q_ERR_LAUNCH, "moe_route: %s", cudaGetErrorString(e));
    }
    return B200Q_OK;
  }
  B200Q_REQUIRE(a->expert_idx != nullptr && a->row_idx != nullptr, B200Q_ERR_BAD_ARG, "moe_route: expert_idx or row_idx is NULL");
  B200Q_REQUIRE(a->hidden == 0 || (a->x != nullptr && (a->out != nullptr || a->out_rows == 0)), B200Q_ERR_BAD_ARG, "moe_route: x or out is NULL");
  B200Q_REQUIRE(!a->quantise || a->out_scale != nullptr, B200Q_ERR_BAD_ARG, "moe_route: out_scale is NULL");
  const int es = a->quantise ? 2 : element_bytes(a->x_dtype);
  B200Q_REQUIRE(aligned(a->x, es) && aligned(a->out, a->quantise ? 1 : es) && aligned(a->expert_idx, a->idx_dtype == B200Q_I64 ? 8 : 4) &&
                    aligned(a->row_idx, 4) && aligned(a->row_src, 4) && aligned(a->expert_tokens, 8) && aligned(a->out_scale, 4) &&
                    aligned(a->scale, a->scale == nullptr || a->scale_dtype == B200Q_F32 ? 4 : 2),
                B200Q_ERR_BAD_ARG, "moe_route: misaligned buffer");
  const size_t need = route_workspace(n, a->quantise);
  B200Q_REQUIRE(need == 0 || (a->workspace != nullptr && a->workspace_bytes >= need && aligned(a->workspace, 256)), B200Q_ERR_WORKSPACE,
                "moe_route: needs %zu bytes of 256-byte aligned workspace, got %zu", need, a->workspace_bytes);
  int32_t* valid_rows = static_cast<int32_t*>(a->workspace);
  int2* row_info = a->quantise && need != 0 ? reinterpret_cast<int2*>(static_cast<uint8_t*>(a->workspace) + 256) : nullptr;
  RouteIds r{a->expert_idx, n, a->expert_begin, (int)(a->expert_end - a->expert_begin), (int)a->topk, a->strict ? a->expert_end : 0};
  return a->idx_dtype == B200Q_I64 ? route<int64_t>(*a, r, row_info, valid_rows, st) : route<int32_t>(*a, r, row_info, valid_rows, st);
}

extern "C" int b200q_moe_combine(const void* rows, int dtype, int64_t num_rows, const int32_t* row_idx, const void* weights, int weight_dtype,
                                 void* out, int64_t tokens, int64_t topk, int64_t hidden, void* stream) {
  using namespace b200q;
  clear_error();
  B200Q_REQUIRE(num_rows >= 0 && tokens >= 0 && topk >= 1 && hidden >= 0, B200Q_ERR_BAD_ARG, "moe_combine: negative size, or no slot");
  B200Q_REQUIRE(float_dtype(dtype), B200Q_ERR_UNSUPPORTED, "moe_combine: rows must be bf16, f16 or f32 (dtype enum %d)", dtype);
  B200Q_REQUIRE(weights == nullptr || float_dtype(weight_dtype), B200Q_ERR_UNSUPPORTED, "moe_combine: weights must be bf16, f16 or f32");
  B200Q_REQUIRE(topk <= 1024 && tokens <= 0x7fffffffLL && num_rows <= 0x7fffffffLL && hidden <= (1LL << 28), B200Q_ERR_UNSUPPORTED,
                "moe_combine: size out of range");
  if (tokens == 0 || hidden == 0) return B200Q_OK;
  B200Q_REQUIRE((rows != nullptr || num_rows == 0) && row_idx != nullptr && out != nullptr, B200Q_ERR_BAD_ARG, "moe_combine: NULL buffer");
  const int es = element_bytes(dtype);
  B200Q_REQUIRE(aligned(rows, es) && aligned(out, es) && aligned(row_idx, 4) && (weights == nullptr || aligned(weights, element_bytes(weight_dtype))),
                B200Q_ERR_BAD_ARG, "moe_combine: misaligned buffer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == B200Q_BF16) return combine<__nv_bfloat16>(rows, num_rows, row_idx, weights, weight_dtype, out, tokens, (int)topk, hidden, st);
  if (dtype == B200Q_F16) return combine<__half>(rows, num_rows, row_idx, weights, weight_dtype, out, tokens, (int)topk, hidden, st);
  return combine<float>(rows, num_rows, row_idx, weights, weight_dtype, out, tokens, (int)topk, hidden, st);
}

extern "C" size_t b200q_moe_combine_grad_workspace_bytes(int64_t num_rows) {
  return num_rows > 0 ? ((size_t)b200q::ceil_div(num_rows, 32) * 4 + 255) & ~size_t(255) : 0;
}

extern "C" int b200q_moe_combine_grad(const b200q_moe_combine_grad_args* a, void* stream) {
  using namespace b200q;
  clear_error();
  B200Q_REQUIRE(a != nullptr, B200Q_ERR_BAD_ARG, "moe_combine_grad: args is NULL");
  B200Q_REQUIRE(a->num_rows >= 0 && a->tokens >= 0 && a->topk >= 1 && a->hidden >= 0, B200Q_ERR_BAD_ARG,
                "moe_combine_grad: negative size, or no slot");
  B200Q_REQUIRE(float_dtype(a->dtype), B200Q_ERR_UNSUPPORTED, "moe_combine_grad: rows must be bf16, f16 or f32 (dtype enum %d)", a->dtype);
  B200Q_REQUIRE((a->weights == nullptr && a->dweights == nullptr) || float_dtype(a->weight_dtype), B200Q_ERR_UNSUPPORTED,
                "moe_combine_grad: weights must be bf16, f16 or f32");
  B200Q_REQUIRE(a->topk <= 1024 && a->tokens <= 0x7fffffffLL && a->num_rows <= 0x7fffffffLL && a->hidden <= (1LL << 28), B200Q_ERR_UNSUPPORTED,
                "moe_combine_grad: size out of range");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->num_rows == 0 || a->hidden == 0) {
    if (a->dweights != nullptr && a->tokens > 0) {
      cudaError_t e = cudaMemsetAsync(a->dweights, 0, (size_t)(a->tokens * a->topk) * element_bytes(a->weight_dtype), st);
      if (e != cudaSuccess) return fail(B200Q_ERR_LAUNCH, "moe_combine_grad: %s", cudaGetErrorString(e));
    }
    return B200Q_OK;
  }
  B200Q_REQUIRE(a->drows != nullptr && (a->tokens == 0 || (a->dy != nullptr && a->row_idx != nullptr)) &&
                    (a->dweights == nullptr || a->rows != nullptr || a->tokens == 0),
                B200Q_ERR_BAD_ARG, "moe_combine_grad: NULL buffer");
  const int es = element_bytes(a->dtype), ws = element_bytes(a->weight_dtype);
  B200Q_REQUIRE(aligned(a->dy, es) && aligned(a->rows, es) && aligned(a->drows, es) && aligned(a->row_idx, 4) &&
                    (ws == 0 || (aligned(a->weights, ws) && aligned(a->dweights, ws))),
                B200Q_ERR_BAD_ARG, "moe_combine_grad: misaligned buffer");
  const size_t need = b200q_moe_combine_grad_workspace_bytes(a->num_rows);
  B200Q_REQUIRE(a->workspace != nullptr && a->workspace_bytes >= need && aligned(a->workspace, 256), B200Q_ERR_WORKSPACE,
                "moe_combine_grad: needs %zu bytes of 256-byte aligned workspace, got %zu", need, a->workspace_bytes);
  if (a->dtype == B200Q_BF16) return combine_grad<__nv_bfloat16>(*a, st);
  if (a->dtype == B200Q_F16) return combine_grad<__half>(*a, st);
  return combine_grad<float>(*a, st);
}
