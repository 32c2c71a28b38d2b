// npu_grouped_matmul, W8A8 form: the products of a mixture of experts.  Rows of x sorted by expert, expert e's rows
// times its own int8 weight, with the dequantising epilogue of npu_quant_matmul:
//
//   out[m,n] = cast( float(sum_k x[m,k] * w[e,n,k] + bias_i32[e,n]) * scale[e,n] * row_scale[m] + bias_float[e,n] )
//
// where e is the group of row m.  How many rows an expert has is known on the device only.
//
// One persistent kernel on tcgen05 (kind::i8).  The weight rows are the MMA's 128 (256 for a CTA pair) rows and the
// tokens its columns, because the number of columns may change from one instruction to the next: a group of m rows is cut
// into ceil(m / kMaxTokens) tiles of equal width, rounded up to the instruction's step (16, or 32 for a pair), so at most
// a step's worth of columns is computed for nothing, where tiles with tokens on the row axis would pad every group to a
// multiple of 128 or 256 rows.  Every CTA builds the same list of non-empty groups and their tiles from the group list in
// shared memory and walks it with a stride of the grid; token tiles of one weight tile are neighbours, so a weight tile
// is fetched from HBM once and its other readers find it in L2.
//   warp 0      TMA producer: a 128 x 128-byte weight tile and the tokens' rows a stage, one copy each (a tensor map for
//               every number of rows a tile can have)
//   warp 1      MMA issuer; accumulators in TMEM, two buffers, so that one tile's epilogue overlaps the next one's products
//   warps 2-9   epilogue: a lane owns a channel; neighbouring lanes exchange tokens so that a lane stores two channels
// Three instantiations: CTA pairs and single CTAs with up to 256 tokens a tile (bound by the tensor cores), and single CTAs
// with up to 64 and a deeper ring (few rows an expert: bound by reading the weights).  Two rows for each of 64 weights of 4096 x 4096
// take 159 us (6.75 TB/s of weights); 16384 rows over 8 weights of 4096 x 22016 1058 us in a burst (2790 TOP/s) and 1230 under the
// power cap; 1531 very unequal rows over 24 weights of 5120 x 1416 46 us (up to 128 tokens a tile and six stages: 44 there, but
// 270 against 245 with 64 groups of 128 rows and 60 against 51 with 8 of 256).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ptx.cuh"
#include "tensormap.cuh"

namespace b200q {
namespace {

constexpr int kMaxGroups = 1024;
constexpr int kGroupedEpiThreads = 256;
constexpr int kGroupedThreads = 64 + kGroupedEpiThreads;

// AND of a predicate over the epilogue warps (named barrier 1): a barrier, and the common decision whether to go on.
__device__ __forceinline__ bool grouped_epilogue_all(bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)pred), "r"(kGroupedEpiThreads)
      : "memory");
  return r != 0;
}

struct GroupedArgs {
  const int64_t* group_list;   // [groups] ends (cumulative) or counts
  int counts;                  // group_list holds counts
  int groups;
  int64_t m;                   // rows of x and out
  int64_t k;
  int n, tiles_n, kblocks;
  const void* scale;           // [groups, n]; NULL for int32 output
  const void* bias;            // [groups, n] or NULL
  const float* row_scale;      // [m] or NULL
  void* out;                   // [m, n]
  int scale_dtype, bias_dtype, out_dtype;
};

__device__ __forceinline__ bool aligned_word(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// The non-empty groups, in order.
struct GroupTable {
  int start[kMaxGroups];       // first row
  int rows[kMaxGroups];
  int unit[kMaxGroups];        // first unit (token tile x channel tile)
  uint16_t group[kMaxGroups];
  int count, units, total;     // non-empty groups, units of all, rows of all
};

__device__ __forceinline__ int64_t warp_incl_sum(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Built by one warp.  Ends are clamped to [previous end, m], counts to what is left, so no list leads out of x.
template <int MAX_TOKENS>
__device__ void build_group_table(const GroupedArgs& a, GroupTable& t, int lane) {
  int64_t done = 0;            // rows of the groups before this batch
  int count = 0;
  int64_t units = 0;
  for (int g0 = 0; g0 < a.groups; g0 += 32) {
    const int g = g0 + lane;
    int64_t v = g < a.groups ? a.group_list[g] : (a.counts ? 0 : a.m);
    v = v < 0 ? 0 : v > a.m ? a.m : v;
    if (a.counts) {
      v = done + warp_incl_sum(v, lane);
      if (v > a.m) v = a.m;
    } else {
      if (v < done) v = done;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o && u > v) v = u;
      }
    }
    const int64_t before = __shfl_up_sync(0xffffffffu, v, 1);
    const int64_t first = lane == 0 ? done : before;
    const int rows = g < a.groups ? (int)(v - first) : 0;
    const int64_t mine = (int64_t)((rows + MAX_TOKENS - 1) / MAX_TOKENS) * a.tiles_n;
    const int64_t incl = units + warp_incl_sum(mine, lane);
    const unsigned live = __ballot_sync(0xffffffffu, rows > 0);
    if (rows > 0) {
      const int at = count + __popc(live & ((1u << lane) - 1));
      t.start[at] = (int)first;
      t.rows[at] = rows;
      t.unit[at] = (int)(incl - mine);
      t.group[at] = (uint16_t)g;
    }
    count += __popc(live);
    units = __shfl_sync(0xffffffffu, incl, 31);
    const int last = min(31, a.groups - 1 - g0);
    done = __shfl_sync(0xffffffffu, v, last);
  }
  if (lane == 0) {
    t.count = count;
    t.units = (int)units;
    t.total = (int)done;
  }
}

// A unit's place: group, channel tile, rows [row0, row0 + live) computed as `width` columns.  A group's rows, in steps of
// STEP, are dealt out evenly: the first tiles get one step more, and only the last step of the group can have idle columns.
struct Unit {
  int group, tile_n, row0, live, width;
};
template <int MAX_TOKENS, int STEP>
__device__ __forceinline__ Unit find_unit(const GroupTable& t, int u, int& at) {
  while (at + 1 < t.count && u >= t.unit[at + 1]) ++at;
  const int rows = t.rows[at], tiles = (rows + MAX_TOKENS - 1) / MAX_TOKENS, steps = (rows + STEP - 1) / STEP;
  const int local = u - t.unit[at], tile_n = local / tiles, tt = local - tile_n * tiles;
  const int per = steps / tiles, more = steps - per * tiles;
  const int first = (tt * per + min(tt, more)) * STEP;
  Unit r;
  r.group = t.group[at];
  r.tile_n = tile_n;
  r.row0 = t.start[at] + first;
  r.width = (per + (tt < more ? 1 : 0)) * STEP;
  r.live = min(r.width, rows - first);
  return r;
}

// Finishes CH accumulator columns (tokens) of a lane's channel for a 16-bit output without bias, all columns live: scale and
// row scale as packed two-wide products (each rounded like the scalar one), one conversion for two tokens, one exchange with
// the neighbouring lane.  Even lanes then hold token j of channels n, n + 1, odd lanes token j + 1 of channels n - 1, n: a
// 32-bit store each.  The tensor cores keep shared memory and its crossbar busy, so every LDS and shuffle here costs them
// time: four row scales a load, half a shuffle an element.
template <bool BF16, int CH>
__device__ __forceinline__ void store_columns(const uint32_t (&r)[CH], const float* row_scale, float sc, bool scaled, uint8_t* out, int64_t pitch,
                                              bool live) {
  const float2 sc2 = make_float2(sc, sc);
  const uint32_t pick = (threadIdx.x & 1) ? 0x3276u : 0x5410u;
#pragma unroll
  for (int j = 0; j < CH; j += 4) {
    float4 rs = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
    if (scaled) rs = *reinterpret_cast<const float4*>(row_scale + j);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      float2 v = __fmul2_rn(make_float2(__int2float_rn((int)r[j + 2 * q]), __int2float_rn((int)r[j + 2 * q + 1])), sc2);
      if (scaled) v = __fmul2_rn(v, q == 0 ? make_float2(rs.x, rs.y) : make_float2(rs.z, rs.w));
      uint32_t w;
      if constexpr (BF16) {
        const __nv_bfloat162 h = __float22bfloat162_rn(v);
        w = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __float22half2_rn(v);
        w = *reinterpret_cast<const uint32_t*>(&h);
      }
      w = __byte_perm(w, __shfl_xor_sync(0xffffffffu, w, 1), pick);
      if (live) *reinterpret_cast<uint32_t*>(out + (j + 2 * q) * pitch) = w;
    }
  }
}

template <int CTAS, int MAX_TOKENS, int STAGES>
struct GroupedLayout {
  static constexpr int kBRows = MAX_TOKENS / CTAS;             // token rows a CTA holds
  static constexpr int kBTileBytes = kBRows * kBK;
  static constexpr int kTiles = STAGES * (kATileBytes + kBTileBytes);
  static constexpr int kBarOff = kTiles;                       // full[S], empty[S], tfull[2], tempty[2]
  static constexpr int kMiscOff = kBarOff + (2 * STAGES + 4) * 8;
  static constexpr int kRowScaleOff = kMiscOff + 16;           // 2 x MAX_TOKENS floats
  static constexpr int kTableOff = kRowScaleOff + 2 * MAX_TOKENS * 4;
  static constexpr int kTotal = kTableOff + (int)sizeof(GroupTable);
  static constexpr int kDynamic = kTotal + 1024;
};

template <int B_ROWS>
struct GroupedMaps {
  CUtensorMap w;               // weight [groups, n, k]: box 1 x 128 x 128
  CUtensorMap x[B_ROWS / 16];  // x [m, k]: a box for every number of rows a tile can have, 16 (i + 1)
};

// STREAM: weights are read once (evicted first from L2, so that they do not push out the tokens; measured 144 us for 56
// weights of 4096 x 4096 where builds without the hint took between 144 and 160).
template <int CTAS, int MAX_TOKENS, int STAGES, bool STREAM>
__device__ __forceinline__ void
grouped_matmul_body(const GroupedMaps<MAX_TOKENS / CTAS>& maps, const GroupedArgs& a) {
  using L = GroupedLayout<CTAS, MAX_TOKENS, STAGES>;
  constexpr int kStep = 16 * CTAS;
  constexpr uint32_t kTmemCols = 2 * MAX_TOKENS;
  static_assert(kTmemCols <= 512 && (kTmemCols & (kTmemCols - 1)) == 0, "TMEM columns: power of two <= 512");
  static_assert(L::kDynamic > 116 * 1024 && L::kDynamic <= 227 * 1024, "one CTA per SM; shared memory budget");

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * kATileBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);
  float* row_scale = reinterpret_cast<float*>(smem + L::kRowScaleOff);
  GroupTable& table = *reinterpret_cast<GroupTable*>(smem + L::kTableOff);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CTAS == 2 ? (int)cluster_ctarank() : 0;         // 0 = leader
  const int first = blockIdx.x / CTAS, stride = gridDim.x / CTAS;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], CTAS * (kGroupedEpiThreads / 32));     // epilogue warps of all CTAs
    }
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tensormap(&maps.w);
  }
  if (warp == 1) {
    if constexpr (CTAS == 2) {
      tmem_alloc_pair(tmem_holder, kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_holder, kTmemCols);
      tmem_relinquish();
    }
  }
  if (warp == 2) build_group_table<MAX_TOKENS>(a, table, lane);
  tc_fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) cluster_sync_all();                     // the peer's barriers exist before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const int units = table.units;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (every CTA loads its own rows)
    if (lane == 0) {
      const uint64_t once = policy_evict_first();
      int stage = 0, at = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = first; u < units && ok; u += stride) {
        const Unit t = find_unit<MAX_TOKENS, kStep>(table, u, at);
        const int b_rows = t.width / CTAS, n0 = (t.tile_n * CTAS + rank) * kTileA, m0 = t.row0 + rank * b_rows;
        const uint32_t bytes = (uint32_t)(CTAS * (kATileBytes + b_rows * kBK));
        for (int kb = 0; kb < a.kblocks; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, kDevTimeoutProducer)) { ok = false; break; }
          uint8_t* dst_a = sA + stage * kATileBytes;
          uint8_t* dst_b = sB + stage * L::kBTileBytes;
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], bytes);
          uint32_t bar = smem_u32(&full[stage]);
          if constexpr (CTAS == 2) bar = map_to_cta(bar, 0);
          if constexpr (STREAM) tma_load_3d_hint(dst_a, &maps.w, bar, kb * kBK, n0, t.group, once);
          else tma_load_3d<CTAS>(dst_a, &maps.w, bar, kb * kBK, n0, t.group);
          tma_load_2d_to<CTAS>(dst_b, &maps.x[b_rows / 16 - 1], bar, kb * kBK, m0);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // Give copies that are still in flight time to land before shared memory is released.
      if (!ok)
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    }
  } else if (warp == 1) {
    // -------------------------------------------------------------- MMA issuer (leader)
    if (lane == 0 && rank == 0) {
      int stage = 0, buf = 0, at = 0;
      uint32_t phase = 0, tphase = 0;
      bool ok = true;
      for (int u = first; u < units && ok; u += stride) {
        const Unit t = find_unit<MAX_TOKENS, kStep>(table, u, at);
        const uint32_t idesc = make_idesc(2 /*s32*/, 1 /*s8*/, 1 /*s8*/, 0, 0, kTileA * CTAS, (uint32_t)t.width);
        if (!mbar_wait(&tempty[buf], tphase ^ 1, abort_flag, kDevTimeoutMma)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * MAX_TOKENS;
        for (int kb = 0; kb < a.kblocks; ++kb) {
          if (!mbar_wait(&full[stage], phase, abort_flag, kDevTimeoutMma)) { ok = false; break; }
          tc_fence_after();
          const uint64_t adesc = make_smem_desc(smem_u32(sA + stage * kATileBytes), 16, 1024, kSwizzle128B);
          const uint64_t bdesc = make_smem_desc(smem_u32(sB + stage * L::kBTileBytes), 16, 1024, kSwizzle128B);
#pragma unroll
          for (int k4 = 0; k4 < kBK / 32; ++k4) {
            const uint32_t acc = (kb > 0 || k4 > 0) ? 1u : 0u;
            if constexpr (CTAS == 2) umma_i8_pair(d_tmem, adesc + 2 * k4, bdesc + 2 * k4, idesc, acc);
            else umma_i8(d_tmem, adesc + 2 * k4, bdesc + 2 * k4, idesc, acc);
          }
          if constexpr (CTAS == 2) {
            umma_commit_pair(map_to_cta(smem_u32(&empty[stage]), 0));
            umma_commit_pair(map_to_cta(smem_u32(&empty[stage]), 1));
          } else {
            umma_commit(&empty[stage]);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        if constexpr (CTAS == 2) {
          umma_commit_pair(map_to_cta(smem_u32(&tfull[buf]), 0));
          umma_commit_pair(map_to_cta(smem_u32(&tfull[buf]), 1));
        } else {
          umma_commit(&tfull[buf]);
        }
        if (++buf == 2) { buf = 0; tphase ^= 1; }
      }
    }
  } else {
    // ---------------------------------------------------------------- epilogue: this CTA's 128 channels, all columns.
    // Two warps a quadrant of TMEM lanes, chunks of CH columns in turn.  The next tile's scales are loaded during this tile's
    // work; one barrier a tile stands between the row scales' writers and readers (two buffers) and makes the warps agree on
    // whether the accumulator came.
    constexpr int CH = 32;                                         // accumulator columns per tcgen05.ld
    const int et = threadIdx.x - 64;
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const bool two_byte = a.out_dtype == B200Q_BF16 || a.out_dtype == B200Q_F16;
    const bool words = two_byte && a.n % 2 == 0 && aligned_word(a.out);   // two channels of a row make an aligned word
    const bool plain = words && a.bias == nullptr;
    const bool scaled = a.row_scale != nullptr;
    Epi e{};
    e.scale = a.scale; e.scale_dtype = a.scale_dtype;
    e.bias = a.bias; e.bias_dtype = a.bias_dtype;
    e.out = a.out; e.out_dtype = a.out_dtype;
    e.flags = (scaled ? (uint32_t)kHasPt : 0u) |
              (a.bias != nullptr ? (a.bias_dtype == B200Q_I32 ? (uint32_t)kHasIntBias : (uint32_t)kHasFloatBias) : 0u);
    const int lane_n = rank * kTileA + quad * 32 + lane;           // this lane's channel within a tile
    int buf = 0, at = 0;
    uint32_t tphase = 0;
    Unit t{};
    float sc = 0.0f, rs = 1.0f;
    auto look = [&](int u) {                                       // unit u's place, this lane's scale and row scale
      if (u >= units) return;
      t = find_unit<MAX_TOKENS, kStep>(table, u, at);
      const int n = t.tile_n * CTAS * kTileA + lane_n;
      sc = n < a.n && a.scale != nullptr ? load_scale(e, (int64_t)t.group * a.n + n) : 0.0f;
      rs = scaled && et < t.live ? __ldg(a.row_scale + t.row0 + et) : 1.0f;
    };
    look(first);
    for (int u = first; u < units; u += stride) {
      float* scales = row_scale + buf * MAX_TOKENS;
      if (et < MAX_TOKENS) scales[et] = rs;
      const Unit now = t;
      const float sc_now = sc;
      const int n = now.tile_n * CTAS * kTileA + lane_n;
      const bool nv = n < a.n;
      const int64_t gn = (int64_t)now.group * a.n + n;
      const float fb = nv ? load_float_bias(e, gn) : 0.0f;
      const int ib = nv ? load_int_bias(e, gn) : 0;
      if (!grouped_epilogue_all(mbar_wait(&tfull[buf], tphase, abort_flag, kDevTimeoutEpilogue))) break;
      tc_fence_after();
      look(u + stride);
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + buf * MAX_TOKENS;
#pragma unroll 1
      for (int c = half * CH; c < now.live; c += 2 * CH) {
        uint32_t r[CH];
        __syncwarp();
        tmem_ld_chunk<CH>(taddr + c, r);
        tmem_ld_wait();
        if (plain && c + CH <= now.live) {
          // this lane's first word: token c (even lanes) or c + 1, channels n & ~1 and the next
          uint8_t* at_out = static_cast<uint8_t*>(a.out) + ((now.row0 + c + (lane & 1)) * (int64_t)a.n + (n & ~1)) * 2;
          if (a.out_dtype == B200Q_BF16) store_columns<true, CH>(r, scales + c, sc_now, scaled, at_out, (int64_t)a.n * 2, nv);
          else store_columns<false, CH>(r, scales + c, sc_now, scaled, at_out, (int64_t)a.n * 2, nv);
          continue;
        }
#pragma unroll
        for (int j = 0; j < CH; j += 2) {
          if (c + j >= now.live) break;                            // the same in every lane
          const float v0 = dequant((int)r[j], ib, sc_now, scales[c + j], fb, 0.0f, e.flags);
          const float v1 = dequant((int)r[j + 1], ib, sc_now, scales[c + j + 1], fb, 0.0f, e.flags);
          const int64_t row = now.row0 + c + j;
          if (words) {
            const uint32_t b0 = to_bits16(v0, a.out_dtype), b1 = to_bits16(v1, a.out_dtype);
            const uint32_t other = __shfl_xor_sync(0xffffffffu, (lane & 1) ? b0 : b1, 1);
            const uint32_t w = (lane & 1) ? (other | (b1 << 16)) : (b0 | (other << 16));
            if (c + j + (lane & 1) < now.live && nv)               // n is even: n < N for both or for neither
              *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + (row + (lane & 1)) * a.n + (n & ~1)) = w;
          } else if (nv) {
            store_one(e, row * a.n + n, (int)r[j], ib, v0);
            if (c + j + 1 < now.live) store_one(e, (row + 1) * a.n + n, (int)r[j + 1], ib, v1);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CTAS == 2) mbar_arrive_cluster(map_to_cta(smem_u32(&tempty[buf]), 0));
        else mbar_arrive(&tempty[buf]);
      }
      if (++buf == 2) { buf = 0; tphase ^= 1; }
    }
    // Rows behind the last group.
    const int ob = two_byte ? 2 : 4;
    for (int64_t row = (int64_t)table.total + blockIdx.x; row < a.m; row += gridDim.x)
      for (int c = et; c < a.n; c += kGroupedEpiThreads) {
        if (ob == 2) static_cast<uint16_t*>(a.out)[row * a.n + c] = 0;
        else static_cast<uint32_t*>(a.out)[row * a.n + c] = 0;
      }
  }

  // Teardown: no CTA of a pair may leave while the other can still signal its barriers or read its operands.
  tc_fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) cluster_sync_all();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    if constexpr (CTAS == 2) tmem_dealloc_pair(tmem_base, kTmemCols);
    else tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <int MAX_TOKENS, int STAGES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGroupedThreads, 1)
grouped_matmul_pair_kernel(const __grid_constant__ GroupedMaps<MAX_TOKENS / 2> maps, const GroupedArgs a) {
  grouped_matmul_body<2, MAX_TOKENS, STAGES, false>(maps, a);
}
template <int MAX_TOKENS, int STAGES>
__global__ void __launch_bounds__(kGroupedThreads, 1)
grouped_matmul_kernel(const __grid_constant__ GroupedMaps<MAX_TOKENS> maps, const GroupedArgs a) {
  grouped_matmul_body<1, MAX_TOKENS, STAGES, MAX_TOKENS <= 64>(maps, a);
}

// Any k, strides and alignment: one thread an output element, which walks k byte by byte.  It is here so that every layout has an
// answer, not for speed: 128 rows over 64 contiguous [k, n] weights of 4096 x 4096 take 1664 us where the transposed views of [n, k] take
// 159, 2048 rows over eight of them 12570 against 41.
__global__ void __launch_bounds__(256)
grouped_matmul_simt_kernel(const int8_t* __restrict__ x, const int8_t* __restrict__ w, int64_t w_stride_g, int64_t w_stride_k, int64_t w_stride_n,
                           const GroupedArgs a) {
  extern __shared__ uint8_t simt_smem[];
  GroupTable& table = *reinterpret_cast<GroupTable*>(simt_smem);
  if (threadIdx.y == 0) build_group_table<64>(a, table, threadIdx.x);
  __syncthreads();
  const int64_t n = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (n >= a.n) return;
  Epi e{};
  e.scale = a.scale; e.scale_dtype = a.scale_dtype;
  e.bias = a.bias; e.bias_dtype = a.bias_dtype;
  e.out = a.out; e.out_dtype = a.out_dtype;
  e.flags = (a.row_scale != nullptr ? (uint32_t)kHasPt : 0u) |
            (a.bias != nullptr ? (a.bias_dtype == B200Q_I32 ? (uint32_t)kHasIntBias : (uint32_t)kHasFloatBias) : 0u);
  int at = 0;
  for (int64_t m = blockIdx.y * (int64_t)blockDim.y + threadIdx.y; m < a.m; m += (int64_t)gridDim.y * blockDim.y) {
    if (m >= table.total) {
      store_one(e, m * a.n + n, 0, 0, 0.0f);
      continue;
    }
    while (at + 1 < table.count && m >= table.start[at + 1]) ++at;
    const int g = table.group[at];
    const int8_t* xr = x + m * a.k;
    const int8_t* wr = w + g * w_stride_g + n * w_stride_n;
    int acc = 0;
    for (int64_t i = 0; i < a.k; ++i) acc += (int)xr[i] * (int)wr[i * w_stride_k];
    const int64_t gn = (int64_t)g * a.n + n;
    const int ib = load_int_bias(e, gn);
    const float pt = a.row_scale != nullptr ? a.row_scale[m] : 1.0f;
    store_one(e, m * a.n + n, acc, ib, dequant(acc, ib, a.scale != nullptr ? load_scale(e, gn) : 0.0f, pt, load_float_bias(e, gn), 0.0f, e.flags));
  }
}

template <int CTAS, int MAX_TOKENS, int STAGES>
int launch_grouped(const b200q_grouped_matmul_args& in, const GroupedArgs& a, cudaStream_t st) {
  using L = GroupedLayout<CTAS, MAX_TOKENS, STAGES>;
  GroupedMaps<L::kBRows> maps;
  if (int rc = make_tmap_3d(&maps.w, in.weight, (uint64_t)in.k, (uint64_t)in.n, (uint64_t)in.groups, (uint64_t)in.w_stride_n,
                            (uint64_t)in.w_stride_g, kBK, kTileA, "grouped_matmul (weight)"))
    return rc;
  for (int i = 0; i < L::kBRows / 16; ++i)
    if (int rc = make_tmap_2d(&maps.x[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, in.x, (uint64_t)in.k, (uint64_t)in.m, (uint64_t)in.k, kBK,
                              16 * (i + 1), CU_TENSOR_MAP_SWIZZLE_128B, "grouped_matmul (x)"))
      return rc;
  // No more CTAs than there can be units.
  const int64_t tiles = in.m / MAX_TOKENS + (in.groups < in.m ? in.groups : in.m);
  const int64_t most = tiles * a.tiles_n;
  B200Q_REQUIRE(most < (1LL << 31), B200Q_ERR_UNSUPPORTED, "grouped_matmul: too many tiles");
  if constexpr (CTAS == 2) {
    constexpr auto kern = grouped_matmul_pair_kernel<MAX_TOKENS, STAGES>;
    if (int rc = ensure_dynamic_smem<kern>(L::kDynamic, "grouped_matmul")) return rc;
    const int64_t fit = resident_clusters<kern>(2, L::kDynamic, kGroupedThreads);
    kern<<<(unsigned)(2 * (most < fit ? most : fit)), kGroupedThreads, L::kDynamic, st>>>(maps, a);
  } else {
    constexpr auto kern = grouped_matmul_kernel<MAX_TOKENS, STAGES>;
    if (int rc = ensure_dynamic_smem<kern>(L::kDynamic, "grouped_matmul")) return rc;
    kern<<<(unsigned)(most < sm_count() ? most : sm_count()), kGroupedThreads, L::kDynamic, st>>>(maps, a);
  }
  return check_launch("grouped_matmul (tcgen05)");
}

}  // namespace
}  // namespace b200q

extern "C" int b200q_grouped_matmul(const b200q_grouped_matmul_args* a, void* stream) {
  using namespace b200q;
  clear_error();
  B200Q_REQUIRE(a != nullptr, B200Q_ERR_BAD_ARG, "grouped_matmul: args is NULL");
  B200Q_REQUIRE(a->m >= 0 && a->k >= 0 && a->n >= 0, B200Q_ERR_BAD_ARG, "grouped_matmul: negative size");
  B200Q_REQUIRE(a->groups >= 1 && a->groups <= kMaxGroups, B200Q_ERR_UNSUPPORTED, "grouped_matmul: %lld groups (1 to %d)", (long long)a->groups, kMaxGroups);
  B200Q_REQUIRE(a->m < 0x7fffffffLL && a->n < (1LL << 28) && a->k < (1LL << 28), B200Q_ERR_UNSUPPORTED, "grouped_matmul: size out of range");
  B200Q_REQUIRE(a->out_dtype == B200Q_F16 || a->out_dtype == B200Q_BF16 || a->out_dtype == B200Q_I32, B200Q_ERR_UNSUPPORTED,
                "grouped_matmul: output dtype enum %d is not f16, bf16 or int32", a->out_dtype);
  const bool acc_only = a->out_dtype == B200Q_I32;
  B200Q_REQUIRE(acc_only || a->scale_dtype == B200Q_F32 || a->scale_dtype == B200Q_BF16 || a->scale_dtype == B200Q_I64, B200Q_ERR_UNSUPPORTED,
                "grouped_matmul: scale must be f32, bf16 or i64 (dtype enum %d)", a->scale_dtype);
  B200Q_REQUIRE(a->bias == nullptr || a->bias_dtype == B200Q_I32 ||
                    (!acc_only && (a->bias_dtype == B200Q_BF16 || a->bias_dtype == B200Q_F16 || a->bias_dtype == B200Q_F32)),
                B200Q_ERR_UNSUPPORTED, "grouped_matmul: bias must be i32, or (not for int32 output) bf16, f16 or f32");
  if (a->m == 0 || a->n == 0) return B200Q_OK;
  B200Q_REQUIRE(a->group_list != nullptr && a->out != nullptr && (acc_only || a->scale != nullptr) && (a->k == 0 || (a->x != nullptr && a->weight != nullptr)),
                B200Q_ERR_BAD_ARG, "grouped_matmul: NULL buffer");
  auto fits = [](const void* p, int dtype) {
    return p == nullptr || aligned(p, dtype == B200Q_I64 ? 8 : dtype == B200Q_F32 || dtype == B200Q_I32 ? 4 : 2);
  };
  B200Q_REQUIRE(aligned(a->group_list, 8) && fits(a->out, a->out_dtype) && (acc_only || fits(a->scale, a->scale_dtype)) &&
                    fits(a->bias, a->bias_dtype) && aligned(a->row_scale, 4),
                B200Q_ERR_BAD_ARG, "grouped_matmul: misaligned buffer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  GroupedArgs g{};
  g.group_list = a->group_list; g.counts = a->counts; g.groups = (int)a->groups;
  g.m = a->m; g.k = a->k; g.n = (int)a->n; g.kblocks = (int)ceil_div(a->k, kBK);
  g.scale = acc_only ? nullptr : a->scale; g.scale_dtype = a->scale_dtype;
  g.bias = a->bias; g.bias_dtype = a->bias != nullptr ? a->bias_dtype : B200Q_NONE;
  g.row_scale = acc_only ? nullptr : a->row_scale;
  g.out = a->out; g.out_dtype = a->out_dtype;
  const bool tensor = a->k >= 16 && a->k % 16 == 0 && a->w_stride_k == 1 && a->w_stride_n >= a->k && a->w_stride_n % 16 == 0 &&
                      a->w_stride_g % 16 == 0 && (a->groups == 1 || a->w_stride_g >= a->k) && aligned(a->x, 16) && aligned(a->weight, 16);
  if (!tensor) {
    if (int rc = ensure_dynamic_smem<grouped_matmul_simt_kernel>((int)sizeof(GroupTable), "grouped_matmul")) return rc;
    g.tiles_n = 1;
    const int64_t gy = ceil_div(a->m, 8);
    dim3 grid((unsigned)ceil_div(a->n, 32), (unsigned)(gy < 4096 ? gy : 4096));
    grouped_matmul_simt_kernel<<<grid, dim3(32, 8), sizeof(GroupTable), st>>>(a->x, a->weight, a->w_stride_g, a->w_stride_k, a->w_stride_n, g);
    return check_launch("grouped_matmul (simt)");
  }
  // Few rows a group: the time goes into reading the weights, which small tiles with a deep ring do best.  Between: single CTAs,
  // whose tiles are half a pair's, waste less at the end of a group and of the launch.  Many rows: pairs, which read each
  // weight and token tile from L2 half as often and draw less power for it.  Measured for weights of 4096 x 4096 (us; small
  // tiles / single CTAs / pairs): 64 groups of 2 rows 146 / 166 / 178, of 32 rows 193 / 209 / 220, of 64 rows 244 / 232 / 243, of
  // 256 rows 655 / 368 / 390; 8 groups of 1024 rows 280 / 145 / 153; 8 groups of 2048 rows and 4096 x 22016 - / 1220 / 1180.
  if (a->m <= 48 * a->groups) {
    g.tiles_n = (int)ceil_div(a->n, kTileA);
    return launch_grouped<1, 64, 8>(*a, g, st);
  }
  if (a->m < 1536 * a->groups) {
    g.tiles_n = (int)ceil_div(a->n, kTileA);
    return launch_grouped<1, 256, 4>(*a, g, st);
  }
  g.tiles_n = (int)ceil_div(a->n, 2 * kTileA);
  return launch_grouped<2, 256, 6>(*a, g, st);
}
