// Matrix products grouped by expert over 16-bit weights [E][N][K], with ragged
// group sizes that only the device knows: y[r] = x[r] w[e]^T for the rows of
// expert e, optionally silu(gate) * up over the two halves of w's rows.
//
// Layout of the work. The tensor core's M side takes weights, its N side takes tokens:
// N may be any multiple of 16 (32 for a CTA pair), so a ragged group costs what its
// rows cost, where tokens on the M side would round every group up to 128 rows. A
// group's rows are cut into equal token tiles; a tile is (expert, token tile,
// feature tile), the tiles of one weight tile following one another so that its
// later reads hit L2. CTAs are persistent and take tiles round-robin; every CTA
// finds a tile's expert by bisection in a prefix sum of tile counts that it builds
// from the offsets at its start, so the host never waits for them. A TMA producer
// warp, an MMA warp (tcgen05, fp32 accumulators in tensor memory) and epilogue warps
// work side by side.
//
// Two kernels. Up to 24 rows per expert on average the weights' bytes bound the work:
// one CTA per tile of 128 features x up to 64 tokens, eight stages in flight. Above,
// the tensor cores and their power do: a CTA pair takes 256 features x up to 256
// tokens with two accumulators, so that a tile is stored while the next one is
// multiplied. (512 features with one accumulator fetch a quarter less from L2, but
// all pairs then store at the same time and wait for it: 16 % of their time, 806 us
// against 752 in turn for eight experts of 4096 -> 14336 over 8111 rows.)
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "awqb200.h"
#include "awqb_common.h"
#include "awqb_ptx.cuh"
#include "awqb_tma.h"
#include "awqb_vec.cuh"

namespace awqb {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kFeat = 128;        // features per CTA and tile
constexpr int kK = 64;            // k per stage: one 128-byte swizzled row
constexpr int kWBytes = kFeat * kK * 2;
constexpr uint32_t kErrWait = 128u;  // a bounded wait of these kernels gave up

// The few-rows kernel.
struct Few {
  static constexpr int kTok = 64;      // tokens per tile
  static constexpr int kRound = 16;    // granularity of the MMA's N
  static constexpr int kStages = 8;    // 128 KB of weights in flight
  static constexpr int kStageBytes = kWBytes + kTok * kK * 2;
  static constexpr int kEpiWarps = 4;
  static constexpr int kThreads = 32 * (kEpiWarps + 2);
  static constexpr int kChunk = 32;    // tokens per epilogue turn
};
// The many-rows kernel; a CTA of the pair loads its 128 weight rows and half the
// tokens.
struct Many {
  static constexpr int kTok = 256;
  static constexpr int kRound = 32;
  static constexpr int kStages = 6;
  static constexpr int kStageBytes = kWBytes + kTok / 2 * kK * 2;
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 32 * (kEpiWarps + 2);
};

// Boxes of token rows: a quarter, a half and all of what a CTA may load per stage.
struct TokenMaps {
  CUtensorMap box[3];
};

struct Params {
  const int32_t *offsets, *row_map;
  const float* row_scale;
  void* out;
  uint32_t* err;
  int64_t ldo, out_rows;
  int rows, E, K, N, n_out, silu, feat_tiles, tile_out;  // output features of a tile
};

struct Tile {
  int e, row0, rows, n, feat;  // expert, first row, rows, rows rounded up for the MMA, first output feature
};

// Shared-memory tables of the groups: first row and first tile of each.
struct Groups {
  int* row0;
  int* tile0;  // [E + 1]
};

template <typename C>
__device__ __forceinline__ Tile find_tile(const Groups& g, const Params& p, int t) {
  int lo = 0, hi = p.E;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (g.tile0[mid] <= t) lo = mid; else hi = mid;
  }
  const int local = t - g.tile0[lo];
  const int mt = (g.tile0[lo + 1] - g.tile0[lo]) / p.feat_tiles;
  const int ft = local / mt, tt = local - ft * mt;
  const int rows = g.row0[p.E + lo];
  // equal token tiles, rounded up to what the MMA takes
  const int per = ((rows + mt - 1) / mt + C::kRound - 1) / C::kRound * C::kRound;
  Tile r;
  r.e = lo;
  r.row0 = g.row0[lo] + tt * per;
  r.rows = min(per, rows - tt * per);
  r.n = (r.rows + C::kRound - 1) / C::kRound * C::kRound;
  r.feat = ft * p.tile_out;
  return r;
}

// Builds the tables of the groups from the offsets (clamped to the rows); all
// threads, with a barrier still to come before they are read.
template <typename C>
__device__ __forceinline__ void build_groups(const Groups& g, const Params& p) {
  for (int e = threadIdx.x; e < p.E; e += C::kThreads) {
    const int r0 = min(max(p.offsets[e], 0), p.rows), r1 = min(max(p.offsets[e + 1], 0), p.rows);
    g.row0[e] = r0;
    g.row0[p.E + e] = max(r1 - r0, 0);
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    int run = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + threadIdx.x;
      int v = e < p.E ? (g.row0[p.E + e] + C::kTok - 1) / C::kTok * p.feat_tiles : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if ((int)threadIdx.x >= o) v += u;
      }
      if (e < p.E) g.tile0[e + 1] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
    if (threadIdx.x == 0) g.tile0[0] = 0;
  }
}

// Where a tile's rows go in out, and their factors, into shared memory.
__device__ __forceinline__ void load_rows(const Params& p, const Tile& tile, int first, int step, int* dst, float* scl) {
  for (int i = first; i < tile.rows; i += step) {
    const int to = p.row_map ? p.row_map[tile.row0 + i] : tile.row0 + i;
    const bool in = to >= 0 && to < p.out_rows;
    dst[i] = in ? to : -1;
    if (p.row_scale) scl[i] = in ? p.row_scale[to] : 0.f;
  }
}

// silu(g) * u with the approximate exponential and division: right to
// (6 + 1.173 |g|) 2^-23 of the value (1.2e-5 at g = -80; 16-bit results keep 2^-11 at
// best), and 0 below g = -87.3, where |silu(g)| < 88 * 2^-126.
__device__ __forceinline__ float silu_mul(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// Eight lanes, kStep apart, hold eight values each: v[t] of feature l, l = 0..7 their
// number. Afterwards lane l holds value l of all eight features, rounded to 16 bits.
template <typename T, int kStep>
__device__ __forceinline__ uint4 transpose8(const float* v, int lane) {
  const bool b2 = lane & (4 * kStep), b1 = lane & (2 * kStep), b0 = lane & kStep;
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = Pair<T>::pack(v[2 * i], v[2 * i + 1]);
  // values 0..3 to the lower four lanes, 4..7 to the upper ones; x[feature bit 2][pair]
  const uint32_t g0 = __shfl_xor_sync(0xffffffffu, b2 ? r[0] : r[2], 4 * kStep);
  const uint32_t g1 = __shfl_xor_sync(0xffffffffu, b2 ? r[1] : r[3], 4 * kStep);
  const uint32_t x00 = b2 ? g0 : r[0], x01 = b2 ? g1 : r[1], x10 = b2 ? r[2] : g0, x11 = b2 ? r[3] : g1;
  // the pair of this lane's value; y[feature bit 2][feature bit 1]
  const uint32_t h0 = __shfl_xor_sync(0xffffffffu, b1 ? x00 : x01, 2 * kStep);
  const uint32_t h1 = __shfl_xor_sync(0xffffffffu, b1 ? x10 : x11, 2 * kStep);
  const uint32_t y00 = b1 ? h0 : x00, y01 = b1 ? x01 : h0, y10 = b1 ? h1 : x10, y11 = b1 ? x11 : h1;
  // the half of the pair; the neighbour's goes as the other feature of each word
  const uint32_t send = b0 ? 0x5410u : 0x7632u;  // lower halves, or upper ones
  const uint32_t k0 = __shfl_xor_sync(0xffffffffu, __byte_perm(y00, y01, send), kStep);
  const uint32_t k1 = __shfl_xor_sync(0xffffffffu, __byte_perm(y10, y11, send), kStep);
  const uint32_t low = b0 ? 0x3254u : 0x5410u, high = b0 ? 0x3276u : 0x7610u;
  return make_uint4(__byte_perm(y00, k0, low), __byte_perm(y01, k0, high), __byte_perm(y10, k1, low),
                    __byte_perm(y11, k1, high));
}

// The smallest box that holds `rows` token rows.
__device__ __forceinline__ int box_of(int rows, int most) { return rows * 4 <= most ? 0 : rows * 2 <= most ? 1 : 2; }

template <typename T>
__global__ void __launch_bounds__(Few::kThreads, 1)
grouped_gemm_few_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ TokenMaps tm_x,
                        const __grid_constant__ Params p) {
  using C = Few;
  extern __shared__ uint8_t raw[];
  uint8_t* ring = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  float* turn = reinterpret_cast<float*>(ring + C::kStages * C::kStageBytes);  // [kChunk][kFeat]
  int* dst = reinterpret_cast<int*>(turn + C::kChunk * kFeat);                 // [2][kTok] out row of a token
  float* scl = reinterpret_cast<float*>(dst + 2 * C::kTok);                    // [2][kTok]
  Groups g;
  g.row0 = reinterpret_cast<int*>(scl + 2 * C::kTok);  // [E] first rows, [E] row counts
  g.tile0 = g.row0 + 2 * p.E;
  __shared__ uint64_t full[C::kStages], empty[C::kStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&acc_full[b]), 1);
      mbar_init(smem_u32(&acc_empty[b]), C::kEpiWarps);
    }
    failed = 0;
    fence_barrier_init();
    prefetch_tmap(&tm_w);
  }
  if (warp == C::kEpiWarps + 1) {
    tmem_alloc(smem_u32(&tmem_slot), 2 * C::kTok);
    tmem_relinquish();
  }
  grid_dep_wait();
  grid_dep_launch();
  build_groups<C>(g, p);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int total = g.tile0[p.E];
  const int nk = (p.K + kK - 1) / kK;
  bool ok = true;

  if (warp == C::kEpiWarps) {  // ------------------------------------- producer
    const uint64_t keep = policy_evict_normal(), once = policy_evict_first();
    int it = 0;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      const Tile tile = find_tile<C>(g, p, t);
      const int box = box_of(tile.n, C::kTok);
      // weights that one token tile reads once need not stay in L2
      const uint64_t wpol = tile.rows == g.row0[p.E + tile.e] ? once : keep;
      const int wrow = tile.e * p.N + tile.feat;
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const int s = it % C::kStages;
        ok = mbar_wait(smem_u32(&empty[s]), ((it / C::kStages) & 1) ^ 1);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t base = smem_u32(ring + s * C::kStageBytes), bar = smem_u32(&full[s]);
          mbar_arrive_expect_tx(bar, kWBytes + (C::kTok >> (2 - box)) * kK * 2);
          tma_load_2d(base, &tm_w, kb * kK, wrow, bar, wpol);
          if (p.silu) tma_load_2d(base + kWBytes / 2, &tm_w, kb * kK, wrow + p.n_out, bar, wpol);
          tma_load_2d(base + kWBytes, &tm_x.box[box], kb * kK, tile.row0, bar, keep);
        }
        __syncwarp();
      }
    }
  } else if (warp == C::kEpiWarps + 1) {  // ---------------------------- MMA
    int it = 0, n_tile = 0;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x, ++n_tile) {
      const Tile tile = find_tile<C>(g, p, t);
      const uint32_t idesc = make_idesc_f16(kFeat, tile.n, std::is_same<T, __nv_bfloat16>::value);
      const int b = n_tile & 1;
      ok = mbar_wait(smem_u32(&acc_empty[b]), ((n_tile >> 1) & 1) ^ 1);
      tc_fence_after();
      const uint32_t d = tmem + b * C::kTok;
      for (int kb = 0; kb < nk && ok; ++kb, ++it) {
        const int s = it % C::kStages;
        ok = mbar_wait(smem_u32(&full[s]), (it / C::kStages) & 1);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t base = smem_u32(ring + s * C::kStageBytes);
          const uint64_t ad = make_sw128_kmajor_desc(base), bd = make_sw128_kmajor_desc(base + kWBytes);
          const int steps = min(kK, p.K - kb * kK + 15) / 16;
          for (int j = 0; j < steps; ++j) tc_mma_f16(d, ad + 2 * j, bd + 2 * j, idesc, kb + j > 0);
          tc_commit(smem_u32(&empty[s]));
          if (kb == nk - 1) tc_commit(smem_u32(&acc_full[b]));
        }
        __syncwarp();
      }
    }
  } else {  // -------------------------------------------------------- epilogue
    // The accumulator (features on lanes, tokens on columns) turns through shared
    // memory, 32 tokens at a time in fp32, where gate and up (two halves of the
    // lanes) also meet; a token's features leave as 16-byte vectors.
    const int tid = threadIdx.x;  // 0..127, TMEM lane = feature
    const int feats = p.silu ? kFeat / 2 : kFeat;
    const int per_row = feats / 8;                      // threads that write one token
    const int fl = (tid % per_row) * 8, tk = tid / per_row;
    const int tok_step = 128 / per_row;
    // Feature c stands at c, its halves of eight swapped where bit 5 is set: the
    // 16-byte reads of eight lanes then hit all banks.
    const int put = tid ^ ((tid >> 3) & 4), get = fl + ((fl >> 3) & 4);
    int n_tile = 0;
    for (int t = blockIdx.x; t < total; t += gridDim.x, ++n_tile) {
      const Tile tile = find_tile<C>(g, p, t);
      const int b = n_tile & 1;
      load_rows(p, tile, tid, 128, dst + b * C::kTok, scl + b * C::kTok);
      ok = named_bar_and(1, 128, mbar_wait(smem_u32(&acc_full[b]), (n_tile >> 1) & 1));
      if (!ok) break;
      tc_fence_after();
      const int f = tile.feat + fl;
      for (int c = 0; c < tile.rows; c += C::kChunk) {
        uint32_t v[2][16];
        tmem_ld16(tmem + b * C::kTok + c + ((uint32_t)warp << 21), v[0]);
        tmem_ld16(tmem + b * C::kTok + c + 16 + ((uint32_t)warp << 21), v[1]);
        tmem_ld_wait();
        if (c + C::kChunk >= tile.rows) {  // the accumulator is read: the MMA warp may reuse it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&acc_empty[b]));
        }
#pragma unroll
        for (int j = 0; j < C::kChunk; ++j) turn[j * kFeat + put] = __uint_as_float(v[j / 16][j % 16]);
        named_bar_sync(1, 128);
        const int m = min(C::kChunk, tile.rows - c);
        for (int j = tk; j < m; j += tok_step) {
          const int to = dst[b * C::kTok + c + j];
          if (to < 0 || f >= p.n_out) continue;
          const float* src = turn + j * kFeat;
          float y[8];
          *reinterpret_cast<float4*>(y) = *reinterpret_cast<const float4*>(src + get);
          *reinterpret_cast<float4*>(y + 4) = *reinterpret_cast<const float4*>(src + (get ^ 4));
          if (p.silu) {
            float u[8];
            *reinterpret_cast<float4*>(u) = *reinterpret_cast<const float4*>(src + kFeat / 2 + get);
            *reinterpret_cast<float4*>(u + 4) = *reinterpret_cast<const float4*>(src + kFeat / 2 + (get ^ 4));
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = silu_mul(y[i], u[i]);
          }
          if (p.row_scale) {
            const float w = scl[b * C::kTok + c + j];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] *= w;
          }
          *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (int64_t)to * p.ldo + f) = pack_vec<T>(y);
        }
        named_bar_sync(1, 128);
      }
    }
  }
  if (!ok && lane == 0) {
    failed = 1;
    atomicOr(p.err, kErrWait);
  }
  __syncwarp();
  __syncthreads();
  if (failed) linger();
  tc_fence_before();
  __syncthreads();
  if (warp == C::kEpiWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * C::kTok);
  }
}

template <typename T>
__global__ void __launch_bounds__(Many::kThreads, 1)
grouped_gemm_many_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ TokenMaps tm_x,
                         const __grid_constant__ Params p) {
  using C = Many;
  extern __shared__ uint8_t raw[];
  uint8_t* ring = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  int* dst = reinterpret_cast<int*>(ring + C::kStages * C::kStageBytes);  // [2][kTok] out row of a token
  float* scl = reinterpret_cast<float*>(dst + 2 * C::kTok);               // [2][kTok]
  Groups g;
  g.row0 = reinterpret_cast<int*>(scl + 2 * C::kTok);
  g.tile0 = g.row0 + 2 * p.E;
  __shared__ uint64_t full[C::kStages], empty[C::kStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&acc_full[b]), 1);
      mbar_init(smem_u32(&acc_empty[b]), 2 * C::kEpiWarps);
    }
    failed = 0;
    fence_barrier_init();
    prefetch_tmap(&tm_w);
  }
  if (warp == C::kEpiWarps + 1) {
    tmem_alloc_pair(smem_u32(&tmem_slot), 2 * C::kTok);
    tmem_relinquish_pair();
  }
  grid_dep_wait();
  grid_dep_launch();
  build_groups<C>(g, p);
  tc_fence_before();
  cluster_sync_all();  // the peer's barriers are ready before anything arrives on them
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int total = g.tile0[p.E];
  const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;
  const int nk = (p.K + kK - 1) / kK;
  bool ok = true;

  if (warp == C::kEpiWarps) {  // ------------------------------------- producer
    const uint64_t keep = policy_evict_normal(), once = policy_evict_first();
    int it = 0;
    for (int t = pair; t < total && ok; t += pairs) {
      const Tile tile = find_tile<C>(g, p, t);
      const int box = box_of(tile.n / 2, C::kTok / 2);
      // weights that one token tile reads once need not stay in L2
      const uint64_t wpol = tile.rows == g.row0[p.E + tile.e] ? once : keep;
      const int feat = tile.feat + (int)rank * p.tile_out / 2, row = tile.row0 + (int)rank * (tile.n / 2);
      const uint32_t bytes = 2 * (kWBytes + (C::kTok / 2 >> (2 - box)) * kK * 2);
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const int s = it % C::kStages;
        ok = mbar_wait(smem_u32(&empty[s]), ((it / C::kStages) & 1) ^ 1);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t base = smem_u32(ring + s * C::kStageBytes), bar = mapa_shared(smem_u32(&full[s]), 0);
          if (rank == 0) mbar_arrive_expect_tx(smem_u32(&full[s]), bytes);
          if (p.silu)
            tma_load_4d_pair(base, &tm_w, kb * kK, 0, feat, tile.e, bar, wpol);
          else
            tma_load_2d_pair(base, &tm_w, kb * kK, tile.e * p.N + feat, bar, wpol);
          tma_load_2d_pair(base + kWBytes, &tm_x.box[box], kb * kK, row, bar, keep);
        }
        __syncwarp();
      }
    }
    // the last stages' releases arrive from the pair's leader before this CTA may leave
    for (int i = max(0, it - C::kStages); i < it && ok; ++i)
      ok = mbar_wait(smem_u32(&empty[i % C::kStages]), (i / C::kStages) & 1);
  } else if (warp == C::kEpiWarps + 1) {  // ---------------------------- MMA, the leader's
    int it = 0, n_tile = 0;
    for (int t = pair; t < total && ok && rank == 0; t += pairs, ++n_tile) {
      const Tile tile = find_tile<C>(g, p, t);
      const uint32_t idesc = make_idesc_f16(2 * kFeat, tile.n, std::is_same<T, __nv_bfloat16>::value);
      const int b = n_tile & 1;
      ok = mbar_wait(smem_u32(&acc_empty[b]), ((n_tile >> 1) & 1) ^ 1);
      tc_fence_after();
      for (int kb = 0; kb < nk && ok; ++kb, ++it) {
        const int s = it % C::kStages;
        ok = mbar_wait(smem_u32(&full[s]), (it / C::kStages) & 1);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t base = smem_u32(ring + s * C::kStageBytes);
          const uint64_t ad = make_sw128_kmajor_desc(base), bd = make_sw128_kmajor_desc(base + kWBytes);
          const int steps = min(kK, p.K - kb * kK + 15) / 16;
          for (int j = 0; j < steps; ++j)
            tc_mma_f16_pair(tmem + b * C::kTok, ad + 2 * j, bd + 2 * j, idesc, kb + j > 0);
          tc_commit_pair(smem_u32(&empty[s]));
          if (kb == nk - 1) tc_commit_pair(smem_u32(&acc_full[b]));
        }
        __syncwarp();
      }
    }
  } else {  // -------------------------------------------------------- epilogue
    // Two groups of four warps take turns over 32 tokens. A lane holds a feature's
    // tokens; eight lanes transpose eight tokens among them in registers, so that
    // each writes eight features of a token: no shared memory and no barrier on the
    // way. With silu_mul even lanes hold gate and odd lanes up rows (the copies
    // interleave them): a lane keeps 16 tokens and gives its neighbour the other 16.
    const int group = warp >> 2, quarter = warp & 3, odd = lane & 1;
    const uint32_t at = tmem + ((uint32_t)quarter << 21);
    int n_tile = 0;
    for (int t = pair; t < total; t += pairs, ++n_tile) {
      const Tile tile = find_tile<C>(g, p, t);
      const int b = n_tile & 1;
      int* rows = dst + b * C::kTok;
      float* scales = scl + b * C::kTok;
      load_rows(p, tile, threadIdx.x, 32 * C::kEpiWarps, rows, scales);
      ok = named_bar_and(1, 32 * C::kEpiWarps, mbar_wait(smem_u32(&acc_full[b]), (n_tile >> 1) & 1));
      if (!ok) break;
      tc_fence_after();
      const int f = tile.feat + (int)rank * p.tile_out / 2 +
                    (p.silu ? quarter * 16 + (lane & 16) / 2 : quarter * 32 + (lane & 24));
      const auto put = [&](uint4 o, int i) {  // token i's features f ..
        const int to = rows[i];
        if (i < tile.rows && to >= 0 && f < p.n_out)
          *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (int64_t)to * p.ldo + f) = o;
      };
      for (int c = group * 32; c < tile.rows; c += 64) {
        uint32_t lo[16], hi[16];
        tmem_ld16(at + b * C::kTok + c, lo);
        tmem_ld16(at + b * C::kTok + c + 16, hi);
        tmem_ld_wait();
        if (c + 64 >= tile.rows) {  // this warp has read its part of the accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&acc_empty[b]), 0));
        }
        if (p.silu) {
          float v[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float own = __uint_as_float(odd ? hi[j] : lo[j]);
            const float got = __shfl_xor_sync(0xffffffffu, __uint_as_float(odd ? lo[j] : hi[j]), 1);
            v[j] = silu_mul(odd ? got : own, odd ? own : got);
            if (p.row_scale) v[j] *= scales[c + 16 * odd + j];
          }
#pragma unroll
          for (int j = 0; j < 16; j += 8) put(transpose8<T, 2>(v + j, lane), c + 16 * odd + j + ((lane >> 1) & 7));
        } else {
          float v[32];
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(lo[j]), v[16 + j] = __uint_as_float(hi[j]);
          if (p.row_scale)
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= scales[c + j];
#pragma unroll
          for (int j = 0; j < 32; j += 8) put(transpose8<T, 1>(v + j, lane), c + j + (lane & 7));
        }
      }
      if (group * 32 >= tile.rows) {  // no tokens for this group
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&acc_empty[b]), 0));
      }
    }
  }
  if (!ok && lane == 0) {
    failed = 1;
    atomicOr(p.err, kErrWait);
  }
  __syncwarp();
  __syncthreads();
  if (failed) linger();
  tc_fence_before();
  cluster_sync_all();  // the peer may still write or arrive here
  __syncthreads();
  if (warp == C::kEpiWarps + 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 2 * C::kTok);
  }
}

// w as [expert][feature][gate, up][k]: a box of 64 features brings gate and up rows
// by turns. Features past the last one read as zero.
int make_gate_up_map(CUtensorMap* tm, const void* w, const Params& p) {
  const auto enc = tensor_map_encoder();
  AWQB_REQUIRE(enc != nullptr, kCudaError, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t row = (cuuint64_t)p.K * 2;
  const cuuint64_t dim[4] = {(cuuint64_t)p.K, 2, (cuuint64_t)p.n_out, (cuuint64_t)p.E};
  const cuuint64_t stride[3] = {row * p.n_out, row, row * p.N};
  const cuuint32_t box[4] = {kK, 2, kFeat / 2, 1}, step[4] = {1, 1, 1, 1};
  const CUresult r = enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void*>(w), dim, stride, box, step,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  AWQB_REQUIRE(r == CUDA_SUCCESS, kCudaError, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return kOk;
}

// Clusters that run at once (a GPC with an odd number of SMs leaves one idle),
// per device; the persistent grid must not exceed it.
template <typename Kernel>
int max_clusters(Kernel kernel, const cudaLaunchConfig_t& cfg, std::atomic<int>* cached, int64_t* out) {
  int dev = 0;
  AWQB_CUDA(cudaGetDevice(&dev));
  int n = dev < 64 ? cached[dev].load() : 0;
  if (n == 0) {
    AWQB_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
    AWQB_REQUIRE(n > 0, kCudaError, "the kernel does not fit this GPU");
    if (dev < 64) cached[dev].store(n);
  }
  *out = n;
  return kOk;
}

template <typename T, bool kMany>
int launch(const void* x, int64_t ldx, const void* w, Params p, cudaStream_t stream) {
  using C = typename std::conditional<kMany, Many, Few>::type;
  const auto kernel = kMany ? grouped_gemm_many_kernel<T> : grouped_gemm_few_kernel<T>;
  constexpr int kCluster = kMany ? 2 : 1, kTokCta = C::kTok / kCluster;
  p.tile_out = kFeat * kCluster / (p.silu ? 2 : 1);
  p.feat_tiles = (p.n_out + p.tile_out - 1) / p.tile_out;
  CUtensorMap tw;
  TokenMaps tx;
  int st = kMany && p.silu ? make_gate_up_map(&tw, w, p)
                           : make_rows_map(&tw, w, (int64_t)p.E * p.N, p.K, p.K, p.silu ? kFeat / 2 : kFeat);
  for (int i = 0; i < 3 && st == kOk; ++i) st = make_rows_map(&tx.box[i], x, p.rows, p.K, ldx, kTokCta >> (2 - i));
  if (st != kOk) return st;
  const auto smem_for = [](int E) {
    return 1024 + C::kStages * C::kStageBytes + (kMany ? 0 : Few::kChunk * kFeat * 4) + 4 * C::kTok * 4 + (3 * E + 1) * 4;
  };
  const int smem = smem_for(p.E);
  // (the most that any call wants: another thread's call may set it before this launch)
  AWQB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_for(kMaxExperts)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kCluster);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static std::atomic<int> cached[64];
  int64_t clusters = 0;
  st = max_clusters(kernel, cfg, cached, &clusters);
  if (st != kOk) return st;
  // every tile there could be: a group adds at most one partly filled token tile
  const int64_t tiles = ((p.rows + C::kTok - 1) / C::kTok + std::min<int64_t>(p.E, p.rows)) * p.feat_tiles;
  AWQB_REQUIRE(tiles < (1ll << 31), kUnsupported, "too many tiles (%lld)", (long long)tiles);
  cfg.gridDim = dim3((unsigned)(std::min(tiles, clusters) * kCluster));
  cfg.numAttrs = 2;
  AWQB_CUDA(cudaLaunchKernelEx(&cfg, kernel, tw, tx, p));
  return kOk;
}

}  // namespace
}  // namespace awqb

using namespace awqb;

extern "C" int awqb_grouped_gemm(const awqb_grouped_gemm_args* args, void* stream) {
  AWQB_REQUIRE(args != nullptr, kInvalidArgument, "args is null");
  const auto [x, rows, ldx, w, E, K, N, offsets, dtype, silu_mul, row_map, row_scale, out, out_rows, ldo] = *args;
  AWQB_REQUIRE(dtype == AWQB_DTYPE_F16 || dtype == AWQB_DTYPE_BF16, kInvalidArgument, "bad dtype %d", dtype);
  AWQB_REQUIRE(E >= 1 && E <= kMaxExperts, kInvalidArgument, "%lld experts: 1..%d are supported", (long long)E,
               kMaxExperts);
  AWQB_REQUIRE(K > 0 && K % 8 == 0 && K <= (1 << 20), kInvalidArgument, "K=%lld must be a positive multiple of 8",
               (long long)K);
  AWQB_REQUIRE(N > 0 && N % (silu_mul ? 16 : 8) == 0 && N <= (1 << 20), kInvalidArgument,
               "N=%lld must be a positive multiple of %d", (long long)N, silu_mul ? 16 : 8);
  AWQB_REQUIRE(rows >= 0 && rows < (1 << 30) && out_rows >= 0 && out_rows < (1ll << 31), kInvalidArgument,
               "bad number of rows %lld -> %lld", (long long)rows, (long long)out_rows);
  const int64_t n_out = silu_mul ? N / 2 : N;
  AWQB_REQUIRE(ldx >= K && ldo >= n_out && ldx % 8 == 0 && ldo % 8 == 0, kInvalidArgument,
               "row strides must be at least the row's length and multiples of 8");
  AWQB_REQUIRE(row_map != nullptr || out_rows >= rows, kInvalidArgument, "out has %lld rows, x %lld",
               (long long)out_rows, (long long)rows);
  if (rows == 0 || out_rows == 0) return kOk;
  AWQB_REQUIRE(x && w && offsets && out, kInvalidArgument, "null pointer");
  AWQB_REQUIRE(aligned16(x) && aligned16(w) && aligned16(out), kInvalidArgument, "tensors must be 16-byte aligned");
  Params p = {};
  p.offsets = offsets, p.row_map = row_map, p.row_scale = row_scale, p.out = out;
  p.err = device_error_word();
  AWQB_REQUIRE(p.err != nullptr, kCudaError, "cannot resolve the device error word");
  p.ldo = ldo, p.out_rows = out_rows;
  p.rows = (int)rows, p.E = (int)E, p.K = (int)K, p.N = (int)N, p.n_out = (int)n_out, p.silu = silu_mul != 0;
  // By the rows of the buffer, the only count that the host has: padding and rows of no
  // group count too. A large buffer with few live rows so takes the many-rows kernel,
  // which costs it 1 to 5 % (128 experts 2048 -> 1536, one row each: 123 / 126 us; eight
  // 4096 -> 14336: 156 / 161). Measured, few / many in us: 128 experts 2048 -> 1536 at 16, 32, 64 rows per expert
  // 126 / 129, 141 / 130, 178 / 138; 768 -> 2048 65 / 66, 78 / 67, 100 / 76; eight experts
  // 4096 -> 14336 161 / 167, 158 / 168, 207 / 168.
  const bool many = rows > 24 * E;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == AWQB_DTYPE_F16)
    return many ? launch<__half, true>(x, ldx, w, p, st) : launch<__half, false>(x, ldx, w, p, st);
  return many ? launch<__nv_bfloat16, true>(x, ldx, w, p, st) : launch<__nv_bfloat16, false>(x, ldx, w, p, st);
}
