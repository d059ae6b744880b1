// Products of microscaled 4-bit rows and weights (awqb_fp4.cuh has the formats), whole
// or grouped by expert: y[r] = x_scale w_scale[e] x[r] w[e]^T, with bias, SiLU-and-mul,
// scatter and router weights in the epilogue.
//
// The block-scaled tensor-core instructions take e2m1 operands from shared memory and
// their scales from tensor memory, so nothing is dequantised: TMA brings the operands,
// tcgen05.cp the scales. As in the 16-bit grouped kernels the M side takes weights (128
// rows), the N side tokens, in steps of 16.
//
// Scales. An instruction takes 64 k and wants row r's scales on lane r % 32 of column
// r / 32. The weights' scales are laid out so once, at load. The rows' scales are kept
// as rows, [granule][row][16 bytes], since a group may begin at any row: the copy of a
// tile's scales then is one contiguous bulk copy, and one warp turns four rows' words
// among a lane's registers, in place, on the way to tensor memory.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "awqb200.h"
#include "awqb_common.h"
#include "awqb_grouped.cuh"
#include "awqb_ptx.cuh"
#include "awqb_tma.h"
#include "awqb_vec.cuh"

namespace awqb {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kFeat = 128;            // weight rows per CTA and tile
constexpr int kK = 256;               // k per stage: one 128-byte swizzled row
constexpr int kWBytes = kFeat * kK / 2;
constexpr uint32_t kErrWait = 512u;   // a bounded wait of these kernels gave up

struct Params {
  const int32_t *offsets, *row_map;
  const float *row_scale, *x_scale, *w_scale;
  const uint8_t *x_scales, *w_scales;
  const void* bias;
  void* out;
  uint32_t* err;
  int64_t ldo, out_rows;
  int rows, E, K, N, n_out, silu, feat_tiles, tile_out;  // tile_out: weight rows of a tile
};

struct Few {
  static constexpr int kTok = 64;   // tokens per tile
  static constexpr int kRound = 16;
  static constexpr int kStages = 6;
  static constexpr int kEpiWarps = 4;
  static constexpr int kThreads = 32 * (kEpiWarps + 3);
  // of a stage: weights, rows (both swizzled: 1024-byte aligned), the weights' and the rows' scales
  static constexpr int kAtX = kWBytes, kAtWs = kAtX + kTok * kK / 2, kAtXs = kAtWs + 2048;
  static constexpr int kStageBytes = kAtXs + 2048;
  // tensor memory: two accumulators, two sets of scales
  static constexpr int kSets = 2 * kTok, kSetColumns = 32, kColumns = 256;
};

// A CTA pair; each loads its 128 weight rows and half the tokens, and the scales of all tokens.
struct Many {
  static constexpr int kTok = 224;  // two accumulators and the scales fill tensor memory
  static constexpr int kRound = 32;
  static constexpr int kStages = 5;
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 32 * (kEpiWarps + 3);
  static constexpr int kAtX = kWBytes, kAtWs = kAtX + kTok / 2 * kK / 2, kAtXs = kAtWs + 2048;
  static constexpr int kStageBytes = kAtXs + 4096;
  static constexpr int kSets = 2 * kTok, kColumns = 512;
};

// Bytes of a stage's weight scales.
template <bool kNv>
constexpr int kWsBytes = kNv ? 2048 : 1024;

// The granule of a row's scales that a stage needs, and the first of its words in it.
template <bool kNv>
__device__ __forceinline__ int granule_of(int kb) { return kNv ? kb : kb >> 1; }
template <bool kNv>
__device__ __forceinline__ int first_word(int kb) { return kNv ? 0 : 2 * (kb & 1); }

// Rows of 16 bytes of scales, as they stand in memory, into tiles of 32 x 16 bytes, in
// place: of 128 rows, lane l holds l, l + 32, l + 64 and l + 96, four words each; word w
// of the four goes to tile w.
__device__ __forceinline__ void turn_scales(uint8_t* at, int rows, int lane) {
  for (int r = 0; r < rows; r += 128, at += 2048) {
    uint4* p = reinterpret_cast<uint4*>(at) + lane;
    const uint4 a = p[0], b = p[32], c = p[64], d = p[96];
    p[0] = make_uint4(a.x, b.x, c.x, d.x);
    p[32] = make_uint4(a.y, b.y, c.y, d.y);
    p[64] = make_uint4(a.z, b.z, c.z, d.z);
    p[96] = make_uint4(a.w, b.w, c.w, d.w);
  }
}

template <typename T, bool kNv>
__global__ void __launch_bounds__(Few::kThreads, 1)
fp4_gemm_few_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ TokenMaps tm_x,
                    const __grid_constant__ Params p) {
  using C = Few;
  extern __shared__ uint8_t raw[];
  uint8_t* ring = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  int* dst = reinterpret_cast<int*>(ring + C::kStages * C::kStageBytes);  // [2][kTok] out row of a token
  float* scl = reinterpret_cast<float*>(dst + 2 * C::kTok);               // [2][kTok]
  Groups g;
  g.row0 = reinterpret_cast<int*>(scl + 2 * C::kTok);  // [E] first rows, [E] row counts
  g.tile0 = g.row0 + 2 * p.E;
  __shared__ uint64_t full[C::kStages], raw_scales[C::kStages], scaled[C::kStages], empty[C::kStages];
  __shared__ uint64_t acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&raw_scales[s]), 1);
      mbar_init(smem_u32(&scaled[s]), 1);
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
    tmem_alloc(smem_u32(&tmem_slot), C::kColumns);
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
      const uint8_t* ws = p.w_scales + ((int64_t)tile.e * p.feat_tiles + tile.feat / kFeat) * nk * kWsBytes<kNv>;
      const int scale_rows = min(tile.n, p.rows - tile.row0);
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const int s = it % C::kStages;
        ok = mbar_wait(smem_u32(&empty[s]), ((it / C::kStages) & 1) ^ 1);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t base = smem_u32(ring + s * C::kStageBytes);
          const uint32_t bar = smem_u32(&full[s]), sbar = smem_u32(&raw_scales[s]);
          mbar_arrive_expect_tx(bar, kWBytes + kWsBytes<kNv> + (C::kTok >> (2 - box)) * kK / 2);
          tma_load_2d(base, &tm_w, kb * kK / 2, wrow, bar, wpol);
          bulk_g2s(base + C::kAtWs, ws + (int64_t)kb * kWsBytes<kNv>, kWsBytes<kNv>, bar, wpol);
          tma_load_2d(base + C::kAtX, &tm_x.box[box], kb * kK / 2, tile.row0, bar, keep);
          mbar_arrive_expect_tx(sbar, scale_rows * 16);
          bulk_g2s(base + C::kAtXs, p.x_scales + ((int64_t)granule_of<kNv>(kb) * p.rows + tile.row0) * 16,
                   scale_rows * 16, sbar, keep);
        }
        __syncwarp();
      }
    }
  } else if (warp == C::kEpiWarps + 2) {  // ---------------------------- scales of the rows
    int it = 0;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const int s = it % C::kStages;
        ok = mbar_wait(smem_u32(&raw_scales[s]), (it / C::kStages) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        turn_scales(ring + s * C::kStageBytes + C::kAtXs, C::kTok, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&scaled[s]));
      }
    }
  } else if (warp == C::kEpiWarps + 1) {  // ---------------------------- MMA
    int it = 0, n_tile = 0;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x, ++n_tile) {
      const Tile tile = find_tile<C>(g, p, t);
      const int b = n_tile & 1;
      ok = mbar_wait(smem_u32(&acc_empty[b]), ((n_tile >> 1) & 1) ^ 1);
      tc_fence_after();
      const uint32_t d = tmem + b * C::kTok;
      for (int kb = 0; kb < nk && ok; ++kb, ++it) {
        const int s = it % C::kStages;
        ok = mbar_wait(smem_u32(&full[s]), (it / C::kStages) & 1) && mbar_wait(smem_u32(&scaled[s]), (it / C::kStages) & 1);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t base = smem_u32(ring + s * C::kStageBytes);
          const uint64_t ad = make_sw128_kmajor_desc(base), bd = make_sw128_kmajor_desc(base + C::kAtX);
          const uint32_t sa = tmem + C::kSets + (it & 1) * C::kSetColumns, sb = sa + 16;
          const int steps = min(kK, p.K - kb * kK + 63) / 64;
          const int words = kNv ? steps : (steps + 1) / 2;
          for (int j = 0; j < words; ++j) {
            tc_copy_scales<false>(sa + 4 * j, base + C::kAtWs + 512 * j);
            tc_copy_scales<false>(sb + 4 * j, base + C::kAtXs + 512 * (first_word<kNv>(kb) + j));
          }
          for (int j = 0; j < steps; ++j) {
            const int w = kNv ? j : j >> 1, half = kNv ? 0 : j & 1;
            tc_mma_fp4<kNv, false>(d, ad + 2 * j, bd + 2 * j, make_idesc_fp4(kFeat, tile.n, kNv, half), sa + 4 * w,
                                   sb + 4 * w, kb + j > 0);
          }
          tc_commit(smem_u32(&empty[s]));
          if (kb == nk - 1) tc_commit(smem_u32(&acc_full[b]));
        }
        __syncwarp();
      }
    }
  } else {  // -------------------------------------------------------- epilogue
    // A lane holds a weight row's tokens. Neighbouring lanes write neighbouring features
    // of a token. With silu_mul even lanes hold gate and odd lanes up rows: a lane keeps
    // eight of 16 tokens and gives its neighbour the others.
    const int tid = threadIdx.x, odd = lane & 1;
    const float xs = p.x_scale ? *p.x_scale : 1.f;
    int n_tile = 0;
    for (int t = blockIdx.x; t < total; t += gridDim.x, ++n_tile) {
      const Tile tile = find_tile<C>(g, p, t);
      const int b = n_tile & 1;
      int* rows = dst + b * C::kTok;
      float* scales = scl + b * C::kTok;
      load_rows(p, tile, tid, 128, rows, scales);
      const int row = tile.feat + tid;  // of the weights
      const float alpha = xs * (p.w_scale ? p.w_scale[tile.e] : 1.f);
      const float bias = p.bias && row < p.N ? (float)static_cast<const T*>(p.bias)[row] : 0.f;
      ok = named_bar_and(1, 128, mbar_wait(smem_u32(&acc_full[b]), (n_tile >> 1) & 1));
      if (!ok) break;
      tc_fence_after();
      T* out = static_cast<T*>(p.out) + (p.silu ? row / 2 : row);
      for (int c = 0; c < tile.n; c += 16) {
        uint32_t v[16];
        tmem_ld16(tmem + b * C::kTok + c + ((uint32_t)warp << 21), v);
        tmem_ld_wait();
        if (c + 16 >= tile.n) {  // the accumulator is read: the MMA warp may reuse it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&acc_empty[b]));
        }
        float y[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = __uint_as_float(v[j]) * alpha + bias;
        const int count = p.silu ? 8 : 16, first = p.silu ? c + 8 * odd : c;
        if (p.silu) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float keep = odd ? y[8 + j] : y[j];
            const float got = __shfl_xor_sync(0xffffffffu, odd ? y[j] : y[8 + j], 1);
            y[j] = odd ? silu_mul(got, keep) : silu_mul(keep, got);
          }
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (j >= count || first + j >= tile.rows || row >= p.N) continue;
          const int to = rows[first + j];
          if (to < 0) continue;
          const float w = p.row_scale ? y[j] * scales[first + j] : y[j];
          out[(int64_t)to * p.ldo] = (T)w;
        }
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
    tmem_dealloc(tmem, C::kColumns);
  }
}

template <typename T, bool kNv>
__global__ void __launch_bounds__(Many::kThreads, 1)
fp4_gemm_many_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ TokenMaps tm_x,
                     const __grid_constant__ Params p) {
  using C = Many;
  extern __shared__ uint8_t raw[];
  uint8_t* ring = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  int* dst = reinterpret_cast<int*>(ring + C::kStages * C::kStageBytes);  // [2][kTok] out row of a token
  float* scl = reinterpret_cast<float*>(dst + 2 * C::kTok);               // [2][kTok]
  Groups g;
  g.row0 = reinterpret_cast<int*>(scl + 2 * C::kTok);
  g.tile0 = g.row0 + 2 * p.E;
  __shared__ uint64_t full[C::kStages], raw_scales[C::kStages], scaled[C::kStages], empty[C::kStages];
  __shared__ uint64_t acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&raw_scales[s]), 1);
      mbar_init(smem_u32(&scaled[s]), 2);  // both CTAs' scales
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
    tmem_alloc_pair(smem_u32(&tmem_slot), C::kColumns);
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
    const int scale_tiles = (p.N + kFeat - 1) / kFeat;
    int it = 0;
    for (int t = pair; t < total && ok; t += pairs) {
      const Tile tile = find_tile<C>(g, p, t);
      const int box = box_of(tile.n / 2, C::kTok / 2);
      // weights that one token tile reads once need not stay in L2
      const uint64_t wpol = tile.rows == g.row0[p.E + tile.e] ? once : keep;
      const int feat = tile.feat + (int)rank * kFeat, row = tile.row0 + (int)rank * (tile.n / 2);
      // (rows past N are multiplied, by whatever scales, and not stored)
      const uint8_t* ws =
          p.w_scales + ((int64_t)tile.e * scale_tiles + min(feat / kFeat, scale_tiles - 1)) * nk * kWsBytes<kNv>;
      const int scale_rows = min(tile.n, p.rows - tile.row0);
      const uint32_t bytes = 2 * (kWBytes + (C::kTok / 2 >> (2 - box)) * kK / 2);
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const int s = it % C::kStages;
        ok = mbar_wait(smem_u32(&empty[s]), ((it / C::kStages) & 1) ^ 1);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t base = smem_u32(ring + s * C::kStageBytes), bar = mapa_shared(smem_u32(&full[s]), 0);
          const uint32_t sbar = smem_u32(&raw_scales[s]);
          mbar_arrive_expect_tx(sbar, kWsBytes<kNv> + scale_rows * 16);
          bulk_g2s(base + C::kAtXs, p.x_scales + ((int64_t)granule_of<kNv>(kb) * p.rows + tile.row0) * 16,
                   scale_rows * 16, sbar, keep);
          bulk_g2s(base + C::kAtWs, ws + (int64_t)kb * kWsBytes<kNv>, kWsBytes<kNv>, sbar, wpol);
          if (rank == 0) mbar_arrive_expect_tx(smem_u32(&full[s]), bytes);
          tma_load_2d_pair(base, &tm_w, kb * kK / 2, tile.e * p.N + feat, bar, wpol);
          tma_load_2d_pair(base + C::kAtX, &tm_x.box[box], kb * kK / 2, row, bar, keep);
        }
        __syncwarp();
      }
    }
    // the last stages' releases arrive from the pair's leader before this CTA may leave
    for (int i = max(0, it - C::kStages); i < it && ok; ++i)
      ok = mbar_wait(smem_u32(&empty[i % C::kStages]), (i / C::kStages) & 1);
  } else if (warp == C::kEpiWarps + 2) {  // ---------------------------- scales of the rows
    int it = 0;
    for (int t = pair; t < total && ok; t += pairs) {
      const Tile tile = find_tile<C>(g, p, t);
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const int s = it % C::kStages;
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&raw_scales[s]), (it / C::kStages) & 1));
        if (!ok) break;
        turn_scales(ring + s * C::kStageBytes + C::kAtXs, tile.n, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_peer(mapa_shared(smem_u32(&scaled[s]), 0));
      }
    }
  } else if (warp == C::kEpiWarps + 1) {  // ---------------------------- MMA, the leader's
    int it = 0, n_tile = 0;
    for (int t = pair; t < total && ok && rank == 0; t += pairs, ++n_tile) {
      const Tile tile = find_tile<C>(g, p, t);
      const int b = n_tile & 1;
      ok = mbar_wait(smem_u32(&acc_empty[b]), ((n_tile >> 1) & 1) ^ 1);
      tc_fence_after();
      const uint32_t sa = tmem + C::kSets, sb = sa + 16;  // a word's column of row scales: 8 for 256 rows
      for (int kb = 0; kb < nk && ok; ++kb, ++it) {
        const int s = it % C::kStages;
        ok = mbar_wait(smem_u32(&full[s]), (it / C::kStages) & 1) && mbar_wait(smem_u32(&scaled[s]), (it / C::kStages) & 1);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t base = smem_u32(ring + s * C::kStageBytes);
          const uint64_t ad = make_sw128_kmajor_desc(base), bd = make_sw128_kmajor_desc(base + C::kAtX);
          const int steps = min(kK, p.K - kb * kK + 63) / 64;
          const int words = kNv ? steps : (steps + 1) / 2;
          for (int j = 0; j < words; ++j) {
            tc_copy_scales<true>(sa + 4 * j, base + C::kAtWs + 512 * j);
            const uint32_t at = base + C::kAtXs + 512 * (first_word<kNv>(kb) + j);
            tc_copy_scales<true>(sb + 8 * j, at);
            if (tile.n > 128) tc_copy_scales<true>(sb + 8 * j + 4, at + 2048);
          }
          for (int j = 0; j < steps; ++j) {
            const int w = kNv ? j : j >> 1, half = kNv ? 0 : j & 1;
            tc_mma_fp4<kNv, true>(tmem + b * C::kTok, ad + 2 * j, bd + 2 * j, make_idesc_fp4(2 * kFeat, tile.n, kNv, half),
                                  sa + 4 * w, sb + 8 * w, kb + j > 0);
          }
          tc_commit_pair(smem_u32(&empty[s]));
          if (kb == nk - 1) tc_commit_pair(smem_u32(&acc_full[b]));
        }
        __syncwarp();
      }
    }
  } else {  // -------------------------------------------------------- epilogue
    // Two groups of four warps take turns over 32 tokens. A lane holds a weight row's
    // tokens; eight lanes transpose eight tokens among them in registers, so that each
    // writes eight features of a token. With silu_mul even lanes hold gate and odd lanes
    // up rows: a lane keeps 16 tokens and gives its neighbour the other 16.
    const int group = warp >> 2, quarter = warp & 3, odd = lane & 1;
    const uint32_t at = tmem + ((uint32_t)quarter << 21);
    const float xs = p.x_scale ? *p.x_scale : 1.f;
    int n_tile = 0;
    for (int t = pair; t < total; t += pairs, ++n_tile) {
      const Tile tile = find_tile<C>(g, p, t);
      const int b = n_tile & 1;
      int* rows = dst + b * C::kTok;
      float* scales = scl + b * C::kTok;
      load_rows(p, tile, threadIdx.x, 32 * C::kEpiWarps, rows, scales);
      const int row = tile.feat + (int)rank * kFeat + quarter * 32;  // of the weights, the warp's first
      const float alpha = xs * (p.w_scale ? p.w_scale[tile.e] : 1.f);
      const float bias = p.bias && row + lane < p.N ? (float)static_cast<const T*>(p.bias)[row + lane] : 0.f;
      ok = named_bar_and(1, 32 * C::kEpiWarps, mbar_wait(smem_u32(&acc_full[b]), (n_tile >> 1) & 1));
      if (!ok) break;
      tc_fence_after();
      const int f = p.silu ? (row + (lane & 16)) / 2 : row + (lane & 24);
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
          if (lane == 0) mbar_arrive_peer(mapa_shared(smem_u32(&acc_empty[b]), 0));
        }
        float v[32];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          v[j] = __uint_as_float(lo[j]) * alpha + bias;
          v[16 + j] = __uint_as_float(hi[j]) * alpha + bias;
        }
        if (p.silu) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float own = odd ? v[16 + j] : v[j];
            const float got = __shfl_xor_sync(0xffffffffu, odd ? v[j] : v[16 + j], 1);
            v[j] = silu_mul(odd ? got : own, odd ? own : got);
            if (p.row_scale) v[j] *= scales[c + 16 * odd + j];
          }
#pragma unroll
          for (int j = 0; j < 16; j += 8) put(transpose8<T, 2>(v + j, lane), c + 16 * odd + j + ((lane >> 1) & 7));
        } else {
          if (p.row_scale)
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= scales[c + j];
#pragma unroll
          for (int j = 0; j < 32; j += 8) put(transpose8<T, 1>(v + j, lane), c + j + (lane & 7));
        }
      }
      if (group * 32 >= tile.rows) {  // no tokens for this group
        __syncwarp();
        if (lane == 0) mbar_arrive_peer(mapa_shared(smem_u32(&acc_empty[b]), 0));
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
    tmem_dealloc_pair(tmem, C::kColumns);
  }
}

template <typename T, bool kNv, bool kMany>
int launch(const void* codes, const void* w, Params p, cudaStream_t stream) {
  using C = typename std::conditional<kMany, Many, Few>::type;
  const auto kernel = kMany ? fp4_gemm_many_kernel<T, kNv> : fp4_gemm_few_kernel<T, kNv>;
  constexpr int kCluster = kMany ? 2 : 1, kTokCta = C::kTok / kCluster;
  p.tile_out = kFeat * kCluster;
  p.feat_tiles = (p.N + p.tile_out - 1) / p.tile_out;
  CUtensorMap tw;
  TokenMaps tx;
  const int64_t row_bytes = p.K / 2;
  int st = make_bytes_map(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, (int64_t)p.E * p.N, row_bytes, row_bytes, kFeat);
  for (int i = 0; i < 3 && st == kOk; ++i)
    st = make_bytes_map(&tx.box[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes, p.rows, row_bytes, row_bytes,
                        kTokCta >> (2 - i));
  if (st != kOk) return st;
  const auto smem_for = [](int E) { return 1024 + C::kStages * C::kStageBytes + 4 * C::kTok * 4 + (3 * E + 1) * 4; };
  // (the most that any call wants: another thread's call may set it before this launch)
  AWQB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_for(kMaxExperts)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kCluster);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = smem_for(p.E);
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
  const int64_t tiles = ((p.rows + C::kTok - 1) / C::kTok + (p.offsets ? std::min<int64_t>(p.E, p.rows) : 0)) * p.feat_tiles;
  AWQB_REQUIRE(tiles < (1ll << 31), kUnsupported, "too many tiles (%lld)", (long long)tiles);
  cfg.gridDim = dim3((unsigned)(std::min(tiles, clusters) * kCluster));
  cfg.numAttrs = 2;
  AWQB_CUDA(cudaLaunchKernelEx(&cfg, kernel, tw, tx, p));
  return kOk;
}

template <typename T, bool kNv>
int pick(const void* codes, const void* w, const Params& p, cudaStream_t stream) {
  if (p.rows > 24 * p.E) return launch<T, kNv, true>(codes, w, p, stream);
  return launch<T, kNv, false>(codes, w, p, stream);
}

}  // namespace
}  // namespace awqb

using namespace awqb;

extern "C" int awqb_fp4_gemm(const awqb_fp4_gemm_args* args, void* stream) {
  AWQB_REQUIRE(args != nullptr, kInvalidArgument, "args is null");
  const auto [codes, scales, rows, K, w, w_scales, E, N, offsets, format, dtype, x_scale, w_scale, bias, silu_mul, row_map,
              row_scale, out, out_rows, ldo] = *args;
  AWQB_REQUIRE(dtype == AWQB_DTYPE_F16 || dtype == AWQB_DTYPE_BF16, kInvalidArgument, "bad dtype %d", dtype);
  AWQB_REQUIRE(format == AWQB_FP4_NV || format == AWQB_FP4_MX, kInvalidArgument, "bad format %d", format);
  AWQB_REQUIRE(format != AWQB_FP4_MX || (x_scale == nullptr && w_scale == nullptr), kInvalidArgument,
               "mxfp4 has no scale but its blocks'");
  AWQB_REQUIRE(E >= 1 && E <= kMaxExperts, kInvalidArgument, "%lld experts: 1..%d are supported", (long long)E,
               kMaxExperts);
  AWQB_REQUIRE(offsets != nullptr || E == 1, kInvalidArgument, "several groups need offsets");
  AWQB_REQUIRE(offsets == nullptr || bias == nullptr, kInvalidArgument, "a bias is for a product without groups");
  AWQB_REQUIRE(K > 0 && K % 32 == 0 && K <= (1 << 20), kInvalidArgument, "K=%lld must be a positive multiple of 32",
               (long long)K);
  AWQB_REQUIRE(N > 0 && N % (silu_mul ? 16 : 8) == 0 && E * N <= 0x7fffffff, kInvalidArgument,
               "N=%lld must be a positive multiple of %d", (long long)N, silu_mul ? 16 : 8);
  AWQB_REQUIRE(rows >= 0 && rows <= (1 << 30) && out_rows >= 0, kInvalidArgument, "bad row count %lld", (long long)rows);
  const int64_t n_out = silu_mul ? N / 2 : N;
  AWQB_REQUIRE(ldo >= n_out && ldo % 8 == 0, kInvalidArgument, "the row stride of out must be >= %lld and a multiple of 8",
               (long long)n_out);
  AWQB_REQUIRE(row_map != nullptr || out_rows >= rows, kInvalidArgument, "out has %lld rows, x has %lld",
               (long long)out_rows, (long long)rows);
  if (rows == 0 || out_rows == 0) return kOk;
  AWQB_REQUIRE(codes && scales && w && w_scales && out, kInvalidArgument, "null pointer");
  AWQB_REQUIRE(aligned16(codes) && aligned16(scales) && aligned16(w) && aligned16(w_scales) && aligned16(out),
               kInvalidArgument, "tensors must be 16-byte aligned");
  Params p = {};
  p.offsets = offsets, p.row_map = row_map, p.row_scale = row_scale, p.x_scale = x_scale, p.w_scale = w_scale;
  p.x_scales = scales, p.w_scales = w_scales, p.bias = bias, p.out = out, p.ldo = ldo, p.out_rows = out_rows;
  p.rows = (int)rows, p.E = (int)E, p.K = (int)K, p.N = (int)N, p.n_out = (int)n_out, p.silu = silu_mul ? 1 : 0;
  p.err = device_error_word();
  AWQB_REQUIRE(p.err != nullptr, kCudaError, "no device error word");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool nv = format == AWQB_FP4_NV;
  if (dtype == AWQB_DTYPE_F16) return nv ? pick<__half, true>(codes, w, p, st) : pick<__half, false>(codes, w, p, st);
  return nv ? pick<__nv_bfloat16, true>(codes, w, p, st) : pick<__nv_bfloat16, false>(codes, w, p, st);
}
