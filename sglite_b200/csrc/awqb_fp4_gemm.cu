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
// tile's scales then is one contiguous bulk copy, and a warp turns four rows' words
// among a lane's registers, in place, on the way to tensor memory. A stage is 256 k, one
// swizzled row of 128 bytes.
//
// Roles of a CTA's warps: a producer of copies, one that issues the tensor-core work, the
// scale turners, one that finds tiles and where their rows go ahead of the others (the
// rows' places come from memory, two loads one after the other; with that and two CTAs to an SM
// 256 tokens' experts 768 -> 2048 went from 52 to 28 us),
// and the epilogue. A role's code and waits are a whole warp's, and the issuing lane is
// a predicate: with branches around them each instruction's operands pass through a move
// to the uniform registers (4096 tokens 8192 -> 28672: 414 -> 378 us for roles and waits by the whole
// warp).
//
// Two kernels. Few rows: the weights' bytes bound it; a CTA takes 128 weight rows x up to 32
// tokens, two CTAs to an SM, eight stages of 23 KB in flight there. Where the tiles of a
// product do not fill the GPU, two to eight CTAs of a cluster share a tile's K, and each adds
// its share of the tokens from what the others send to its shared memory (1 token
// 4096 -> 4096: 7.7 us whole, 5.3 by four). Many rows: a CTA pair takes 256 weight rows x up to
// 208 tokens, what two accumulators and two sets of scales leave of tensor memory; K is
// shared by two or four pairs where tiles are few. On a B200: 1 token 4096 -> 6144 in 6.1 us, 32
// tokens 4096 -> 28672 with SiLU-and-mul in 13.8 (4.9 TB/s), 4096 tokens 8192 -> 28672 in 383
// (5.0 PFLOP/s; 443 when repeated for seconds, under the power cap) and in 360 in mxfp4.
// Copies of that kernel which leave work out (374 us whole on that GPU): 321 without the scales'
// copies to tensor memory, 289 without the products, 323 without both. The last is slower than the
// one before it, so the series says that neither alone bounds it, and not what the loop waits for.
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
  int tok_tiles, tok_per;  // without offsets: token tiles, rows of each
  int box_rows;  // without offsets: rows of the box that all tiles take
  int split;  // CTAs (pairs) of a cluster that share a tile's K; above 1, a cluster has one tile
};

// One CTA per tile of 128 weight rows x up to 32 tokens, two CTAs to an SM. Of a stage:
// weights, rows (both swizzled: 1024-byte aligned), the weights' and the rows' scales.
// Tensor memory: two accumulators, two sets of scales. Where K is shared, the parts of a
// tile's sum land behind the stages, of which there are fewer then.
struct Few {
  static constexpr int kTok = 32;
  static constexpr int kRound = 16;
  static constexpr int kStages = 4, kSplitStages = 3;
  static constexpr int kEpiWarps = 4;
  static constexpr int kThreads = 32 * (kEpiWarps + 4);
  static constexpr int kPlans = 4, kPlanReaders = kEpiWarps, kCtasPerSm = 2;
  static constexpr int kAtX = kWBytes, kAtWs = kAtX + kTok * kK / 2, kAtXs = kAtWs + 2048;
  static constexpr int kStageBytes = kAtXs + 2048;
  static constexpr int kSets = 2 * kTok, kSetColumns = 32, kColumns = 128;
  static constexpr int kTurn = 16 * 272;  // bytes of the epilogue's transposition
  static __host__ __device__ constexpr int ring_bytes(int split) {
    return split > 1 ? kSplitStages * kStageBytes + kTok * kFeat * 4 : kStages * kStageBytes + kTurn;
  }
};
// A CTA pair; each loads its 128 weight rows and half the tokens, and the scales of all
// tokens. The accumulators and scales of 208 tokens fill tensor memory. Three groups of
// epilogue warps: a tile of few stages is bound by them (4096 tokens' experts 768 -> 2048:
// 82 us with two, 77 with three or four).
struct Many {
  static constexpr int kTok = 208;
  static constexpr int kRound = 16;
  static constexpr int kStages = 5;
  static constexpr int kEpiWarps = 12, kGroups = kEpiWarps / 4;
  static constexpr int kThreads = 32 * (kEpiWarps + 5);
  // the epilogue, and the scale turners: a tile of few stages may need nothing of one of them
  static constexpr int kPlans = 4, kPlanReaders = kEpiWarps + 2, kCtasPerSm = 1;
  static constexpr int kAtX = kWBytes, kAtWs = kAtX + kTok / 2 * kK / 2, kAtXs = kAtWs + 2048;
  static constexpr int kStageBytes = kAtXs + 4096;
  static constexpr int kSets = 2 * kTok, kSetColumns = 48, kColumns = 512;
  static constexpr int kTurn = 16 * 272;  // bytes of a group's transposition
  // the stages and the groups' transpositions
  static __host__ __device__ constexpr int ring_bytes(int) { return kStages * kStageBytes + kGroups * kTurn; }
};

// What the roles need to know of a tile, found by one warp ahead of them: the tile, then
// (a barrier later, since they come from memory) where its rows go.
template <typename C>
struct Plans {
  uint64_t tile_full[C::kPlans], rows_full[C::kPlans], free[C::kPlans];
  Tile tile[C::kPlans];
  float alpha[C::kPlans];
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
// of the four goes to tile w. (Tiles of up to 32 rows take it too: an instruction's scales
// have to begin at a column that is a multiple of four, so a row's four words cannot be
// left in neighbouring columns.)
template <int kBlocks>
__device__ __forceinline__ void turn_scales(uint8_t* at, int rows, int lane) {
  uint4* p = reinterpret_cast<uint4*>(at) + lane;
  if (rows <= 32) {
    const uint4 a = p[0];
    uint32_t* q = reinterpret_cast<uint32_t*>(p);
    q[0] = a.x, q[128] = a.y, q[256] = a.z, q[384] = a.w;
  } else if (rows <= 64) {
    const uint4 a = p[0], b = p[32];
    uint2* q = reinterpret_cast<uint2*>(p);
    q[0] = make_uint2(a.x, b.x), q[64] = make_uint2(a.y, b.y), q[128] = make_uint2(a.z, b.z), q[192] = make_uint2(a.w, b.w);
  } else {
    uint4 v[kBlocks][4];  // all loads before the first store
#pragma unroll
    for (int i = 0; i < 4 * kBlocks; ++i)
      if (i < 4 || rows > 128) v[i / 4][i % 4] = p[32 * i];
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      if (i > 0 && rows <= 128) break;
      const uint4 a = v[i][0], b = v[i][1], c = v[i][2], d = v[i][3];
      p[128 * i] = make_uint4(a.x, b.x, c.x, d.x);
      p[128 * i + 32] = make_uint4(a.y, b.y, c.y, d.y);
      p[128 * i + 64] = make_uint4(a.z, b.z, c.z, d.z);
      p[128 * i + 96] = make_uint4(a.w, b.w, c.w, d.w);
    }
  }
}

// Stores a weight row's values of 2 kPairs tokens from c on. Neighbouring lanes write
// neighbouring features of a token. Where rows are gate and up by turns, of each two tokens
// a lane keeps one and gives its neighbour the other.
template <typename T, int kPairs>
__device__ __forceinline__ void store_tokens(const Params& p, float (&y)[2 * kPairs], const int* to, const float* factor,
                                             int c, int rows, bool real, int odd, T* out) {
  int at[2 * kPairs];
  float f[2 * kPairs];
#pragma unroll
  for (int i = 0; i < 2 * kPairs; ++i) {  // (all of them before the first store)
    at[i] = to[c + i];
    f[i] = p.row_scale ? factor[c + i] : 1.f;
  }
#pragma unroll
  for (int i = 0; i < 2 * kPairs; i += 2) {
    if (c + i >= rows) break;
    if (p.silu) {
      const float got = __shfl_xor_sync(0xffffffffu, odd ? y[i] : y[i + 1], 1);
      y[i] = y[i + 1] = odd ? silu_mul(got, y[i + 1]) : silu_mul(y[i], got);
    }
#pragma unroll
    for (int k = i; k < i + 2; ++k) {
      if (!real || at[k] < 0 || (p.silu && k - i != odd)) continue;  // (-1 behind the rows)
      out[(int64_t)at[k] * p.ldo] = (T)(y[k] * f[k]);
    }
  }
}

// Initialises `n` barriers by one warp's lanes.
__device__ __forceinline__ void init_barriers(uint64_t* bars, int n, uint32_t count, int lane) {
  for (int i = lane; i < n; i += 32) mbar_init(smem_u32(bars + i), count);
}
template <typename C>
__device__ __forceinline__ void init_plans(Plans<C>& plans, int lane) {
  init_barriers(plans.tile_full, C::kPlans, 1, lane);
  init_barriers(plans.rows_full, C::kPlans, 1, lane);
  init_barriers(plans.free, C::kPlans, C::kPlanReaders, lane);
}

// Tile t where all rows are one group.
template <typename C>
__device__ __forceinline__ Tile whole_tile(const Params& p, int t) {
  const int ft = p.tok_tiles == 1 ? t : t / p.tok_tiles, tt = t - ft * p.tok_tiles;
  Tile r;
  r.e = 0;
  r.row0 = tt * p.tok_per;
  r.rows = min(p.tok_per, p.rows - r.row0);
  r.n = (r.rows + C::kRound - 1) / C::kRound * C::kRound;
  r.feat = ft * p.tile_out;
  return r;
}

// The planning warp: tiles first_tile, first_tile + tile_step .. A plan is free again when
// the epilogue is done with it, and whoever else may still have it to read: the roles that
// every tile needs something of have read it before the epilogue gets the tile.
template <typename C>
__device__ __forceinline__ bool plan_tiles(Plans<C>& plans, const Groups& g, const Params& p, int first_tile,
                                           int tile_step, int total, int* dst, float* scl, int lane) {
  int i = 0;
  for (int t = first_tile; t < total; t += tile_step, ++i) {
    const int at = i % C::kPlans;
    if (!mbar_wait_warp(smem_u32(&plans.free[at]), ((i / C::kPlans) & 1) ^ 1)) return false;
    const Tile tile = p.offsets ? find_tile<C>(g, p, t) : whole_tile<C>(p, t);
    if (lane == 0) {
      plans.tile[at] = tile;
      mbar_arrive(smem_u32(&plans.tile_full[at]));
    }
    float alpha = p.x_scale ? *p.x_scale : 1.f;
    if (p.w_scale) alpha *= p.w_scale[tile.e];
    constexpr int kMine = (C::kTok + 31) / 32;  // rows of a lane: all their loads in flight
    int to[kMine];
    float factor[kMine];
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int r = 32 * j + lane;
      to[j] = r >= tile.rows ? -1 : p.row_map ? p.row_map[tile.row0 + r] : tile.row0 + r;
    }
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      if (to[j] >= p.out_rows) to[j] = -1;
      factor[j] = p.row_scale && to[j] >= 0 ? p.row_scale[to[j]] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kMine; ++j)
      if (32 * j + lane < C::kTok) {
        dst[at * C::kTok + 32 * j + lane] = to[j];
        scl[at * C::kTok + 32 * j + lane] = factor[j];
      }
    if (lane == 0) plans.alpha[at] = alpha;
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&plans.rows_full[at]));
  }
  return true;
}

// A role's turn to tile t, number i of this CTA (false: the wait gave up). Without groups
// it is known at once.
template <typename C>
__device__ __forceinline__ bool next_tile(Plans<C>& plans, const Params& p, int t, int i, Tile* tile) {
  if (p.offsets == nullptr) {
    *tile = whole_tile<C>(p, t);
    return true;
  }
  const int at = i % C::kPlans;
  if (!mbar_wait_warp(smem_u32(&plans.tile_full[at]), (i / C::kPlans) & 1)) return false;
  *tile = plans.tile[at];
  return true;
}

// The number of tiles; builds the groups' tables where there are groups. All threads, a
// barrier among them, but for one group.
template <typename C>
__device__ __forceinline__ void find_groups(const Groups& g, const Params& p) {
  if (p.offsets != nullptr) build_groups<C>(g, p);
}
__device__ __forceinline__ int count_tiles(const Groups& g, const Params& p) {
  return __shfl_sync(0xffffffffu, p.offsets ? g.tile0[p.E] : p.tok_tiles * p.feat_tiles, 0);
}

// A role's place in the ring of stages.
struct Place {
  int s = 0, lap = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++s == stages) s = 0, lap ^= 1;
  }
};

// Stages of K that part `part` of p.split works on.
__device__ __forceinline__ void stages_of(const Params& p, int nk, int part, int* first, int* last) {
  *first = nk * part / p.split;
  *last = nk * (part + 1) / p.split;
}

// Stores tokens of a group of four warps' 128 weight rows, 8 G at a time. The accumulator
// comes as fragments (rows l / 4 and l / 4 + 8 of each half of a warp's rows, tokens
// 2 (l % 4) and the next), which stmatrix transposes on the way through the group's
// [16 tokens][128 features] of shared memory (rows of 272 bytes: no bank twice for eight of
// them), so that a token's features leave as 256 contiguous bytes. (64 bytes a warp, without
// the group's barriers, kept the stores at 14 bytes a clock and SM.) Where rows are gate and
// up by turns, neighbouring rows are four lanes apart: the even one takes the first eight
// rows' four products and the odd one the last eight's, which come out as features
// 0, 4, 1, 5 .. and are put in order behind the transposition.
template <typename T>
struct TileStore {
  static constexpr int kPitch = 272;
  float alpha, bias[2][2];
  int f, lane, quarter, group;  // f: the CTA's first feature
  uint32_t turn;
  // row: of the weights, the CTA's first
  __device__ __forceinline__ TileStore(const Params& p, int row, float alpha_, int warp, int lane_, uint8_t* turn_)
      : alpha(alpha_), lane(lane_), quarter(warp & 3), group(warp >> 2), turn(smem_u32(turn_)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = row + 32 * quarter + 8 * i + (lane >> 2);
      bias[i / 2][i % 2] = p.bias && r < p.N ? (float)static_cast<const T*>(p.bias)[r] : 0.f;
    }
    f = p.silu ? row / 2 : row;
  }
  // tokens c .. c + 8 G - 1 of the tile, v[half of the rows][eight tokens]
  template <int G>
  __device__ __forceinline__ void tokens(const Params& p, int rows, uint32_t (&v)[2][G][4], int c, const int* to,
                                         const float* factor) const {
    const int odd = (lane >> 2) & 1;
    uint32_t m[G][4];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float2 s = make_float2(1.f, 1.f);
      if (p.row_scale) s = *reinterpret_cast<const float2*>(factor + c + 8 * g + 2 * (lane & 3));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = __uint_as_float(v[h][g][k]) * alpha + bias[h][k / 2];
        if (p.silu) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {  // even lanes keep rows 0..7 (gate) and get their up; odd ones 8..15 (up) and get gate
            const float got = __shfl_xor_sync(0xffffffffu, odd ? y[k] : y[2 + k], 4);
            y[k] = odd ? silu_mul(got, y[2 + k]) : silu_mul(y[k], got);
          }
          m[g][h] = Pair<T>::pack(y[0] * s.x, y[1] * s.y);
        } else {
          m[g][2 * h] = Pair<T>::pack(y[0] * s.x, y[1] * s.y);
          m[g][2 * h + 1] = Pair<T>::pack(y[2] * s.x, y[3] * s.y);
        }
      }
    }
    named_bar_sync(2 + group, 128);  // (the last tokens are read)
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint32_t at = turn + (8 * g + (lane & 7)) * kPitch;
      if (p.silu)  // two matrices of eight features
        asm volatile("stmatrix.sync.aligned.m8n8.x2.trans.shared.b16 [%0], {%1, %2};" ::"r"(
                         at + quarter * 32 + ((lane >> 3) & 1) * 16),
                     "r"(m[g][0]), "r"(m[g][1])
                     : "memory");
      else
        st_matrix_trans(at + quarter * 64 + (lane >> 3) * 16, m[g]);
    }
    named_bar_sync(2 + group, 128);
    // vector `piece` of every step-th token from t0 on
    const int tid = quarter * 32 + lane, shift = p.silu ? 3 : 4, t0 = tid >> shift, piece = tid & ((1 << shift) - 1);
    const int step = 128 >> shift;
    T* out = static_cast<T*>(p.out) + f + 8 * piece;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int t = step * i + t0;
      if (step * i >= 8 * G || c + t >= rows || f + 8 * piece >= p.n_out) break;
      const int row = to[c + t];
      uint4 o;
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(o.x), "=r"(o.y), "=r"(o.z), "=r"(o.w)
                   : "r"(turn + t * kPitch + piece * 16)
                   : "memory");
      if (p.silu)
        o = make_uint4(__byte_perm(o.x, o.y, 0x5410), __byte_perm(o.z, o.w, 0x5410), __byte_perm(o.x, o.y, 0x7632),
                       __byte_perm(o.z, o.w, 0x7632));
      if (row >= 0) *reinterpret_cast<uint4*>(out + (int64_t)row * p.ldo) = o;
    }
  }
};

// The first stages of weight rows feat .. on their way to L2 while the kernel in front ends,
// where there are no groups to wait for. (Its outputs, this product's rows, are not
// touched before the wait.) One thread.
template <bool kNv>
__device__ __forceinline__ void prefetch_weights(const CUtensorMap* tm_w, const CUtensorMap* tm_x, const Params& p,
                                                 int feat, int nk, int kb0, int kb1) {
  prefetch_tmap(tm_w);
  prefetch_tmap(tm_x);
  if (feat >= p.N) return;
  bulk_prefetch(p.w_scales + ((int64_t)(feat / kFeat) * nk + kb0) * kWsBytes<kNv>, (kb1 - kb0) * kWsBytes<kNv>);
  for (int kb = kb0; kb < kb1; ++kb) tma_prefetch_2d(tm_w, kb * kK / 2, feat);
}

template <typename T, bool kNv>
__global__ void __launch_bounds__(Few::kThreads, Few::kCtasPerSm)
fp4_gemm_few_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ TokenMaps tm_x,
                    const __grid_constant__ Params p) {
  using C = Few;
  extern __shared__ uint8_t raw[];
  uint8_t* ring = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  int* dst = reinterpret_cast<int*>(ring + C::ring_bytes(p.split));  // [kPlans][C::kTok] out row of a token
  float* scl = reinterpret_cast<float*>(dst + C::kPlans * C::kTok);          // [kPlans][C::kTok] its factor
  Groups g;
  g.row0 = reinterpret_cast<int*>(scl + C::kPlans * C::kTok);  // [E] first rows, [E] row counts
  g.tile0 = g.row0 + 2 * p.E;
  __shared__ uint64_t full[C::kStages], raw_scales[C::kStages], empty[C::kStages];
  __shared__ uint64_t acc_full[2], acc_empty[2], landed;
  __shared__ Plans<C> plans;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;

  // (from lane 0: the compiler then takes the roles' code as the whole warp's)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int part = p.split > 1 ? (int)cluster_ctarank() : 0;
  const int first_tile = blockIdx.x / p.split, tile_step = gridDim.x / p.split;
  const int nk = (p.K + kK - 1) / kK;
  int kb0, kb1;
  stages_of(p, nk, part, &kb0, &kb1);
  const int stages = p.split > 1 ? C::kSplitStages : C::kStages;
  // Where K is shared: four tokens at a time go by turns to the parts; this one's, and where they land
  const int fours = p.split > 1 ? (whole_tile<C>(p, first_tile).rows + 3) / 4 : 0;
  const int my_fours = (fours - part + p.split - 1) / p.split;
  float4* landing = reinterpret_cast<float4*>(ring + C::kSplitStages * C::kStageBytes);  // [turn][part][weight row]
  if (warp == C::kEpiWarps) {
    init_barriers(full, stages, 2, lane);  // the producer's expectation and the turned scales
    init_barriers(raw_scales, stages, 1, lane);
    init_barriers(empty, stages, 1, lane);
    init_barriers(acc_full, 2, 1, lane);
    init_barriers(acc_empty, 2, C::kEpiWarps, lane);
    init_plans(plans, lane);
    if (lane == 0) {
      mbar_init(smem_u32(&landed), 1);
      failed = 0;
    }
    fence_barrier_init();
    __syncwarp();
    if (p.split > 1 && lane == 0) mbar_arrive_expect_tx(smem_u32(&landed), my_fours * p.split * kFeat * 16);
  }
  if (warp == C::kEpiWarps + 1) {
    tmem_alloc(smem_u32(&tmem_slot), C::kColumns);
    tmem_relinquish();
  }
  grid_dep_launch();
  if (p.offsets == nullptr && warp == C::kEpiWarps && elect_one())
    prefetch_weights<kNv>(&tm_w, &tm_x.box[0], p, whole_tile<C>(p, first_tile).feat, nk, kb0,
                          min(kb1, kb0 + C::kStages));
  __syncwarp();
  if (p.split > 1) cluster_arrive();  // the barrier for landing parts is ready
  grid_dep_wait();
  find_groups<C>(g, p);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int total = count_tiles(g, p);
  bool ok = true, waited = p.split == 1;

  if (warp == C::kEpiWarps) {  // ------------------------------------- producer
    const uint64_t keep = policy_evict_normal(), once = policy_evict_first();
    Place at;
    int n_tile = 0;
    for (int t = first_tile; t < total && ok; t += tile_step, ++n_tile) {
      Tile tile;
      ok = next_tile(plans, p, t, n_tile, &tile);
      if (!ok) break;
      const int box = p.offsets ? box_of(tile.rows, C::kTok) : 0;
      const uint32_t x_bytes = (p.offsets ? C::kTok >> (2 - box) : p.box_rows) * kK / 2;
      // weights that one token tile reads once need not stay in L2
      const uint64_t wpol = (p.offsets ? tile.rows == g.row0[p.E + tile.e] : p.tok_tiles == 1) ? once : keep;
      const int wrow = tile.e * p.N + tile.feat;
      const uint8_t* ws = p.w_scales + ((int64_t)tile.e * p.feat_tiles + tile.feat / kFeat) * nk * kWsBytes<kNv>;
      const int scale_rows = min(tile.n, p.rows - tile.row0);
      for (int kb = kb0; kb < kb1; ++kb, at.next(stages)) {
        const int s = at.s, lap = at.lap;
        ok = mbar_wait_warp(smem_u32(&empty[s]), lap ^ 1);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t base = smem_u32(ring + s * C::kStageBytes), bar = smem_u32(&full[s]);
          const uint32_t sbar = smem_u32(&raw_scales[s]);
          mbar_arrive_expect_tx(bar, kWBytes + kWsBytes<kNv> + x_bytes);
          mbar_arrive_expect_tx(sbar, scale_rows * 16);
          tma_load_2d(base, &tm_w, kb * kK / 2, wrow, bar, wpol);
          bulk_g2s(base + C::kAtWs, ws + (int64_t)kb * kWsBytes<kNv>, kWsBytes<kNv>, bar, wpol);
          bulk_g2s(base + C::kAtXs, p.x_scales + ((int64_t)granule_of<kNv>(kb) * p.rows + tile.row0) * 16,
                   scale_rows * 16, sbar, keep);
          tma_load_2d(base + C::kAtX, &tm_x.box[box], kb * kK / 2, tile.row0, bar, keep);
        }
        __syncwarp();
      }
    }
  } else if (warp == C::kEpiWarps + 2) {  // ---------------------------- scales of the rows
    Place at;
    int n_tile = 0;
    for (int t = first_tile; t < total && ok; t += tile_step, ++n_tile) {
      Tile tile;
      ok = next_tile(plans, p, t, n_tile, &tile);
      if (!ok) break;
      for (int kb = kb0; kb < kb1; ++kb, at.next(stages)) {
        const int s = at.s, lap = at.lap;
        ok = mbar_wait_warp(smem_u32(&raw_scales[s]), lap);
        if (!ok) break;
        turn_scales<1>(ring + s * C::kStageBytes + C::kAtXs, tile.n, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&full[s]));
      }
    }
  } else if (warp == C::kEpiWarps + 1) {  // ---------------------------- MMA
    const uint32_t issue = elect_one();
    // (what the compiler cannot see to be the same for all lanes)
    const uint32_t tmem0 = __shfl_sync(0xffffffffu, tmem, 0), ring0 = __shfl_sync(0xffffffffu, smem_u32(ring), 0);
    Place at;
    int it = 0, n_tile = 0;
    for (int t = first_tile; t < total && ok; t += tile_step, ++n_tile) {
      Tile tile;
      const int b = n_tile & 1;
      ok = next_tile(plans, p, t, n_tile, &tile) &&
           mbar_wait_warp(smem_u32(&acc_empty[b]), ((n_tile >> 1) & 1) ^ 1);
      if (!ok) break;
      tc_fence_after();
      const uint32_t d = tmem0 + b * C::kTok;
      const uint32_t idesc = make_idesc_fp4(kFeat, __shfl_sync(0xffffffffu, tile.n, 0), kNv, 0);
      for (int kb = kb0; kb < kb1; ++kb, ++it, at.next(stages)) {
        const int s = at.s;
        ok = mbar_wait_warp(smem_u32(&full[s]), at.lap);
        if (!ok) break;
        tc_fence_after();
        const uint32_t base = ring0 + s * C::kStageBytes;
        const uint32_t ad = desc_low(base), bd = desc_low(base + C::kAtX);
        const uint32_t sa = tmem0 + C::kSets + (it & 1) * C::kSetColumns, sb = sa + 16;
        const int steps = min(kK, p.K - kb * kK + 63) / 64;
        const int words = kNv ? steps : (steps + 1) / 2;
#pragma unroll
        for (int j = 0; j < (kNv ? 4 : 2); ++j) {
          const uint32_t want = issue && j < words;
          tc_copy_scales<false>(want, sa + 4 * j, base + C::kAtWs + 512 * j);
          tc_copy_scales<false>(want, sb + 4 * j, base + C::kAtXs + 512 * (first_word<kNv>(kb) + j));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int w = kNv ? j : j >> 1, half = kNv ? 0 : j & 1;
          tc_mma_fp4<kNv, false>(issue && j < steps, d, ad + 2 * j, bd + 2 * j, idesc | make_idesc_fp4(0, 0, kNv, half),
                                 sa + 4 * w, sb + 4 * w, kb > kb0 || j > 0);
        }
        tc_commit_if(issue, smem_u32(&empty[s]));
      }
      if (ok) tc_commit_if(issue, smem_u32(&acc_full[b]));
    }
  } else if (warp == C::kEpiWarps + 3) {  // ---------------------------- plans
    ok = plan_tiles(plans, g, p, first_tile, tile_step, total, dst, scl, lane);
  } else {  // -------------------------------------------------------- epilogue
    // A lane holds a weight row's tokens. Where K is shared, each four tokens are sent to
    // the part whose turn it is, which adds what landed in the parts' order.
    const int tid = threadIdx.x, odd = lane & 1;
    int n_tile = 0;
    for (int t = first_tile; t < total; t += tile_step, ++n_tile) {
      const int b = n_tile & 1, at = n_tile % C::kPlans;
      ok = mbar_wait(smem_u32(&plans.rows_full[at]), (n_tile / C::kPlans) & 1);
      const Tile tile = plans.tile[at];
      const float alpha = plans.alpha[at];
      const int row = tile.feat + tid;  // of the weights
      const float bias = p.bias && row < p.N ? (float)static_cast<const T*>(p.bias)[row] : 0.f;
      ok = named_bar_and(1, 128, ok && mbar_wait(smem_u32(&acc_full[b]), (n_tile >> 1) & 1));
      if (!ok) break;
      tc_fence_after();
      const int* to = dst + at * C::kTok;
      const float* factor = scl + at * C::kTok;
      T* out = static_cast<T*>(p.out) + (p.silu ? row / 2 : row);
      if (!waited) cluster_wait();
      waited = true;
      for (int c = 0; c < tile.rows && p.split > 1; c += 16) {
        uint32_t v[16];
        tmem_ld16(tmem + b * C::kTok + c + ((uint32_t)warp << 21), v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const int four = (c + j) / 4, turn = four / p.split, who = four - turn * p.split;
          if (four < fours)
            st_async_v4(mapa_shared(smem_u32(landing + (turn * p.split + part) * kFeat + tid), who), v + j,
                        mapa_shared(smem_u32(&landed), who));
        }
      }
      if (p.split > 1) {
        ok = named_bar_and(1, 128, mbar_wait(smem_u32(&landed), 0));
        if (!ok) break;
        for (int turn = 0; turn < my_fours; ++turn) {
          const float4* part0 = landing + turn * p.split * kFeat + tid;
          float4 sum = part0[0];
          for (int q = 1; q < p.split; ++q) {
            const float4 v = part0[q * kFeat];
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
          }
          float y[4] = {sum.x * alpha + bias, sum.y * alpha + bias, sum.z * alpha + bias, sum.w * alpha + bias};
          store_tokens<T, 2>(p, y, to, factor, 4 * (turn * p.split + part), tile.rows, row < p.N, odd, out);
        }
        break;
      }
      const TileStore<T> store(p, tile.feat, alpha, warp, lane, ring + C::kStages * C::kStageBytes);
      for (int c = 0; c < tile.rows; c += 16) {
        uint32_t v[2][2][4];
        const uint32_t from = tmem + b * C::kTok + c + ((uint32_t)warp << 21);
        tmem_ld_fragments(from, v[0]);
        tmem_ld_fragments(from + (16u << 16), v[1]);
        tmem_ld_wait();
        if (c + 16 >= tile.rows) {  // the accumulator is read: the MMA warp may reuse it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&acc_empty[b]));
        }
        store.tokens(p, tile.rows, v, c, to, factor);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&plans.free[at]));
    }
  }
  if (!ok && lane == 0) {
    failed = 1;
    atomicOr(p.err, kErrWait);
  }
  __syncwarp();
  if (!waited) cluster_wait();
  __syncthreads();
  // (where K is shared, until nobody can still be sending a part here)
  for (int i = 0; failed && i < (p.split > 1 ? 250 : 1); ++i) linger();
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
  int* dst = reinterpret_cast<int*>(ring + C::ring_bytes(1));  // [kPlans][kTok] out row of a token
  float* scl = reinterpret_cast<float*>(dst + C::kPlans * C::kTok);  // [kPlans][kTok] its factor
  Groups g;
  g.row0 = reinterpret_cast<int*>(scl + C::kPlans * C::kTok);
  g.tile0 = g.row0 + 2 * p.E;
  __shared__ uint64_t full[C::kStages], raw_scales[C::kStages], empty[C::kStages];
  __shared__ uint64_t acc_full[2], acc_empty[2], landed;
  __shared__ Plans<C> plans;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;

  // (from lane 0: the compiler then takes the roles' code as the whole warp's)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // a cluster is p.split pairs; rank: in the pair, whose leader is CTA `leader` of the cluster
  const uint32_t rank = cluster_ctarank() & 1, leader = cluster_ctarank() & ~1u;
  const int part = cluster_ctarank() >> 1;
  const uint16_t pair_mask = (uint16_t)(3u << leader);
  const int first_tile = blockIdx.x / (2 * p.split), tile_step = gridDim.x / (2 * p.split);
  const int nk = (p.K + kK - 1) / kK;
  int kb0, kb1;
  stages_of(p, nk, part, &kb0, &kb1);
  // Where K is shared: 16 tokens at a time go by turns to the parts, this one's among them,
  // and land in the ring, [turn][part, without this one][fragment][lane of the warps' 128]
  const int turns = p.split > 1 ? (whole_tile<C>(p, first_tile).rows + 15) / 16 : 0;
  const int my_turns = (turns - part + p.split - 1) / p.split;
  float4* landing = reinterpret_cast<float4*>(ring);
  if (warp == C::kEpiWarps) {
    init_barriers(full, C::kStages, 3, lane);  // the leader's expectation and both CTAs' turned scales
    init_barriers(raw_scales, C::kStages, 1, lane);
    init_barriers(empty, C::kStages, 1, lane);
    init_barriers(acc_full, 2, 1, lane);
    init_barriers(acc_empty, 2, 2 * C::kEpiWarps, lane);
    init_plans(plans, lane);
    if (lane == 0) {
      mbar_init(smem_u32(&landed), 1);
      failed = 0;
    }
    fence_barrier_init();
    __syncwarp();
    if (p.split > 1 && lane == 0)
      mbar_arrive_expect_tx(smem_u32(&landed), my_turns * (p.split - 1) * 16 * kFeat * 4);
  }
  if (warp == C::kEpiWarps + 1) {
    tmem_alloc_pair(smem_u32(&tmem_slot), C::kColumns);
    tmem_relinquish_pair();
  }
  grid_dep_launch();
  if (p.offsets == nullptr && warp == C::kEpiWarps && elect_one())
    prefetch_weights<kNv>(&tm_w, &tm_x.box[0], p, whole_tile<C>(p, first_tile).feat + (int)rank * kFeat, nk, kb0,
                          min(kb1, kb0 + C::kStages));
  __syncwarp();
  grid_dep_wait();
  find_groups<C>(g, p);
  tc_fence_before();
  cluster_sync_all();  // the peer's barriers are ready before anything arrives on them
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  uint8_t* turn_bytes = ring + C::kStages * C::kStageBytes + (warp >> 2) % C::kGroups * C::kTurn;
  const int total = count_tiles(g, p);
  bool ok = true;

  if (warp == C::kEpiWarps) {  // ------------------------------------- producer
    const uint64_t keep = policy_evict_normal(), once = policy_evict_first();
    const int scale_tiles = (p.N + kFeat - 1) / kFeat;
    Place at;
    int n_tile = 0;
    for (int t = first_tile; t < total && ok; t += tile_step, ++n_tile) {
      Tile tile;
      ok = next_tile(plans, p, t, n_tile, &tile);
      if (!ok) break;
      const int box = p.offsets ? box_of(min(tile.rows, tile.n / 2), C::kTok / 2) : 0;
      // weights that one token tile reads once need not stay in L2
      const uint64_t wpol = (p.offsets ? tile.rows == g.row0[p.E + tile.e] : p.tok_tiles == 1) ? once : keep;
      const int feat = tile.feat + (int)rank * kFeat, row = tile.row0 + (int)rank * (tile.n / 2);
      // (rows past N are multiplied, by whatever scales, and not stored)
      const uint8_t* ws =
          p.w_scales + ((int64_t)tile.e * scale_tiles + min(feat / kFeat, scale_tiles - 1)) * nk * kWsBytes<kNv>;
      const int scale_rows = min(tile.n, p.rows - tile.row0);
      const uint32_t bytes = 2 * (kWBytes + (p.offsets ? C::kTok / 2 >> (2 - box) : p.box_rows) * kK / 2);
      for (int kb = kb0; kb < kb1; ++kb, at.next(C::kStages)) {
        const int s = at.s, lap = at.lap;
        ok = mbar_wait_warp(smem_u32(&empty[s]), lap ^ 1);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t base = smem_u32(ring + s * C::kStageBytes), bar = mapa_shared(smem_u32(&full[s]), leader);
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
    for (int i = 0; i < C::kStages && ok; ++i, at.next(C::kStages))
      ok = mbar_wait_warp(smem_u32(&empty[at.s]), at.lap ^ 1);
  } else if (warp == C::kEpiWarps + 2 || warp == C::kEpiWarps + 4) {  // -- scales of the rows
    // A slot of the ring is always the same warp's: copies may land out of order, and a wait
    // for a lap of a slot tells it from the one before only if that one has been seen to end.
    // Where tiles have few stages, one may have none in this warp's slots and be done without
    // it: the plan is read and given back all the same.
    const int odd = warp == C::kEpiWarps + 4;
    Place at;
    int n_tile = 0;
    for (int t = first_tile; t < total && ok; t += tile_step, ++n_tile) {
      Tile tile;
      ok = next_tile(plans, p, t, n_tile, &tile);
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&plans.free[n_tile % C::kPlans]));
      for (int kb = kb0; kb < kb1; ++kb, at.next(C::kStages)) {
        const int s = at.s, lap = at.lap;
        if ((s & 1) != odd) continue;
        ok = mbar_wait_warp(smem_u32(&raw_scales[s]), lap);
        if (!ok) break;
        turn_scales<2>(ring + s * C::kStageBytes + C::kAtXs, tile.n, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_peer(mapa_shared(smem_u32(&full[s]), leader));
      }
    }
  } else if (warp == C::kEpiWarps + 1) {  // ---------------------------- MMA, the leader's
    const uint32_t issue = elect_one();
    // (what the compiler cannot see to be the same for all lanes)
    const uint32_t tmem0 = __shfl_sync(0xffffffffu, tmem, 0), ring0 = __shfl_sync(0xffffffffu, smem_u32(ring), 0);
    Place at;
    int it = 0, n_tile = 0;
    for (int t = first_tile; t < total && ok && rank == 0; t += tile_step, ++n_tile) {
      Tile tile;
      const int b = n_tile & 1;
      ok = next_tile(plans, p, t, n_tile, &tile) &&
           mbar_wait_warp(smem_u32(&acc_empty[b]), ((n_tile >> 1) & 1) ^ 1);
      if (!ok) break;
      tc_fence_after();
      const int n = __shfl_sync(0xffffffffu, tile.n, 0);
      const uint32_t d = tmem0 + b * C::kTok, idesc = make_idesc_fp4(2 * kFeat, n, kNv, 0);
      for (int kb = kb0; kb < kb1; ++kb, ++it, at.next(C::kStages)) {
        const int s = at.s;
        ok = mbar_wait_warp(smem_u32(&full[s]), at.lap);
        if (!ok) break;
        tc_fence_after();
        const uint32_t base = ring0 + s * C::kStageBytes;
        const uint32_t ad = desc_low(base), bd = desc_low(base + C::kAtX);
        // a word's columns of row scales: 8, for up to 256 rows
        const uint32_t sa = tmem0 + C::kSets + (it & 1) * C::kSetColumns, sb = sa + 16;
        const int steps = min(kK, p.K - kb * kK + 63) / 64;
        const int words = kNv ? steps : (steps + 1) / 2;
#pragma unroll
        for (int j = 0; j < (kNv ? 4 : 2); ++j) {
          const uint32_t want = issue && j < words;
          const uint32_t at = base + C::kAtXs + 512 * (first_word<kNv>(kb) + j);
          tc_copy_scales<true>(want, sa + 4 * j, base + C::kAtWs + 512 * j);
          tc_copy_scales<true>(want, sb + 8 * j, at);
          tc_copy_scales<true>(want && n > 128, sb + 8 * j + 4, at + 2048);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int w = kNv ? j : j >> 1, half = kNv ? 0 : j & 1;
          tc_mma_fp4<kNv, true>(issue && j < steps, d, ad + 2 * j, bd + 2 * j, idesc | make_idesc_fp4(0, 0, kNv, half),
                                sa + 4 * w, sb + 8 * w, kb > kb0 || j > 0);
        }
        tc_commit_pair_if(issue, smem_u32(&empty[s]), pair_mask);
      }
      if (ok) tc_commit_pair_if(issue, smem_u32(&acc_full[b]), pair_mask);
    }
  } else if (warp == C::kEpiWarps + 3) {  // ---------------------------- plans
    ok = plan_tiles(plans, g, p, first_tile, tile_step, total, dst, scl, lane);
  } else {  // -------------------------------------------------------- epilogue
    // The groups of four warps take turns over 16 tokens.
    const int quarter = warp & 3;
    const uint32_t at = tmem + ((uint32_t)quarter << 21);
    int n_tile = 0;
    for (int t = first_tile; t < total; t += tile_step, ++n_tile) {
      const int b = n_tile & 1, slot = n_tile % C::kPlans;
      ok = mbar_wait(smem_u32(&plans.rows_full[slot]), (n_tile / C::kPlans) & 1);
      const Tile tile = plans.tile[slot];
      const TileStore<T> store(p, tile.feat + (int)rank * kFeat, plans.alpha[slot], warp, lane, turn_bytes);
      ok = named_bar_and(1, 32 * C::kEpiWarps, ok && mbar_wait(smem_u32(&acc_full[b]), (n_tile >> 1) & 1));
      if (!ok) break;
      tc_fence_after();
      if (p.split > 1) break;  // the accumulator is summed below
      for (int c = (warp >> 2) * 16; c < tile.rows; c += 16 * C::kGroups) {
        uint32_t v[2][2][4];
        tmem_ld_fragments(at + b * C::kTok + c, v[0]);
        tmem_ld_fragments(at + b * C::kTok + c + (16u << 16), v[1]);
        tmem_ld_wait();
        if (c + 16 * C::kGroups >= tile.rows) {  // this warp has read its part of the accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_peer(mapa_shared(smem_u32(&acc_empty[b]), leader));
        }
        store.tokens(p, tile.rows, v, c, dst + slot * C::kTok, scl + slot * C::kTok);
      }
      if ((warp >> 2) * 16 >= tile.rows) {  // no tokens for this group
        __syncwarp();
        if (lane == 0) mbar_arrive_peer(mapa_shared(smem_u32(&acc_empty[b]), leader));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&plans.free[slot]));
    }
  }
  if (!ok && lane == 0) {
    failed = 1;
    atomicOr(p.err, kErrWait);
  }
  __syncwarp();
  if (p.split > 1) {
    cluster_sync_all();  // every ring is idle: parts may land there
    if (warp < C::kEpiWarps && first_tile < total && ok) {
      const Tile tile = plans.tile[0];
      const int quarter = warp & 3, group = warp >> 2, place = quarter * 32 + lane;
      const uint32_t at = tmem + ((uint32_t)quarter << 21);
      tc_fence_after();
      for (int i = group; i < turns; i += C::kGroups) {
        const int turn = i / p.split, who = i - turn * p.split;
        if (who == part) continue;
        uint32_t v[2][2][4];
        tmem_ld_fragments(at + 16 * i, v[0]);
        tmem_ld_fragments(at + 16 * i + (16u << 16), v[1]);
        tmem_ld_wait();
        const int slot = turn * (p.split - 1) + (part < who ? part : part - 1);
        const uint32_t to = mapa_shared(smem_u32(landing + slot * 4 * kFeat + place), 2 * who + rank);
        const uint32_t bar = mapa_shared(smem_u32(&landed), 2 * who + rank);
#pragma unroll
        for (int j = 0; j < 4; ++j) st_async_v4(to + j * kFeat * 16, v[j / 2][j % 2], bar);
      }
      const TileStore<T> store(p, tile.feat + (int)rank * kFeat, plans.alpha[0], warp, lane, turn_bytes);
      // (all of them or none: a group's warps meet at barriers when they store)
      ok = named_bar_and(1, 32 * C::kEpiWarps, mbar_wait(smem_u32(&landed), 0));
      for (int turn = group; turn < my_turns && ok; turn += C::kGroups) {
        const int c = 16 * (turn * p.split + part);
        uint32_t own[2][2][4];
        tmem_ld_fragments(at + c, own[0]);
        tmem_ld_fragments(at + c + (16u << 16), own[1]);
        tmem_ld_wait();
        float sum[4][4] = {};
        for (int q = 0; q < p.split; ++q) {  // in the parts' order
          const float4* from = landing + (turn * (p.split - 1) + (q < part ? q : q - 1)) * 4 * kFeat + place;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t* o = own[j / 2][j % 2];
            const float4 f = q == part ? make_float4(__uint_as_float(o[0]), __uint_as_float(o[1]), __uint_as_float(o[2]),
                                                     __uint_as_float(o[3]))
                                       : from[j * kFeat];
            sum[j][0] += f.x, sum[j][1] += f.y, sum[j][2] += f.z, sum[j][3] += f.w;
          }
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) own[j / 8][j / 4 % 2][j % 4] = __float_as_uint(sum[j / 4][j % 4]);
        store.tokens(p, tile.rows, own, c, dst, scl);
      }
      if (!ok && lane == 0) {
        failed = 1;
        atomicOr(p.err, kErrWait);
      }
    }
  }
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

template <typename C, auto kernel>
int launch(int pair, const void* codes, const void* w, Params p, int max_split, cudaStream_t stream) {
  const int tok_cta = C::kTok / pair;
  p.tile_out = kFeat * pair;
  p.feat_tiles = (p.N + p.tile_out - 1) / p.tile_out;
  CUtensorMap tw;
  TokenMaps tx;
  const int64_t row_bytes = p.K / 2;
  int st = make_bytes_map(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, (int64_t)p.E * p.N, row_bytes, row_bytes, kFeat);
  // without groups all tiles take the first, largest tile's box
  p.tok_tiles = (p.rows + C::kTok - 1) / C::kTok;
  p.tok_per = ((p.rows + p.tok_tiles - 1) / p.tok_tiles + C::kRound - 1) / C::kRound * C::kRound;
  // without groups, a box of just the rows of a tile: rows that a box reads past the last
  // one cost as much as real ones and more (1 token 4096 -> 28672: 16.2 us in a box of 16, 14.0 in one of 8)
  p.box_rows = std::min(p.rows, p.tok_per / pair);
  for (int i = 0; i < (p.offsets ? 3 : 1) && st == kOk; ++i)
    st = make_bytes_map(&tx.box[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes, p.rows, row_bytes, row_bytes,
                        p.offsets ? tok_cta >> (2 - i) : p.box_rows);
  if (st != kOk) return st;
  const auto smem_for = [](int E, int split) {
    return 1024 + C::ring_bytes(split) + 2 * C::kPlans * C::kTok * 4 + (3 * E + 1) * 4;
  };
  static std::atomic<bool> ready[64];  // the kernel's attributes, set once for a device
  int dev = 0;
  AWQB_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !ready[dev].load()) {
    AWQB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   std::max(smem_for(kMaxExperts, 1), smem_for(1, 2))));
    // all of it, so that two CTAs of the few-rows kernel fit an SM
    AWQB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100));
    if (dev < 64) ready[dev].store(true);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(C::kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  // every tile there could be: a group adds at most one partly filled token tile
  const int64_t tiles = (p.tok_tiles + (p.offsets ? std::min<int64_t>(p.E, p.rows) : 0)) * p.feat_tiles;
  AWQB_REQUIRE(tiles < (1ll << 31), kUnsupported, "too many tiles (%lld)", (long long)tiles);
  // K is shared by as many CTAs (pairs) as leave each tile a cluster of its own at once, and
  // each of them two stages
  static std::atomic<int> cached[4][64];
  const int nk = (p.K + kK - 1) / kK;
  int64_t clusters = 0;
  int log = 3;  // up to 8
  if (p.offsets != nullptr) max_split = 1;
  for (;; --log) {
    p.split = 1 << log;
    if (p.split > max_split || (p.split > 1 && nk < 2 * p.split)) continue;
    attr[0].val.clusterDim.x = (unsigned)(pair * p.split);
    cfg.gridDim = dim3((unsigned)(pair * p.split));
    cfg.numAttrs = 1;
    cfg.dynamicSmemBytes = smem_for(p.E, p.split);
    st = max_clusters(kernel, cfg, cached[log], &clusters);
    if (st != kOk) return st;
    clusters *= C::kCtasPerSm;  // (the query counts one for kernels with tensor memory)
    if (log == 0 || tiles <= clusters) break;
  }
  cfg.gridDim = dim3((unsigned)(std::min(tiles, clusters) * pair * p.split));
  cfg.numAttrs = 2;
  AWQB_CUDA(cudaLaunchKernelEx(&cfg, kernel, tw, tx, p));
  return kOk;
}

template <typename T, bool kNv>
int pick(const void* codes, const void* w, const Params& p, cudaStream_t stream) {
  // Groups: by their mean rows, since the CTA pairs' epilogue and start cost more and are
  // spread over K's stages (us, few-rows and many-rows kernel, 2048 -> 1536 x 128 experts: 39 and 40 for
  // 12 rows, 43 and 41 for 16, 53 and 44 for 48; 768 -> 2048: 31 and 33 for 32, 39 and 36 for 48. The
  // border, 20, is past that of the first series: 16 rows take the slower kernel, by 5 %). The rows
  // are the buffer's, the only count that the host has: rows behind the last group count too. One group:
  // above 32 rows, unless the few-rows kernel's tiles are few as well (4096 -> 28672, 48 rows: 22
  // and 17; 8192 -> 1024, 128 rows: 7.9 and 9.0).
  const int nk = (p.K + kK - 1) / kK;
  const int64_t mean = (p.rows + p.E - 1) / p.E;
  const int64_t tiles = (int64_t)((p.N + kFeat - 1) / kFeat) * ((p.rows + Few::kTok - 1) / Few::kTok);
  const bool many = p.offsets ? mean > (nk >= 4 ? 20 : 40) : p.rows > Few::kTok && tiles > device_sm_count() / 2;
  if (many) return launch<Many, fp4_gemm_many_kernel<T, kNv>>(2, codes, w, p, 4, stream);
  return launch<Few, fp4_gemm_few_kernel<T, kNv>>(1, codes, w, p, 8, stream);
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
  // (a pair's rows behind the last one still have 32-bit coordinates; N first, so that E * N cannot overflow)
  AWQB_REQUIRE(N > 0 && N % (silu_mul ? 16 : 8) == 0 && N <= 0x7fffff00 && E * N <= 0x7fffff00, kInvalidArgument,
               "N=%lld must be a positive multiple of %d, and all experts' rows fewer than 2^31 - 255", (long long)N,
               silu_mul ? 16 : 8);
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
