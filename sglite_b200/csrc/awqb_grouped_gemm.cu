// Matrix products grouped by expert over 16-bit weights [E][N][K], with ragged
// group sizes that only the device knows: y[r] = x[r] w[e]^T for the rows of
// expert e, optionally silu(gate) * up over the two halves of w's rows.
//
// Layout of the work. The tensor core's M side takes weights (128 features per
// CTA), its N side takes tokens: N may be any multiple of 16 (32 for a CTA
// pair), so a ragged group costs what its rows cost, where tokens on the M side
// would round every group up to 128 rows. A group's rows are cut into equal
// token tiles of at most kTok; a tile is (expert, token tile, feature tile), the
// tiles of one weight tile following one another so that its later reads hit L2.
// CTAs are persistent and take tiles round-robin; every CTA finds a tile's
// expert by bisection in a prefix sum of tile counts that it builds from the
// offsets at its start, so the host never waits for them.
//
// Per CTA: a TMA producer warp, an MMA warp (tcgen05, fp32 accumulators in tensor
// memory, two buffers so that the epilogue overlaps the next tile) and four
// epilogue warps. The accumulator has features on lanes and tokens on columns:
// the epilogue turns 32 tokens at a time through shared memory in fp32, where
// gate and up (two halves of the lanes) also meet, and writes 16-byte vectors of
// a token's features.
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
constexpr int kEpiWarps = 4;
constexpr int kThreads = 32 * (kEpiWarps + 2);
constexpr int kWBytes = kFeat * kK * 2;
constexpr int kChunk = 32;        // tokens per epilogue turn
constexpr uint32_t kErrWait = 128u;  // a bounded wait of this kernel gave up

// kPair = 2: a CTA pair shares a tile of 256 features x up to 256 tokens, each CTA
// loading its 128 features and half the tokens: per 64 k a CTA moves 32 KB for
// 2 * 128 * 256 * 64 flops, within what shared memory feeds. kPair = 1: one
// CTA, 128 features x up to 64 tokens, for groups so small that the weights'
// bytes bound them; eight stages keep 128 KB of weights in flight.
template <int kPair>
struct Cfg {
  static constexpr int kTok = kPair == 2 ? 256 : 64;       // tokens per tile
  static constexpr int kTokCta = kTok / kPair;             // tokens a CTA loads
  static constexpr int kStageBytes = kWBytes + kTokCta * kK * 2;
  static constexpr int kStages = kPair == 2 ? 6 : 8;
  static constexpr int kCols = kTok < 32 ? 32 : kTok;      // accumulator columns per buffer
  static constexpr int kRound = 16 * kPair;                // MMA N granularity
};

struct Params {
  const int32_t *offsets, *row_map;
  const float* row_scale;
  void* out;
  uint32_t* err;
  int64_t ldo, out_rows;
  int rows, E, K, N, n_out, silu, feat_tiles;
};

struct Tile {
  int e, row0, rows, feat;  // expert, first row, rows, first output feature of the cluster's tile
};

// Shared-memory tables of the groups: first row and first tile of each.
struct Groups {
  int* row0;
  int* tile0;  // [E + 1]
};

template <int kPair>
__device__ __forceinline__ int token_tiles(int rows) {
  return (rows + Cfg<kPair>::kTok - 1) / Cfg<kPair>::kTok;
}

template <int kPair>
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
  const int per = ((rows + mt - 1) / mt + Cfg<kPair>::kRound - 1) / Cfg<kPair>::kRound * Cfg<kPair>::kRound;
  Tile r;
  r.e = lo;
  r.row0 = g.row0[lo] + tt * per;
  r.rows = min(per, rows - tt * per);
  r.feat = ft * kFeat * kPair / (p.silu ? 2 : 1);
  return r;
}

template <typename T, int kPair>
__global__ void __launch_bounds__(kThreads, 1)
grouped_gemm_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                    const __grid_constant__ CUtensorMap tm_x16, const __grid_constant__ Params p) {
  using C = Cfg<kPair>;
  extern __shared__ uint8_t raw[];
  uint8_t* ring = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  float* turn = reinterpret_cast<float*>(ring + C::kStages * C::kStageBytes);  // [kChunk][kFeat]
  int* dst = reinterpret_cast<int*>(turn + kChunk * kFeat);                     // [2][kTok] out row of a token
  float* scl = reinterpret_cast<float*>(dst + 2 * C::kTok);                     // [2][kTok]
  Groups g;
  g.row0 = reinterpret_cast<int*>(scl + 2 * C::kTok);  // [E] first rows, [E] row counts
  g.tile0 = g.row0 + 2 * p.E;
  __shared__ uint64_t full[C::kStages], empty[C::kStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = kPair == 2 ? cluster_ctarank() : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&acc_full[b]), 1);
      mbar_init(smem_u32(&acc_empty[b]), kEpiWarps * kPair);
    }
    failed = 0;
    fence_barrier_init();
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_x);
  }
  if (warp == kEpiWarps + 1) {
    if (kPair == 2) {
      tmem_alloc_pair(smem_u32(&tmem_slot), 2 * C::kCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(&tmem_slot), 2 * C::kCols);
      tmem_relinquish();
    }
  }
  grid_dep_wait();
  for (int e = threadIdx.x; e < p.E; e += kThreads) {
    const int r0 = min(max(p.offsets[e], 0), p.rows), r1 = min(max(p.offsets[e + 1], 0), p.rows);
    g.row0[e] = r0;
    g.row0[p.E + e] = max(r1 - r0, 0);
  }
  __syncthreads();
  if (warp == 0) {
    int run = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane;
      int v = e < p.E ? token_tiles<kPair>(g.row0[p.E + e]) * p.feat_tiles : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (e < p.E) g.tile0[e + 1] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) g.tile0[0] = 0;
  }
  tc_fence_before();
  if (kPair == 2) cluster_sync_all();  // the peer's barriers are ready before anything arrives on them
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int total = g.tile0[p.E];
  const int cta = blockIdx.x / kPair, ctas = gridDim.x / kPair;
  const int nk = (p.K + kK - 1) / kK;

  if (warp == kEpiWarps) {  // ---------------------------------------- producer
    const uint64_t keep = policy_evict_normal();
    const uint64_t once = policy_evict_first();
    int it = 0;
    bool ok = true;
    for (int t = cta; t < total && ok; t += ctas) {
      const Tile tile = find_tile<kPair>(g, p, t);
      const int n = (tile.rows + C::kRound - 1) / C::kRound * C::kRound;
      const int row = tile.row0 + (int)rank * (n / kPair);
      const bool few = kPair == 1 && tile.rows <= 16;
      const uint32_t tok_bytes = few ? 16 * kK * 2 : C::kTokCta * kK * 2;
      // weights that one token tile reads once need not stay in L2
      const uint64_t wpol = tile.rows == g.row0[p.E + tile.e] ? once : keep;
      const int half = kFeat / 2;
      const int wrow = tile.e * p.N + tile.feat + (int)rank * (p.silu ? half : kFeat);
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const int s = it % C::kStages;
        if (!mbar_wait(smem_u32(&empty[s]), ((it / C::kStages) & 1) ^ 1)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          const uint32_t base = smem_u32(ring + s * C::kStageBytes);
          uint32_t bar = smem_u32(&full[s]);
          if (kPair == 2) bar = mapa_shared(bar, 0);
          if (rank == 0) mbar_arrive_expect_tx(smem_u32(&full[s]), kPair * (kWBytes + tok_bytes));
          if (kPair == 2) {
            if (p.silu) {
              tma_load_2d_pair(base, &tm_w, kb * kK, wrow, bar, wpol);
              tma_load_2d_pair(base + kWBytes / 2, &tm_w, kb * kK, wrow + p.n_out, bar, wpol);
            } else {
              tma_load_2d_pair(base, &tm_w, kb * kK, wrow, bar, wpol);
            }
            tma_load_2d_pair(base + kWBytes, &tm_x, kb * kK, row, bar, keep);
          } else {
            tma_load_2d(base, &tm_w, kb * kK, wrow, bar, wpol);
            if (p.silu) tma_load_2d(base + kWBytes / 2, &tm_w, kb * kK, wrow + p.n_out, bar, wpol);
            tma_load_2d(base + kWBytes, few ? &tm_x16 : &tm_x, kb * kK, row, bar, keep);
          }
        }
        __syncwarp();
      }
    }
    // the last stages' releases arrive (from the pair's leader, too) before this CTA may leave
    for (int i = max(0, it - C::kStages); i < it && ok; ++i)
      ok = mbar_wait(smem_u32(&empty[i % C::kStages]), (i / C::kStages) & 1);
    if (!ok && lane == 0) {
      failed = 1;
      atomicOr(p.err, kErrWait);
    }
  } else if (warp == kEpiWarps + 1) {  // ------------------------------- MMA
    if (rank == 0) {
      int it = 0, n_tile = 0;
      bool ok = true;
      for (int t = cta; t < total && ok; t += ctas, ++n_tile) {
        const Tile tile = find_tile<kPair>(g, p, t);
        const int n = (tile.rows + C::kRound - 1) / C::kRound * C::kRound;
        const uint32_t idesc = make_idesc_f16(kFeat * kPair, n, std::is_same<T, __nv_bfloat16>::value);
        const int b = n_tile & 1;
        if (!mbar_wait(smem_u32(&acc_empty[b]), ((n_tile >> 1) & 1) ^ 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + b * C::kCols;
        for (int kb = 0; kb < nk; ++kb, ++it) {
          const int s = it % C::kStages;
          if (!mbar_wait(smem_u32(&full[s]), (it / C::kStages) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint32_t base = smem_u32(ring + s * C::kStageBytes);
            const uint64_t ad = make_sw128_kmajor_desc(base), bd = make_sw128_kmajor_desc(base + kWBytes);
            const int steps = min(kK, p.K - kb * kK + 15) / 16;
            for (int j = 0; j < steps; ++j) {
              if (kPair == 2)
                tc_mma_f16_pair(d, ad + 2 * j, bd + 2 * j, idesc, kb + j > 0);
              else
                tc_mma_f16(d, ad + 2 * j, bd + 2 * j, idesc, kb + j > 0);
            }
            if (kPair == 2) tc_commit_pair(smem_u32(&empty[s])); else tc_commit(smem_u32(&empty[s]));
            if (kb == nk - 1) {
              if (kPair == 2) tc_commit_pair(smem_u32(&acc_full[b])); else tc_commit(smem_u32(&acc_full[b]));
            }
          }
          __syncwarp();
        }
      }
      if (!ok && lane == 0) {
        failed = 1;
        atomicOr(p.err, kErrWait);
      }
    }
  } else {  // -------------------------------------------------------- epilogue
    const int tid = threadIdx.x;  // 0..127, TMEM lane = feature
    const int feats = p.silu ? kFeat / 2 : kFeat;
    const int per_row = feats / 8;                      // threads that write one token
    const int fl = (tid % per_row) * 8, tk = tid / per_row;
    const int tok_step = 128 / per_row;
    // Feature c stands at c, its halves of eight swapped where bit 5 is set: the
    // 16-byte reads of eight lanes then hit all banks.
    const int put = tid ^ ((tid >> 3) & 4), get = fl + ((fl >> 3) & 4);
    int n_tile = 0;
    bool ok = true;
    for (int t = cta; t < total; t += ctas, ++n_tile) {
      const Tile tile = find_tile<kPair>(g, p, t);
      const int b = n_tile & 1;
      // where the tile's rows go, loaded while its products are still running
      for (int i = tid; i < tile.rows; i += 128) {
        const int to = p.row_map ? p.row_map[tile.row0 + i] : tile.row0 + i;
        const bool in = to >= 0 && to < p.out_rows;
        dst[b * C::kTok + i] = in ? to : -1;
        if (p.row_scale) scl[b * C::kTok + i] = in ? p.row_scale[to] : 0.f;
      }
      ok = mbar_wait(smem_u32(&acc_full[b]), (n_tile >> 1) & 1);
      if (!named_bar_and(1, 128, ok)) break;
      tc_fence_after();
      const int f = tile.feat + (int)rank * feats + fl;
      for (int c = 0; c < tile.rows; c += kChunk) {
        uint32_t v[2][16];
        tmem_ld16(tmem + b * C::kCols + c + ((uint32_t)warp << 21), v[0]);
        tmem_ld16(tmem + b * C::kCols + c + 16 + ((uint32_t)warp << 21), v[1]);
        tmem_ld_wait();
        if (c + kChunk >= tile.rows) {  // the accumulator is read: the MMA warp may reuse it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (kPair == 2) mbar_arrive_cluster(mapa_shared(smem_u32(&acc_empty[b]), 0));
            else mbar_arrive(smem_u32(&acc_empty[b]));
          }
        }
#pragma unroll
        for (int j = 0; j < kChunk; ++j) turn[j * kFeat + put] = __uint_as_float(v[j / 16][j % 16]);
        named_bar_sync(1, 128);
        const int m = min(kChunk, tile.rows - c);
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
            for (int i = 0; i < 8; ++i) y[i] = y[i] / (1.f + __expf(-y[i])) * u[i];
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
    if (!ok && lane == 0) {
      failed = 1;
      atomicOr(p.err, kErrWait);
    }
  }
  __syncwarp();
  __syncthreads();
  if (failed) {  // a wait gave up: leave copies and products in flight time to end
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 10000000ull) {
    }
  }
  tc_fence_before();
  if (kPair == 2) cluster_sync_all();  // the peer may still write or arrive here
  __syncthreads();
  if (warp == kEpiWarps + 1) {
    tc_fence_after();
    if (kPair == 2) tmem_dealloc_pair(tmem, 2 * C::kCols); else tmem_dealloc(tmem, 2 * C::kCols);
  }
  grid_dep_launch();
}

int make_map(CUtensorMap* tm, const void* base, int64_t rows, int64_t K, int64_t ld, int box_rows) {
  const auto enc = tensor_map_encoder();
  AWQB_REQUIRE(enc != nullptr, kCudaError, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t dim[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t stride[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {kK, (cuuint32_t)box_rows}, step[2] = {1, 1};
  const CUresult r = enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base), dim, stride, box, step,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  AWQB_REQUIRE(r == CUDA_SUCCESS, kCudaError, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return kOk;
}

// Clusters that run at once (a GPC with an odd number of SMs leaves one idle),
// per device; the persistent grid must not exceed it.
template <typename T, int kPair>
int max_clusters(cudaLaunchConfig_t cfg, int64_t* out) {
  static std::atomic<int> cached[64];
  int dev = 0;
  AWQB_CUDA(cudaGetDevice(&dev));
  int n = dev < 64 ? cached[dev].load() : 0;
  if (n == 0) {
    cfg.gridDim = dim3(kPair);
    AWQB_CUDA(cudaOccupancyMaxActiveClusters(&n, grouped_gemm_kernel<T, kPair>, &cfg));
    AWQB_REQUIRE(n > 0, kCudaError, "the kernel does not fit this GPU");
    if (dev < 64) cached[dev].store(n);
  }
  *out = n;
  return kOk;
}

template <typename T, int kPair>
int launch(const void* x, int64_t ldx, const void* w, const Params& p, cudaStream_t stream) {
  using C = Cfg<kPair>;
  CUtensorMap tw, tx, tx16;
  int st = make_map(&tw, w, (int64_t)p.E * p.N, p.K, p.K, p.silu ? kFeat / 2 : kFeat);
  if (st == kOk) st = make_map(&tx, x, p.rows, p.K, ldx, C::kTokCta);
  if (st == kOk) st = make_map(&tx16, x, p.rows, p.K, ldx, 16);
  if (st != kOk) return st;
  const int smem = 1024 + C::kStages * C::kStageBytes + kChunk * kFeat * 4 + 4 * C::kTok * 4 + (3 * p.E + 1) * 4;
  const auto kernel = grouped_gemm_kernel<T, kPair>;
  AWQB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kPair;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int64_t clusters = 0;
  st = max_clusters<T, kPair>(cfg, &clusters);
  if (st != kOk) return st;
  // every tile there could be: a group adds at most one partly filled token tile
  const int64_t tiles = ((p.rows + C::kTok - 1) / C::kTok + std::min<int64_t>(p.E, p.rows)) * p.feat_tiles;
  AWQB_REQUIRE(tiles < (1ll << 31), kUnsupported, "too many tiles (%lld)", (long long)tiles);
  cfg.gridDim = dim3((unsigned)(std::min(tiles, clusters) * kPair));
  cfg.numAttrs = 2;
  AWQB_CUDA(cudaLaunchKernelEx(&cfg, kernel, tw, tx, tx16, p));
  return kOk;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace
}  // namespace awqb

using namespace awqb;

static int awqb_grouped_gemm_impl(const void* x, int64_t rows, int64_t ldx, const void* w, int64_t E, int64_t K,
                                 int64_t N, const int32_t* offsets, int dtype, int silu_mul, const int32_t* row_map,
                                 const float* row_scale, void* out, int64_t out_rows, int64_t ldo, void* stream) {
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
  const bool pair = rows > 64 * E;
  p.feat_tiles = (int)((N + kFeat * (pair ? 2 : 1) - 1) / (kFeat * (pair ? 2 : 1)));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == AWQB_DTYPE_F16)
    return pair ? launch<__half, 2>(x, ldx, w, p, st) : launch<__half, 1>(x, ldx, w, p, st);
  return pair ? launch<__nv_bfloat16, 2>(x, ldx, w, p, st) : launch<__nv_bfloat16, 1>(x, ldx, w, p, st);
}

extern "C" int awqb_grouped_gemm(const awqb_grouped_gemm_args* a, void* stream) {
  AWQB_REQUIRE(a != nullptr, kInvalidArgument, "args is null");
  return awqb_grouped_gemm_impl(a->x, a->rows, a->ldx, a->w, a->E, a->K, a->N, a->offsets, a->dtype, a->silu_mul, a->row_map,
                                a->row_scale, a->out, a->out_rows, a->ldo, stream);
}
