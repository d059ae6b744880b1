// What the kernels over ragged groups of rows share: a group's rows cut into equal
// token tiles, tiles found on the device from the groups' offsets, SiLU-and-mul. P is a
// kernel's parameter structure (offsets, rows, E, feat_tiles, tile_out), C its
// constants (kTok, kRound, kThreads).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "awqb_common.h"
#include "awqb_ptx.cuh"

namespace awqb {
namespace {

// Boxes of token rows: a quarter, a half and all of what a CTA may load per stage.
struct TokenMaps {
  CUtensorMap box[3];
};

struct Tile {
  int e, row0, rows, n, feat;  // expert, first row, rows, rows rounded up for the MMA, first output feature
};

// Shared-memory tables of the groups: first row and first tile of each.
struct Groups {
  int* row0;
  int* tile0;  // [E + 1]
};

template <typename C, typename P>
__device__ __forceinline__ Tile find_tile(const Groups& g, const P& p, int t) {
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
template <typename C, typename P>
__device__ __forceinline__ void build_groups(const Groups& g, const P& p) {
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

// silu(g) * u with the approximate exponential and division: right to
// (6 + 1.173 |g|) 2^-23 of the value (1.2e-5 at g = -80; 16-bit results keep 2^-11 at
// best), and 0 below g = -87.3, where |silu(g)| < 88 * 2^-126.
__device__ __forceinline__ float silu_mul(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// The smallest box that holds `rows` token rows.
__device__ __forceinline__ int box_of(int rows, int most) { return rows * 4 <= most ? 0 : rows * 2 <= most ? 1 : 2; }

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

}  // namespace
}  // namespace awqb
