// What the kernels over ragged groups of rows share: a group's rows cut into equal
// token tiles, tiles found on the device from the groups' offsets, and the epilogues'
// small parts. P is a kernel's parameter structure (offsets, row_map, row_scale,
// out_rows, rows, E, feat_tiles, tile_out), C its constants (kTok, kRound, kThreads).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "awqb_common.h"
#include "awqb_ptx.cuh"
#include "awqb_vec.cuh"

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

// Builds the tables of the groups from the offsets (clamped to the rows; without
// offsets, one group of all rows); all threads, with a barrier still to come before
// they are read.
template <typename C, typename P>
__device__ __forceinline__ void build_groups(const Groups& g, const P& p) {
  for (int e = threadIdx.x; e < p.E; e += C::kThreads) {
    const int r0 = p.offsets ? min(max(p.offsets[e], 0), p.rows) : 0;
    const int r1 = p.offsets ? min(max(p.offsets[e + 1], 0), p.rows) : p.rows;
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
template <typename P>
__device__ __forceinline__ void load_rows(const P& p, const Tile& tile, int first, int step, int* dst, float* scl) {
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
__host__ __device__ __forceinline__ int box_of(int rows, int most) { return rows * 4 <= most ? 0 : rows * 2 <= most ? 1 : 2; }

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
