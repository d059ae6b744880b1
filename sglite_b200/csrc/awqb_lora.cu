// Low-rank adapters of many requests beside a shared projection:
//   out[t] = base[t] + scale_a * (x[t] A_a^T) B_a^T,  a the row's adapter.
//
// Rows come grouped by adapter (order, offsets), so both products run on tiles
// of rows of one adapter: the ranks are so small that the bytes of x, base and out
// (prompts) or A and B (decoding) bound the work, not the products. Decode batches
// take the two kernels of this file, on mma.sync, the second launched as a
// programmatic dependent; prompts those of awqb_lora_wide.cuh.
//   first:  h = x A^T, fp32. A CTA takes a tile of rows x columns of A over a
//           part of K; its warps split that part, so that every byte of x and A is
//           loaded once per CTA, straight into operand registers (16 bytes per
//           lane: the order of k inside a product is free as long as both
//           operands share it), and meet in shared memory at the end. Parts of
//           K are kept apart and added in order by the second kernel: no atomics,
//           the same bits every time.
//   second: out = base + scale * h B^T. h enters as two 16-bit halves
//           (h = hi + lo, each rounded to nearest), so what is lost is 2^-16 of each
//           value for bf16, not 2^-8. fp16 gets a power-of-two scale per row and slice
//           that brings the largest value to 2^14 .. 2^15: 2^-22 of each value is lost,
//           or 2^-39 of the largest where that is more (values under 2^-17 of it). A
//           third half would be half as many products again for bits that the result's
//           own rounding drops. Features are dealt to the product's
//           columns so that a lane ends with 8 neighbouring ones: base and out move
//           as 16-byte vectors.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "awqb200.h"
#include "awqb_common.h"
#include "awqb_ptx.cuh"
#include "awqb_tma.h"
#include "awqb_vec.cuh"

namespace awqb {
namespace {

constexpr int kMaxAdapters = 1024;
constexpr int kMaxRank = 128;
constexpr int kMaxSlices = 4;
constexpr int kMaxParts = 8;      // parts of K
constexpr int kFirstWarps = 8;
constexpr int kSecondWarps = 4;
// The prompt kernels cost about 14 us more at the start (three launches, tcgen05
// tiles of 128 rows) and then move base and out at HBM speed; the decode kernels
// cost about 2.4e-8 us per unit of M * (N * (50 + rank) + K * columns). Measured,
// decode / prompt in us at K = 4096, N = 28672, rank 16: M = 256 23 / 27, 512 39 / 30,
// 2048 137 / 65; K = 14336, N = 4096, rank 64: 512 25 / 25, 1024 37 / 27; K = N = 4096,
// rank 16: 512 11 / 22, 2048 26 / 28.
constexpr double kPromptWork = 8e8;

struct Args {
  const void *x, *a, *b, *base;
  const int32_t *order, *offsets;
  const float* scales;
  void* out;
  float* h;      // [parts][M][R]
  void* halves;  // prompts: [slices][2][M][rank], see the join kernel
  float* up;     // prompts: [slices][M]
  uint32_t* err;
  int64_t ldx, ld_base, ld_out;
  int M, K, L, rank, R, N, S, parts, k_part;
  int slice_end[kMaxSlices];
};

struct Rows {
  int adapter, p0, n;  // -1: no adapter; first place, rows (0: no such tile)
};

// The rows of tile `tile` of kRows places: the groups are [0, offsets[0]) without an
// adapter, the adapters', and the rest without one. With adapters_only the first
// and last kind have no tiles. *total gets the number of tiles, if asked for. All
// threads of the CTA take part.
template <int kThreads, int kRows>
__device__ __forceinline__ Rows find_rows(const Args& g, int tile, bool adapters_only, int* total) {
  __shared__ int warp_tot[kThreads / 32];
  __shared__ Rows found;
  const int groups = g.L + 2;
  const int per = (groups + kThreads - 1) / kThreads;
  const int e0 = threadIdx.x * per, e1 = min(groups, e0 + per);
  const auto bound = [&](int e) {  // first place of group e
    return e <= 0 ? 0 : e > g.L + 1 ? g.M : min(max(g.offsets[e - 1], 0), g.M);
  };
  const auto tiles_of = [&](int e) {
    const bool none = e == 0 || e == g.L + 1;
    return none && adapters_only ? 0 : (max(bound(e + 1) - bound(e), 0) + kRows - 1) / kRows;
  };
  int sum = 0;
  for (int e = e0; e < e1; ++e) sum += tiles_of(e);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) warp_tot[warp] = incl;
  if (threadIdx.x == 0) found.n = 0;
  __syncthreads();
  int before = incl - sum;
  for (int w = 0; w < warp; ++w) before += warp_tot[w];
  if (tile >= before && tile < before + sum) {
    int t = tile - before, e = e0;
    while (e + 1 < e1 && t >= tiles_of(e)) t -= tiles_of(e++);
    const int p0 = bound(e) + t * kRows;
    found.adapter = e == 0 || e == g.L + 1 ? -1 : e - 1;
    found.p0 = p0;
    found.n = min(kRows, bound(e + 1) - p0);
  }
  if (total != nullptr) {
    *total = 0;
    for (int w = 0; w < kThreads / 32; ++w) *total += warp_tot[w];
  }
  __syncthreads();
  const Rows r = found;
  __syncthreads();  // found may be written again
  return r;
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if (std::is_same<T, __half>::value)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 32 k of both operands, 8 per lane: two products of 16 k.
template <typename T>
__device__ __forceinline__ void mma32(float (&d)[4], const uint4& lo_row, const uint4& hi_row, const uint4& b) {
  mma16816<T>(d, lo_row.x, hi_row.x, lo_row.y, hi_row.y, b.x, b.y);
  mma16816<T>(d, lo_row.z, hi_row.z, lo_row.w, hi_row.w, b.z, b.w);
}

// Decode batches: 16 rows x 16 columns of A.
template <typename T>
__global__ void __launch_bounds__(kFirstWarps * 32) lora_first_kernel(const __grid_constant__ Args g) {
  constexpr int kRows = 16, kN = 2, kCols = kN * 8;
  __shared__ float meet[kFirstWarps / 2 * kN * 4 * 32];
  grid_dep_wait();
  grid_dep_launch();
  const int col_tiles = (g.R + kCols - 1) / kCols;
  const int part = blockIdx.x % g.parts, ct = blockIdx.x / g.parts % col_tiles;
  const Rows r = find_rows<kFirstWarps * 32, kRows>(g, blockIdx.x / (g.parts * col_tiles), true, nullptr);
  if (r.n <= 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, t = lane & 3;
  const T* x[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = i * 8 + gr;
    const int tok = row < r.n ? g.order[r.p0 + row] : -1;
    x[i] = tok >= 0 && tok < g.M ? static_cast<const T*>(g.x) + tok * g.ldx + t * 8 : nullptr;
  }
  const T* w = static_cast<const T*>(g.a) + ((int64_t)r.adapter * g.R + ct * kCols + gr) * g.K + t * 8;
  const int cols_left = g.R - ct * kCols;
  float d[kN][4] = {};
  const int k_end = min(g.K, (part + 1) * g.k_part);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  constexpr int kAhead = 4;  // steps whose loads are in flight together
  for (int k0 = part * g.k_part + warp * 32; k0 < k_end; k0 += kAhead * kFirstWarps * 32) {
    uint4 xa[kAhead][2], wb[kAhead][kN];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int k = k0 + j * kFirstWarps * 32;
      const bool in = k + t * 8 < k_end;
#pragma unroll
      for (int n = 0; n < kN; ++n)
        wb[j][n] = in && n * 8 < cols_left ? __ldg(reinterpret_cast<const uint4*>(w + (int64_t)n * 8 * g.K + k)) : zero;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        xa[j][i] = in && x[i] != nullptr ? __ldg(reinterpret_cast<const uint4*>(x[i] + k)) : zero;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
#pragma unroll
      for (int n = 0; n < kN; ++n) mma32<T>(d[n], xa[j][0], xa[j][1], wb[j][n]);
  }
  // the warps' sums, halving the number of warps each time
#pragma unroll
  for (int half = kFirstWarps / 2; half > 0; half /= 2) {
    if (warp >= half && warp < 2 * half)
#pragma unroll
      for (int i = 0; i < kN * 4; ++i) meet[((warp - half) * kN * 4 + i) * 32 + lane] = d[i / 4][i % 4];
    __syncthreads();
    if (warp < half)
#pragma unroll
      for (int i = 0; i < kN * 4; ++i) d[i / 4][i % 4] += meet[(warp * kN * 4 + i) * 32 + lane];
    __syncthreads();
  }
  if (warp != 0) return;
  float* h = g.h + (int64_t)part * g.M * g.R + ct * kCols + t * 2;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = i * 8 + gr;
    if (row >= r.n) continue;
#pragma unroll
    for (int n = 0; n < kN; ++n)
      if (n * 8 < cols_left)
        *reinterpret_cast<float2*>(h + (int64_t)(r.p0 + row) * g.R + n * 8) = make_float2(d[n][2 * i], d[n][2 * i + 1]);
  }
}

// The two 16-bit halves of a value.
template <typename T>
__device__ __forceinline__ void halves(float v, T* hi, T* lo) {
  *hi = (T)v;
  const float rest = v - (float)*hi;
  *lo = (T)(fabsf((float)*hi) < INFINITY ? rest : 0.f);
}

// The power of two that a row of h is divided by before it is split: fp16 gets the
// row's largest value to 2^14 .. 2^15 (exact), bf16 has fp32's range. Whole warps.
template <typename T>
__device__ __forceinline__ int row_exponent(float top) {
  if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    return top > 0.f && top < INFINITY ? min(max(ilogbf(top) - 14, -100), 100) : 0;
  } else {
    return 0;
  }
}

constexpr int kBlock = 32;                      // features of a warp
constexpr int kChunk = kSecondWarps * kBlock;   // features of a CTA

// The chunk of features that CTA c of a tile takes: chunks of `chunk` features,
// slice after slice, none of them over two slices.
struct Feats {
  int slice, begin, end;
};
__device__ __forceinline__ Feats find_feats(const Args& g, int c, int chunk) {
  int s = 0, s0 = 0;
  for (;; ++s) {
    const int here = (g.slice_end[s] - s0 + chunk - 1) / chunk;
    if (c < here) break;
    c -= here;
    s0 = g.slice_end[s];
  }
  return {s, s0 + c * chunk, min(g.slice_end[s], s0 + (c + 1) * chunk)};
}

// Decode batches: 16 rows, 32 features per warp. kRank32: the rank in blocks of 32.
template <typename T, int kRank32>
__global__ void __launch_bounds__(kSecondWarps * 32) lora_second_kernel(const __grid_constant__ Args g, int chunks) {
  constexpr int kRows = 16;
  // 64 bytes past a multiple of 128: the 16-byte loads of 8 lanes hit all banks
  constexpr int kHStride = (kRank32 + 1) / 2 * 64 + 32;
  __shared__ __align__(16) T hs[2][kRows][kHStride];
  __shared__ float row_scale[kRows];
  const Rows r = find_rows<kSecondWarps * 32, kRows>(g, blockIdx.x / chunks, g.out == g.base, nullptr);
  if (r.n <= 0) {
    grid_dep_wait();
    return;
  }
  const bool adapted = r.adapter >= 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, t = lane & 3;
  const Feats feats = find_feats(g, blockIdx.x % chunks, kChunk);
  const int f = feats.begin + warp * kBlock;
  // What the first kernel does not write is loaded before it has ended: it let
  // this kernel start only after everything in front of it was complete.
  uint4 y[2], wb[kRank32][4];
  int tok[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    tok[i] = i * 8 + gr < r.n && f + t * 8 < feats.end ? g.order[r.p0 + i * 8 + gr] : -1;
    if (tok[i] >= g.M) tok[i] = -1;
    if (tok[i] >= 0)
      y[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(g.base) + tok[i] * g.ld_base + f + t * 8);
  }
  // Columns of the four 8-column products are dealt so that lane t of a row ends
  // with features 8t .. 8t + 7.
  const int col = (gr >> 1) * 8 + (gr & 1);
#pragma unroll
  for (int k = 0; k < kRank32; ++k)
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int feat = f + col + 2 * n;
      wb[k][n] = adapted && feat < feats.end && k * 32 + t * 8 < g.rank
                     ? __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(g.b) +
                                                            ((int64_t)r.adapter * g.N + feat) * g.rank + k * 32 + t * 8))
                     : make_uint4(0, 0, 0, 0);
    }
  const float scale = adapted && g.scales ? g.scales[r.adapter] : 1.f;
  grid_dep_wait();
  if (adapted) {
    for (int row = warp; row < r.n; row += kSecondWarps) {
      const float* src = g.h + (int64_t)(r.p0 + row) * g.R + feats.slice * g.rank + lane;
      float u[kMaxParts][kRank32], v[kRank32] = {}, top = 0.f;
#pragma unroll
      for (int part = 0; part < kMaxParts; ++part)
#pragma unroll
        for (int i = 0; i < kRank32; ++i)
          u[part][i] = part < g.parts && i * 32 + lane < g.rank ? src[(int64_t)part * g.M * g.R + i * 32] : 0.f;
#pragma unroll
      for (int i = 0; i < kRank32; ++i) {
#pragma unroll
        for (int part = 0; part < kMaxParts; ++part) v[i] += u[part][i];
        top = fmaxf(top, fabsf(v[i]));
      }
      const int e = row_exponent<T>(top);
      const float down = ldexpf(1.f, -e);
#pragma unroll
      for (int i = 0; i < kRank32; ++i)
        halves<T>(v[i] * down, &hs[0][row][i * 32 + lane], &hs[1][row][i * 32 + lane]);
      if (lane == 0) row_scale[row] = scale * ldexpf(1.f, e);
    }
  }
  __syncthreads();
  float d[4][4] = {};
  if (adapted) {
#pragma unroll
    for (int k = 0; k < kRank32; ++k)
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        const uint4 lo = *reinterpret_cast<const uint4*>(&hs[part][gr][k * 32 + t * 8]);
        const uint4 hi = *reinterpret_cast<const uint4*>(&hs[part][8 + gr][k * 32 + t * 8]);
#pragma unroll
        for (int n = 0; n < 4; ++n) mma32<T>(d[n], lo, hi, wb[k][n]);
      }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (tok[i] < 0) continue;
    uint4 o = y[i];
    if (adapted) {
      float v[8];
      unpack_vec<T>(o, v);
      const float w = row_scale[i * 8 + gr];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        v[2 * n] += w * d[n][2 * i];
        v[2 * n + 1] += w * d[n][2 * i + 1];
      }
      o = pack_vec<T>(v);
    }
    *reinterpret_cast<uint4*>(static_cast<T*>(g.out) + tok[i] * g.ld_out + f + t * 8) = o;
  }
}

}  // namespace
}  // namespace awqb

#include "awqb_lora_wide.cuh"

namespace awqb {
namespace {

struct Sizes {
  int64_t M, K, N, L, rank, S, R;
};

bool for_prompt(const Sizes& z) {
  return (double)z.M * ((double)z.N * (50 + z.rank) + (double)z.K * z.R) > kPromptWork;
}

// Parts of K: enough CTAs to fill the GPU, each part long enough to be worth its
// sums (64 k per warp of a decode batch's CTA, eight stages of a prompt's).
int parts_of_k(const Sizes& z) {
  const bool wide = for_prompt(z);
  // a decode batch may have a tile for every adapter, a prompt has few partial ones
  const int64_t rows = wide ? (z.M + kWideRows - 1) / kWideRows : std::min(z.M, z.M / 16 + z.L);
  const int64_t tiles = rows * (wide ? (z.R + 127) / 128 : (z.R + 15) / 16);
  const int64_t want = 296 / std::max<int64_t>(tiles, 1), most = z.K / 512;
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, (int64_t)kMaxParts}));
}

// The workspace: parts of h, then for prompts the halves and their powers of two.
struct Layout {
  int64_t halves, up, bytes;
};
Layout layout(const Sizes& z) {
  const auto round = [](int64_t v) { return (v + 255) / 256 * 256; };
  const bool wide = for_prompt(z);
  Layout l = {};
  l.halves = round(z.M * z.R * 4 * parts_of_k(z));
  l.up = l.halves + (wide ? round(z.M * z.R * 4) : 0);
  l.bytes = l.up + (wide ? round(z.M * z.S * 4) : 0);
  return l;
}

int64_t max_tiles(const Args& g, int rows) { return std::min<int64_t>(g.M, g.M / rows + g.L + 2); }

// Chunks of `chunk` features over all slices.
int64_t count_chunks(const Args& g, int64_t chunk) {
  int64_t chunks = 0;
  for (int s = 0, s0 = 0; s < g.S; s0 = g.slice_end[s++]) chunks += (g.slice_end[s] - s0 + chunk - 1) / chunk;
  return chunks;
}

template <typename T>
int launch_decode(const Args& g, cudaLaunchConfig_t cfg) {
  cfg.gridDim = dim3((unsigned)(max_tiles(g, 16) * ((g.R + 15) / 16) * g.parts));
  cfg.blockDim = dim3(kFirstWarps * 32);
  AWQB_CUDA(cudaLaunchKernelEx(&cfg, lora_first_kernel<T>, g));
  const int64_t chunks = count_chunks(g, kChunk);
  cfg.gridDim = dim3((unsigned)(max_tiles(g, 16) * chunks));
  cfg.blockDim = dim3(kSecondWarps * 32);
  const auto second = g.rank <= 32   ? lora_second_kernel<T, 1>
                      : g.rank <= 64 ? lora_second_kernel<T, 2>
                                     : lora_second_kernel<T, 4>;
  AWQB_CUDA(cudaLaunchKernelEx(&cfg, second, g, (int)chunks));
  return kOk;
}

template <typename T>
int launch_prompt(const Args& g, cudaLaunchConfig_t cfg) {
  const int col_box = std::min(128, g.R), atoms = (g.rank + 63) / 64;
  CUtensorMap tx, ta, tb, th;
  int st = make_rows_map(&tx, g.x, g.M, g.K, g.ldx, kWideRows);
  if (st == kOk) st = make_rows_map(&ta, g.a, (int64_t)g.L * g.R, g.K, g.K, col_box);
  if (st == kOk) st = make_rows_map(&tb, g.b, (int64_t)g.L * g.N, g.rank, g.rank, kWideFeat);
  if (st == kOk) st = make_rows_map(&th, g.halves, (int64_t)g.S * 2 * g.M, g.rank, g.rank, kWideRows);
  if (st != kOk) return st;
  cfg.gridDim = dim3((unsigned)(max_tiles(g, kWideRows) * ((g.R + 127) / 128) * g.parts));
  cfg.blockDim = dim3(kFirstWideThreads);
  cfg.dynamicSmemBytes = first_wide_smem();
  AWQB_CUDA(cudaFuncSetAttribute(lora_first_wide_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, first_wide_smem()));
  AWQB_CUDA(cudaLaunchKernelEx(&cfg, lora_first_wide_kernel<T>, tx, ta, g, col_box));
  cfg.gridDim = dim3((unsigned)(((int64_t)g.M * g.S + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  AWQB_CUDA(cudaLaunchKernelEx(&cfg, lora_join_kernel<T>, g));
  const int64_t blocks_per_tile = count_chunks(g, kWideFeat);
  cfg.gridDim = dim3((unsigned)std::min<int64_t>(max_tiles(g, kWideRows) * blocks_per_tile, device_sm_count()));
  cfg.blockDim = dim3(kSecondWideThreads);
  cfg.dynamicSmemBytes = second_wide_smem(atoms);
  AWQB_CUDA(cudaFuncSetAttribute(lora_second_wide_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 std::max(second_wide_smem(1), second_wide_smem(2))));
  AWQB_CUDA(cudaLaunchKernelEx(&cfg, lora_second_wide_kernel<T>, tb, th, g, (int)blocks_per_tile, atoms));
  return kOk;
}

template <typename T>
int launch(const Args& g, bool prompt, cudaStream_t st) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return prompt ? launch_prompt<T>(g, cfg) : launch_decode<T>(g, cfg);
}

int check_sizes(int64_t M, int64_t K, int64_t N, int64_t L, int64_t rank, int64_t S) {
  AWQB_REQUIRE(M >= 0 && M < (1ll << 24), kInvalidArgument, "bad number of rows %lld", (long long)M);
  AWQB_REQUIRE(K > 0 && K % 8 == 0 && K <= (1 << 20), kInvalidArgument, "K=%lld must be a positive multiple of 8",
               (long long)K);
  AWQB_REQUIRE(N > 0 && N % 8 == 0 && N <= (1 << 20), kInvalidArgument, "N=%lld must be a positive multiple of 8",
               (long long)N);
  AWQB_REQUIRE(L >= 1 && L <= kMaxAdapters, kInvalidArgument, "%lld adapters: 1..%d are supported", (long long)L,
               kMaxAdapters);
  AWQB_REQUIRE(rank >= 8 && rank % 8 == 0 && rank <= kMaxRank, kInvalidArgument,
               "rank %lld must be a multiple of 8, at most %d", (long long)rank, kMaxRank);
  AWQB_REQUIRE(S >= 1 && S <= kMaxSlices, kInvalidArgument, "%lld slices: 1..%d are supported", (long long)S,
               kMaxSlices);
  return kOk;
}

}  // namespace
}  // namespace awqb

using namespace awqb;

extern "C" int awqb_lora_workspace_bytes(int64_t M, int64_t K, int64_t N, int64_t L, int64_t rank, int64_t num_slices,
                                         int64_t* bytes) {
  AWQB_REQUIRE(bytes != nullptr, kInvalidArgument, "bytes is null");
  const int st = check_sizes(M, K, N, L, rank, num_slices);
  if (st != kOk) return st;
  *bytes = layout({M, K, N, L, rank, num_slices, rank * num_slices}).bytes;
  return kOk;
}

extern "C" int awqb_lora(const awqb_lora_args* args, void* stream) {
  AWQB_REQUIRE(args != nullptr, kInvalidArgument, "args is null");
  const auto [x, M, ldx, K, a, b, L, rank, N, num_slices, slices, order, offsets, scales, base, ld_base, out, ld_out,
              dtype, workspace, workspace_bytes] = *args;
  AWQB_REQUIRE(dtype == AWQB_DTYPE_F16 || dtype == AWQB_DTYPE_BF16, kInvalidArgument, "bad dtype %d", dtype);
  int64_t need = 0;
  const int st = awqb_lora_workspace_bytes(M, K, N, L, rank, num_slices, &need);
  if (st != kOk) return st;
  Args g = {};
  int64_t end = 0;
  for (int s = 0; s < num_slices; ++s) {
    const int64_t w = slices[s];
    AWQB_REQUIRE(w > 0 && w % 8 == 0 && w <= N, kInvalidArgument, "slice width %lld must be a positive multiple of 8",
                 (long long)w);
    end += w;
    g.slice_end[s] = (int)end;
  }
  AWQB_REQUIRE(end == N, kInvalidArgument, "the slices' widths add up to %lld, not N=%lld", (long long)end,
               (long long)N);
  AWQB_REQUIRE(ldx >= K && ld_base >= N && ld_out >= N && ldx % 8 == 0 && ld_base % 8 == 0 && ld_out % 8 == 0,
               kInvalidArgument, "row strides must be at least the row's length and multiples of 8");
  if (M == 0) return kOk;
  AWQB_REQUIRE(x && a && b && order && offsets && base && out, kInvalidArgument, "null pointer");
  AWQB_REQUIRE(out != base || ld_out == ld_base, kInvalidArgument,
               "out is base with another row stride: in place, the strides must agree");
  AWQB_REQUIRE(aligned16(x) && aligned16(a) && aligned16(b) && aligned16(base) && aligned16(out) &&
                   aligned16(workspace),
               kInvalidArgument, "tensors must be 16-byte aligned");
  AWQB_REQUIRE(workspace != nullptr && workspace_bytes >= need, kInvalidArgument,
               "workspace too small: %lld < %lld bytes", (long long)workspace_bytes, (long long)need);
  g.err = device_error_word();
  AWQB_REQUIRE(g.err != nullptr, kCudaError, "cannot resolve the device error word");
  g.x = x, g.a = a, g.b = b, g.base = base, g.order = order, g.offsets = offsets, g.scales = scales, g.out = out;
  g.h = static_cast<float*>(workspace);
  g.ldx = ldx, g.ld_base = ld_base, g.ld_out = ld_out;
  g.M = (int)M, g.K = (int)K, g.L = (int)L, g.rank = (int)rank, g.R = (int)(rank * num_slices), g.N = (int)N;
  g.S = (int)num_slices;
  const Sizes z = {M, K, N, L, rank, num_slices, g.R};
  g.parts = parts_of_k(z);
  g.k_part = (int)((K + g.parts - 1) / g.parts + 63) / 64 * 64;
  const Layout at = layout(z);
  g.halves = static_cast<uint8_t*>(workspace) + at.halves;
  g.up = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + at.up);
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  return dtype == AWQB_DTYPE_F16 ? launch<__half>(g, for_prompt(z), cs) : launch<__nv_bfloat16>(g, for_prompt(z), cs);
}
