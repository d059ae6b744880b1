// Low-rank adapters of many requests beside a shared projection:
//   out[t] = base[t] + scale_a * (x[t] A_a^T) B_a^T,  a the row's adapter.
//
// Rows come grouped by adapter (order, offsets), so both products run on tiles
// of rows of one adapter, on mma.sync: the ranks are so small that the bytes of
// x, base and out (prompts) or A and B (decoding) bound the work, not the
// products. Two kernels, the second launched as a programmatic dependent:
//   first:  h = x A^T, fp32. A CTA takes a tile of rows x columns of A over a
//           part of K; its warps split that part, so that every byte of x and A is
//           loaded once per CTA, straight into operand registers (16 bytes per
//           lane: the order of k inside a product is free as long as both
//           operands share it), and meet in shared memory at the end. Parts of
//           K are kept apart and added in order by the second kernel: no atomics,
//           the same bits every time.
//   second: out = base + scale * h B^T. h enters as two 16-bit halves
//           (h = hi + lo, each rounded to nearest, after a power-of-two scale per
//           row that keeps fp16 in range), so what is lost is 2^-16 (bf16) or
//           2^-22 (fp16) of h, not 2^-8. Features are dealt to the product's
//           columns so that a lane ends with 8 neighbouring ones: base and out move
//           as 16-byte vectors.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "awqb200.h"
#include "awqb_common.h"
#include "awqb_ptx.cuh"
#include "awqb_vec.cuh"

namespace awqb {
namespace {

constexpr int kMaxAdapters = 1024;
constexpr int kMaxRank = 128;
constexpr int kMaxSlices = 4;
constexpr int kMaxParts = 8;      // parts of K
constexpr int kFirstWarps = 8;
constexpr int kSecondWarps = 4;
// Rows from which the 64-row tiles are taken: below, 16-row tiles keep more CTAs
// in flight and pad the few rows of a decode batch's adapters less.
constexpr int64_t kWideRows = 512;

struct Args {
  const void *x, *a, *b, *base;
  const int32_t *order, *offsets;
  const float* scales;
  void* out;
  float* h;  // [parts][M][R]
  int64_t ldx, ld_base, ld_out;
  int M, K, L, rank, R, N, S, parts, k_part;
  int slice_end[kMaxSlices];
};

struct Rows {
  int adapter, p0, n;  // -1: no adapter; first place, rows (0: no such tile)
};

// The rows of tile `tile` of kRows places: the groups are [0, offsets[0]) without an
// adapter, the adapters', and the rest without one. With adapters_only the first
// and last kind have no tiles. All threads of the CTA take part.
template <int kThreads, int kRows>
__device__ __forceinline__ Rows find_rows(const Args& g, int tile, bool adapters_only) {
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
    while (t >= tiles_of(e)) t -= tiles_of(e++);
    const int p0 = bound(e) + t * kRows;
    found.adapter = e == 0 || e == g.L + 1 ? -1 : e - 1;
    found.p0 = p0;
    found.n = min(kRows, bound(e + 1) - p0);
  }
  __syncthreads();
  return found;
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

// kM row tiles of 16, kN column tiles of 8.
template <typename T, int kM, int kN>
__global__ void __launch_bounds__(kFirstWarps * 32) lora_first_kernel(const __grid_constant__ Args g) {
  constexpr int kRows = kM * 16, kCols = kN * 8;
  extern __shared__ float4 meet4[];
  float* meet = reinterpret_cast<float*>(meet4);  // [kFirstWarps / 2][kM * kN * 4][32]
  grid_dep_wait();
  grid_dep_launch();
  const int col_tiles = (g.R + kCols - 1) / kCols;
  const int part = blockIdx.x % g.parts, ct = blockIdx.x / g.parts % col_tiles;
  const Rows r = find_rows<kFirstWarps * 32, kRows>(g, blockIdx.x / (g.parts * col_tiles), true);
  if (r.n <= 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, t = lane & 3;
  const T* x[kM][2];
#pragma unroll
  for (int m = 0; m < kM; ++m)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = m * 16 + i * 8 + gr;
      const int tok = row < r.n ? g.order[r.p0 + row] : -1;
      x[m][i] = tok >= 0 && tok < g.M ? static_cast<const T*>(g.x) + tok * g.ldx + t * 8 : nullptr;
    }
  const T* w = static_cast<const T*>(g.a) + ((int64_t)r.adapter * g.R + ct * kCols + gr) * g.K + t * 8;
  const int cols_left = g.R - ct * kCols;
  float d[kM][kN][4] = {};
  const int k_end = min(g.K, (part + 1) * g.k_part);
  const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll(kM == 1 ? 4 : 1)
  for (int k = part * g.k_part + warp * 32; k < k_end; k += kFirstWarps * 32) {
    const bool in = k + t * 8 < k_end;
    uint4 xa[kM][2], wb[kN];
#pragma unroll
    for (int n = 0; n < kN; ++n)
      wb[n] = in && n * 8 < cols_left ? __ldg(reinterpret_cast<const uint4*>(w + (int64_t)n * 8 * g.K + k)) : zero;
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        xa[m][i] = in && x[m][i] != nullptr ? __ldg(reinterpret_cast<const uint4*>(x[m][i] + k)) : zero;
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int n = 0; n < kN; ++n) mma32<T>(d[m][n], xa[m][0], xa[m][1], wb[n]);
  }
  // the warps' sums, halving the number of warps each time
#pragma unroll
  for (int half = kFirstWarps / 2; half > 0; half /= 2) {
    if (warp >= half && warp < 2 * half)
#pragma unroll
      for (int i = 0; i < kM * kN * 4; ++i)
        meet[((warp - half) * kM * kN * 4 + i) * 32 + lane] = d[i / (kN * 4)][i / 4 % kN][i % 4];
    __syncthreads();
    if (warp < half)
#pragma unroll
      for (int i = 0; i < kM * kN * 4; ++i) d[i / (kN * 4)][i / 4 % kN][i % 4] += meet[(warp * kM * kN * 4 + i) * 32 + lane];
    __syncthreads();
  }
  if (warp != 0) return;
  float* h = g.h + (int64_t)part * g.M * g.R + ct * kCols + t * 2;
#pragma unroll
  for (int m = 0; m < kM; ++m)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = m * 16 + i * 8 + gr;
      if (row >= r.n) continue;
#pragma unroll
      for (int n = 0; n < kN; ++n)
        if (n * 8 < cols_left)
          *reinterpret_cast<float2*>(h + (int64_t)(r.p0 + row) * g.R + n * 8) = make_float2(d[m][n][2 * i], d[m][n][2 * i + 1]);
    }
}

// The two 16-bit halves of a value.
template <typename T>
__device__ __forceinline__ void halves(float v, T* hi, T* lo) {
  *hi = (T)v;
  const float rest = v - (float)*hi;
  *lo = (T)(fabsf((float)*hi) < INFINITY ? rest : 0.f);
}

constexpr int kBlock = 32;  // features of a warp's step
constexpr int kHStride = kMaxRank + 32;  // halves per row of h in shared memory: 16-byte loads of 8 lanes hit all banks

template <typename T, int kM>
__global__ void __launch_bounds__(kSecondWarps * 32) lora_second_kernel(const __grid_constant__ Args g, int chunks, int chunk) {
  constexpr int kRows = kM * 16;
  __shared__ __align__(16) T hs[2][kRows][kHStride];
  __shared__ float row_scale[kRows];
  __shared__ int row_of[kRows];
  const bool in_place = g.out == g.base;
  const Rows r = find_rows<kSecondWarps * 32, kRows>(g, blockIdx.x / chunks, in_place);
  if (r.n <= 0) {
    grid_dep_wait();
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, t = lane & 3;
  // this CTA's features: chunk blockIdx.x % chunks of some slice
  int c = blockIdx.x % chunks, s = 0, s0 = 0;
  for (;; ++s) {
    const int here = (g.slice_end[s] - s0 + chunk - 1) / chunk;
    if (c < here) break;
    c -= here;
    s0 = g.slice_end[s];
  }
  const int f_begin = s0 + c * chunk, f_end = min(g.slice_end[s], f_begin + chunk);
  for (int i = threadIdx.x; i < kRows; i += kSecondWarps * 32) {
    const int tok = i < r.n ? g.order[r.p0 + i] : -1;
    row_of[i] = tok >= 0 && tok < g.M ? tok : -1;
  }
  const float scale = r.adapter >= 0 && g.scales ? g.scales[r.adapter] : 1.f;
  const int blocks32 = (g.rank + 31) / 32;
  grid_dep_wait();
  if (r.adapter >= 0) {
    for (int row = warp; row < kRows; row += kSecondWarps) {
      float v[kMaxRank / 32];
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < kMaxRank / 32; ++i) {
        const int j = i * 32 + lane;
        v[i] = 0.f;
        if (row < r.n && j < g.rank) {
          const float* src = g.h + (int64_t)(r.p0 + row) * g.R + s * g.rank + j;
          for (int q = 0; q < g.parts; ++q) v[i] += src[(int64_t)q * g.M * g.R];
        }
        top = fmaxf(top, fabsf(v[i]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // fp16: bring the row's largest value to 2^14 (exact: a power of two)
      const int e = std::is_same<T, __half>::value && top > 0.f && top < INFINITY ? min(max(ilogbf(top) - 14, -100), 100) : 0;
      const float down = ldexpf(1.f, -e);
#pragma unroll
      for (int i = 0; i < kMaxRank / 32; ++i)
        if (i < blocks32) halves<T>(v[i] * down, &hs[0][row][i * 32 + lane], &hs[1][row][i * 32 + lane]);
      if (lane == 0) row_scale[row] = scale * ldexpf(1.f, e);
    }
  }
  __syncthreads();
  // Columns of the four 8-column products of a block are dealt so that lane t of
  // a row ends with features 8t .. 8t + 7.
  const int col = (gr >> 1) * 8 + (gr & 1);
  const T* b = static_cast<const T*>(g.b) + (int64_t)(r.adapter >= 0 ? r.adapter : 0) * g.N * g.rank + t * 8;
  for (int f = f_begin + warp * kBlock; f < f_end; f += kSecondWarps * kBlock) {
    uint4 y[kM][2];
    const bool mine = f + t * 8 < f_end;
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int tok = row_of[m * 16 + i * 8 + gr];
        if (tok >= 0 && mine)
          y[m][i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(g.base) + tok * g.ld_base + f + t * 8);
      }
    float d[kM][4][4] = {};
    if (r.adapter >= 0) {
      for (int k = 0; k < blocks32; ++k) {
        uint4 wb[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int feat = f + col + 2 * n;
          wb[n] = feat < f_end && k * 32 + t * 8 < g.rank
                      ? __ldg(reinterpret_cast<const uint4*>(b + (int64_t)feat * g.rank + k * 32))
                      : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            const uint4 lo = *reinterpret_cast<const uint4*>(&hs[part][m * 16 + gr][k * 32 + t * 8]);
            const uint4 hi = *reinterpret_cast<const uint4*>(&hs[part][m * 16 + 8 + gr][k * 32 + t * 8]);
#pragma unroll
            for (int n = 0; n < 4; ++n) mma32<T>(d[m][n], lo, hi, wb[n]);
          }
      }
    }
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int tok = row_of[m * 16 + i * 8 + gr];
        if (tok < 0 || !mine) continue;
        uint4 o = y[m][i];
        if (r.adapter >= 0) {
          float v[8];
          unpack_vec<T>(o, v);
          const float w = row_scale[m * 16 + i * 8 + gr];
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            v[2 * n] += w * d[m][n][2 * i];
            v[2 * n + 1] += w * d[m][n][2 * i + 1];
          }
          o = pack_vec<T>(v);
        }
        *reinterpret_cast<uint4*>(static_cast<T*>(g.out) + tok * g.ld_out + f + t * 8) = o;
      }
  }
}

bool wide_tiles(int64_t M) { return M >= kWideRows; }

// Parts of K: enough CTAs for about two per SM, each part at least 64 k per warp.
int parts_of_k(int64_t M, int64_t K, int64_t R) {
  const int rows = wide_tiles(M) ? 64 : 16, cols = wide_tiles(M) ? 64 : 16;
  const int64_t tiles = (M + rows - 1) / rows * ((R + cols - 1) / cols);
  const int64_t want = 296 / std::max<int64_t>(tiles, 1), most = K / (kFirstWarps * 64);
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, (int64_t)kMaxParts}));
}

int64_t max_tiles(const Args& g, int rows) { return std::min<int64_t>(g.M, g.M / rows + g.L + 2); }

template <typename T, int kM, int kN>
int launch_tiles(const Args& g, cudaStream_t st) {
  const int cols = kN * 8, col_tiles = (g.R + cols - 1) / cols;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)(max_tiles(g, kM * 16) * col_tiles * g.parts));
  cfg.blockDim = dim3(kFirstWarps * 32);
  cfg.dynamicSmemBytes = kFirstWarps / 2 * kM * kN * 4 * 32 * 4;
  const auto first = lora_first_kernel<T, kM, kN>;
  if (cfg.dynamicSmemBytes > 32 * 1024)
    AWQB_CUDA(cudaFuncSetAttribute(first, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cfg.dynamicSmemBytes));
  AWQB_CUDA(cudaLaunchKernelEx(&cfg, first, g));
  // features per CTA: one block per warp for decode batches, four for prompts
  const int chunk = kSecondWarps * kBlock * (kM == 1 ? 1 : 4);
  int chunks = 0;
  for (int s = 0, s0 = 0; s < g.S; s0 = g.slice_end[s++]) chunks += (g.slice_end[s] - s0 + chunk - 1) / chunk;
  cfg.gridDim = dim3((unsigned)(max_tiles(g, kM * 16) * chunks));
  cfg.blockDim = dim3(kSecondWarps * 32);
  cfg.dynamicSmemBytes = 0;
  AWQB_CUDA(cudaLaunchKernelEx(&cfg, lora_second_kernel<T, kM>, g, chunks, chunk));
  return kOk;
}

template <typename T>
int launch(const Args& g, cudaStream_t st) {
  return wide_tiles(g.M) ? launch_tiles<T, 4, 8>(g, st) : launch_tiles<T, 1, 2>(g, st);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_sizes(int64_t M, int64_t K, int64_t L, int64_t rank, int64_t S) {
  AWQB_REQUIRE(M >= 0 && M < (1ll << 24), kInvalidArgument, "bad number of rows %lld", (long long)M);
  AWQB_REQUIRE(K > 0 && K % 8 == 0 && K <= (1 << 20), kInvalidArgument, "K=%lld must be a positive multiple of 8",
               (long long)K);
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

extern "C" int awqb_lora_workspace_bytes(int64_t M, int64_t K, int64_t L, int64_t rank, int64_t num_slices,
                                         int64_t* bytes) {
  AWQB_REQUIRE(bytes != nullptr, kInvalidArgument, "bytes is null");
  const int st = check_sizes(M, K, L, rank, num_slices);
  if (st != kOk) return st;
  *bytes = M * rank * num_slices * 4 * parts_of_k(M, K, rank * num_slices);
  return kOk;
}

extern "C" int awqb_lora(const void* x, int64_t M, int64_t ldx, int64_t K, const void* a, const void* b, int64_t L,
                         int64_t rank, int64_t N, const int64_t* slices, int64_t num_slices, const int32_t* order,
                         const int32_t* offsets, const float* scales, const void* base, int64_t ld_base, void* out,
                         int64_t ld_out, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  AWQB_REQUIRE(dtype == AWQB_DTYPE_F16 || dtype == AWQB_DTYPE_BF16, kInvalidArgument, "bad dtype %d", dtype);
  int64_t need = 0;
  const int st = awqb_lora_workspace_bytes(M, K, L, rank, num_slices, &need);
  if (st != kOk) return st;
  AWQB_REQUIRE(N > 0 && N % 8 == 0 && N <= (1 << 20), kInvalidArgument, "N=%lld must be a positive multiple of 8",
               (long long)N);
  AWQB_REQUIRE(slices != nullptr || num_slices == 1, kInvalidArgument, "the slices' widths are missing");
  Args g = {};
  int64_t end = 0;
  for (int s = 0; s < num_slices; ++s) {
    const int64_t w = slices ? slices[s] : N;
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
  AWQB_REQUIRE(aligned16(x) && aligned16(a) && aligned16(b) && aligned16(base) && aligned16(out) &&
                   aligned16(workspace),
               kInvalidArgument, "tensors must be 16-byte aligned");
  AWQB_REQUIRE(workspace != nullptr && workspace_bytes >= need, kInvalidArgument,
               "workspace too small: %lld < %lld bytes", (long long)workspace_bytes, (long long)need);
  g.x = x, g.a = a, g.b = b, g.base = base, g.order = order, g.offsets = offsets, g.scales = scales, g.out = out;
  g.h = static_cast<float*>(workspace);
  g.ldx = ldx, g.ld_base = ld_base, g.ld_out = ld_out;
  g.M = (int)M, g.K = (int)K, g.L = (int)L, g.rank = (int)rank, g.R = (int)(rank * num_slices), g.N = (int)N;
  g.S = (int)num_slices;
  g.parts = parts_of_k(M, K, g.R);
  g.k_part = (int)((K + g.parts - 1) / g.parts + 31) / 32 * 32;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  return dtype == AWQB_DTYPE_F16 ? launch<__half>(g, cs) : launch<__nv_bfloat16>(g, cs);
}
