// Matrix products grouped by expert over 16-bit weights [E][N][K], with ragged
// group sizes that only the device knows: y[r] = x[r] w[e]^T for the rows of
// expert e, optionally silu(gate) * up over the two halves of w's rows.
#include <cuda_runtime.h>

#include "awqb200.h"
#include "awqb_common.h"
#include "awqb_vec.cuh"

namespace awqb {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kTile = 64, kStep = 32;

struct Args {
  const void *x, *w;
  const int32_t *offsets, *row_map;
  const float* row_scale;
  void* out;
  int64_t ldx, ldo, out_rows;
  int rows, E, K, N, silu;
};

// A 64 x 64 tile per CTA of 256 threads (4 x 4 values each), fp32.
template <typename T>
__global__ void __launch_bounds__(256) grouped_gemm_kernel(const Args a) {
  __shared__ float xs[kStep][kTile + 1], ws[2][kStep][kTile + 1];
  __shared__ int where[3];
  if (threadIdx.x == 0) {
    int tile = blockIdx.x, e = 0, r0 = 0, r1 = 0, prev = min(max(a.offsets[0], 0), a.rows);
    for (; e < a.E; ++e) {
      r0 = prev;
      r1 = prev = max(r0, min(a.offsets[e + 1], a.rows));
      const int tiles = (r1 - r0 + kTile - 1) / kTile;
      if (tile < tiles) break;
      tile -= tiles;
    }
    where[0] = e, where[1] = r0 + tile * kTile, where[2] = r1;
  }
  __syncthreads();
  const int e = where[0], m0 = where[1], m1 = where[2];
  if (e >= a.E) return;
  const int n_out = a.silu ? a.N / 2 : a.N, n0 = blockIdx.y * kTile;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const T* w = static_cast<const T*>(a.w) + (int64_t)e * a.N * a.K;
  float acc[2][4][4] = {};
  for (int k0 = 0; k0 < a.K; k0 += kStep) {
    for (int i = threadIdx.x; i < kTile * kStep; i += 256) {
      const int r = i / kStep, k = i % kStep, kk = k0 + k;
      xs[k][r] = m0 + r < m1 && kk < a.K ? (float)static_cast<const T*>(a.x)[(m0 + r) * a.ldx + kk] : 0.f;
      const bool in = n0 + r < n_out && kk < a.K;
      ws[0][k][r] = in ? (float)w[(int64_t)(n0 + r) * a.K + kk] : 0.f;
      if (a.silu) ws[1][k][r] = in ? (float)w[(int64_t)(n_out + n0 + r) * a.K + kk] : 0.f;
    }
    __syncthreads();
    for (int k = 0; k < kStep; ++k)
      for (int half = 0; half < 1 + a.silu; ++half)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = xs[k][ty * 4 + i] * ws[half][k][tx * 4 + j];
            if (half) acc[1][i][j] += p; else acc[0][i][j] += p;
          }
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int r = m0 + ty * 4 + i;
    if (r >= m1) break;
    const int64_t to = a.row_map ? a.row_map[r] : r;
    if (to < 0 || to >= a.out_rows) continue;
    const float scale = a.row_scale ? a.row_scale[to] : 1.f;
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx * 4 + j;
      float y = acc[0][i][j];
      if (a.silu) y = y / (1.f + expf(-y)) * acc[1][i][j];
      if (n < n_out) static_cast<T*>(a.out)[to * a.ldo + n] = (T)(y * scale);
    }
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace
}  // namespace awqb

using namespace awqb;

extern "C" int awqb_grouped_gemm(const void* x, int64_t rows, int64_t ldx, const void* w, int64_t E, int64_t K,
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
  Args a = {x, w, offsets, row_map, row_scale, out, ldx, ldo, out_rows, (int)rows, (int)E, (int)K, (int)N, silu_mul != 0};
  const dim3 grid((unsigned)(rows / kTile + E), (unsigned)((n_out + kTile - 1) / kTile));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == AWQB_DTYPE_F16)
    grouped_gemm_kernel<__half><<<grid, 256, 0, st>>>(a);
  else
    grouped_gemm_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
  AWQB_LAUNCH_CHECK();
  return kOk;
}
