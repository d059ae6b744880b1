// Low-rank adapters of many requests beside a shared projection:
//   out[t] = base[t] + scale_a * (x[t] A_a^T) B_a^T,  a the row's adapter.
// Two kernels: the first factor's products h (fp32, one row per place in the
// grouped order), then the second factor's, added to the projection's output.
#include <cuda_runtime.h>

#include "awqb200.h"
#include "awqb_common.h"
#include "awqb_vec.cuh"

namespace awqb {
namespace {

constexpr int kMaxAdapters = 1024;
constexpr int kMaxRank = 128;
constexpr int kMaxSlices = 4;

struct Args {
  const void *x, *a, *b, *base;
  const int32_t *order, *offsets;
  const float* scales;
  void* out;
  float* h;
  int64_t ldx, ld_base, ld_out;
  int M, K, L, rank, R, N, S;
  int slice_end[kMaxSlices];
};

// The adapter of place p (the last group whose first place is <= p), or -1.
__device__ __forceinline__ int adapter_of(const int32_t* __restrict__ offsets, int L, int p) {
  if (p < offsets[0] || p >= offsets[L]) return -1;
  int lo = 0, hi = L;  // offsets[lo] <= p < offsets[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (offsets[mid] <= p) lo = mid; else hi = mid;
  }
  return lo;
}

// One warp per (place, row of A).
template <typename T>
__global__ void __launch_bounds__(256) lora_first_kernel(const Args a) {
  const int p = blockIdx.x;
  const int ad = adapter_of(a.offsets, a.L, p);
  if (ad < 0) return;
  const int t = a.order[p];
  if (t < 0 || t >= a.M) return;
  const int lane = threadIdx.x & 31;
  const T* x = static_cast<const T*>(a.x) + t * a.ldx;
  for (int j = threadIdx.x >> 5; j < a.R; j += 8) {
    const T* w = static_cast<const T*>(a.a) + ((int64_t)ad * a.R + j) * a.K;
    float s = 0.f;
    for (int k = lane * 8; k < a.K; k += 256) {
      float u[8], v[8];
      unpack_vec<T>(*reinterpret_cast<const uint4*>(x + k), u);
      unpack_vec<T>(*reinterpret_cast<const uint4*>(w + k), v);
#pragma unroll
      for (int i = 0; i < 8; ++i) s += u[i] * v[i];
    }
    s = warp_sum(s);
    if (lane == 0) a.h[(int64_t)p * a.R + j] = s;
  }
}

// One thread per eight output features of a place.
template <typename T>
__global__ void __launch_bounds__(256) lora_second_kernel(const Args a) {
  const int p = blockIdx.x;
  const int t = a.order[p];
  if (t < 0 || t >= a.M) return;
  const int ad = adapter_of(a.offsets, a.L, p);
  const T* base = static_cast<const T*>(a.base) + t * a.ld_base;
  T* out = static_cast<T*>(a.out) + t * a.ld_out;
  const float scale = ad >= 0 && a.scales ? a.scales[ad] : 1.f;
  for (int n = (blockIdx.y * 256 + threadIdx.x) * 8; n < a.N; n += gridDim.y * 256 * 8) {
    float y[8];
    unpack_vec<T>(*reinterpret_cast<const uint4*>(base + n), y);
    if (ad >= 0) {
      int s = 0;
      while (n >= a.slice_end[s]) ++s;
      const float* h = a.h + (int64_t)p * a.R + s * a.rank;
      for (int i = 0; i < 8; ++i) {
        const T* w = static_cast<const T*>(a.b) + ((int64_t)ad * a.N + n + i) * a.rank;
        float d = 0.f;
        for (int j = 0; j < a.rank; ++j) d += h[j] * (float)w[j];
        y[i] += scale * d;
      }
    }
    *reinterpret_cast<uint4*>(out + n) = pack_vec<T>(y);
  }
}

template <typename T>
int launch(const Args& a, cudaStream_t st) {
  lora_first_kernel<T><<<a.M, 256, 0, st>>>(a);
  lora_second_kernel<T><<<dim3(a.M, (a.N + 2047) / 2048), 256, 0, st>>>(a);
  AWQB_LAUNCH_CHECK();
  return kOk;
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
  *bytes = M * rank * num_slices * 4;
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
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  return dtype == AWQB_DTYPE_F16 ? launch<__half>(g, cs) : launch<__nv_bfloat16>(g, cs);
}
