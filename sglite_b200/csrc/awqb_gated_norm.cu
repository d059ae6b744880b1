// The norms around a block, fused with its gate and residual scale:
//   b = post ? x * rsqrt(mean(x^2) + eps) * (offset + post) : x
//   h = residual + scale * act(gate) * b            (stored rounded)
//   y = h * rsqrt(mean(h^2) + eps) * (offset + pre)
//
// Bound by HBM: x, residual and gate are read once, h and y written once. A CTA
// takes a row and holds it in registers from its loads to its last store; all of
// a row's loads are issued before the first sum, the weights' (L1 and L2 hits)
// before the sum that they follow, so a row waits for memory once. Both sums are
// over fp32 values, in a fixed order. Launched with programmatic dependent
// launch, like the other norms.
#include <cuda_runtime.h>

#include <algorithm>

#include "awqb200.h"
#include "awqb_common.h"
#include "awqb_ptx.cuh"
#include "awqb_vec.cuh"

namespace awqb {
namespace {

constexpr int kMaxThreads = 512;
constexpr int kMaxVec = 4;  // 16-byte vectors per thread
constexpr int kMaxN = kMaxThreads * 8 * kMaxVec;

struct Args {
  const void *x, *residual, *post, *gate, *pre;
  void *out, *residual_out;
  int64_t ld_x, ld_res, gate_row, gate_col, ld_out, ld_res_out;
  int N, act;
  float scale, offset, eps;
};

// Sum over the CTA; every thread gets the same value. `red` is used once per call site.
__device__ __forceinline__ float block_sum(float v, float* red) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  v = warp_sum(v);
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return warp_sum(lane < (int)blockDim.x / 32 ? red[lane] : 0.f);
}

// The sigmoid by the approximate exponential and division (exact division would make
// this copy-like kernel issue-bound): right to (6 + 1.173 |g|) 2^-23 of the value, 1.2e-5
// at g = -80 and 9e-7 at |g| = 1, and 0 below g = -87.3, where it is under 2^-125.
__device__ __forceinline__ float activate(float g, int act) {
  if (act == 1) return __fdividef(1.f, 1.f + __expf(-g));
  if (act == 2) return tanhf(g);
  if (act == 3) return __fdividef(g, 1.f + __expf(-g));
  return g;
}

template <typename T, bool kResF32, int kVec>
__global__ void __launch_bounds__(kMaxThreads, kVec <= 2 ? 2 : 1) gated_norm_kernel(const __grid_constant__ Args a) {
  __shared__ float red[2][kMaxThreads / 32];
  grid_dep_wait();
  grid_dep_launch();
  const int64_t row = blockIdx.x;
  const int nvec = a.N / 8;
  const uint4* xp = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + row * a.ld_x);
  const uint4* rp = reinterpret_cast<const uint4*>(static_cast<const char*>(a.residual) + row * a.ld_res * (kResF32 ? 4 : 2));
  const T* gp = static_cast<const T*>(a.gate) + row * a.gate_row;
  constexpr int kRes = kResF32 ? 2 : 1;  // vectors of residual per vector of x
  uint4 x[kVec], r[kVec][kRes], g[kVec], w[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    if (v < nvec) {
      x[i] = xp[v];
#pragma unroll
      for (int j = 0; j < kRes; ++j) r[i][j] = rp[kRes * v + j];
      if (a.gate != nullptr && a.gate_col) g[i] = reinterpret_cast<const uint4*>(gp)[v];
    }
  }
  float one_gate = a.scale;
  if (a.gate != nullptr && !a.gate_col) one_gate *= activate((float)gp[0], a.act);
  float rms = 1.f;
  if (a.post != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int v = i * blockDim.x + threadIdx.x;
      if (v < nvec) {
        w[i] = static_cast<const uint4*>(a.post)[v];
        float b[8];
        unpack_vec<T>(x[i], b);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += b[j] * b[j];
      }
    }
    rms = rsqrtf(block_sum(ss, red[0]) / (float)a.N + a.eps);
  }
  float h[kVec][8], ss = 0.f;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    if (v < nvec) {
      float b[8];
      unpack_vec<T>(x[i], b);
      if (a.post != nullptr) {
        float p[8];
        unpack_vec<T>(w[i], p);
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] *= rms * (a.offset + p[j]);
      }
      if (a.pre != nullptr) w[i] = static_cast<const uint4*>(a.pre)[v];
      if (a.gate != nullptr && a.gate_col) {
        float t[8];
        unpack_vec<T>(g[i], t);
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] *= activate(t[j], a.act);
      }
      if (kResF32) {
#pragma unroll
        for (int j = 0; j < kRes; ++j) {
          h[i][4 * j] = __uint_as_float(r[i][j].x), h[i][4 * j + 1] = __uint_as_float(r[i][j].y);
          h[i][4 * j + 2] = __uint_as_float(r[i][j].z), h[i][4 * j + 3] = __uint_as_float(r[i][j].w);
        }
      } else {
        unpack_vec<T>(r[i][0], h[i]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[i][j] += one_gate * b[j];
        ss += h[i][j] * h[i][j];
      }
      uint4* to = reinterpret_cast<uint4*>(static_cast<char*>(a.residual_out) + row * a.ld_res_out * (kResF32 ? 4 : 2));
      if (kResF32) {
#pragma unroll
        for (int j = 0; j < kRes; ++j)
          to[kRes * v + j] = make_uint4(__float_as_uint(h[i][4 * j]), __float_as_uint(h[i][4 * j + 1]),
                                        __float_as_uint(h[i][4 * j + 2]), __float_as_uint(h[i][4 * j + 3]));
      } else {
        to[v] = pack_vec<T>(h[i]);
      }
    }
  }
  if (a.pre == nullptr) return;
  rms = rsqrtf(block_sum(ss, red[1]) / (float)a.N + a.eps);
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    if (v < nvec) {
      float p[8];
      unpack_vec<T>(w[i], p);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] *= rms * (a.offset + p[j]);
      reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * a.ld_out)[v] = pack_vec<T>(h[i]);
    }
  }
}

template <typename T, bool kResF32>
int launch(const Args& a, int64_t M, cudaStream_t stream) {
  // one vector per thread up to 4096 features, then two, then four
  const int nvec = a.N / 8, vecs = nvec <= kMaxThreads ? 1 : nvec <= 2 * kMaxThreads ? 2 : 4;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)M);
  cfg.blockDim = dim3((unsigned)(((nvec + vecs - 1) / vecs + 31) / 32 * 32));
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const auto kernel = vecs == 1   ? gated_norm_kernel<T, kResF32, 1>
                      : vecs == 2 ? gated_norm_kernel<T, kResF32, 2>
                                  : gated_norm_kernel<T, kResF32, 4>;
  AWQB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  return kOk;
}

}  // namespace
}  // namespace awqb

using namespace awqb;

extern "C" int awqb_gated_add_rmsnorm(const awqb_gated_norm_args* args, void* stream) {
  AWQB_REQUIRE(args != nullptr, kInvalidArgument, "args is null");
  const auto [x, ld_x, residual, ld_res, residual_f32, post_weight, gate, gate_row, gate_col, gate_act, scale,
              weight, weight_offset, out, ld_out, residual_out, ld_res_out, M, N, eps, dtype] = *args;
  AWQB_REQUIRE(dtype == AWQB_DTYPE_F16 || dtype == AWQB_DTYPE_BF16, kInvalidArgument, "bad dtype %d", dtype);
  AWQB_REQUIRE(M >= 0 && M <= 0x7fffffff && N > 0 && N % 8 == 0 && N <= kMaxN, kInvalidArgument,
               "N=%lld must be a positive multiple of 8, at most %d", (long long)N, kMaxN);
  AWQB_REQUIRE(ld_x >= N && ld_res >= N && ld_res_out >= N && (weight == nullptr || ld_out >= N) && ld_x % 8 == 0 &&
                   ld_res % 8 == 0 && ld_res_out % 8 == 0 && ld_out % 8 == 0,
               kInvalidArgument, "row strides must be >= N and multiples of 8");
  AWQB_REQUIRE(gate_act >= 0 && gate_act <= 3, kInvalidArgument, "bad gate activation %d", gate_act);
  AWQB_REQUIRE(eps >= 0.f, kInvalidArgument, "eps must be >= 0");
  AWQB_REQUIRE(gate == nullptr || gate_col == 0 || gate_col == 1, kInvalidArgument, "gate_col must be 0 or 1");
  AWQB_REQUIRE(gate == nullptr || gate_row == 0 || (gate_row > 0 && (gate_col == 0 || (gate_row >= N && gate_row % 8 == 0))),
               kInvalidArgument, "the gate's row stride must be 0, or at least N and a multiple of 8");
  AWQB_REQUIRE(post_weight != nullptr || weight != nullptr, kInvalidArgument,
               "one of the two norms' weights must be given");
  if (M == 0) return kOk;
  AWQB_REQUIRE(x && residual && residual_out && (out != nullptr || weight == nullptr), kInvalidArgument,
               "null pointer");
  AWQB_REQUIRE(aligned16(x) && aligned16(residual) && aligned16(post_weight) && aligned16(weight) && aligned16(out) &&
                   aligned16(residual_out) && (gate_col == 0 || aligned16(gate)),
               kInvalidArgument, "tensors must be 16-byte aligned");
  Args a = {x,      residual, post_weight, gate,   weight, out,    residual_out, ld_x,         ld_res, gate_row,
            gate_col, ld_out, ld_res_out,  (int)N, gate_act, scale, weight_offset, eps};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == AWQB_DTYPE_F16) return residual_f32 ? launch<__half, true>(a, M, st) : launch<__half, false>(a, M, st);
  return residual_f32 ? launch<__nv_bfloat16, true>(a, M, st) : launch<__nv_bfloat16, false>(a, M, st);
}
