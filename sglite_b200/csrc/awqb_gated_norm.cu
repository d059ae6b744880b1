// The norms around a block, fused with its gate and residual scale:
//   b = post ? x * rsqrt(mean(x^2) + eps) * (offset + post) : x
//   h = residual + scale * act(gate) * b            (stored rounded)
//   y = h * rsqrt(mean(h^2) + eps) * (offset + pre)
// A row stays in registers from its loads to its last store, so x, residual and
// gate are read once and h, y written once; both sums are over fp32 values.
#include <cuda_runtime.h>

#include "awqb200.h"
#include "awqb_common.h"
#include "awqb_vec.cuh"

namespace awqb {
namespace {

constexpr int kThreads = 512;
constexpr int kMaxVec = 4;  // 16-byte vectors per thread
constexpr int kMaxN = kThreads * 8 * kMaxVec;

struct Args {
  const void *x, *residual, *post, *gate, *pre;
  void *out, *residual_out;
  int64_t ld_x, ld_res, gate_row, gate_col, ld_out, ld_res_out;
  int N, act;
  float scale, offset, eps;
};

// Sum over the CTA; every thread gets the same value.
__device__ __forceinline__ float block_sum(float v, float* red) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  v = warp_sum(v);
  __syncthreads();  // an earlier sum may still be read
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return warp_sum(lane < kThreads / 32 ? red[lane] : 0.f);
}

__device__ __forceinline__ float activate(float g, int act) {
  if (act == 1) return 1.f / (1.f + expf(-g));
  if (act == 2) return tanhf(g);
  if (act == 3) return g / (1.f + expf(-g));
  return g;
}

template <typename T, bool kResF32>
__global__ void __launch_bounds__(kThreads) gated_norm_kernel(const Args a) {
  __shared__ float red[kThreads / 32];
  const int64_t row = blockIdx.x;
  const int nvec = a.N / 8;
  float b[kMaxVec][8], h[kMaxVec][8];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxVec; ++i) {
    const int v = i * kThreads + threadIdx.x;
    if (v < nvec) {
      unpack_vec<T>(reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + row * a.ld_x)[v], b[i]);
      if (kResF32) {
        const float4* r = reinterpret_cast<const float4*>(static_cast<const float*>(a.residual) + row * a.ld_res);
        const float4 lo = r[2 * v], hi = r[2 * v + 1];
        h[i][0] = lo.x, h[i][1] = lo.y, h[i][2] = lo.z, h[i][3] = lo.w;
        h[i][4] = hi.x, h[i][5] = hi.y, h[i][6] = hi.z, h[i][7] = hi.w;
      } else {
        unpack_vec<T>(reinterpret_cast<const uint4*>(static_cast<const T*>(a.residual) + row * a.ld_res)[v], h[i]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += b[i][j] * b[i][j];
    }
  }
  float rms = 1.f;
  if (a.post != nullptr) rms = rsqrtf(block_sum(ss, red) / (float)a.N + a.eps);
  ss = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxVec; ++i) {
    const int v = i * kThreads + threadIdx.x;
    if (v < nvec) {
      if (a.post != nullptr) {
        float w[8];
        unpack_vec<T>(static_cast<const uint4*>(a.post)[v], w);
#pragma unroll
        for (int j = 0; j < 8; ++j) b[i][j] *= rms * (a.offset + w[j]);
      }
      if (a.gate != nullptr) {
        const T* gp = static_cast<const T*>(a.gate) + row * a.gate_row;
        float g[8];
        if (a.gate_col) {
          unpack_vec<T>(reinterpret_cast<const uint4*>(gp)[v], g);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) g[j] = (float)gp[0];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) b[i][j] *= activate(g[j], a.act);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[i][j] += a.scale * b[i][j];
        ss += h[i][j] * h[i][j];
      }
      if (kResF32) {
        float4* r = reinterpret_cast<float4*>(static_cast<float*>(a.residual_out) + row * a.ld_res_out);
        r[2 * v] = make_float4(h[i][0], h[i][1], h[i][2], h[i][3]);
        r[2 * v + 1] = make_float4(h[i][4], h[i][5], h[i][6], h[i][7]);
      } else {
        reinterpret_cast<uint4*>(static_cast<T*>(a.residual_out) + row * a.ld_res_out)[v] = pack_vec<T>(h[i]);
      }
    }
  }
  if (a.pre == nullptr) return;
  rms = rsqrtf(block_sum(ss, red) / (float)a.N + a.eps);
#pragma unroll
  for (int i = 0; i < kMaxVec; ++i) {
    const int v = i * kThreads + threadIdx.x;
    if (v < nvec) {
      float w[8];
      unpack_vec<T>(static_cast<const uint4*>(a.pre)[v], w);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] *= rms * (a.offset + w[j]);
      reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * a.ld_out)[v] = pack_vec<T>(h[i]);
    }
  }
}

template <typename T>
int launch(const Args& a, int64_t M, bool res_f32, cudaStream_t stream) {
  if (res_f32)
    gated_norm_kernel<T, true><<<(unsigned)M, kThreads, 0, stream>>>(a);
  else
    gated_norm_kernel<T, false><<<(unsigned)M, kThreads, 0, stream>>>(a);
  AWQB_LAUNCH_CHECK();
  return kOk;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace
}  // namespace awqb

using namespace awqb;

extern "C" int awqb_gated_add_rmsnorm(const void* x, int64_t ld_x, const void* residual, int64_t ld_res,
                                      int residual_f32, const void* post_weight, const void* gate, int64_t gate_row,
                                      int64_t gate_col, int gate_act, float scale, const void* weight,
                                      float weight_offset, void* out, int64_t ld_out, void* residual_out,
                                      int64_t ld_res_out, int64_t M, int64_t N, float eps, int dtype, void* stream) {
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
  return dtype == AWQB_DTYPE_F16 ? launch<__half>(a, M, residual_f32 != 0, st)
                                 : launch<__nv_bfloat16>(a, M, residual_f32 != 0, st);
}
