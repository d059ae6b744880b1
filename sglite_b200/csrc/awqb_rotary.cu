// Rotary positions of q and k, with their per-head RMSNorm folded in.
//
// Pair j of a head turns by the angle positions[m] * inv_freq[j]. The angle is
// taken in turns (inv_freq / 2 pi, fp64) and reduced to a fraction of a turn in
// fp64, so a position of millions loses nothing before the fp32 sine.
#include <cuda_runtime.h>

#include "awqb200.h"
#include "awqb_common.h"
#include "awqb_vec.cuh"

namespace awqb {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxD = 256;

struct Side {  // q or k
  const void *in, *weight;
  void* out;
  int64_t row, head, out_row, out_head;
};

struct Args {
  Side side[2];
  const void* positions;
  const double* inv_freq;
  int Hq, H, D, rot, pos64, interleaved;
  float scale, eps;
};

// One CTA per token: cos and sin of its pairs once, then a warp per head.
template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Args a) {
  __shared__ float2 cs[kMaxD / 2];
  const int64_t m = blockIdx.x;
  const int64_t pos = a.pos64 ? static_cast<const int64_t*>(a.positions)[m]
                              : (int64_t) static_cast<const int32_t*>(a.positions)[m];
  if (pos < 0) return;  // padding
  const int half = a.rot / 2;
  for (int j = threadIdx.x; j < half; j += kThreads) {
    const double turns = (double)pos * (a.inv_freq[j] * 0.15915494309189533577);  // 1 / (2 pi)
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    cs[j] = make_float2(a.scale * c, a.scale * s);
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int hh = warp; hh < a.H; hh += kThreads / 32) {
    const Side& s = a.side[hh >= a.Hq];
    const int h = hh >= a.Hq ? hh - a.Hq : hh;
    const T* in = static_cast<const T*>(s.in) + m * s.row + h * s.head;
    T* out = static_cast<T*>(s.out) + m * s.out_row + h * s.out_head;
    const T* w = static_cast<const T*>(s.weight);
    float rms = 1.f;
    if (w != nullptr) {
      float ss = 0.f;
      for (int d = lane; d < a.D; d += 32) ss += (float)in[d] * (float)in[d];
      rms = rsqrtf(warp_sum(ss) / (float)a.D + a.eps);
    }
    for (int j = lane; j < half; j += 32) {
      const int i0 = a.interleaved ? 2 * j : j, i1 = a.interleaved ? 2 * j + 1 : j + half;
      float x = (float)in[i0], y = (float)in[i1];
      if (w != nullptr) x *= rms * (float)w[i0], y *= rms * (float)w[i1];
      const float2 t = cs[j];
      out[i0] = (T)(x * t.x - y * t.y);
      out[i1] = (T)(x * t.y + y * t.x);
    }
    for (int d = a.rot + lane; d < a.D; d += 32) {
      float x = (float)in[d];
      if (w != nullptr) x *= rms * (float)w[d];
      out[d] = (T)x;
    }
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace
}  // namespace awqb

using namespace awqb;

extern "C" int awqb_rotary(const void* q, int64_t q_row, int64_t q_head, int64_t Hq, const void* k, int64_t k_row,
                           int64_t k_head, int64_t Hk, const void* positions, int positions_i64,
                           const double* inv_freq, int64_t rot_dim, int64_t head_dim, int64_t M, int interleaved,
                           float scale, const void* q_weight, const void* k_weight, float eps, void* q_out,
                           int64_t q_out_row, int64_t q_out_head, void* k_out, int64_t k_out_row, int64_t k_out_head,
                           int dtype, void* stream) {
  AWQB_REQUIRE(dtype == AWQB_DTYPE_F16 || dtype == AWQB_DTYPE_BF16, kInvalidArgument, "bad dtype %d", dtype);
  AWQB_REQUIRE(head_dim > 0 && head_dim % 8 == 0 && head_dim <= kMaxD, kInvalidArgument,
               "head_dim=%lld must be a positive multiple of 8, at most %d", (long long)head_dim, kMaxD);
  AWQB_REQUIRE(rot_dim >= 2 && rot_dim % 2 == 0 && rot_dim <= head_dim, kInvalidArgument,
               "rot_dim=%lld must be even, 2..head_dim", (long long)rot_dim);
  AWQB_REQUIRE(M >= 0 && M <= 0x7fffffff && Hq >= 1 && Hq <= 65536 && Hk >= 0 && Hk <= 65536, kInvalidArgument,
               "bad sizes: %lld tokens, %lld q heads, %lld k heads", (long long)M, (long long)Hq, (long long)Hk);
  AWQB_REQUIRE((q_row | q_head | q_out_row | q_out_head) % 8 == 0 &&
                   (Hk == 0 || (k_row | k_head | k_out_row | k_out_head) % 8 == 0),
               kInvalidArgument, "strides must be multiples of 8");
  AWQB_REQUIRE(eps >= 0.f, kInvalidArgument, "eps must be >= 0");
  if (M == 0) return kOk;
  AWQB_REQUIRE(q && q_out && positions && inv_freq && (Hk == 0 || (k && k_out)), kInvalidArgument, "null pointer");
  AWQB_REQUIRE(aligned16(q) && aligned16(q_out) && aligned16(q_weight) &&
                   (Hk == 0 || (aligned16(k) && aligned16(k_out) && aligned16(k_weight))),
               kInvalidArgument, "tensors must be 16-byte aligned");
  Args a = {};
  a.side[0] = {q, q_weight, q_out, q_row, q_head, q_out_row, q_out_head};
  a.side[1] = {k, k_weight, k_out, k_row, k_head, k_out_row, k_out_head};
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.Hq = (int)Hq;
  a.H = (int)(Hq + Hk);
  a.D = (int)head_dim;
  a.rot = (int)rot_dim;
  a.pos64 = positions_i64 != 0;
  a.interleaved = interleaved != 0;
  a.scale = scale;
  a.eps = eps;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == AWQB_DTYPE_F16)
    rotary_kernel<__half><<<(unsigned)M, kThreads, 0, st>>>(a);
  else
    rotary_kernel<__nv_bfloat16><<<(unsigned)M, kThreads, 0, st>>>(a);
  AWQB_LAUNCH_CHECK();
  return kOk;
}
