// Rotary positions of q and k, with their per-head RMSNorm folded in.
//
// Pair j of a head turns by the angle positions[m] * inv_freq[j]. The angle is
// taken in turns (inv_freq / 2 pi, fp64) and reduced to a fraction of a turn in
// fp64, so a position of millions loses nothing before the fp32 sine. Nothing is
// tabulated: a token's sines are made once and serve all its heads.
//
// Bound by HBM (q and k in and out). A CTA takes a token. A thread keeps one piece
// of a head for all the heads it serves, with the sines in registers: the vectors
// of eight at d and d + rot_dim / 2 (or one vector of four neighbouring pairs);
// its first head's loads are issued before the sines are made. The lanes of a
// head (a power of two) add up its squares by shuffles.
#include <cuda_runtime.h>

#include <algorithm>

#include "awqb200.h"
#include "awqb_common.h"
#include "awqb_ptx.cuh"
#include "awqb_vec.cuh"

namespace awqb {
namespace {

constexpr int kThreads = 256;      // of the general kernel
constexpr int kVecThreads = 320;   // at most, of the vector kernel
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

// scale * (cos, sin) of the token's pairs into shared memory, cos at [pair], sin at
// [kMaxD / 2 + pair]; `place` is where a pair stands.
template <typename Place>
__device__ __forceinline__ void make_sines(const Args& a, int64_t pos, float* cs, Place place) {
  for (int j = threadIdx.x; j < a.rot / 2; j += blockDim.x) {
    const double turns = (double)pos * (a.inv_freq[j] * 0.15915494309189533577);  // 1 / (2 pi)
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    cs[place(j)] = a.scale * c;
    cs[kMaxD / 2 + place(j)] = a.scale * s;
  }
}

__device__ __forceinline__ int64_t position_of(const Args& a, int64_t m) {
  return a.pos64 ? static_cast<const int64_t*>(a.positions)[m] : (int64_t) static_cast<const int32_t*>(a.positions)[m];
}

// kInterleaved: piece u is the vector at 8u. Otherwise pieces below rot / 16 are the
// vectors at 8u and 8u + rot / 2, the others the vectors past rot. `lanes` lanes
// (a power of two) per head, the last ones idle if a head has fewer pieces.
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kVecThreads) rotary_vec_kernel(const __grid_constant__ Args a, int lanes, int pieces) {
  __shared__ __align__(16) float cs[kMaxD];
  grid_dep_wait();
  grid_dep_launch();
  const int64_t m = blockIdx.x;
  const int64_t pos = position_of(a, m);
  if (pos < 0) return;  // padding
  const int u = threadIdx.x & (lanes - 1), per_pass = blockDim.x / lanes, half = a.rot / 2;
  const bool turns = kInterleaved ? u * 8 < a.rot : u * 16 < a.rot;
  const bool two = !kInterleaved && turns;
  const int at0 = kInterleaved || two ? u * 8 : a.rot + (u - a.rot / 16) * 8, at1 = u * 8 + half;
  const auto side_of = [&](int hh) -> const Side& { return a.side[hh >= a.Hq]; };
  const auto load = [&](int hh, uint4& v0, uint4& v1) {
    if (hh >= a.H || u >= pieces) return;
    const Side& s = side_of(hh);
    const T* in = static_cast<const T*>(s.in) + m * s.row + (hh >= a.Hq ? hh - a.Hq : hh) * s.head;
    v0 = *reinterpret_cast<const uint4*>(in + at0);
    if (two) v1 = *reinterpret_cast<const uint4*>(in + at1);
  };
  int hh = threadIdx.x / lanes;
  uint4 v0 = {}, v1 = {};
  load(hh, v0, v1);
  // Pair j stands at j, its halves of eight swapped where bit 5 is set: the
  // 16-byte reads of eight lanes then hit all banks.
  make_sines(a, pos, cs, [](int j) { return kInterleaved ? j : j ^ ((j >> 3) & 4); });
  __syncthreads();
  constexpr int kPairs = kInterleaved ? 4 : 8;
  float c[kPairs], sn[kPairs];
  if (turns) {
    const int first = kInterleaved ? u * 4 : u * 8, get = kInterleaved ? first : first + ((first >> 3) & 4);
#pragma unroll
    for (int i = 0; i < kPairs; i += 4) {
      *reinterpret_cast<float4*>(c + i) = *reinterpret_cast<const float4*>(cs + (get ^ i));
      *reinterpret_cast<float4*>(sn + i) = *reinterpret_cast<const float4*>(cs + kMaxD / 2 + (get ^ i));
    }
  }
  for (int h0 = 0; h0 < a.H; h0 += per_pass, hh += per_pass) {
    uint4 n0 = {}, n1 = {};
    load(hh + per_pass, n0, n1);
    const bool live = hh < a.H && u < pieces;
    const Side& s = side_of(min(hh, a.H - 1));
    float x[8], y[8];
    unpack_vec<T>(v0, x);
    unpack_vec<T>(v1, y);
    if (a.side[0].weight != nullptr || a.side[1].weight != nullptr) {  // uniform: all lanes shuffle
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i] + (two ? y[i] * y[i] : 0.f);
      for (int o = lanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (live && s.weight != nullptr) {
        const float rms = rsqrtf(ss / (float)a.D + a.eps);
        float w[8];
        unpack_vec<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(s.weight) + at0), w);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= rms * w[i];
        if (two) {
          unpack_vec<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(s.weight) + at1), w);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] *= rms * w[i];
        }
      }
    }
    if (live) {
      T* out = static_cast<T*>(s.out) + m * s.out_row + (hh >= a.Hq ? hh - a.Hq : hh) * s.out_head;
      if (kInterleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (u * 4 + i < half) {
            const float p = x[2 * i], q = x[2 * i + 1];
            x[2 * i] = p * c[i] - q * sn[i];
            x[2 * i + 1] = p * sn[i] + q * c[i];
          }
      } else if (two) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const float p = x[i], q = y[i];
          x[i] = p * c[i] - q * sn[i];
          y[i] = p * sn[i] + q * c[i];
        }
        *reinterpret_cast<uint4*>(out + at1) = pack_vec<T>(y);
      }
      *reinterpret_cast<uint4*>(out + at0) = pack_vec<T>(x);
    }
    v0 = n0, v1 = n1;
  }
}

// Any layout: a CTA per token, a warp per head, element by element. Taken where the
// two halves of the turned part do not split into whole vectors.
template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ Args a) {
  __shared__ float cs[kMaxD];
  grid_dep_wait();
  grid_dep_launch();
  const int64_t m = blockIdx.x;
  const int64_t pos = position_of(a, m);
  if (pos < 0) return;  // padding
  const int half = a.rot / 2;
  make_sines(a, pos, cs, [](int j) { return j; });
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
      const float c = cs[j], sn = cs[kMaxD / 2 + j];
      out[i0] = (T)(x * c - y * sn);
      out[i1] = (T)(x * sn + y * c);
    }
    for (int d = a.rot + lane; d < a.D; d += 32) {
      float x = (float)in[d];
      if (w != nullptr) x *= rms * (float)w[d];
      out[d] = (T)x;
    }
  }
}

template <typename T>
int launch(const Args& a, int64_t M, cudaStream_t st) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)M);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (!a.interleaved && a.rot % 16 != 0) {
    cfg.blockDim = dim3(kThreads);
    AWQB_CUDA(cudaLaunchKernelEx(&cfg, rotary_kernel<T>, a));
    return kOk;
  }
  const int pieces = a.interleaved ? a.D / 8 : a.rot / 16 + (a.D - a.rot) / 8;
  int lanes = 1;
  while (lanes < pieces) lanes *= 2;
  // equal passes over the heads, whole warps
  const int most = kVecThreads / lanes, passes = (a.H + most - 1) / most, heads = (a.H + passes - 1) / passes;
  cfg.blockDim = dim3((unsigned)((heads * lanes + 31) / 32 * 32));
  AWQB_CUDA(a.interleaved ? cudaLaunchKernelEx(&cfg, rotary_vec_kernel<T, true>, a, lanes, pieces)
                          : cudaLaunchKernelEx(&cfg, rotary_vec_kernel<T, false>, a, lanes, pieces));
  return kOk;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace
}  // namespace awqb

using namespace awqb;

static int awqb_rotary_impl(const void* q, int64_t q_row, int64_t q_head, int64_t Hq, const void* k, int64_t k_row,
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
  return dtype == AWQB_DTYPE_F16 ? launch<__half>(a, M, st) : launch<__nv_bfloat16>(a, M, st);
}

extern "C" int awqb_rotary(const awqb_rotary_args* a, void* stream) {
  AWQB_REQUIRE(a != nullptr, kInvalidArgument, "args is null");
  return awqb_rotary_impl(a->q, a->q_row, a->q_head, a->Hq, a->k, a->k_row, a->k_head, a->Hk, a->positions,
                          a->positions_i64, a->inv_freq, a->rot_dim, a->head_dim, a->M, a->interleaved, a->scale, a->q_weight,
                          a->k_weight, a->eps, a->q_out, a->q_out_row, a->q_out_head, a->k_out, a->k_out_row,
                          a->k_out_head, a->dtype, stream);
}
