// Rotary positions of q and k, with their per-head RMSNorm folded in.
//
// Pair j of a head turns by the angle positions[m] * inv_freq[j]. Whole turns do not
// matter, so the angle is kept as a 64-bit fraction of a turn: inv_freq / 2 pi
// modulo 1, times the position modulo 2^64. That integer product is exact; the
// fraction comes from fp64 and is off by 2^-53 of inv_freq / 2 pi, which the position
// multiplies (2^-24 of a turn at 2^29). Its upper 32 bits go to the fp32 sine.
// Nothing is tabulated by position: a token's sines are made once and serve all
// its heads.
//
// Bound by HBM (q and k in and out), and by instruction issue next to it. Warps work
// by themselves: one takes a token (or, where tokens are few, a batch of its
// heads), makes its sines, and turns batches of heads in packed fp32 arithmetic
// (two values per instruction), a piece of a head per lane: the vectors of eight at
// d and d + rot_dim / 2, or one vector of four neighbouring pairs. A batch's
// loads are issued together. The lanes of a head (a power of two) add up its squares
// by shuffles. With CTAs that shared a token's sines, their barriers and starts
// left memory idle (8192 tokens of 32 + 8 heads of 128 with q/k norm: 37 us).
#include <cuda_runtime.h>

#include <algorithm>

#include "awqb200.h"
#include "awqb_common.h"
#include "awqb_ptx.cuh"
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
  float scale, eps, inv_d;
};

// The 64-bit fraction of a turn that a pair advances per position.
__device__ __forceinline__ uint64_t turn_fraction(double inv_freq) {
  const double turns = inv_freq * 0.15915494309189533577;  // 1 / (2 pi)
  return (uint64_t)((turns - floor(turns)) * 18446744073709551616.0);  // 2^64
}

// scale * cos of the angle fraction * pos into *at, scale * sin kMaxD / 2 further.
__device__ __forceinline__ void make_sine(const Args& a, uint64_t fraction, int64_t pos, float* at) {
  const int upper = (int)((fraction * (uint64_t)pos) >> 32);  // in 2^-32 turns, -1/2 .. 1/2
  float s, c;
  sincospif((float)upper * 4.656612873077392578125e-10f, &s, &c);  // 2^-31
  at[0] = a.scale * c;
  at[kMaxD / 2] = a.scale * s;
}

__device__ __forceinline__ int64_t position_of(const Args& a, int64_t m) {
  return a.pos64 ? static_cast<const int64_t*>(a.positions)[m] : (int64_t) static_cast<const int32_t*>(a.positions)[m];
}

// Two fp32 values per instruction.
__device__ __forceinline__ uint64_t bits(float2 v) { return *reinterpret_cast<const uint64_t*>(&v); }
__device__ __forceinline__ float2 floats(uint64_t v) { return *reinterpret_cast<const float2*>(&v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
  return floats(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)));
  return floats(d);
}
// (x, y) turned by the angles of cosine c and sine s.
__device__ __forceinline__ void turn2(float2& x, float2& y, float2 c, float2 s) {
  const float2 minus = make_float2(-s.x, -s.y), p = x;
  x = fma2(y, minus, mul2(x, c));
  y = fma2(p, s, mul2(y, c));
}
template <typename T>
__device__ __forceinline__ void unpack_pairs(const uint4& v, float2 (&f)[4]) {
  f[0] = Pair<T>::unpack(v.x), f[1] = Pair<T>::unpack(v.y), f[2] = Pair<T>::unpack(v.z), f[3] = Pair<T>::unpack(v.w);
}
template <typename T>
__device__ __forceinline__ uint4 pack_pairs(const float2 (&f)[4]) {
  return make_uint4(Pair<T>::pack(f[0].x, f[0].y), Pair<T>::pack(f[1].x, f[1].y), Pair<T>::pack(f[2].x, f[2].y),
                    Pair<T>::pack(f[3].x, f[3].y));
}

// Which elements a piece u of a head holds: kWhole, the vectors at 8u and
// 8u + rot / 2 (the whole head turns); kPart, the same below rot / 16, then the
// vectors past rot; kNext, the vector at 8u (interleaved).
enum Pieces { kWhole, kPart, kNext };

// `lanes` lanes (a power of two) per head, the last ones idle if a head has fewer
// pieces.
// kBatch: steps (32 / lanes heads each) whose loads are in flight together.
template <typename T, Pieces kKind, bool kNorm, int kBatch>
__global__ void __launch_bounds__(kThreads, 2)
rotary_vec_kernel(const __grid_constant__ Args a, int64_t M, int lanes, int pieces, int q_batches, int k_batches, int per_unit) {
  constexpr bool kInterleaved = kKind == kNext;
  __shared__ __align__(16) float cs[kThreads / 32][kMaxD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int u = lane & (lanes - 1), per_step = 32 / lanes, half = a.rot / 2;
  const bool turns = kKind == kWhole || (kInterleaved ? u * 8 < a.rot : u * 16 < a.rot);
  const bool two = kKind == kWhole || (kKind == kPart && turns);
  const int at0 = kInterleaved || two ? u * 8 : a.rot + (u - a.rot / 16) * 8, at1 = u * 8 + half;
  const int first = kInterleaved ? u * 4 : u * 8, get = kInterleaved ? first : first + ((first >> 3) & 4);
  grid_dep_wait();
  grid_dep_launch();
  // this lane's pairs for the sines: lane, lane + 32, ...; the loads' latency passes
  // while the first token is fetched
  uint64_t fraction[kMaxD / 64];  // the bits of inv_freq until they are first used
  bool fractions = false;
#pragma unroll
  for (int i = 0; i < kMaxD / 64; ++i)
    fraction[i] = lane + 32 * i < half ? (uint64_t)__double_as_longlong(a.inv_freq[lane + 32 * i]) : 0;
  const int batches = q_batches + k_batches, splits = (batches + per_unit - 1) / per_unit;
  const int64_t units = M * splits;
  float* sines = cs[warp];
  for (int64_t unit = (int64_t)blockIdx.x * (kThreads / 32) + warp; unit < units; unit += (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t m = splits == 1 ? unit : unit / splits;
    const int b0 = splits == 1 ? 0 : (int)(unit - m * splits) * per_unit, b1 = min(batches, b0 + per_unit);
    const int64_t pos = position_of(a, m);
    float2 c[4], sn[4];  // interleaved: four pairs in the first two
    for (int b = b0; b < b1; ++b) {
      const bool is_k = b >= q_batches;
      const Side& s = a.side[is_k];
      const int heads = is_k ? a.H - a.Hq : a.Hq;
      const int h0 = (is_k ? b - q_batches : b) * kBatch * per_step + lane / lanes;
      const T* in = static_cast<const T*>(s.in) + m * s.row + h0 * s.head;
      uint4 v0[kBatch] = {}, v1[kBatch] = {};
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (h0 + i * per_step < heads && u < pieces) {
          const T* at = in + i * per_step * s.head;
          v0[i] = *reinterpret_cast<const uint4*>(at + at0);
          if (two) v1[i] = *reinterpret_cast<const uint4*>(at + at1);
        }
      if (pos < 0) break;  // padding (the same for the whole warp)
      if (b == b0) {
        // Pair j stands at j, its halves of eight swapped where bit 5 is set: the
        // 16-byte reads of eight lanes then hit all banks.
        if (!fractions) {
          fractions = true;
#pragma unroll
          for (int i = 0; i < kMaxD / 64; ++i) fraction[i] = turn_fraction(__longlong_as_double((long long)fraction[i]));
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kMaxD / 64; ++i) {
          const int j = lane + 32 * i;
          if (32 * i < half && j < half)
            make_sine(a, fraction[i], pos, sines + (kInterleaved ? j : j ^ ((j >> 3) & 4)));
        }
        __syncwarp();
        if (turns) {
#pragma unroll
          for (int i = 0; i < (kInterleaved ? 2 : 4); i += 2) {
            const float4 p = *reinterpret_cast<const float4*>(sines + (get ^ (2 * i)));
            const float4 q = *reinterpret_cast<const float4*>(sines + kMaxD / 2 + (get ^ (2 * i)));
            c[i] = make_float2(p.x, p.y), c[i + 1] = make_float2(p.z, p.w);
            sn[i] = make_float2(q.x, q.y), sn[i + 1] = make_float2(q.z, q.w);
          }
        }
      }
      float2 w0[4], w1[4];  // this piece's norm weights
      const bool normed = kNorm && s.weight != nullptr;
      if (normed && u < pieces) {
        const T* w = static_cast<const T*>(s.weight);
        unpack_pairs<T>(*reinterpret_cast<const uint4*>(w + at0), w0);
        if (two) unpack_pairs<T>(*reinterpret_cast<const uint4*>(w + at1), w1);
      }
      T* out = static_cast<T*>(s.out) + m * s.out_row + h0 * s.out_head;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (h0 - lane / lanes + i * per_step >= heads) break;  // no lane has a head
        float2 x[4], y[4];
        unpack_pairs<T>(v0[i], x);
        unpack_pairs<T>(v1[i], y);
        if (normed) {  // all lanes shuffle; those without a piece hold zeros
          float2 sq = make_float2(0.f, 0.f);
#pragma unroll
          for (int j = 0; j < 4; ++j) sq = fma2(x[j], x[j], sq);
          if (two)
#pragma unroll
            for (int j = 0; j < 4; ++j) sq = fma2(y[j], y[j], sq);
          float ss = sq.x + sq.y;
          for (int o = lanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float rms = rsqrtf(ss * a.inv_d + a.eps);
          const float2 both = make_float2(rms, rms);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = mul2(mul2(x[j], both), w0[j]);
          if (two)
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = mul2(mul2(y[j], both), w1[j]);
        }
        if (h0 + i * per_step >= heads || u >= pieces) continue;
        T* to = out + i * per_step * s.out_head;
        if (kInterleaved) {
          const float cc[4] = {c[0].x, c[0].y, c[1].x, c[1].y}, ss[4] = {sn[0].x, sn[0].y, sn[1].x, sn[1].y};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (u * 4 + j < half)
              x[j] = make_float2(x[j].x * cc[j] - x[j].y * ss[j], x[j].x * ss[j] + x[j].y * cc[j]);
        } else if (two) {
#pragma unroll
          for (int j = 0; j < 4; ++j) turn2(x[j], y[j], c[j], sn[j]);
          *reinterpret_cast<uint4*>(to + at1) = pack_pairs<T>(y);
        }
        *reinterpret_cast<uint4*>(to + at0) = pack_pairs<T>(x);
      }
    }
  }
}

// A CTA per token, a warp per head, element by element: where the two halves of the
// turned part do not split into whole vectors (never interleaved pairs, whose vectors
// hold whole pairs). Two bytes per access: 8192 tokens of 32 + 8 heads of 128, 20 of
// them turned, in place: 135 us, 1.2 TB/s (64 turned, by whole vectors: 44 us).
template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ Args a) {
  __shared__ float cs[kMaxD];
  grid_dep_wait();
  grid_dep_launch();
  const int64_t m = blockIdx.x;
  const int64_t pos = position_of(a, m);
  if (pos < 0) return;  // padding
  const int half = a.rot / 2;
  for (int j = threadIdx.x; j < half; j += kThreads) make_sine(a, turn_fraction(a.inv_freq[j]), pos, &cs[j]);
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
      rms = rsqrtf(warp_sum(ss) * a.inv_d + a.eps);
    }
    for (int j = lane; j < half; j += 32) {
      float x = (float)in[j], y = (float)in[j + half];
      if (w != nullptr) x *= rms * (float)w[j], y *= rms * (float)w[j + half];
      const float c = cs[j], sn = cs[kMaxD / 2 + j];
      out[j] = (T)(x * c - y * sn);
      out[j + half] = (T)(x * sn + y * c);
    }
    for (int d = a.rot + lane; d < a.D; d += 32) {
      float x = (float)in[d];
      if (w != nullptr) x *= rms * (float)w[d];
      out[d] = (T)x;
    }
  }
}

template <typename T, Pieces kKind>
auto pick(bool norm, bool few) {
  return norm ? (few ? rotary_vec_kernel<T, kKind, true, 1> : rotary_vec_kernel<T, kKind, true, 4>)
              : (few ? rotary_vec_kernel<T, kKind, false, 1> : rotary_vec_kernel<T, kKind, false, 4>);
}

template <typename T>
int launch(const Args& a, int64_t M, cudaStream_t st) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)M);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (!a.interleaved && a.rot % 16 != 0) {
    AWQB_CUDA(cudaLaunchKernelEx(&cfg, rotary_kernel<T>, a));
    return kOk;
  }
  const int pieces = a.interleaved ? a.D / 8 : a.rot / 16 + (a.D - a.rot) / 8;
  int lanes = 1;
  while (lanes < pieces) lanes *= 2;
  // Few tokens: a warp per step, all at once. Else batches of four steps, and whole
  // tokens once they give every warp of a full GPU one.
  const int64_t warps = (int64_t)device_sm_count() * 2 * (kThreads / 32);
  const int steps = (a.Hq * lanes + 31) / 32 + ((a.H - a.Hq) * lanes + 31) / 32;
  const bool few = M * steps <= warps;
  const int per_batch = (few ? 1 : 4) * 32 / lanes;
  const int q_batches = (a.Hq + per_batch - 1) / per_batch, k_batches = (a.H - a.Hq + per_batch - 1) / per_batch;
  const int per_unit = M >= warps ? q_batches + k_batches : 1;
  const int64_t units = M * ((q_batches + k_batches + per_unit - 1) / per_unit);
  cfg.gridDim = dim3((unsigned)((std::min(units, warps) + kThreads / 32 - 1) / (kThreads / 32)));
  const bool norm = a.side[0].weight != nullptr || a.side[1].weight != nullptr;
  const auto kernel = a.interleaved  ? pick<T, kNext>(norm, few)
                      : a.rot == a.D ? pick<T, kWhole>(norm, few)
                                     : pick<T, kPart>(norm, few);
  AWQB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, M, lanes, pieces, q_batches, k_batches, per_unit));
  return kOk;
}

// No element of [rows, heads, D] stands where another does.
bool apart(int64_t rows, int64_t row, int64_t heads, int64_t head, int64_t D) {
  if (rows <= 1) return heads <= 1 || head >= D;
  if (heads <= 1) return row >= D;
  return (head >= D && row >= (heads - 1) * head + D) || (row >= D && head >= (rows - 1) * row + D);
}

}  // namespace
}  // namespace awqb

using namespace awqb;

extern "C" int awqb_rotary(const awqb_rotary_args* args, void* stream) {
  AWQB_REQUIRE(args != nullptr, kInvalidArgument, "args is null");
  const auto [q, q_row, q_head, Hq, k, k_row, k_head, Hk, positions, positions_i64, inv_freq, rot_dim, head_dim, M,
              interleaved, scale, q_weight, k_weight, eps, q_out, q_out_row, q_out_head, k_out, k_out_row,
              k_out_head, dtype] = *args;
  AWQB_REQUIRE(dtype == AWQB_DTYPE_F16 || dtype == AWQB_DTYPE_BF16, kInvalidArgument, "bad dtype %d", dtype);
  AWQB_REQUIRE(head_dim > 0 && head_dim % 8 == 0 && head_dim <= kMaxD, kInvalidArgument,
               "head_dim=%lld must be a positive multiple of 8, at most %d", (long long)head_dim, kMaxD);
  AWQB_REQUIRE(rot_dim >= 2 && rot_dim % 2 == 0 && rot_dim <= head_dim, kInvalidArgument,
               "rot_dim=%lld must be even, 2..head_dim", (long long)rot_dim);
  AWQB_REQUIRE(M >= 0 && M < (1 << 30) && Hq >= 1 && Hq <= 65536 && Hk >= 0 && Hk <= 65536, kInvalidArgument,
               "bad sizes: %lld tokens, %lld q heads, %lld k heads", (long long)M, (long long)Hq, (long long)Hk);
  AWQB_REQUIRE((q_row | q_head | q_out_row | q_out_head) % 8 == 0 &&
                   (Hk == 0 || (k_row | k_head | k_out_row | k_out_head) % 8 == 0),
               kInvalidArgument, "strides must be multiples of 8");
  AWQB_REQUIRE(eps >= 0.f, kInvalidArgument, "eps must be >= 0");
  AWQB_REQUIRE(apart(M, q_out_row, Hq, q_out_head, head_dim) && (Hk == 0 || apart(M, k_out_row, Hk, k_out_head, head_dim)),
               kInvalidArgument, "the outputs' tokens or heads overlap");
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
  a.inv_d = 1.f / (float)head_dim;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == AWQB_DTYPE_F16 ? launch<__half>(a, M, st) : launch<__nv_bfloat16>(a, M, st);
}
