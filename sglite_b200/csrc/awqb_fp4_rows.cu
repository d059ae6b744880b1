// Rows of 16-bit values to microscaled 4-bit floating point and back, and the
// residual-add RMSNorm that writes its result in four bits (awqb_fp4.cuh has the
// formats).
//
// All three are bound by HBM. A lane takes vectors of eight values (16-byte loads, whole
// sectors by neighbouring lanes), two of them at a time where it only quantises; all of a
// thread's loads are issued before the first is used. Launched with programmatic dependent
// launch, like the other norms. On a B200, 4096 bf16 rows of 14336: mxfp4 quantised in 24.4 us
// (6.1 TB/s), nvfp4 in 30.7 (4.9), read back in 26 (5.8); norms of 8192 values in 40.4 in mxfp4
// and 43.6 in nvfp4 (5.4 and 5.1 TB/s).
#include <cuda_runtime.h>

#include <algorithm>

#include "awqb200.h"
#include "awqb_common.h"
#include "awqb_ptx.cuh"
#include "awqb_vec.cuh"
#include "awqb_fp4.cuh"

namespace awqb {
namespace {

constexpr int kThreads = 256;

struct RowsArgs {
  const void* x;
  const float* scale;
  const int32_t *index, *count;
  void* codes;
  uint8_t* scales;
  int64_t ldx, rows_in, rows;
  int K, vecs, per_row;
};

// Threads (x: vectors, y: rows) of a CTA of about kThreads, and CTAs over a row.
struct Shape {
  int x, y, over;
};
inline Shape shape_of(int vecs) {
  Shape s;
  s.over = (vecs + kThreads - 1) / kThreads;
  s.x = ((vecs + s.over - 1) / s.over + 31) / 32 * 32;
  s.y = std::max(1, kThreads / s.x);
  return s;
}

// The largest magnitude of the 16-bit values of some words, NaN if one is.
template <typename T>
struct Most;
template <>
struct Most<__half> {
  static __device__ __forceinline__ uint32_t pair(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a & 0x7fff7fffu), "r"(b & 0x7fff7fffu));
    return r;
  }
};
template <>
struct Most<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pair(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a & 0x7fff7fffu), "r"(b & 0x7fff7fffu));
    return r;
  }
};

// kRows rows of a CTA's thread, blockDim.y apart, 16 values of each. The largest magnitude
// is taken of the 16-bit values, two at a time: multiplying by 1 / scale rounds, and
// rounding keeps the order.
template <typename T, bool kNv, int kRows>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const __grid_constant__ RowsArgs a) {
  grid_dep_wait();
  grid_dep_launch();
  const int v = blockIdx.y * blockDim.x + threadIdx.x;
  const int64_t row0 = (int64_t)blockIdx.x * (kRows * blockDim.y) + threadIdx.y;
  bool real[kRows];
  uint4 x[kRows][2];
  const int64_t limit = a.count != nullptr ? min(a.rows, (int64_t)*a.count) : a.rows;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int64_t row = row0 + i * blockDim.y;
    real[i] = row < limit && v < a.vecs;
    int64_t from = row;
    if (a.index != nullptr && real[i]) {
      from = a.index[row];
      real[i] = from >= 0;
      from = (uint32_t)from / (uint32_t)a.per_row;
    }
    real[i] = real[i] && from < a.rows_in;
    x[i][0] = x[i][1] = make_uint4(0u, 0u, 0u, 0u);
    if (real[i] && v * 16 < a.K) {
      const uint4* xp = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + from * a.ldx) + 2 * v;
      x[i][0] = xp[0];
      x[i][1] = xp[1];
    }
  }
  const float inv = kNv && a.scale != nullptr ? __frcp_rn(*a.scale) : 1.f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    float f[2][8], u[16];
    unpack_vec<T>(x[i][0], f[0]);
    unpack_vec<T>(x[i][1], f[1]);
    const uint4 p = x[i][0], q = x[i][1];
    const uint32_t m = Most<T>::pair(Most<T>::pair(Most<T>::pair(p.x, p.y), Most<T>::pair(p.z, p.w)),
                                     Most<T>::pair(Most<T>::pair(q.x, q.y), Most<T>::pair(q.z, q.w)));
    const float2 both = Pair<T>::unpack(m);
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      const float2 t = make_float2(f[j / 8][j % 8], f[j / 8][j % 8 + 1]), s = kNv ? mul2(t, make_float2(inv, inv)) : t;
      u[j] = s.x, u[j + 1] = s.y;
    }
    const float most = max_nan(both.x, both.y);
    store_vector<kNv, 2>(u, kNv ? most * inv : most, a.codes, a.scales, a.rows, row0 + i * blockDim.y, a.K, v, real[i]);
  }
}

struct BackArgs {
  const void* codes;
  const uint8_t* scales;
  const float* scale;
  void* out;
  int64_t ldo, rows;
  int K;
};

template <typename T, bool kNv, int kRows>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const __grid_constant__ BackArgs a) {
  grid_dep_wait();
  grid_dep_launch();
  const int v = blockIdx.y * blockDim.x + threadIdx.x;
  if (v * 8 >= a.K) return;
  const int64_t row0 = (int64_t)blockIdx.x * (kRows * blockDim.y) + threadIdx.y;
  uint32_t codes[kRows], byte[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int64_t row = row0 + i * blockDim.y;
    if (row < a.rows) {
      codes[i] = static_cast<const uint32_t*>(a.codes)[row * (a.K / 8) + v];
      byte[i] = a.scales[Vectors<kNv, 1>::at(a.rows, row, v)];
    }
  }
  const float scale = kNv && a.scale != nullptr ? *a.scale : 1.f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int64_t row = row0 + i * blockDim.y;
    if (row >= a.rows) return;
    const float s = scale_value<kNv>(byte[i]);
    float f[8];
    e2m1x8_values(codes[i], f);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = f[j] * s * scale;  // f * s is exact
    reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * a.ldo)[v] = pack_vec<T>(f);
  }
}

struct NormArgs {
  const void *x, *residual, *weight;
  const float* scale;
  void *residual_out, *codes;
  uint8_t* scales;
  int64_t ldx, ldr, ldro, rows;
  int K, vecs;
  float eps;
  double inv_K;
};

constexpr int kNormThreads = 512;
constexpr int kNormVec = 4;  // vectors per thread
constexpr int kNormMaxK = kNormThreads * kNormVec * 8;

// A CTA takes a row and holds it in registers between the sum of squares and the
// quantisation. h = x + residual is stored rounded; the norm is of the unrounded sum and
// goes into four bits with no rounding to 16 bits between. A code depends on which side of
// a border its value lies, so little is lost on the way: a thread adds its squares (at most
// 32) and a warp its lanes' sums in fp32, the warps' sums are added in 64 bits; the row's
// factor (over the tensor's scale) is kept as two fp32 numbers, and so is h * weight. h is
// rounded to fp32. A square goes through at most 8 + 4 + 5 additions in fp32, 2^-24 each: less
// than 2^-19.9 of the sum and half of that of its root. With h's rounding and the result's, what
// is quantised is within 2^-20 of the exact value.
// h of the thread's vector v, stored; returns its sum of squares.
template <typename T>
__device__ __forceinline__ float add_vector(const NormArgs& a, int64_t row, int v, const uint4& x, const uint4& r,
                                            float (&h)[8]) {
  unpack_vec<T>(x, h);
  if (a.residual != nullptr) {
    float f[8];
    unpack_vec<T>(r, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] += f[j];
    reinterpret_cast<uint4*>(static_cast<T*>(a.residual_out) + row * a.ldro)[v] = pack_vec<T>(h);
  }
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) ss += h[j] * h[j];
  return ss;
}

// 1 / x of a positive x, from the 64-bit approximation (within 2^-20) by two Newton steps.
// Every fp32 number is in its range, and it has no path of its own for the ends of the range:
// the rounded fp32 reciprocal does, and held up the rows' loads (4096 nvfp4 rows of 8192
// features: 50.7 us with it, 42.4 so).
__device__ __forceinline__ double inverse(float x) {
  double y;
  asm("rcp.approx.ftz.f64 %0, %1;" : "=d"(y) : "d"((double)x));
  y = fma(fma(-(double)x, y, 1.0), y, y);
  return fma(fma(-(double)x, y, 1.0), y, y);
}

// The row's mean square plus eps. Each warp adds the warps' sums for itself, so that one
// barrier is enough.
__device__ __forceinline__ double mean_square(const NormArgs& a, float ss, double eps, float* red) {
  const int warps = blockDim.x / 32, lane = threadIdx.x & 31;
  ss = warp_sum(ss);
  if (lane == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  double sum = (lane & 15) < warps ? (double)red[lane & 15] : 0.0;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return fma(sum, a.inv_K, eps);
}

// over / sqrt(m) as two fp32 numbers, the root from its fp32 approximation by one Newton
// step; over: 1 / scale.
__device__ __forceinline__ float2 row_factor(double m, double over) {
  const double y = (double)rsqrtf((float)m);
  const double f = fma(fma(-m * y, y, 1.0), 0.5 * y, y) * over;
  const float high = (float)f;
  return make_float2(high, (float)(f - (double)high));
}

template <typename T, bool kNv>
__device__ __forceinline__ void norm_vector(const NormArgs& a, int64_t row, int v, const float (&h)[8], const uint4& w,
                                            float2 factor) {
  float u[8] = {}, most = 0.f;
  if (v * 8 < a.K) {
    float f[8];
    unpack_vec<T>(w, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float p = h[j] * f[j], rest = fmaf(h[j], f[j], -p);
      u[j] = fmaf(p, factor.x, fmaf(rest, factor.x, p * factor.y));
      most = max_nan(most, fabsf(u[j]));
    }
  }
  store_vector<kNv, 1>(u, most, a.codes, a.scales, a.rows, row, a.K, v, v < a.vecs);
}

// (mxfp4, two vectors: registers for three CTAs to an SM, 4096 rows of 8192 features 45.2 -> 40.2
// us; nvfp4 is better off with two CTAs and 48 registers: 8192 rows of 4096 features 41.5, 42.1 with three.)
template <typename T, bool kNv, int kVec>
__global__ void __launch_bounds__(kNormThreads, kVec > 2 ? 1 : kVec == 2 && !kNv ? 3 : 2)
norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[2][kNormThreads / 32];
  grid_dep_wait();
  grid_dep_launch();
  const int64_t row = blockIdx.x;
  const int nvec = a.K / 8;
  const uint4* xp = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + row * a.ldx);
  const uint4* rp = reinterpret_cast<const uint4*>(static_cast<const T*>(a.residual) + row * a.ldr);
  double over = kNv && a.scale != nullptr ? inverse(*a.scale) : 1.0;
  uint4 x[kVec], r[kVec], w[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    if (v < nvec) {
      x[i] = xp[v];
      if (a.residual != nullptr) r[i] = rp[v];
    }
  }
  float h[kVec][8], ss = 0.f;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    if (v < nvec) {
      ss += add_vector<T>(a, row, v, x[i], r[i], h[i]);
    }
  }
  double m = mean_square(a, ss, a.eps, red[0]);
  if (__builtin_expect(!((float)m >= 0x1p-90f && (float)m <= 0x1p120f), 0)) {
    // bf16 reaches from 2^-133 to 2^128, where fp32 squares end at half of that: once more with h
    // times a power of two, which the quotient does not see. (The same branch for the whole row.)
    const float by = m < 1.0 ? 0x1p80f : 0x1p-80f;
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[i][j] *= by;
        if (i * blockDim.x + threadIdx.x < nvec) ss += h[i][j] * h[i][j];
      }
    }
    m = mean_square(a, ss, (double)a.eps * by * by, red[1]);
    if (m > 0x1p127) m = 1.0, over = 0.0;  // an infinity in the row: all else is 0
  }
  const float2 factor = row_factor(m, over);
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    if (v < nvec) w[i] = static_cast<const uint4*>(a.weight)[v];
    norm_vector<T, kNv>(a, row, v, h[i], w[i], factor);
  }
}

template <typename Kernel, typename A>
int launch(Kernel kernel, dim3 grid, dim3 threads, void* stream, const A& a) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = threads;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  AWQB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  return kOk;
}

// The row kernels' grid: CTAs of a shape, so many rows to a thread as leave every SM
// several CTAs.
constexpr int kQuantizeRows = 2, kBackRows = 4;
inline bool many_rows(const Shape& s, int64_t rows, int per_thread) {
  return rows * s.over >= (int64_t)8 * per_thread * s.y * device_sm_count();
}
inline dim3 grid_of(const Shape& s, int64_t rows, int per_thread) {
  return dim3((unsigned)((rows + s.y * per_thread - 1) / (s.y * per_thread)), (unsigned)s.over);
}

// kernel<T, kNv> of the dtype and format, with further template arguments behind.
#define AWQB_FP4_PICK(kernel, ...)                                                                  \
  (dtype == AWQB_DTYPE_F16 ? (nv ? kernel<__half, true __VA_ARGS__> : kernel<__half, false __VA_ARGS__>) \
                           : (nv ? kernel<__nv_bfloat16, true __VA_ARGS__> : kernel<__nv_bfloat16, false __VA_ARGS__>))

#define AWQB_FP4_CHECK(K, format, dtype, scale)                                                                     \
  AWQB_REQUIRE(format != AWQB_FP4_MX || scale == nullptr, kInvalidArgument, "mxfp4 has no scale but its blocks'");    \
  AWQB_REQUIRE(dtype == AWQB_DTYPE_F16 || dtype == AWQB_DTYPE_BF16, kInvalidArgument, "bad dtype %d", dtype);       \
  AWQB_REQUIRE(format == AWQB_FP4_NV || format == AWQB_FP4_MX, kInvalidArgument, "bad format %d", format);          \
  AWQB_REQUIRE(K > 0 && K % 32 == 0 && K <= (1 << 20), kInvalidArgument, "K=%lld must be a positive multiple of 32", \
               (long long)K);

}  // namespace
}  // namespace awqb

using namespace awqb;

extern "C" int awqb_fp4_quantize(const awqb_fp4_quantize_args* args, void* stream) {
  AWQB_REQUIRE(args != nullptr, kInvalidArgument, "args is null");
  const auto [x, rows_in, ldx, K, format, dtype, scale, index, per_row, count, rows, codes, scales] = *args;
  AWQB_FP4_CHECK(K, format, dtype, scale);
  AWQB_REQUIRE(rows >= 0 && rows <= 0x7fffffff && rows_in >= 0 && rows_in <= 0x7fffffff, kInvalidArgument,
               "too many rows (%lld)", (long long)rows);
  // (an empty index may have no address)
  AWQB_REQUIRE(index != nullptr || rows == rows_in || rows == 0, kInvalidArgument, "without an index, rows are those of x");
  AWQB_REQUIRE(per_row >= 1 && per_row <= 0x7fffffff, kInvalidArgument, "per_row must be at least 1");
  AWQB_REQUIRE(ldx >= K && ldx % 8 == 0, kInvalidArgument, "the row stride of x must be >= K and a multiple of 8");
  if (rows == 0) return kOk;
  AWQB_REQUIRE((x || rows_in == 0) && codes && scales, kInvalidArgument, "null pointer");
  AWQB_REQUIRE(aligned16(x) && aligned16(codes) && aligned16(scales), kInvalidArgument, "tensors must be 16-byte aligned");
  const bool nv = format == AWQB_FP4_NV;
  const int vecs = nv ? Vectors<true, 2>::count((int)K) : Vectors<false, 2>::count((int)K);
  const RowsArgs a = {x, scale, index, count, codes, scales, ldx, rows_in, rows, (int)K, vecs, (int)per_row};
  const Shape s = shape_of(vecs);
  const dim3 threads(s.x, s.y);
  if (many_rows(s, rows, kQuantizeRows))
    return launch(AWQB_FP4_PICK(quantize_kernel, , kQuantizeRows), grid_of(s, rows, kQuantizeRows), threads, stream, a);
  return launch(AWQB_FP4_PICK(quantize_kernel, , 1), grid_of(s, rows, 1), threads, stream, a);
}

extern "C" int awqb_fp4_dequantize(const awqb_fp4_dequantize_args* args, void* stream) {
  AWQB_REQUIRE(args != nullptr, kInvalidArgument, "args is null");
  const auto [codes, scales, rows, K, format, dtype, scale, out, ldo] = *args;
  AWQB_FP4_CHECK(K, format, dtype, scale);
  AWQB_REQUIRE(rows >= 0 && rows <= 0x7fffffff, kInvalidArgument, "too many rows (%lld)", (long long)rows);
  AWQB_REQUIRE(ldo >= K && ldo % 8 == 0, kInvalidArgument, "the row stride of out must be >= K and a multiple of 8");
  if (rows == 0) return kOk;
  AWQB_REQUIRE(codes && scales && out, kInvalidArgument, "null pointer");
  AWQB_REQUIRE(aligned16(codes) && aligned16(scales) && aligned16(out), kInvalidArgument,
               "tensors must be 16-byte aligned");
  const bool nv = format == AWQB_FP4_NV;
  const BackArgs a = {codes, scales, scale, out, ldo, rows, (int)K};
  const Shape s = shape_of((int)K / 8);
  const dim3 threads(s.x, s.y);
  if (many_rows(s, rows, kBackRows))
    return launch(AWQB_FP4_PICK(dequantize_kernel, , kBackRows), grid_of(s, rows, kBackRows), threads, stream, a);
  return launch(AWQB_FP4_PICK(dequantize_kernel, , 1), grid_of(s, rows, 1), threads, stream, a);
}

extern "C" int awqb_fp4_add_rmsnorm(const awqb_fp4_add_rmsnorm_args* args, void* stream) {
  AWQB_REQUIRE(args != nullptr, kInvalidArgument, "args is null");
  const auto [x, ldx, residual, ldr, weight, residual_out, ldro, rows, K, eps, format, dtype, scale, codes, scales] =
      *args;
  AWQB_FP4_CHECK(K, format, dtype, scale);
  AWQB_REQUIRE(K <= kNormMaxK, kInvalidArgument, "K=%lld: at most %d features are supported", (long long)K, kNormMaxK);
  AWQB_REQUIRE(rows >= 0 && rows <= 0x7fffffff, kInvalidArgument, "too many rows (%lld)", (long long)rows);
  AWQB_REQUIRE(ldx >= K && ldx % 8 == 0 && (residual == nullptr || (ldr >= K && ldr % 8 == 0 && ldro >= K && ldro % 8 == 0)),
               kInvalidArgument, "row strides must be >= K and multiples of 8");
  AWQB_REQUIRE(eps >= 0.f, kInvalidArgument, "eps must be >= 0");
  if (rows == 0) return kOk;
  AWQB_REQUIRE(x && weight && codes && scales && (residual_out != nullptr || residual == nullptr), kInvalidArgument,
               "null pointer");
  AWQB_REQUIRE(aligned16(x) && aligned16(residual) && aligned16(weight) && aligned16(residual_out) && aligned16(codes) &&
                   aligned16(scales),
               kInvalidArgument, "tensors must be 16-byte aligned");
  const bool nv = format == AWQB_FP4_NV;
  const int vecs = nv ? Vectors<true, 1>::count((int)K) : Vectors<false, 1>::count((int)K);
  const NormArgs a = {x, residual, weight, scale, residual_out, codes, scales, ldx, ldr, ldro, rows, (int)K, vecs, eps,
                      1.0 / (double)K};
  // Vectors per thread: many rows want small CTAs, more of them to an SM (8192 rows of 4096
  // features: 49.4 us with one, 41.8 with two; 16 rows of 2048: 2.15 and 2.56)
  const bool few = rows <= 2 * device_sm_count();
  const int per = vecs <= (few ? kNormThreads : 128) ? 1 : vecs <= 2 * kNormThreads ? 2 : 4;
  const dim3 grid((unsigned)rows), threads((vecs + per - 1) / per + 31 & ~31);
  if (per == 1) return launch(AWQB_FP4_PICK(norm_kernel, , 1), grid, threads, stream, a);
  if (per == 2) return launch(AWQB_FP4_PICK(norm_kernel, , 2), grid, threads, stream, a);
  return launch(AWQB_FP4_PICK(norm_kernel, , 4), grid, threads, stream, a);
}
