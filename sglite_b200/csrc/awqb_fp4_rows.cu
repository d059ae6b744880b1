// Rows of 16-bit values to microscaled 4-bit floating point and back, and the
// residual-add RMSNorm that writes its result in four bits (awqb_fp4.cuh has the
// formats).
//
// All three are bound by HBM. A thread takes 16 values: two 16-byte loads, eight bytes
// of codes; four scales leave as one word.
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

// Threads of a row: one per 16 values, rounded up to whole granules of scales.
__host__ __device__ constexpr int items_of(int K, bool nv) {
  return nv ? (K + 255) / 256 * 16 : (K + 511) / 512 * 32;
}

struct RowsArgs {
  const void* x;
  const float* scale;
  const int32_t *index, *count;
  void* codes;
  uint8_t* scales;
  int64_t ldx, rows_in, rows;
  int K, items, per_row;
};

// Stores a thread's codes and, by the first of four (mxfp4: eight) neighbours, four scales.
template <bool kNv>
__device__ __forceinline__ void store_block(void* codes, uint8_t* scales, int64_t rows, int64_t row, int K, int item,
                                            uint2 c, uint32_t byte, bool real) {
  constexpr int kStep = kNv ? 1 : 2;
  uint32_t w = byte << (8 * (item / kStep % 4));
  w |= __shfl_xor_sync(0xffffffffu, w, kStep);
  w |= __shfl_xor_sync(0xffffffffu, w, 2 * kStep);
  if (!real) return;
  if (item * 16 < K) reinterpret_cast<uint2*>(codes)[row * (K / 16) + item] = c;
  if (item % (4 * kStep) == 0) *reinterpret_cast<uint32_t*>(scales + scale_at<kNv>(rows, row, item)) = w;
}

template <typename T, bool kNv>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const __grid_constant__ RowsArgs a) {
  grid_dep_wait();
  grid_dep_launch();
  const int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t row = t / a.items;
  const int item = (int)(t - row * a.items);
  int64_t from = row;
  bool real = row < a.rows && (a.count == nullptr || row < *a.count);
  if (real && a.index != nullptr) {
    from = a.index[row];
    real = from >= 0;
    from /= a.per_row;
  }
  real = real && from < a.rows_in;
  float u[16] = {}, most = 0.f;
  if (real && item * 16 < a.K) {
    const uint4* xp = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + from * a.ldx) + 2 * item;
    const uint4 x0 = xp[0], x1 = xp[1];
    float f[2][8];
    unpack_vec<T>(x0, f[0]);
    unpack_vec<T>(x1, f[1]);
    const float inv = kNv && a.scale != nullptr ? __frcp_rn(*a.scale) : 1.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      u[j] = f[j / 8][j % 8] * inv;
      most = max_nan(most, fabsf(u[j]));
    }
  }
  if (!kNv) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, 1));
  const uint32_t byte = item * 16 < a.K ? block_scale<kNv>(most) : 0u;
  store_block<kNv>(a.codes, a.scales, a.rows, row, a.K, item, block_codes<kNv>(u, byte), byte, real);
}

struct BackArgs {
  const void* codes;
  const uint8_t* scales;
  const float* scale;
  void* out;
  int64_t ldo, rows;
  int K;
};

template <typename T, bool kNv>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const __grid_constant__ BackArgs a) {
  grid_dep_wait();
  grid_dep_launch();
  const int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int items = a.K / 16;
  const int64_t row = t / items;
  const int item = (int)(t - row * items);
  if (row >= a.rows) return;
  const uint2 c = reinterpret_cast<const uint2*>(a.codes)[row * items + item];
  const float s = scale_value<kNv>(a.scales[scale_at<kNv>(a.rows, row, item)]);
  const float scale = kNv && a.scale != nullptr ? *a.scale : 1.f;
  uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * a.ldo) + 2 * item;
  float v[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    e2m1x8_values(h ? c.y : c.x, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] * s * scale;  // v * s is exact
    to[h] = pack_vec<T>(v);
  }
}

struct NormArgs {
  const void *x, *residual, *weight;
  const float* scale;
  void *residual_out, *codes;
  uint8_t* scales;
  int64_t ldx, ldr, ldro, rows;
  int K, items;
  float eps;
};

constexpr int kNormThreads = 512;
constexpr int kNormVec = 2;
constexpr int kNormMaxK = kNormThreads * kNormVec * 16;

// A CTA takes a row and holds it in registers between the sum of squares and the
// quantisation. h = x + residual is stored rounded; the norm is of the unrounded sum and
// goes from fp32 into four bits with no rounding between. The threads' sums of squares
// are added in 64 bits, so that a row's factor is right to its last bits: a block's
// codes then differ from the exact ones only within 2^-23 of a border.
template <typename T, bool kNv, int kVec>
__global__ void __launch_bounds__(kNormThreads, kVec == 1 ? 2 : 1) norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ double red[kNormThreads / 32];
  grid_dep_wait();
  grid_dep_launch();
  const int64_t row = blockIdx.x;
  const int nreal = a.K / 16;
  const T* xp = static_cast<const T*>(a.x) + row * a.ldx;
  const T* rp = static_cast<const T*>(a.residual) + row * a.ldr;
  float h[kVec][16];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int item = i * blockDim.x + threadIdx.x;
    if (item < nreal) {
      const uint4* xv = reinterpret_cast<const uint4*>(xp) + 2 * item;
      const uint4 x0 = xv[0], x1 = xv[1];
      float f[2][8];
      unpack_vec<T>(x0, f[0]);
      unpack_vec<T>(x1, f[1]);
      if (a.residual != nullptr) {
        const uint4* rv = reinterpret_cast<const uint4*>(rp) + 2 * item;
        const uint4 r0 = rv[0], r1 = rv[1];
        float r[2][8];
        unpack_vec<T>(r0, r[0]);
        unpack_vec<T>(r1, r[1]);
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j / 8][j % 8] += r[j / 8][j % 8];
        uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(a.residual_out) + row * a.ldro) + 2 * item;
        to[0] = pack_vec<T>(f[0]);
        to[1] = pack_vec<T>(f[1]);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        h[i][j] = f[j / 8][j % 8];
        ss += h[i][j] * h[i][j];
      }
    }
  }
  double sum = ss;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) sum += red[w];
  const float rms = (float)(1.0 / sqrt(sum / a.K + (double)a.eps));
  const float inv = kNv && a.scale != nullptr ? __frcp_rn(*a.scale) : 1.f;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int item = i * blockDim.x + threadIdx.x;
    float most = 0.f;
    if (item < nreal) {
      const uint4* wv = static_cast<const uint4*>(a.weight) + 2 * item;
      const uint4 w0 = wv[0], w1 = wv[1];
      float w[2][8];
      unpack_vec<T>(w0, w[0]);
      unpack_vec<T>(w1, w[1]);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        h[i][j] = h[i][j] * rms * w[j / 8][j % 8] * inv;
        most = max_nan(most, fabsf(h[i][j]));
      }
    }
    if (!kNv) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, 1));
    const uint32_t byte = item < nreal ? block_scale<kNv>(most) : 0u;
    store_block<kNv>(a.codes, a.scales, a.rows, row, a.K, item, block_codes<kNv>(h[i], byte), byte, item < a.items);
  }
}

template <typename Kernel, typename A>
int launch(Kernel kernel, const A& a, int64_t blocks, int threads, void* stream) {
  AWQB_REQUIRE(blocks <= 0x7fffffff, kUnsupported, "too many rows");
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  AWQB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  return kOk;
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
  AWQB_REQUIRE(index != nullptr || rows == rows_in, kInvalidArgument, "without an index, rows are those of x");
  AWQB_REQUIRE(per_row >= 1 && per_row <= 0x7fffffff, kInvalidArgument, "per_row must be at least 1");
  AWQB_REQUIRE(ldx >= K && ldx % 8 == 0, kInvalidArgument, "the row stride of x must be >= K and a multiple of 8");
  if (rows == 0) return kOk;
  AWQB_REQUIRE((x || rows_in == 0) && codes && scales, kInvalidArgument, "null pointer");
  AWQB_REQUIRE(aligned16(x) && aligned16(codes) && aligned16(scales), kInvalidArgument, "tensors must be 16-byte aligned");
  const bool nv = format == AWQB_FP4_NV;
  const int items = items_of((int)K, nv);
  const RowsArgs a = {x, scale, index, count, codes, scales, ldx, rows_in, rows, (int)K, items, (int)per_row};
  return launch(AWQB_FP4_PICK(quantize_kernel), a, (rows * items + kThreads - 1) / kThreads, kThreads, stream);
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
  return launch(AWQB_FP4_PICK(dequantize_kernel), a, (rows * (K / 16) + kThreads - 1) / kThreads, kThreads, stream);
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
  const int items = items_of((int)K, nv);
  const NormArgs a = {x, residual, weight, scale, residual_out, codes, scales, ldx, ldr, ldro, rows, (int)K, items, eps};
  if (items <= kNormThreads) return launch(AWQB_FP4_PICK(norm_kernel, , 1), a, rows, (items + 31) / 32 * 32, stream);
  return launch(AWQB_FP4_PICK(norm_kernel, , 2), a, rows, (items / 2 + 31) / 32 * 32, stream);
}
