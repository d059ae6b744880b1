// Microscaled 4-bit floating point: e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
// negatives), 16 with an e4m3 scale and one fp32 scale for the tensor (nvfp4), or 32
// with a power of two (mxfp4, OCP MX v1.0). What the kernels share: the formats'
// numbers and the quantisation of a block.
//
// nvfp4: u = x * (1 / scale), both rounded to fp32; s = e4m3(min(max |u| / 6, 448));
// code = e2m1(u / s), 0 where s = 0. mxfp4: s = 2^(floor(log2 max |x|) - 2), at least
// 2^-127; code = e2m1(x / s), saturating. Roundings to nearest, ties to even. A block
// that holds an infinity or a NaN gets the scale NaN, so that it stays visible.
//
// The quotients decide as the real numbers do. u has 24 bits, a midpoint between two
// codes times s at most 7, so u is such a product or differs from it by an ulp of u at
// least; the quotient, rounded correctly to fp32, then falls on the same side of the
// midpoint, or on it. The same holds for max |u| / 6 and the midpoints of e4m3.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "awqb_vec.cuh"

namespace awqb {

// Scales of a row that stand side by side in a granule of 16 bytes.
constexpr int kGranule = 16;

// max that keeps a NaN (fmaxf drops it)
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Eight values to eight codes, the first in the lowest four bits.
__device__ __forceinline__ uint32_t e2m1x8(const float* v) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Eight codes to eight values.
__device__ __forceinline__ void e2m1x8_values(uint32_t codes, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 p = Pair<__half>::unpack(h[j]);
    v[2 * j] = p.x;
    v[2 * j + 1] = p.y;
  }
}

__device__ __forceinline__ uint32_t e4m3_byte(float s) {  // s >= 0, at most 448
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(s));
  return r & 0xffu;
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)byte));
  return Pair<__half>::unpack(h).x;
}
__device__ __forceinline__ float e8m0_value(uint32_t byte) {  // 255 is NaN, 0 is 2^-127
  return __uint_as_float(byte == 255u ? 0x7fc00000u : byte == 0u ? 0x00400000u : byte << 23);
}

template <bool kNv>
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return kNv ? e4m3_value(byte) : e8m0_value(byte);
}

// The scale of a block whose largest magnitude is `most` (NaN or infinite where the
// block holds one), as its byte.
template <bool kNv>
__device__ __forceinline__ uint32_t block_scale(float most) {
  if (!(most <= 3.402823466e38f)) return kNv ? 0x7fu : 0xffu;
  if (kNv) {  // most / 6, correctly rounded as in block_codes
    const float sixth = 1.f / 6.f, q = most * sixth;
    return e4m3_byte(fminf(fmaf(fmaf(-q, 6.f, most), sixth, q), 448.f));
  }
  const int e = (int)(__float_as_uint(most) >> 23) - 2;
  return (uint32_t)max(e, 0);
}

// 8 L values of a block over its scale, as codes.
template <bool kNv, int L>
__device__ __forceinline__ void block_codes(const float (&u)[8 * L], uint32_t byte, uint32_t (&codes)[L]) {
  float v[8 * L];
  const bool none = kNv ? byte == 0u || byte == 0x7fu : byte == 0xffu;
  if (kNv) {
    // u / s, correctly rounded: s has few bits, so one correction of u * (1 / s) is enough
    const float s = e4m3_value(byte), r = __frcp_rn(s);
    const float2 rr = make_float2(r, r), minus = make_float2(-s, -s);
#pragma unroll
    for (int j = 0; j < 8 * L; j += 2) {
      const float2 x = make_float2(u[j], u[j + 1]), y = mul2(x, rr), z = fma2(fma2(y, minus, x), rr, y);
      v[j] = z.x, v[j + 1] = z.y;
    }
  } else {
    // 1 / s = 2^(127 - byte); byte <= 252, so this is a normal number. The product is exact
    // (or far below the smallest value's half)
    const float r = __uint_as_float((254u - byte) << 23);
#pragma unroll
    for (int j = 0; j < 8 * L; ++j) v[j] = u[j] * r;
  }
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const uint32_t c = e2m1x8(v + 8 * i);
    codes[i] = none ? 0u : c;
  }
}

// A row is worked on in vectors of 8 L values, by neighbouring lanes: kBlock of them make
// a block. kPer vectors go with a granule of scales.
template <bool kNv, int L>
struct Vectors {
  static constexpr int kBlock = (kNv ? 2 : 4) / L;
  static constexpr int kPer = kBlock * kGranule;
  // of a row of K values, whole granules
  static __host__ __device__ constexpr int count(int K) { return (K / (8 * L) + kPer - 1) / kPer * kPer; }
  // the byte of vector v's scale, [granule][row][16]
  static __device__ __forceinline__ int64_t at(int64_t rows, int64_t row, int v) {
    const int i = v / kBlock;
    return ((int64_t)(i / kGranule) * rows + row) * kGranule + i % kGranule;
  }
};

// A vector's codes and, by the first of the lanes whose blocks' four scales make a word,
// those. All lanes of a warp; `most` is the vector's own largest magnitude.
template <bool kNv, int L>
__device__ __forceinline__ void store_vector(const float (&u)[8 * L], float most, void* codes, uint8_t* scales,
                                             int64_t rows, int64_t row, int K, int v, bool real) {
  using V = Vectors<kNv, L>;
#pragma unroll
  for (int o = 1; o < V::kBlock; o *= 2) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
  const bool inside = v * 8 * L < K;
  const uint32_t byte = inside ? block_scale<kNv>(most) : 0u;
  uint32_t w = byte << (8 * (v / V::kBlock % 4));
  w |= __shfl_xor_sync(0xffffffffu, w, V::kBlock);
  w |= __shfl_xor_sync(0xffffffffu, w, 2 * V::kBlock);
  if (!real) return;
  if (inside) {
    uint32_t c[L];
    block_codes<kNv, L>(u, byte, c);
    uint32_t* to = static_cast<uint32_t*>(codes) + row * (K / 8) + v * L;
    if (L == 2)
      *reinterpret_cast<uint2*>(to) = make_uint2(c[0], c[L - 1]);
    else
      *to = c[0];
  }
  if (v % (4 * V::kBlock) == 0) *reinterpret_cast<uint32_t*>(scales + V::at(rows, row, v)) = w;
}

}  // namespace awqb
