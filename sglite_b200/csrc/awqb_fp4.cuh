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
  if (kNv) return e4m3_byte(fminf(__fdiv_rn(most, 6.f), 448.f));
  const int e = (int)(__float_as_uint(most) >> 23) - 2;
  return (uint32_t)max(e, 0);
}

// 16 values of one block (mxfp4: half of one) over its scale, as codes.
template <bool kNv>
__device__ __forceinline__ uint2 block_codes(const float (&u)[16], uint32_t byte) {
  float v[16];
  if (kNv) {
    if (byte == 0u || byte == 0x7fu) return make_uint2(0u, 0u);
    // u / s, correctly rounded: s has few bits, so one correction of u * (1 / s) is enough
    const float s = e4m3_value(byte), r = __frcp_rn(s);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float y = u[j] * r;
      v[j] = fmaf(fmaf(-y, s, u[j]), r, y);
    }
  } else {
    if (byte == 0xffu) return make_uint2(0u, 0u);
    // 1 / s = 2^(127 - byte); byte <= 252, so this is a normal number. The product is exact
    // (or far below the smallest value's half)
    const float r = __uint_as_float((254u - byte) << 23);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = u[j] * r;
  }
  return make_uint2(e2m1x8(v), e2m1x8(v + 8));
}

// Where the scales of a row's 16 values number `item` (of 16) stand: granules of 16
// bytes, [granule][row][16]. mxfp4: the second half of a block shares the first one's.
template <bool kNv>
__device__ __forceinline__ int64_t scale_at(int64_t rows, int64_t row, int item) {
  const int i = kNv ? item : item >> 1;
  return ((int64_t)(i / kGranule) * rows + row) * kGranule + i % kGranule;
}

}  // namespace awqb
