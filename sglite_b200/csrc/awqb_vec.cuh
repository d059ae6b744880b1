// Conversions between 16-byte vectors of fp16 / bf16 and fp32 registers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace awqb {

template <typename T>
__device__ __forceinline__ void unpack_vec(const uint4& u, float (&f)[8]) {
  const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (float)h[j];
}

template <typename T>
__device__ __forceinline__ uint4 pack_vec(const float (&f)[8]) {
  uint4 u;
  T* h = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int j = 0; j < 8; ++j) h[j] = (T)f[j];
  return u;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace awqb
