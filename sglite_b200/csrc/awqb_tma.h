// The driver's tensor-map encoder, looked up once (no link against libcuda).
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include "awqb_common.h"

namespace awqb {

// nullptr if the driver lacks it. Binds the current device's context to the calling
// thread if it is the thread's first call.
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

// A row-major matrix in boxes of box_rows x 128 bytes, 128-byte swizzle, zeros outside;
// ld in bytes, a multiple of 16.
inline int make_bytes_map(CUtensorMap* tm, CUtensorMapDataType type, int width, const void* base, int64_t rows,
                          int64_t row_bytes, int64_t ld, int box_rows) {
  const auto enc = tensor_map_encoder();
  AWQB_REQUIRE(enc != nullptr, kCudaError, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t dim[2] = {(cuuint64_t)(row_bytes / width), (cuuint64_t)rows};
  const cuuint64_t stride[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / width), (cuuint32_t)box_rows}, step[2] = {1, 1};
  const CUresult r = enc(tm, type, 2, const_cast<void*>(base), dim, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  AWQB_REQUIRE(r == CUDA_SUCCESS, kCudaError, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return kOk;
}

// Of 16-bit values: k and ld in elements.
inline int make_rows_map(CUtensorMap* tm, const void* base, int64_t rows, int64_t k, int64_t ld, int box_rows) {
  return make_bytes_map(tm, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, base, rows, 2 * k, 2 * ld, box_rows);
}

}  // namespace awqb
