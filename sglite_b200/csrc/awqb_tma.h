// The driver's tensor-map encoder, looked up once (no link against libcuda).
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

namespace awqb {

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();  // nullptr if the driver lacks it

}  // namespace awqb
