// Host services of the tensor-core GEMMs that several translation units share
// (defined in gemm.cu).
#pragma once

#include <cudaTypedefs.h>

#include "common.cuh"

namespace col {

// cuTensorMapEncodeTiled of the loaded driver, or null.
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

// Device-side status word of the bounded waits on device `dev`, or null.
unsigned* gemm_status_ptr(int dev);

}  // namespace col
