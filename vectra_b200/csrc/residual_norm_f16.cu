// residual_norm_f16.cu: the kernels of residual_norm_kernel.cuh for f16.
#include "residual_norm_kernel.cuh"

namespace vectra {

VECTRA_NORM_TYPE(__half)

}  // namespace vectra
