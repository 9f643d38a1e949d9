// residual_norm_f32.cu: the kernels of residual_norm_kernel.cuh for f32.
#include "residual_norm_kernel.cuh"

namespace vectra {

VECTRA_NORM_TYPE(float)

}  // namespace vectra
