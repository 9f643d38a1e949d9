// residual_norm_bf16.cu: the kernels of residual_norm_kernel.cuh for bf16.
#include "residual_norm_kernel.cuh"

namespace vectra {

VECTRA_NORM_TYPE(__nv_bfloat16)

}  // namespace vectra
