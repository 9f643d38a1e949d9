// gemm_tc_linear_f32.cu: tensor-core kernels, products with an epilogue, f32
// (operands in bf16 planes).
#include "gemm_tc_kernel.cuh"

namespace vectra {

template cudaError_t launch_tc_linear<float>(
    int bn, int cg, const CUtensorMap* maps, const TcArgs& g,
    cudaStream_t stream);

}  // namespace vectra
