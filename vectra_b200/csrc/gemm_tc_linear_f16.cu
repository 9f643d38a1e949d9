// gemm_tc_linear_f16.cu: tensor-core kernels, products with an epilogue, f16.
#include "gemm_tc_kernel.cuh"

namespace vectra {

template cudaError_t launch_tc_linear<__half>(
    int bn, int cg, const CUtensorMap* maps, const TcArgs& g,
    cudaStream_t stream);

}  // namespace vectra
