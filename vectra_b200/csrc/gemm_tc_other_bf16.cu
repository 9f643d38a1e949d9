// gemm_tc_other_bf16.cu: tensor-core kernels, gated, bare and partial products, bf16.
#include "gemm_tc_kernel.cuh"

namespace vectra {

template cudaError_t launch_tc_other<__nv_bfloat16>(
    int epilogue, int bn, int cg, const CUtensorMap* maps, const TcArgs& g,
    cudaStream_t stream);

}  // namespace vectra
