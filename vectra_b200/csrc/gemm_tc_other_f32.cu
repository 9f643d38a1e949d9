// gemm_tc_other_f32.cu: tensor-core kernels, gated, bare and partial products, f32
// (operands in bf16 planes).
#include "gemm_tc_kernel.cuh"

namespace vectra {

template cudaError_t launch_tc_other<float>(
    int epilogue, int bn, int cg, const CUtensorMap* maps, const TcArgs& g,
    cudaStream_t stream);

}  // namespace vectra
