// gemm_tc.cuh: interface of the tensor-core matrix products (gemm_tc.cu).
#pragma once

#include "block_common.cuh"

namespace vectra {

// A launch shape: tile columns (accumulator columns; a gated tile has half
// as many outputs), CTAs per tile, and parts of the reduction.
struct TcShape {
  int bn = 256;  // 256, 128 or 64
  int cg = 1;    // 2 only with bn = 256
  int split = 1;
};

// bf16 / f16 products with a non-empty reduction, in any layout.
bool gemm_tc_supports(const GemmProblem& p);
cudaError_t run_gemm_tc(const GemmProblem& p, const TcShape& shape,
                        Workspace& ws, cudaStream_t stream);

}  // namespace vectra
