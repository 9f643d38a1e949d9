// gemm_rows.cuh: interface of the few-row products (gemm_rows.cu).
#pragma once

#include "block_common.cuh"

namespace vectra {

constexpr int64_t kRowsMost = 64;  // rows of x

// One product, operands in 16-byte aligned rows along the reduction, and few
// enough rows for the size.
bool gemm_rows_supports(const GemmProblem& p);
cudaError_t launch_gemm_rows(const GemmProblem& p, cudaStream_t stream);

}  // namespace vectra
