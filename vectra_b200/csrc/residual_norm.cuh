// residual_norm.cuh: problem description of dropout and of the norms, gate and
// residual between two sublayers (residual_norm.cu).
#pragma once

#include "block_common.cuh"
#include "philox.cuh"

namespace vectra {

// Rows `ld` elements apart, whose elements are `inner` apart.
struct RowView {
  const void* p = nullptr;
  int64_t ld = 0, inner = 1;
  template <typename T>
  __device__ __forceinline__ const char* row(int64_t r) const {
    return reinterpret_cast<const char*>(static_cast<const T*>(p) + r * ld);
  }
};

struct NormProblem {
  int32_t dtype = VECTRA_F32;
  int32_t C = 0;
  int64_t M = 0;
  bool layer = false;
  float eps = 0.f, residual_scale = 1.f;
  Drop drop;
  RowView x, branch;  // backward: x is x_out
  RowView weight, bias, branch_weight, gate;
  int64_t gate_rows = 1;   // rows that share a gate row
  int64_t gate_count = 0;  // gate rows
  void* x_out = nullptr;
  void* y = nullptr;
  float* stats = nullptr;  // [M][4]
  // Backward: gradients of x_out (e) and y (f), and the results.
  RowView e, f;
  void* dx = nullptr;
  void* dbranch = nullptr;
  void* dweight = nullptr;
  void* dbias = nullptr;
  void* dbranch_weight = nullptr;
  void* dgate = nullptr;
  // Set at launch.
  int64_t units = 0, units_per_group = 1;
  int32_t unit_rows = 1;
  float* part[3] = {nullptr, nullptr, nullptr};
  float* gate_part = nullptr;
};

constexpr int kMaxNormCols = 16384;

cudaError_t launch_dropout(int32_t dtype, const RowView& x, int64_t rows,
                           int64_t cols, void* y, const Drop& drop,
                           cudaStream_t stream);
cudaError_t launch_norm_forward(const NormProblem& p, cudaStream_t stream);
cudaError_t run_norm_backward(const NormProblem& p, Workspace& ws,
                              cudaStream_t stream);

}  // namespace vectra
