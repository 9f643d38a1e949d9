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
  // x (backward: x_out), the branch, and in the backward pass the gradients of
  // x_out (e) and y (f).
  RowView x, branch, e, f;
  RowView weight, bias, branch_weight, gate;
  int64_t gate_rows = 1;   // rows that share a gate row
  int64_t gate_count = 0;  // gate rows
  void* x_out = nullptr;
  void* y = nullptr;
  float* stats = nullptr;  // [M][4]
  void* rest = nullptr;    // [M][C]: what x_out's rounding left
  // Backward's results.
  void* dx = nullptr;
  void* dbranch = nullptr;
  void* dweight = nullptr;
  void* dbias = nullptr;
  void* dbranch_weight = nullptr;
  void* dgate = nullptr;
  // Set at launch.
  int64_t units = 0, units_per_group = 1;
  int32_t unit_rows = 1;
  int32_t stages = 0;   // rows under way in shared memory
  int32_t tensors = 0;  // read row by row
  float* part[4] = {nullptr, nullptr, nullptr, nullptr};
  float* gate_part = nullptr;
};

constexpr int kMaxNormCols = 16384;

constexpr int kChunk = 8;  // columns a thread reads at once
constexpr int kNormVectors = 4;  // over the columns, the bias last

struct DropArgs {
  const void* x;
  void* y;
  int64_t rows, cols, ld, inner;  // x; y is contiguous
  Drop drop;
};

struct FinishArgs {
  const float* part[4];
  void* out[4];
  int64_t count;   // rows a sum
  int64_t groups;  // sums
  int C;
};

// A team's chunks a thread, its block, and the grid.
struct NormLaunch {
  int chunks;
  dim3 block;
  unsigned blocks;
  bool vec;         // rows in 16-byte pieces
  bool two_blocks;  // backward: two blocks an SM
  size_t bytes;     // of dynamic shared memory
};

// residual_norm_{bf16,f16,f32}.cu.
template <typename T>
cudaError_t dropout_typed(const DropArgs& a, bool vec, unsigned blocks,
                          cudaStream_t stream);
template <typename T>
cudaError_t norm_forward_typed(const NormProblem& p, const NormLaunch& how,
                               cudaStream_t stream);
template <typename T>
cudaError_t norm_backward_typed(const NormProblem& p, const NormLaunch& how,
                                cudaStream_t stream);
template <typename T>
cudaError_t norm_finish_typed(const FinishArgs& a, dim3 grid, int threads,
                              cudaStream_t stream);

cudaError_t launch_dropout(int32_t dtype, const RowView& x, int64_t rows,
                           int64_t cols, void* y, const Drop& drop,
                           cudaStream_t stream);
cudaError_t launch_norm_forward(const NormProblem& p, cudaStream_t stream);
cudaError_t run_norm_backward(const NormProblem& p, Workspace& ws,
                              cudaStream_t stream);

}  // namespace vectra
