// block_checks.cuh: argument checks and the workspace's two passes (sizing and
// running), shared by the C entries of the transformer-block operators.
#pragma once

#include "block_common.cuh"

namespace vectra {

inline bool io_dtype_ok(int32_t d) {
  return d == VECTRA_F32 || d == VECTRA_F16 || d == VECTRA_BF16;
}

// Checks one tensor: rank, sizes, dtype, and the pointer when it holds
// elements.
inline int check(const vectra_tensor& t, int32_t dtype,
                 std::initializer_list<int64_t> sizes) {
  if (t.ndim != int32_t(sizes.size())) return VECTRA_ERR_RANK;
  int64_t count = 1;
  int i = 0;
  for (const int64_t s : sizes) {
    if (t.size[i] != s) return VECTRA_ERR_SHAPE;
    count *= s;
    ++i;
  }
  if (t.dtype != dtype) return VECTRA_ERR_DTYPE;
  if (count > 0 && t.data == nullptr) return VECTRA_ERR_NULL;
  return VECTRA_OK;
}

// Results need a unit inner stride and rows that do not overlap.
inline int check_result(const vectra_tensor& t, int32_t dtype,
                        std::initializer_list<int64_t> sizes) {
  const int st = check(t, dtype, sizes);
  if (st != VECTRA_OK) return st;
  const int last = t.ndim - 1;
  if (t.size[last] > 1 && t.stride[last] != 1) return VECTRA_ERR_LAYOUT;
  if (t.ndim == 2 && t.size[0] > 1 && t.stride[0] < t.size[1])
    return VECTRA_ERR_LAYOUT;
  return VECTRA_OK;
}

inline bool present(const vectra_tensor& t) { return t.data != nullptr; }

#define VECTRA_TRY(expr)                 \
  do {                                   \
    const int st_ = (expr);              \
    if (st_ != VECTRA_OK) return st_;    \
  } while (0)

inline int to_status(cudaError_t e, const Workspace& ws) {
  if (ws.overflow) return VECTRA_ERR_WORKSPACE;
  return e == cudaSuccess ? VECTRA_OK : VECTRA_ERR_CUDA;
}

template <typename Args, typename F>
int run_with_workspace(const Args* a, void* stream, F&& f) {
  if (a == nullptr) return VECTRA_ERR_NULL;
  Workspace ws;
  ws.base = static_cast<char*>(a->workspace);
  ws.size = a->workspace ? a->workspace_bytes : 0;
  ws.dry = false;
  if (reinterpret_cast<uintptr_t>(ws.base) & 255) return VECTRA_ERR_WORKSPACE;
  // Size it first: nothing is launched when it does not fit.
  Workspace need;
  const int st = f(*a, need, nullptr);
  if (st != VECTRA_OK) return st;
  if (need.used > ws.size) return VECTRA_ERR_WORKSPACE;
  return f(*a, ws, static_cast<cudaStream_t>(stream));
}

template <typename Args, typename F>
int64_t workspace_of(const Args* a, F&& f) {
  if (a == nullptr) return VECTRA_ERR_NULL;
  Workspace need;
  const int st = f(*a, need, nullptr);
  return st != VECTRA_OK ? st : int64_t(need.used);
}

}  // namespace vectra
