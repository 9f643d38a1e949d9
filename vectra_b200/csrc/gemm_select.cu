// gemm_select.cu: which kernel computes a matrix product of the
// transformer-block operators.
#include "block_common.cuh"
#include "gemm_rows.cuh"
#include "gemm_tc.cuh"

namespace vectra {
namespace {

// Tile shape and parts of a tensor-core product.
TcShape tc_shape(const GemmProblem& p) {
  const bool gated = p.epilogue == kEpiGated;
  const int64_t sms = device_sm_count();
  const int64_t n = gated ? 2 * p.N : p.N;
  auto tiles = [&](int64_t rows, int64_t cols) {
    return ((p.M + rows - 1) / rows) * ((n + cols - 1) / cols);
  };
  TcShape s;
  if (p.M > 128 && tiles(256, 256) >= sms / 2) {
    s.bn = 256;
    s.cg = 2;
    return s;
  }
  s.bn = gated || tiles(128, 128) >= sms / 2 || p.K >= 4096 ? 128 : 64;
  const int64_t t = tiles(128, s.bn);
  const int64_t steps = (p.K + 63) / 64 * p.segments;
  int64_t split = sms / t;
  if (split > steps / 8) split = steps / 8;
  if (split > 32) split = 32;
  s.split = int(split < 1 ? 1 : split);
  return s;
}

}  // namespace

cudaError_t run_gemm(const GemmProblem& p, Workspace& ws,
                     cudaStream_t stream) {
  if (p.M == 0 || p.N == 0) return cudaSuccess;
  if (gemm_rows_supports(p)) {
    if (ws.dry) return cudaSuccess;
    const cudaError_t e = launch_gemm_rows(p, stream);
    if (e == cudaSuccess) count_launches(1);
    return e;
  }
  if (gemm_tc_supports(p)) return run_gemm_tc(p, tc_shape(p), ws, stream);
  // Split the reduction when the output tiles leave SMs idle: enough parts
  // for one block per SM, at least 256 of the reduction each.
  const bool gated = p.epilogue == kEpiGated;
  const int64_t tiles = ((p.M + 127) / 128) * ((p.N + (gated ? 63 : 127)) /
                                               (gated ? 64 : 128));
  int64_t split = device_sm_count() / tiles;
  const int64_t most = p.K * p.segments / 256;
  if (split > most) split = most;
  if (split > 64) split = 64;
  if (split < 1) split = 1;
  float* partial = nullptr;
  if (split > 1)
    partial = static_cast<float*>(ws.take(
        size_t(split) * (gated ? 2 : 1) * p.M * p.N * sizeof(float)));
  if (ws.dry || ws.overflow) return cudaSuccess;
  cudaError_t e = launch_gemm_generic(p, int(split), partial, stream);
  if (e != cudaSuccess) return e;
  count_launches(1);
  if (split > 1) {
    e = launch_split_finish(p, int(split), partial, stream);
    if (e == cudaSuccess) count_launches(1);
  }
  return e;
}

}  // namespace vectra
