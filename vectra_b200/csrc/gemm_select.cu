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
  if (p.dtype != VECTRA_F32 && p.M > 128 && tiles(256, 256) >= sms / 2) {
    s.bn = 256;
    s.cg = 2;
    return s;
  }
  s.bn = gated || tiles(128, 128) >= sms / 2 || p.K >= 4096 ? 128 : 64;
  const int64_t t = tiles(128, s.bn);
  const int64_t steps =
      (p.K + 63) / 64 * p.segments * (p.dtype == VECTRA_F32 ? 6 : 1);
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
  if (p.K == 0) {
    if (ws.dry) return cudaSuccess;
    const cudaError_t e = launch_split_finish(p, 0, nullptr, stream);
    if (e == cudaSuccess) count_launches(1);
    return e;
  }
  if (gemm_rows_supports(p)) {
    if (ws.dry) return cudaSuccess;
    const cudaError_t e = launch_gemm_rows(p, stream);
    if (e == cudaSuccess) count_launches(1);
    return e;
  }
  return run_gemm_tc(p, tc_shape(p), ws, stream);
}

}  // namespace vectra
