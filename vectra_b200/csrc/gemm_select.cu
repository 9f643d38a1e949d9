// gemm_select.cu: which kernel computes a matrix product of the
// transformer-block operators.
#include "block_common.cuh"

namespace vectra {

cudaError_t run_gemm(const GemmProblem& p, Workspace& ws,
                     cudaStream_t stream) {
  if (p.M == 0 || p.N == 0) return cudaSuccess;
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
