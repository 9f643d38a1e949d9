// qk_norm_rope_axes.cu: the RMS norm and rotation of query and key head
// vectors (qk_norm_rope_kernel.cuh) whose pairs take their position from one
// of several axes.
#include "qk_norm_rope_kernel.cuh"

namespace vectra {

cudaError_t launch_qk_forward_axes(const QkProblem& p, cudaStream_t stream) {
  return forward_with<true>(p, stream);
}
cudaError_t run_qk_backward_axes(const QkProblem& p, Workspace& ws,
                                 cudaStream_t stream) {
  return backward_with<true>(p, ws, stream);
}

}  // namespace vectra
