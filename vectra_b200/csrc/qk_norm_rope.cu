// qk_norm_rope.cu: the RMS norm and rotation of query and key head vectors
// (qk_norm_rope_kernel.cuh), of positions on one axis; qk_norm_rope_axes.cu
// has the kernels of several.
#include "qk_norm_rope_kernel.cuh"

namespace vectra {

cudaError_t launch_qk_forward(const QkProblem& p, cudaStream_t stream) {
  return p.axes > 1 ? launch_qk_forward_axes(p, stream)
                    : forward_with<false>(p, stream);
}
cudaError_t run_qk_backward(const QkProblem& p, Workspace& ws,
                            cudaStream_t stream) {
  return p.axes > 1 ? run_qk_backward_axes(p, ws, stream)
                    : backward_with<false>(p, ws, stream);
}

}  // namespace vectra
