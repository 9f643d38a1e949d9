// qk_norm_rope_axes.cu: the RMS norm and rotation of query and key head
// vectors (qk_norm_rope_kernel.cuh) whose pairs take their position from one
// of several axes. 9,220 tokens of 32 + 8 heads of 128 in bf16 (sections of
// 16, 24 and 24 pairs): 39.5 us, 189 MB at 4.8 TB/s. Training with 66,560
// tokens of 8 + 8 heads of 32 in f16, adjacent pairs, sections of 4, 6 and 6:
// forward 42 us (136 MB), backward 82 us and 8 for the weights' sums; there a
// section ends inside a thread's four pairs, each of which then reads its own
// entries (with the general kernel for such sections the pass took 3033 us).
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
