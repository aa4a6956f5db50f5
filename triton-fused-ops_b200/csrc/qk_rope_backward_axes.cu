// Gradients of the per-head norm with the rotation at positions of several axes (qk_rope_backward.cuh).
#include "qk_rope_backward.cuh"

namespace tfo {

cudaError_t qk_norm_rope_backward_axes_launch(const HeadArgs& a, void* ws, cudaStream_t st) {
  return launch_backward<true>(a, ws, st);
}

}  // namespace tfo
