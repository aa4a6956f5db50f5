// Gradients of the per-head norm with the rotation at positions of several axes
// (qk_rope_backward.cuh), over rows joined beforehand where that is the faster way (qk_rope_axes.cu).
#include "qk_rope_backward.cuh"

namespace tfo {

cudaError_t qk_norm_rope_backward_axes_launch(const HeadArgs& a, void* ws, cudaStream_t st) {
  HeadArgs one = a;
  if (const cudaError_t e = join_axes(&one, true, st); e != cudaSuccess) return e;
  return one.t.axes > 1 ? launch_backward<true>(one, ws, st) : qk_norm_rope_backward_launch(one, ws, st);
}

}  // namespace tfo
