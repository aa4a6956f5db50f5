// Gradients of the per-head norm with the rotation at one position for each token (qk_rope_backward.cuh).
#include "qk_rope_backward.cuh"

namespace tfo {

size_t qk_norm_rope_backward_workspace_bytes(int head_dim) {
  return sizeof(float) * static_cast<size_t>(num_sms() * kBwdCtasPerSm + 1) * head_dim;
}

cudaError_t qk_norm_rope_backward_launch(const HeadArgs& a, void* ws, cudaStream_t st) {
  return a.t.axes > 1 ? qk_norm_rope_backward_axes_launch(a, ws, st) : launch_backward<false>(a, ws, st);
}

}  // namespace tfo
