// The rotation of query and key heads at positions of several axes (qk_rope.cuh).
#include "qk_rope.cuh"

namespace tfo {

cudaError_t qk_rope_axes_launch(const HeadArgs& a, cudaStream_t st) { return launch_rope<true>(a, st); }

}  // namespace tfo
