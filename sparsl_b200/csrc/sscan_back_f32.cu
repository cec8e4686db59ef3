// The gradients of the selective scan for f32 tokens.
#include "sscan_back.cuh"

namespace sparsl {
cudaError_t launch_sscan_backward_f32(const SscanArgs& a, cudaStream_t s) { return by_states<float>(a, s); }
}  // namespace sparsl
