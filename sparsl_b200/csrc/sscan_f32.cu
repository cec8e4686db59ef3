// The selective scan and its step for f32 tokens.
#include "sscan_fwd.cuh"

namespace sparsl {
cudaError_t launch_sscan_f32(const SscanArgs& a, cudaStream_t s) { return by_states<float>(a, s); }
cudaError_t launch_sscan_step_f32(const SscanArgs& a, cudaStream_t s) { return step_by_states<float>(a, s); }
}  // namespace sparsl
