// The selective scan and its step for f16 tokens.
#include "sscan_fwd.cuh"

namespace sparsl {
cudaError_t launch_sscan_f16(const SscanArgs& a, cudaStream_t s) { return by_states<__half>(a, s); }
cudaError_t launch_sscan_step_f16(const SscanArgs& a, cudaStream_t s) { return step_by_states<__half>(a, s); }
}  // namespace sparsl
