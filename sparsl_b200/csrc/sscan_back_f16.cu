// The gradients of the selective scan for f16 tokens.
#include "sscan_back.cuh"

namespace sparsl {
cudaError_t launch_sscan_backward_f16(const SscanArgs& a, cudaStream_t s) { return by_states<__half>(a, s); }
}  // namespace sparsl
