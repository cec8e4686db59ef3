// The gradients of the selective scan for bf16 tokens.
#include "sscan_back.cuh"

namespace sparsl {
cudaError_t launch_sscan_backward_bf16(const SscanArgs& a, cudaStream_t s) { return by_states<__nv_bfloat16>(a, s); }
}  // namespace sparsl
