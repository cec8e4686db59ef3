// The selective scan and its step for bf16 tokens.
#include "sscan_fwd.cuh"

namespace sparsl {
cudaError_t launch_sscan_bf16(const SscanArgs& a, cudaStream_t s) { return by_states<__nv_bfloat16>(a, s); }
cudaError_t launch_sscan_step_bf16(const SscanArgs& a, cudaStream_t s) { return step_by_states<__nv_bfloat16>(a, s); }
}  // namespace sparsl
