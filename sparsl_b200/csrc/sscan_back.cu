// The gradients' workspace, and their entry by the tokens' type; each type's
// kernels are compiled by themselves (sscan_back_{f32,f16,bf16}.cu).
#include "sscan_back.cuh"

namespace sparsl {

size_t sscan_backward_bytes(uint64_t tokens, uint64_t channels, uint32_t states, uint64_t n_seq, uint32_t groups) {
  uint64_t most = 0;
  for (bool ragged : {false, true}) {
    const ScanPlan p = plan_of(tokens, (uint32_t)channels, states, n_seq, groups, ragged);
    const uint64_t b = back_work(p, tokens, (uint32_t)channels, states, groups, nullptr, nullptr);
    if (b > most) most = b;
  }
  return most;
}

ScanLayout sscan_backward_layout(uint64_t tokens, uint32_t channels, uint32_t states, uint64_t n_seq, uint32_t groups, bool ragged) {
  const ScanPlan p = plan_of(tokens, channels, states, n_seq, groups, ragged);
  const uint32_t padded = states <= 8 ? 8 : states <= 16 ? 16 : states <= 32 ? 32 : 64;
  return {p.lanes, p.chunks, p.len, p.carry, p.carry ? chunk_plan(p, channels, groups, padded).lanes : 0};
}

cudaError_t launch_sscan_backward(const SscanArgs& a, cudaStream_t s) {
  switch (a.type) {
    case SEQ_F32: return launch_sscan_backward_f32(a, s);
    case SEQ_F16: return launch_sscan_backward_f16(a, s);
    default: return launch_sscan_backward_bf16(a, s);
  }
}

}  // namespace sparsl
