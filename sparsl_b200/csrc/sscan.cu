// The scan's workspace, and its entries by the tokens' type; each type's kernels
// are compiled by themselves (sscan_{f32,f16,bf16}.cu).
#include "sscan_fwd.cuh"

namespace sparsl {

size_t sscan_bytes(uint64_t tokens, uint64_t channels, uint32_t states, uint64_t n_seq, uint32_t groups) {
  uint64_t most = 0;
  for (bool ragged : {false, true}) {
    const ScanPlan p = scan_plan(tokens, (uint32_t)channels, groups, n_seq, ragged, lanes_of(states));
    if (!p.carry) continue;
    const uint64_t b = scan_work(p, (uint32_t)channels, states, true, nullptr, nullptr);
    if (b > most) most = b;
  }
  return most;
}

size_t sscan_mark_bytes(uint64_t tokens, uint64_t channels, uint32_t states) {
  return (tokens + kMarkEvery - 1) / kMarkEvery * channels * states * 4;
}

ScanLayout sscan_layout(uint64_t tokens, uint32_t channels, uint32_t states, uint64_t n_seq, uint32_t groups, bool ragged) {
  const ScanPlan p = scan_plan(tokens, channels, groups, n_seq, ragged, lanes_of(states));
  return {p.lanes, p.chunks, p.len, p.carry, p.carry ? p.lanes : 0};
}

cudaError_t launch_sscan(const SscanArgs& a, cudaStream_t s) {
  switch (a.type) {
    case SEQ_F32: return launch_sscan_f32(a, s);
    case SEQ_F16: return launch_sscan_f16(a, s);
    default: return launch_sscan_bf16(a, s);
  }
}

cudaError_t launch_sscan_step(const SscanArgs& a, cudaStream_t s) {
  switch (a.type) {
    case SEQ_F32: return launch_sscan_step_f32(a, s);
    case SEQ_F16: return launch_sscan_step_f16(a, s);
    default: return launch_sscan_step_bf16(a, s);
  }
}

cudaError_t launch_sscan_fold_back(const float* a, const ScanWork& w, uint64_t chunks, uint32_t channels, uint32_t states,
                                   cudaStream_t s) {
  const uint64_t cells = (uint64_t)channels * states;
  sscan_fold_kernel<true><<<(unsigned)((cells + 127) / 128), 128, 0, s>>>(a, w, chunks, channels, states);
  return cudaGetLastError();
}

}  // namespace sparsl
