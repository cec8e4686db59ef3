// The selective state space scan.  For channel c with N states,
//
//   s = softplus(dt + dt_bias)        (or dt + dt_bias)
//   h[n] <- exp(s A[c, n]) h[n] + s B[n] x
//   y    =  sum_n C[n] h[n] + D[c] x,   times z sigmoid(z) where there is a gate
//
// token by token within each sequence.  A lane holds a channel's states in
// registers and walks the tokens: rows of x, dt, z are read once, coalesced
// over the channels; B and C are staged in shared memory for all lanes of a
// block.  Where channels and sequences do not fill the GPU the token axis is
// cut into chunks: a first pass computes the state each chunk hands on from
// zero and the sum of its steps (whose exponential is the chunk's decay), a
// fold over the chunks gives the state each starts from, and the main pass
// starts there.
#include "sscan.cuh"

namespace sparsl {
namespace {

constexpr int kAhead = 8;  // tokens loaded at a time

template <class T>
struct Raw3 {
  T x[kAhead], dt[kAhead], z[kAhead];
};

// B and (BOTH) C of the tokens of a tile from tb on that `live` names, as f32
// in shared memory; what does not exist is 0.
template <class T, int NP, bool BOTH>
__device__ __forceinline__ void stage_bc(const SscanArgs& a, uint32_t group, int64_t tb, uint32_t live,
                                         float (*sh)[2][NP]) {
  constexpr int kRows = BOTH ? 2 : 1;
  for (int i = threadIdx.x; i < kScanTile * kRows * NP; i += kScanThreads) {
    const uint32_t n = i % NP, which = i / NP % kRows, k = i / (NP * kRows);
    const int64_t t = tb + k;
    float v = 0.f;
    if ((live >> k & 1) && n < a.states) {
      const T* p = reinterpret_cast<const T*>(which ? a.c : a.b);
      v = to_f32(p[(uint64_t)t * (which ? a.c_stride : a.b_stride) + (uint64_t)group * (which ? a.c_group : a.b_group) + n]);
    }
    sh[k][which][n] = v;
  }
}

// One token of NS states: h <- a h + (s x) B.
template <int NS, bool FULL>
__device__ __forceinline__ void advance(float s, float sx, const float* b, const float (&a2)[NS], uint32_t n0, uint32_t N,
                                        float (&h)[NS]) {
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    float add = sx * b[j];
    if (!FULL && n0 + j >= N) add = 0.f;  // an infinite x must not reach a state that does not exist
    h[j] = __fmaf_rn(ex2(s * a2[j]), h[j], add);
  }
}

// The state that a chunk hands to the next one: its last sequence's, from that
// sequence's start in it or from zero.
template <class T, int NS, int LP, bool FULL>
__global__ void __launch_bounds__(kScanThreads) sscan_chunk_kernel(SscanArgs a, ScanPlan p, ScanWork w) {
  constexpr int NP = NS * LP;
  __shared__ __align__(16) float bc[kScanTile][2][NP];
  const uint32_t N = a.states;
  const ScanLane<NS, LP> me(a.channels, a.groups, p.per_group, blockIdx.x % p.ctiles);
  const int64_t chunk = blockIdx.x / p.ctiles;
  const int64_t t0 = chunk * (int64_t)p.len, t1 = min(t0 + (int64_t)p.len, (int64_t)a.seq.tokens);
  const int64_t seq = a.seq.of(t1 - 1);
  const bool any = seq >= 0 && seq < (int64_t)a.seq.n_seq;
  const int64_t begin = any ? a.seq.begin(seq) : 0, end = any ? a.seq.begin(seq + 1) : 0;
  const bool spans = any && end > t1 && begin < t1;
  if (threadIdx.x == 0 && blockIdx.x % p.ctiles == 0) w.cut[chunk] = !spans ? 2 : begin >= t0 ? 1 : 0;
  if (!spans) return;
  float h[NS], a2[NS];
  load_states<NS, FULL>(a.a + (uint64_t)me.c * N, me.n0, N, a2);
#pragma unroll
  for (int j = 0; j < NS; ++j) a2[j] *= kLog2e;
  zero_states(h);
  const uint64_t row = ((uint64_t)chunk * a.channels + me.c) * N;
  if (begin >= t0 && a.state) {
    const int64_t slot = a.seq.resumes(seq) ? a.seq.slot(seq) : -1;
    if (slot >= 0) load_states<NS, FULL>(a.state + ((uint64_t)slot * a.channels + me.c) * N, me.n0, N, h);
    if (w.start && me.valid) store_states<NS, FULL>(w.start + row, me.n0, N, h);
  }
  const float bias = a.dt_bias ? a.dt_bias[me.c] : 0.f;
  const T* x = reinterpret_cast<const T*>(a.x) + me.c;
  const T* dt = reinterpret_cast<const T*>(a.dt) + me.c;
  float sum = 0.f;
  for (int64_t tb = max(begin, t0); tb < t1; tb += kScanTile) {
    __syncthreads();
    stage_bc<T, NP, false>(a, me.group, tb, t1 - tb >= 32 ? ~0u : (1u << (t1 - tb)) - 1, bc);
    __syncthreads();
    for (int k = 0; k < kScanTile; k += kAhead) {
      T xr[kAhead], dr[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (tb + k + u < t1) {
          xr[u] = x[(uint64_t)(tb + k + u) * a.x_stride];
          dr[u] = dt[(uint64_t)(tb + k + u) * a.dt_stride];
        }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (tb + k + u >= t1) break;
        float s = to_f32(dr[u]) + bias;
        if (a.softplus) s = softplus(s);
        sum += s;
        advance<NS, FULL>(s, s * to_f32(xr[u]), &bc[k + u][0][me.n0], a2, me.n0, N, h);
      }
    }
  }
  if (me.valid) {
    store_states<NS, FULL>(w.state + row, me.n0, N, h);
    if (me.first) w.sum[(uint64_t)chunk * a.channels + me.c] = sum;
  }
}

// What each chunk starts from, in place of what it hands on: ascending for the
// states, descending (BACK) for their gradients.
template <bool BACK>
__global__ void __launch_bounds__(256) sscan_fold_kernel(const float* a, ScanWork w, uint64_t chunks, uint32_t channels,
                                                         uint32_t states) {
  const uint64_t cells = (uint64_t)channels * states;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= cells) return;
  const uint32_t c = i / states;
  const float a2 = a[i] * kLog2e;
  float carry = 0.f;
  constexpr int U = 8;
  for (uint64_t k = 0; k < chunks; k += U) {
    float v[U], s[U];
    int32_t cut[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u < chunks) {
        const uint64_t j = BACK ? chunks - 1 - (k + u) : k + u;
        v[u] = w.state[j * cells + i];
        s[u] = w.sum[j * channels + c];
        cut[u] = w.cut[j];
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u < chunks) {
        const uint64_t j = BACK ? chunks - 1 - (k + u) : k + u;
        w.state[j * cells + i] = carry;
        carry = cut[u] == 2 ? 0.f : cut[u] == 1 ? v[u] : __fmaf_rn(ex2(s[u] * a2), carry, v[u]);
      }
  }
}

// The main pass over one chunk.
template <class T, int NS, int LP, bool FULL>
__global__ void __launch_bounds__(kScanThreads) sscan_kernel(SscanArgs a, ScanPlan p, ScanWork w) {
  constexpr int NP = NS * LP;
  __shared__ __align__(16) float bc[kScanTile][2][NP];
  const uint32_t N = a.states;
  const ScanLane<NS, LP> me(a.channels, a.groups, p.per_group, blockIdx.x % p.ctiles);
  const int64_t chunk = blockIdx.x / p.ctiles;
  const int64_t t0 = chunk * (int64_t)p.len, t1 = min(t0 + (int64_t)p.len, (int64_t)a.seq.tokens);
  float h[NS], a2[NS];
  load_states<NS, FULL>(a.a + (uint64_t)me.c * N, me.n0, N, a2);
#pragma unroll
  for (int j = 0; j < NS; ++j) a2[j] *= kLog2e;
  zero_states(h);
  const uint64_t row = ((uint64_t)chunk * a.channels + me.c) * N;
  if (p.carry) load_states<NS, FULL>(w.state + row, me.n0, N, h);
  const float bias = a.dt_bias ? a.dt_bias[me.c] : 0.f;
  const float dskip = a.d ? a.d[me.c] : 0.f;
  const T* x = reinterpret_cast<const T*>(a.x) + me.c;
  const T* dt = reinterpret_cast<const T*>(a.dt) + me.c;
  const T* z = a.z ? reinterpret_cast<const T*>(a.z) + me.c : nullptr;
  T* y = reinterpret_cast<T*>(a.y) + me.c;

  for (int64_t tb = t0; tb < t1; tb += kScanTile) {
    const TileMarks m = tile_marks(a.seq, tb, t1);
    if (m.live == 0) continue;
    __syncthreads();
    stage_bc<T, NP, true>(a, me.group, tb, m.live, bc);
    __syncthreads();
    for (int k0 = 0; k0 < kScanTile; k0 += kAhead) {
      T xr[kAhead], dr[kAhead], zr[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (m.live >> (k0 + u) & 1) {
          const uint64_t t = (uint64_t)(tb + k0 + u);
          xr[u] = x[t * a.x_stride];
          dr[u] = dt[t * a.dt_stride];
          if (z) zr[u] = z[t * a.z_stride];
        }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int k = k0 + u;
        if (!(m.live >> k & 1)) continue;
        const int64_t t = tb + k;
        if (m.start >> k & 1) {
          const int64_t seq = tile_seq(m, k);
          zero_states(h);
          if (a.state) {
            const int64_t slot = a.seq.resumes(seq) ? a.seq.slot(seq) : -1;
            const bool saved = w.start && p.carry && a.seq.begin(seq + 1) > t1;
            if (saved) load_states<NS, FULL>(w.start + row, me.n0, N, h);
            else if (slot >= 0) load_states<NS, FULL>(a.state + ((uint64_t)slot * a.channels + me.c) * N, me.n0, N, h);
          }
        }
        if (a.marks && t % kMarkEvery == 0 && me.valid)
          store_states<NS, FULL>(a.marks + ((uint64_t)(t / kMarkEvery) * a.channels + me.c) * N, me.n0, N, h);
        const float xv = to_f32(xr[u]);
        float s = to_f32(dr[u]) + bias;
        if (a.softplus) s = softplus(s);
        advance<NS, FULL>(s, s * xv, &bc[k][0][me.n0], a2, me.n0, N, h);
        float o = 0.f;
#pragma unroll
        for (int j = 0; j < NS; ++j) o = __fmaf_rn(bc[k][1][me.n0 + j], h[j], o);
        o = sum_lanes<LP>(o);
        if (a.d) o = __fmaf_rn(dskip, xv, o);
        if (z) {
          const float zv = to_f32(zr[u]);
          o *= zv * sigmoid(zv);
        }
        if (me.valid && me.first) y[(uint64_t)t * a.y_stride] = from_f32<T>(o);
        if ((m.end >> k & 1) && a.final_state) {
          const int64_t slot = a.seq.slot(tile_seq(m, k));
          if (slot >= 0 && me.valid)
            store_states<NS, FULL>(a.final_state + ((uint64_t)slot * a.channels + me.c) * N, me.n0, N, h);
        }
      }
    }
  }
  if (!a.final_state || !me.valid) return;
  // Sequences without tokens end in the state they start from.
  const bool last = t1 >= (int64_t)a.seq.tokens;
  for (int64_t i = a.seq.first_from(t0); i < (int64_t)a.seq.n_seq; ++i) {
    const int64_t begin = a.seq.begin(i);
    if (begin >= t1 && !last) break;
    if (a.seq.begin(i + 1) > begin) continue;
    const int64_t slot = a.seq.slot(i);
    if (slot < 0) continue;
    zero_states(h);
    const uint64_t at = ((uint64_t)slot * a.channels + me.c) * N;
    if (a.state && a.seq.resumes(i)) load_states<NS, FULL>(a.state + at, me.n0, N, h);
    store_states<NS, FULL>(a.final_state + at, me.n0, N, h);
  }
}

// One token of each sequence: LP lanes share a channel, 4 states each, so a
// warp reads 512 contiguous bytes of states.
template <class T, int LP, bool FULL>
__global__ void __launch_bounds__(kScanThreads) sscan_step_kernel(SscanArgs a, uint32_t ctiles) {
  const uint32_t N = a.states;
  const int64_t i = blockIdx.x / ctiles;
  const uint32_t c = (blockIdx.x % ctiles) * (kScanThreads / LP) + threadIdx.x / LP;
  const uint32_t n0 = threadIdx.x % LP * 4;
  const int64_t slot = a.seq.slot(i);
  if (slot < 0) return;  // the whole block's
  const bool valid = c < a.channels;
  const uint32_t cc = valid ? c : a.channels - 1;
  float* st = a.final_state + ((uint64_t)slot * a.channels + cc) * N;
  float h[4], a2[4];
  load_states<4, FULL>(st, n0, N, h);
  load_states<4, FULL>(a.a + (uint64_t)cc * N, n0, N, a2);
  const uint32_t g = cc / (a.channels / a.groups);
  const T* b = reinterpret_cast<const T*>(a.b) + (uint64_t)i * a.b_stride + (uint64_t)g * a.b_group;
  const T* cv = reinterpret_cast<const T*>(a.c) + (uint64_t)i * a.c_stride + (uint64_t)g * a.c_group;
  const float xv = to_f32(reinterpret_cast<const T*>(a.x)[(uint64_t)i * a.x_stride + cc]);
  float s = to_f32(reinterpret_cast<const T*>(a.dt)[(uint64_t)i * a.dt_stride + cc]);
  const float zv = a.z ? to_f32(reinterpret_cast<const T*>(a.z)[(uint64_t)i * a.z_stride + cc]) : 0.f;
  if (a.dt_bias) s += a.dt_bias[cc];
  if (a.softplus) s = softplus(s);
  float o = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (FULL || n0 + j < N) {
      h[j] = __fmaf_rn(ex2(s * (a2[j] * kLog2e)), h[j], s * xv * to_f32(b[n0 + j]));
      o = __fmaf_rn(to_f32(cv[n0 + j]), h[j], o);
    }
  }
  o = sum_lanes<LP>(o);
  if (a.d) o = __fmaf_rn(a.d[cc], xv, o);
  if (a.z) o *= zv * sigmoid(zv);
  if (!valid) return;
  store_states<4, FULL>(st, n0, N, h);
  if (n0 == 0) reinterpret_cast<T*>(a.y)[(uint64_t)i * a.y_stride + c] = from_f32<T>(o);
}

bool aligned16(const void* p) { return reinterpret_cast<uint64_t>(p) % 16 == 0; }

// The states a lane holds: 16, or 8 where there are no more.
constexpr uint32_t lanes_of(uint32_t states) { return states <= 16 ? 1 : states <= 32 ? 2 : 4; }
constexpr uint32_t kWantedBlocks = kSms * 4;

ScanPlan plan_of(const SscanArgs& a) {
  return scan_plan(a.seq.tokens, a.channels, a.groups, a.seq.n_seq, a.seq.seq_ptr != nullptr,
                   kScanThreads / lanes_of(a.states), kWantedBlocks);
}

template <class T, int NS, int LP, bool FULL>
cudaError_t go(const SscanArgs& a, cudaStream_t s) {
  const ScanPlan p = plan_of(a);
  ScanWork w{};
  scan_work(p, a.channels, a.states, true, a.work, &w);
  if (a.state != a.final_state || !a.state) w.start = nullptr;
  const uint64_t grid = p.chunks * p.ctiles;
  if (grid > 0x7fffffffull) return cudaErrorInvalidValue;
  if (p.carry) {
    sscan_chunk_kernel<T, NS, LP, FULL><<<(unsigned)grid, kScanThreads, 0, s>>>(a, p, w);
    const uint64_t cells = (uint64_t)a.channels * a.states;
    sscan_fold_kernel<false><<<(unsigned)((cells + 255) / 256), 256, 0, s>>>(a.a, w, p.chunks, a.channels, a.states);
  }
  sscan_kernel<T, NS, LP, FULL><<<(unsigned)grid, kScanThreads, 0, s>>>(a, p, w);
  return cudaGetLastError();
}

template <class T, int LP, bool FULL>
cudaError_t go_step(const SscanArgs& a, cudaStream_t s) {
  const uint32_t per = kScanThreads / LP, ctiles = (a.channels + per - 1) / per;
  const uint64_t grid = a.seq.n_seq * ctiles;
  if (grid > 0x7fffffffull) return cudaErrorInvalidValue;
  sscan_step_kernel<T, LP, FULL><<<(unsigned)grid, kScanThreads, 0, s>>>(a, ctiles);
  return cudaGetLastError();
}

template <class T>
cudaError_t by_states(const SscanArgs& a, cudaStream_t s) {
  const uint32_t N = a.states;
  const bool al = aligned16(a.a) && aligned16(a.state) && aligned16(a.final_state) && aligned16(a.marks) && aligned16(a.work);
  if (N == 16 && al) return go<T, 16, 1, true>(a, s);
  if (N == 8 && al) return go<T, 8, 1, true>(a, s);
  if (N == 32 && al) return go<T, 16, 2, true>(a, s);
  if (N == 64 && al) return go<T, 16, 4, true>(a, s);
  if (N <= 8) return go<T, 8, 1, false>(a, s);
  if (N <= 16) return go<T, 16, 1, false>(a, s);
  if (N <= 32) return go<T, 16, 2, false>(a, s);
  return go<T, 16, 4, false>(a, s);
}

template <class T>
cudaError_t step_by_states(const SscanArgs& a, cudaStream_t s) {
  const uint32_t N = a.states;
  const bool al = aligned16(a.a) && aligned16(a.final_state);
  if (N == 16 && al) return go_step<T, 4, true>(a, s);
  if (N == 8 && al) return go_step<T, 2, true>(a, s);
  if (N == 32 && al) return go_step<T, 8, true>(a, s);
  if (N == 64 && al) return go_step<T, 16, true>(a, s);
  if (N <= 4) return go_step<T, 1, false>(a, s);
  if (N <= 8) return go_step<T, 2, false>(a, s);
  if (N <= 16) return go_step<T, 4, false>(a, s);
  if (N <= 32) return go_step<T, 8, false>(a, s);
  return go_step<T, 16, false>(a, s);
}

}  // namespace

size_t sscan_bytes(uint64_t tokens, uint64_t channels, uint32_t states, uint64_t n_seq, uint32_t groups) {
  uint64_t most = 0;
  for (bool ragged : {false, true}) {
    const ScanPlan p = scan_plan(tokens, (uint32_t)channels, groups, n_seq, ragged, kScanThreads / lanes_of(states), kWantedBlocks);
    if (!p.carry) continue;
    const uint64_t b = scan_work(p, (uint32_t)channels, states, true, nullptr, nullptr);
    if (b > most) most = b;
  }
  return most;
}

size_t sscan_mark_bytes(uint64_t tokens, uint64_t channels, uint32_t states) {
  return (tokens + kMarkEvery - 1) / kMarkEvery * channels * states * 4;
}

cudaError_t launch_sscan(const SscanArgs& a, cudaStream_t s) {
  switch (a.type) {
    case SEQ_F32: return by_states<float>(a, s);
    case SEQ_F16: return by_states<__half>(a, s);
    default: return by_states<__nv_bfloat16>(a, s);
  }
}

cudaError_t launch_sscan_step(const SscanArgs& a, cudaStream_t s) {
  switch (a.type) {
    case SEQ_F32: return step_by_states<float>(a, s);
    case SEQ_F16: return step_by_states<__half>(a, s);
    default: return step_by_states<__nv_bfloat16>(a, s);
  }
}

cudaError_t launch_sscan_fold_back(const float* a, const ScanWork& w, uint64_t chunks, uint32_t channels, uint32_t states,
                                   cudaStream_t s) {
  const uint64_t cells = (uint64_t)channels * states;
  sscan_fold_kernel<true><<<(unsigned)((cells + 255) / 256), 256, 0, s>>>(a, w, chunks, channels, states);
  return cudaGetLastError();
}

}  // namespace sparsl
