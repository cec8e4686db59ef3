// Gradients of the selective scan.  With e_t = exp(s_t A), dy the gradient
// behind the gate, and r_t the gradient that h_t receives from later tokens,
//
//   g_t = r_t + C_t dy_t          r_{t-1} = e_t g_t
//   dx = D dy + s (g . B)         ds = sum_n g (A e h_{t-1} + B x)
//   dA = sum_t g e h_{t-1} s      dB = sum_c g s x       dC = sum_c dy h
//
// The forward pass saved the states before every kMarkEvery-th token.  A block
// of that many tokens is recomputed forwards from its mark with the decays and
// states kept in registers, and then walked backwards, so each exponential is
// computed once.  Chunks of the token axis run in parallel as in the forward
// pass: the gradient each chunk hands to the one before it is computed first,
// and folded.  dB and dC are summed over a warp's channels by exchanges that
// halve what a lane holds, over a block's warps in shared memory, and over the
// blocks' partial rows in a fixed order, so that results do not change from run
// to run; so are dA, dD and the step bias's gradient over the chunks.
#include "sscan.cuh"

namespace sparsl {

cudaError_t launch_sscan_fold_back(const float* a, const ScanWork& w, uint64_t chunks, uint32_t channels, uint32_t states,
                                   cudaStream_t s);

namespace {

constexpr int kWarps = kScanThreads / 32;

struct BackWork {
  ScanWork scan;
  float* da;  // [chunks, channels, states]
  float* dd;  // [chunks, 2, channels]: dD, then the step bias's
  float* bc;  // [channel tiles of a group, tokens, groups, 2, states]
};

__device__ __forceinline__ float gate_grad(float z, float sig) { return sig * __fmaf_rn(z, 1.0f - sig, 1.0f); }

// The gradient that a chunk hands to the state before it, from the end of the
// sequence that reaches into it, or from zero at its own end.
template <class T, int NS, int LP, bool FULL>
__global__ void __launch_bounds__(kScanThreads) sscan_chunk_back_kernel(SscanArgs a, ScanPlan p, ScanWork w) {
  constexpr int NP = NS * LP;
  constexpr int U = 8;
  __shared__ __align__(16) float sc[kScanTile][NP];
  const uint32_t N = a.states;
  const ScanLane<NS, LP> me(a.channels, a.groups, p.per_group, blockIdx.x % p.ctiles);
  const int64_t chunk = blockIdx.x / p.ctiles;
  const int64_t t0 = chunk * (int64_t)p.len, t1 = min(t0 + (int64_t)p.len, (int64_t)a.seq.tokens);
  const int64_t seq = a.seq.of(t0);
  const bool any = seq >= 0 && seq < (int64_t)a.seq.n_seq;
  const int64_t begin = any ? a.seq.begin(seq) : 0, end = any ? a.seq.begin(seq + 1) : 0;
  const bool spans = any && begin < t0 && end > t0;
  if (threadIdx.x == 0 && blockIdx.x % p.ctiles == 0) w.cut[chunk] = !spans ? 2 : end <= t1 ? 1 : 0;
  if (!spans) return;
  const int64_t hi = min(end, t1);
  float r[NS], a2[NS];
  load_states<NS, FULL>(a.a + (uint64_t)me.c * N, me.n0, N, a2);
#pragma unroll
  for (int j = 0; j < NS; ++j) a2[j] *= kLog2e;
  zero_states(r);
  if (end <= t1 && a.dfinal) {
    const int64_t slot = a.seq.slot(seq);
    if (slot >= 0) load_states<NS, FULL>(a.dfinal + ((uint64_t)slot * a.channels + me.c) * N, me.n0, N, r);
  }
  const float bias = a.dt_bias ? a.dt_bias[me.c] : 0.f;
  const T* dt = reinterpret_cast<const T*>(a.dt) + me.c;
  const T* dy = reinterpret_cast<const T*>(a.dy) + me.c;
  const T* z = a.z ? reinterpret_cast<const T*>(a.z) + me.c : nullptr;
  const T* cp = reinterpret_cast<const T*>(a.c) + (uint64_t)me.group * a.c_group;
  float sum = 0.f;
  for (int64_t te = hi; te > t0; te -= kScanTile) {  // tokens te - 1 down to te - kScanTile
    __syncthreads();
    for (int i = threadIdx.x; i < kScanTile * NP; i += kScanThreads) {
      const uint32_t n = i % NP, k = i / NP;
      const int64_t t = te - 1 - (int64_t)k;
      sc[k][n] = t >= t0 && n < N ? to_f32(cp[(uint64_t)t * a.c_stride + n]) : 0.f;
    }
    __syncthreads();
    for (int k = 0; k < kScanTile; k += U) {
      T dr[U], gr[U], zr[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t t = te - 1 - (k + u);
        if (t >= t0) {
          dr[u] = dt[(uint64_t)t * a.dt_stride];
          gr[u] = dy[(uint64_t)t * a.dy_stride];
          if (z) zr[u] = z[(uint64_t)t * a.z_stride];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (te - 1 - (k + u) < t0) break;
        float s = to_f32(dr[u]) + bias;
        if (a.softplus) s = softplus(s);
        sum += s;
        float g = to_f32(gr[u]);
        if (z) {
          const float zv = to_f32(zr[u]);
          g *= zv * sigmoid(zv);
        }
#pragma unroll
        for (int j = 0; j < NS; ++j) r[j] = ex2(s * a2[j]) * __fmaf_rn(sc[k + u][me.n0 + j], g, r[j]);
      }
    }
  }
  if (!me.valid) return;
  store_states<NS, FULL>(w.state + ((uint64_t)chunk * a.channels + me.c) * N, me.n0, N, r);
  if (me.first) w.sum[(uint64_t)chunk * a.channels + me.c] = sum;
}

// v[i] summed over the lanes that hold the same states of other channels; the
// lane keeps the sums of `kept` of its states from index `at` on.
template <int NS, int LP>
struct LaneSum {
  static constexpr int rounds() {
    int r = 0;
    for (int o = 16, cnt = NS; o >= LP && cnt > 1; o >>= 1, cnt /= 2) ++r;
    return r;
  }
  static constexpr int kept = NS >> rounds();
  uint32_t at;
  bool writes;
  __device__ __forceinline__ LaneSum() {
    const uint32_t lane = threadIdx.x & 31;
    at = 0;
    writes = true;
    int cnt = NS;
#pragma unroll
    for (int o = 16; o >= LP; o >>= 1) {
      if (cnt > 1) {
        cnt /= 2;
        if (lane & o) at += cnt;
      } else if (lane & o) {
        writes = false;
      }
    }
  }
  __device__ __forceinline__ void operator()(float (&v)[NS]) const {
    const uint32_t lane = threadIdx.x & 31;
    int cnt = NS;
#pragma unroll
    for (int o = 16; o >= LP; o >>= 1) {
      if (cnt > 1) {
        cnt /= 2;
        const bool up = lane & o;
#pragma unroll
        for (int j = 0; j < NS / 2; ++j) {
          if (j < cnt) {
            const float send = up ? v[j] : v[j + cnt], keep = up ? v[j + cnt] : v[j];
            v[j] = keep + __shfl_xor_sync(0xffffffffu, send, o);
          }
        }
      } else {
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
      }
    }
  }
};

template <class T, int NS, int LP, bool FULL>
__global__ void __launch_bounds__(kScanThreads) sscan_back_kernel(SscanArgs a, ScanPlan p, BackWork w) {
  constexpr int NP = NS * LP, K = (int)kMarkEvery;
  using Sum = LaneSum<NS, LP>;
  __shared__ __align__(16) float bc[kScanTile][2][NP];
  __shared__ float red[2][kWarps][K][2][NP];
  const uint32_t N = a.states;
  const ScanLane<NS, LP> me(a.channels, a.groups, p.per_group, blockIdx.x % p.ctiles);
  const int64_t chunk = blockIdx.x / p.ctiles;
  const int64_t t0 = chunk * (int64_t)p.len, t1 = min(t0 + (int64_t)p.len, (int64_t)a.seq.tokens);
  const uint32_t warp = threadIdx.x >> 5;
  const Sum lane_sum;
  float a2[NS], r[NS], da[NS];
  load_states<NS, FULL>(a.a + (uint64_t)me.c * N, me.n0, N, a2);
#pragma unroll
  for (int j = 0; j < NS; ++j) a2[j] *= kLog2e;
  zero_states(r);
  zero_states(da);
  const uint64_t row = ((uint64_t)chunk * a.channels + me.c) * N;
  if (p.carry && me.valid) load_states<NS, FULL>(w.scan.state + row, me.n0, N, r);
  const float bias = a.dt_bias ? a.dt_bias[me.c] : 0.f;
  const float dskip = a.d ? a.d[me.c] : 0.f;
  float dd = 0.f, dbias = 0.f;
  const T* x = reinterpret_cast<const T*>(a.x) + me.c;
  const T* dt = reinterpret_cast<const T*>(a.dt) + me.c;
  const T* dy = reinterpret_cast<const T*>(a.dy) + me.c;
  const T* z = a.z ? reinterpret_cast<const T*>(a.z) + me.c : nullptr;
  T* dx = reinterpret_cast<T*>(a.dx) + me.c;
  T* ddt = reinterpret_cast<T*>(a.ddt) + me.c;
  T* dz = a.z ? reinterpret_cast<T*>(a.dz) + me.c : nullptr;
  int buf = 0;

  const int64_t tiles = (t1 - t0 + kScanTile - 1) / kScanTile;
  for (int64_t tile = tiles - 1; tile >= 0; --tile) {
    const int64_t tb = t0 + tile * kScanTile;
    const TileMarks m = tile_marks(a.seq, tb, t1);
    if (m.live == 0) continue;
    __syncthreads();
    for (int i = threadIdx.x; i < kScanTile * 2 * NP; i += kScanThreads) {
      const uint32_t n = i % NP, which = i / NP & 1, k = i / (NP * 2);
      const int64_t t = tb + k;
      float v = 0.f;
      if ((m.live >> k & 1) && n < N) {
        const T* q = reinterpret_cast<const T*>(which ? a.c : a.b);
        v = to_f32(q[(uint64_t)t * (which ? a.c_stride : a.b_stride) + (uint64_t)me.group * (which ? a.c_group : a.b_group) + n]);
      }
      bc[k][which][n] = v;
    }
    __syncthreads();
    for (int k0 = kScanTile - K; k0 >= 0; k0 -= K) {
      const uint32_t live = m.live >> k0 & ((1u << K) - 1);
      if (!live) continue;
      float xv[K], sv[K], up[K], gv[K], slope[K];
      float hp[K][NS], e[K][NS], h[NS];
      // Forwards from the mark.
      zero_states(h);
      if ((live & 1) && me.valid)
        load_states<NS, FULL>(a.marks + ((uint64_t)((tb + k0) / K) * a.channels + me.c) * N, me.n0, N, h);
      float zv[K];
#pragma unroll
      for (int u = 0; u < K; ++u) {
        xv[u] = sv[u] = up[u] = zv[u] = 0.f;
        if ((live >> u & 1) && me.valid) {
          const uint64_t t = (uint64_t)(tb + k0 + u);
          xv[u] = to_f32(x[t * a.x_stride]);
          sv[u] = to_f32(dt[t * a.dt_stride]) + bias;
          up[u] = to_f32(dy[t * a.dy_stride]);
          if (z) zv[u] = to_f32(z[t * a.z_stride]);
        }
      }
#pragma unroll
      for (int u = 0; u < K; ++u) {
        const int k = k0 + u;
        slope[u] = 1.f;
        if (a.softplus) {
          slope[u] = sigmoid(sv[u]);
          sv[u] = softplus(sv[u]);
        }
        if ((m.start >> k & 1) && u) {
          zero_states(h);
          const int64_t slot = a.state ? a.seq.slot(tile_seq(m, k)) : -1;
          if (slot >= 0 && me.valid)
            load_states<NS, FULL>(a.state + ((uint64_t)slot * a.channels + me.c) * N, me.n0, N, h);
        }
        const float sx = sv[u] * xv[u];
        float o = 0.f;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          hp[u][j] = h[j];
          e[u][j] = ex2(sv[u] * a2[j]);
          float add = sx * bc[k][0][me.n0 + j];
          if (!FULL && me.n0 + j >= N) add = 0.f;
          h[j] = __fmaf_rn(e[u][j], h[j], add);
          o = __fmaf_rn(bc[k][1][me.n0 + j], h[j], o);
        }
        if (z) {
          o = sum_lanes<LP>(o);
          if (a.d) o = __fmaf_rn(dskip, xv[u], o);
          const float sig = sigmoid(zv[u]);
          if ((live >> u & 1) && me.valid && me.first)
            dz[(uint64_t)(tb + k) * a.dz_stride] = from_f32<T>(up[u] * o * gate_grad(zv[u], sig));
          up[u] *= zv[u] * sig;
        }
        gv[u] = up[u];
        float v[NS];
#pragma unroll
        for (int j = 0; j < NS; ++j) v[j] = gv[u] * h[j];
        lane_sum(v);
        if (lane_sum.writes)
#pragma unroll
          for (int j = 0; j < Sum::kept; ++j) red[buf][warp][u][1][me.n0 + lane_sum.at + j] = v[j];
      }
      // Backwards.
#pragma unroll
      for (int u = K - 1; u >= 0; --u) {
        const int k = k0 + u;
        if (m.end >> k & 1) {
          zero_states(r);
          const int64_t slot = a.dfinal ? a.seq.slot(tile_seq(m, k)) : -1;
          if (slot >= 0 && me.valid)
            load_states<NS, FULL>(a.dfinal + ((uint64_t)slot * a.channels + me.c) * N, me.n0, N, r);
        }
        const float sx = sv[u] * xv[u];
        float gb = 0.f, ga = 0.f, v[NS];
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          const float g = __fmaf_rn(bc[k][1][me.n0 + j], gv[u], r[j]);
          gb = __fmaf_rn(g, bc[k][0][me.n0 + j], gb);
          r[j] = e[u][j] * g;
          const float through = r[j] * hp[u][j];
          ga = __fmaf_rn(through, a2[j], ga);
          da[j] = __fmaf_rn(through, sv[u], da[j]);
          v[j] = g * sx;
        }
        lane_sum(v);
        if (lane_sum.writes)
#pragma unroll
          for (int j = 0; j < Sum::kept; ++j) red[buf][warp][u][0][me.n0 + lane_sum.at + j] = v[j];
        gb = sum_lanes<LP>(gb);
        ga = sum_lanes<LP>(ga);
        if (live >> u & 1) {
          const float ds = __fmaf_rn(ga, 1.0f / kLog2e, xv[u] * gb) * slope[u];
          dd = __fmaf_rn(gv[u], xv[u], dd);
          dbias += ds;
          if (me.valid && me.first) {
            const uint64_t t = (uint64_t)(tb + k);
            dx[t * a.dx_stride] = from_f32<T>(__fmaf_rn(dskip, gv[u], sv[u] * gb));
            ddt[t * a.ddt_stride] = from_f32<T>(ds);
          }
        }
        if ((m.start >> k & 1) && a.dstate) {
          const int64_t slot = a.seq.slot(tile_seq(m, k));
          if (slot >= 0 && me.valid)
            store_states<NS, FULL>(a.dstate + ((uint64_t)slot * a.channels + me.c) * N, me.n0, N, r);
        }
        if (m.start >> k & 1) zero_states(r);  // rows in front of it belong to no sequence, or end one
      }
      __syncthreads();
      for (int i = threadIdx.x; i < K * 2 * NP; i += kScanThreads) {
        const uint32_t n = i % NP, which = i / NP & 1, u = i / (2 * NP);
        if (n >= N || !(live >> u & 1)) continue;
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < kWarps; ++q) s += red[buf][q][u][which][n];
        const uint64_t t = (uint64_t)(tb + k0 + u);
        w.bc[((((uint64_t)me.channel_tile * a.seq.tokens + t) * a.groups + me.group) * 2 + which) * N + n] = s;
      }
      buf ^= 1;  // the next block of tokens writes the other one while this is read
    }
  }
  if (!me.valid) return;
  store_states<NS, FULL>(w.da + row, me.n0, N, da);
  if (me.first) {
    w.dd[(uint64_t)chunk * 2 * a.channels + me.c] = dd;
    w.dd[((uint64_t)chunk * 2 + 1) * a.channels + me.c] = dbias;
  }
  if (!a.dstate) return;
  // Sequences without tokens hand their final state's gradient on.
  const bool last = t1 >= (int64_t)a.seq.tokens;
  for (int64_t i = a.seq.first_from(t0); i < (int64_t)a.seq.n_seq; ++i) {
    const int64_t begin = a.seq.begin(i);
    if (begin >= t1 && !last) break;
    if (a.seq.begin(i + 1) > begin) continue;
    const int64_t slot = a.seq.slot(i);
    if (slot < 0) continue;
    zero_states(r);
    const uint64_t at = ((uint64_t)slot * a.channels + me.c) * N;
    if (a.dfinal) load_states<NS, FULL>(a.dfinal + at, me.n0, N, r);
    store_states<NS, FULL>(a.dstate + at, me.n0, N, r);
  }
}

// dB and dC from the channel tiles' partial rows, in ascending order.
template <class T>
__global__ void __launch_bounds__(256) sscan_bc_kernel(SscanArgs a, const float* part, uint32_t tiles) {
  const uint64_t per = (uint64_t)a.groups * 2 * a.states;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.seq.tokens * per) return;
  const uint64_t t = i / per;
  const uint32_t j = i % per, n = j % a.states, which = j / a.states & 1, g = j / (2 * a.states);
  const int64_t seq = a.seq.of((int64_t)t);
  if (seq < 0 || seq >= (int64_t)a.seq.n_seq || (int64_t)t >= a.seq.begin(seq + 1)) return;
  float s = 0.f;
  for (uint32_t k = 0; k < tiles; ++k) s += part[(uint64_t)k * a.seq.tokens * per + i];
  T* out = reinterpret_cast<T*>(which ? a.dc : a.db);
  out[t * (which ? a.dc_stride : a.db_stride) + (uint64_t)g * (which ? a.dc_group : a.db_group) + n] = from_f32<T>(s);
}

bool aligned16(const void* p) { return reinterpret_cast<uint64_t>(p) % 16 == 0; }

// 8 states a lane: a block of kMarkEvery tokens of them fits the registers.
constexpr uint32_t lanes_of(uint32_t states) { return states <= 8 ? 1 : states <= 16 ? 2 : states <= 32 ? 4 : 8; }

ScanPlan plan_of(uint64_t tokens, uint32_t channels, uint32_t states, uint64_t n_seq, uint32_t groups, bool ragged) {
  return scan_plan(tokens, channels, groups, n_seq, ragged, {lanes_of(states), lanes_of(states)});
}

uint64_t back_work(const ScanPlan& p, uint64_t tokens, uint32_t channels, uint32_t states, uint32_t groups, void* base,
                   BackWork* w) {
  uint64_t at = scan_work(p, channels, states, false, base, w ? &w->scan : nullptr);
  char* b = static_cast<char*>(base);
  if (w) w->da = reinterpret_cast<float*>(b + at);
  at += scan_round(p.chunks * channels * states * 4);
  if (w) w->dd = reinterpret_cast<float*>(b + at);
  at += scan_round(p.chunks * channels * 2 * 4);
  if (w) w->bc = reinterpret_cast<float*>(b + at);
  return at + scan_round((uint64_t)p.per_group * tokens * groups * 2 * states * 4);
}

template <class T, int NS, int LP, bool FULL>
cudaError_t go(const SscanArgs& a, cudaStream_t s) {
  const ScanPlan p = plan_of(a.seq.tokens, a.channels, a.states, a.seq.n_seq, a.groups, a.seq.seq_ptr != nullptr);
  BackWork w{};
  back_work(p, a.seq.tokens, a.channels, a.states, a.groups, a.work, &w);
  const uint64_t grid = p.chunks * p.ctiles;
  if (grid > 0x7fffffffull) return cudaErrorInvalidValue;
  if (p.carry) {
    sscan_chunk_back_kernel<T, NS, LP, FULL><<<(unsigned)grid, kScanThreads, 0, s>>>(a, p, w.scan);
    launch_sscan_fold_back(a.a, w.scan, p.chunks, a.channels, a.states, s);
  }
  sscan_back_kernel<T, NS, LP, FULL><<<(unsigned)grid, kScanThreads, 0, s>>>(a, p, w);
  const uint64_t cells = a.seq.tokens * a.groups * 2 * a.states;
  if (cells) sscan_bc_kernel<T><<<(unsigned)((cells + 255) / 256), 256, 0, s>>>(a, w.bc, p.per_group);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const uint64_t as = (uint64_t)a.channels * a.states;
  e = launch_reduce_rows(w.da, p.chunks, as, as, a.da, nullptr, s);
  if (e == cudaSuccess && (a.dd || a.ddt_bias))
    e = launch_reduce_rows(w.dd, p.chunks, 2ull * a.channels, a.channels, a.dd, a.ddt_bias, s);
  return e;
}

template <class T>
cudaError_t by_states(const SscanArgs& a, cudaStream_t s) {
  const uint32_t N = a.states;
  const bool al = aligned16(a.a) && aligned16(a.state) && aligned16(a.dstate) && aligned16(a.dfinal) && aligned16(a.marks) &&
                  aligned16(a.work);
  if (N == 8 && al) return go<T, 8, 1, true>(a, s);
  if (N == 16 && al) return go<T, 8, 2, true>(a, s);
  if (N == 32 && al) return go<T, 8, 4, true>(a, s);
  if (N == 64 && al) return go<T, 8, 8, true>(a, s);
  if (N <= 8) return go<T, 8, 1, false>(a, s);
  if (N <= 16) return go<T, 8, 2, false>(a, s);
  if (N <= 32) return go<T, 8, 4, false>(a, s);
  return go<T, 8, 8, false>(a, s);
}

}  // namespace

size_t sscan_backward_bytes(uint64_t tokens, uint64_t channels, uint32_t states, uint64_t n_seq, uint32_t groups) {
  uint64_t most = 0;
  for (bool ragged : {false, true}) {
    const ScanPlan p = plan_of(tokens, (uint32_t)channels, states, n_seq, groups, ragged);
    const uint64_t b = back_work(p, tokens, (uint32_t)channels, states, groups, nullptr, nullptr);
    if (b > most) most = b;
  }
  return most;
}

cudaError_t launch_sscan_backward(const SscanArgs& a, cudaStream_t s) {
  switch (a.type) {
    case SEQ_F32: return by_states<float>(a, s);
    case SEQ_F16: return by_states<__half>(a, s);
    default: return by_states<__nv_bfloat16>(a, s);
  }
}

}  // namespace sparsl
