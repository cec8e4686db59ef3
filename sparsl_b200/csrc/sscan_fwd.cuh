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
//
// What bounds it: the exponentials, 16 a clock and SM, before HBM's bytes.  With
// 16 states and the 3 of step and gate a cell takes 19, so a pass over 32768
// tokens x 2048 channels 0.28 ms against 0.08 for the rows.  One lane holds all
// states of a channel where there are blocks enough: its step, gate and output
// are formed once, and B and C come by broadcasts.  Measured there: the main pass
// 0.40 ms (the unit 70 % busy, 0.6 instructions a clock and scheduler), the pass
// before it 0.31; 12288 tokens in 19 unequal sequences x 4096 channels 0.30 and
// 0.20 ms.
#pragma once

#include "sscan.cuh"

namespace sparsl {
namespace {

constexpr uint32_t kResident = 4;  // blocks an SM holds, at 128 registers a thread

// One token: h <- e h + (s x) B.
template <int NS, bool FULL>
__device__ __forceinline__ void advance(const f32x2 (&e)[NS / 2], float sx, const float* b, uint32_t n0, uint32_t N,
                                        f32x2 (&h)[NS / 2]) {
  const f32x2 xx = pair(sx, sx);
#pragma unroll
  for (int j = 0; j < NS / 2; j += 2) {
    const ulonglong2 bb = *reinterpret_cast<const ulonglong2*>(b + 2 * j);
    f32x2 add0 = mul2(xx, bb.x), add1 = mul2(xx, bb.y);
    if (!FULL) {  // an infinite x must not reach a state that does not exist
      float lo, hi;
      unpair(add0, lo, hi);
      add0 = pair(n0 + 2 * j < N ? lo : 0.f, n0 + 2 * j + 1 < N ? hi : 0.f);
      unpair(add1, lo, hi);
      add1 = pair(n0 + 2 * j + 2 < N ? lo : 0.f, n0 + 2 * j + 3 < N ? hi : 0.f);
    }
    h[j] = fma2(e[j], h[j], add0);
    h[j + 1] = fma2(e[j + 1], h[j + 1], add1);
  }
}

// The state that a chunk hands to the next one: its last sequence's, from that
// sequence's start in it or from zero.
template <class T, int NS, int LP, bool FULL>
__global__ void __launch_bounds__(kScanThreads, kResident) sscan_chunk_kernel(SscanArgs a, ScanPlan p, ScanWork w, int aligned) {
  constexpr int NP = NS * LP, K = kBatch, kOwn = K / LP;
  using Rows = WarpRows<T, LP>;
  __shared__ __align__(16) float bc[2][kScanTile][NP];
  __shared__ __align__(16) T rows[kScanThreads / 32][2][2][K][Rows::kCols];
  const uint32_t N = a.states;
  const ScanLane<NS, LP> me(a.channels, a.groups, p.per_group, blockIdx.x % p.ctiles);
  const uint32_t part = threadIdx.x % LP, col = threadIdx.x % 32 / LP;
  const int64_t chunk = blockIdx.x / p.ctiles;
  const int64_t t0 = chunk * (int64_t)p.len, t1 = min(t0 + (int64_t)p.len, (int64_t)a.seq.tokens);
  const int64_t seq = a.seq.of(t1 - 1);
  const bool any = seq >= 0 && seq < (int64_t)a.seq.n_seq;
  const int64_t begin = any ? a.seq.begin(seq) : 0, end = any ? a.seq.begin(seq + 1) : 0;
  const bool spans = any && end > t1 && begin < t1;
  if (threadIdx.x == 0 && blockIdx.x % p.ctiles == 0) w.cut[chunk] = !spans ? 2 : begin >= t0 ? 1 : 0;
  if (!spans) return;
  f32x2 h[NS / 2], a2[NS / 2];
  load_pairs<NS, FULL>(a.a + (uint64_t)me.c * N, me.n0, N, a2, kLog2e);
  zero_pairs(h);
  const uint64_t row = ((uint64_t)chunk * a.channels + me.c) * N;
  if (begin >= t0 && a.state) {
    const int64_t slot = a.seq.resumes(seq) ? a.seq.slot(seq) : -1;
    if (slot >= 0) load_pairs<NS, FULL>(a.state + ((uint64_t)slot * a.channels + me.c) * N, me.n0, N, h);
    if (w.start && me.valid) store_pairs<NS, FULL>(w.start + row, me.n0, N, h);
  }
  const float bias = a.dt_bias ? a.dt_bias[me.c] : 0.f;
  float sum = 0.f;
  StageBC<T, NP, 1> stage;
  const int64_t from = max(begin, t0);
  const RowsIn arrays[2] = {{a.x, a.x_row}, {a.dt, a.dt_row}};
  T(*const stages)[2][K][Rows::kCols] = rows[threadIdx.x / 32];
  RowsCursor<T, LP, 2, 1> cursor(arrays, from, me.warp_c, me.warp_cols);
  const auto fetch = [&](int at, int64_t t) {
    if (aligned == 2) cursor.copy(stages[at], first_bits(t1 - t));
    else Rows::in(stages[at], arrays, t, first_bits(t1 - t), me.warp_c, me.warp_cols, aligned);
    copies_issued();
  };
  stage.fetch(a, me.group, from, first_bits(t1 - from));
  fetch(0, from);
  stage.put(&bc[0][0][0]);
  __syncthreads();
  int buf = 0, at = 0;
  for (int64_t tb = from; tb < t1; tb += kScanTile, buf ^= 1) {
    stage.fetch(a, me.group, tb + kScanTile, first_bits(t1 - tb - kScanTile));
#pragma unroll 1
    for (int k0 = 0; k0 < kScanTile; k0 += K, at ^= 1) {
      const int64_t left = t1 - tb - k0;  // the tokens not done
      if (left <= 0) break;
      copies_done();
      fetch(at ^ 1, tb + k0 + K);
      const T(&in)[2][K][Rows::kCols] = stages[at];
      float s[kOwn], sx[kOwn];
#pragma unroll
      for (int j = 0; j < kOwn; ++j) {
        s[j] = sx[j] = 0.f;  // a token behind the chunk changes nothing: its decay is 1
        if (j * LP + (int64_t)part < left) {
          s[j] = to_f32(in[1][j * LP + part][col]) + bias;
          if (a.softplus) s[j] = softplus(s[j]);
          sx[j] = s[j] * to_f32(in[0][j * LP + part][col]);
          sum += s[j];
        }
      }
      f32x2 e[NS / 2], en[NS / 2];
      decay<NS>(from_lane<LP>(s[0], 0), a2, e);
#pragma unroll
      for (int k = 0; k < K; ++k) {  // a token's exponentials are under way while the one before it is added
        if (k + 1 < K) decay<NS>(from_lane<LP>(s[(k + 1) / LP], (k + 1) % LP), a2, en);
        advance<NS, FULL>(e, from_lane<LP>(sx[k / LP], k % LP), &bc[buf][k0 + k][me.n0], me.n0, N, h);
#pragma unroll
        for (int i = 0; i < NS / 2; ++i) e[i] = en[i];
      }
    }
    stage.put(&bc[buf ^ 1][0][0]);
    __syncthreads();
  }
  sum = sum_lanes<LP>(sum);
  if (me.valid) {
    store_pairs<NS, FULL>(w.state + row, me.n0, N, h);
    if (me.first) w.sum[(uint64_t)chunk * a.channels + me.c] = sum;
  }
}

// The state behind a chunk: `carry` in front of it decayed by 2^x, and what the
// chunk itself hands on.  2^x may leave f32's range where no token's decay and no
// state does: from 2^120 on it is applied by halves, which stay finite, as a state
// of zero has to stay zero.  No branch, and no pass of its own in front of the
// states': 12 us for 35 chunks x 65536 states, 16 in a pass of its own.
__device__ __forceinline__ float behind_chunk(float x, float carry, float own) {
  const bool far = fabsf(x) >= 120.0f;
  const float e = fminf(ex2(far ? 0.5f * x : x), 3.0e38f);
  return __fmaf_rn(e, (far ? e : 1.0f) * carry, own);
}

// What each chunk starts from, in place of what it hands on: ascending for the
// states, descending (BACK) for their gradients.
template <bool BACK>
__global__ void __launch_bounds__(128) sscan_fold_kernel(const float* a, ScanWork w, uint64_t chunks, uint32_t channels,
                                                         uint32_t states) {
  const uint64_t cells = (uint64_t)channels * states;
  const uint64_t i = (uint64_t)blockIdx.x * 128 + threadIdx.x;
  if (i >= cells) return;
  const uint32_t c = i / states;
  const float a2 = a[i] * kLog2e;
  float carry = 0.f;
  constexpr int U = 16;
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
        carry = cut[u] == 2 ? 0.f : cut[u] == 1 ? v[u] : behind_chunk(s[u] * a2, carry, v[u]);
      }
  }
}

template <int NS>
__device__ __forceinline__ float dot(const float* c, const f32x2 (&h)[NS / 2]) {
  f32x2 o = 0ull, p = 0ull;
#pragma unroll
  for (int i = 0; i < NS / 2; i += 2) {
    const ulonglong2 cc = *reinterpret_cast<const ulonglong2*>(c + 2 * i);
    o = fma2(cc.x, h[i], o);
    p = fma2(cc.y, h[i + 1], p);
  }
  return sum2(add2(o, p));
}

// The main pass over one chunk, in batches of eight tokens.  A batch inside one
// sequence takes the straight path; one in which a sequence begins or ends
// elsewhere than at its edges goes token by token.  128 registers a thread, 16
// warps an SM: a lane holds its states, their exponents and two tokens' decays.
template <class T, int NS, int LP, bool FULL, bool GATE>
__global__ void __launch_bounds__(kScanThreads, kResident) sscan_kernel(SscanArgs a, ScanPlan p, ScanWork w, int aligned) {
  constexpr int NP = NS * LP, K = kBatch, kOwn = K / LP, A = GATE ? 3 : 2;
  using Rows = WarpRows<T, LP>;
  __shared__ __align__(16) float bc[2][kScanTile][2][NP];
  __shared__ __align__(16) T rows[kScanThreads / 32][2][A][K][Rows::kCols];
  __shared__ __align__(16) T results[kScanThreads / 32][K][Rows::kCols];
  const uint32_t N = a.states;
  const ScanLane<NS, LP> me(a.channels, a.groups, p.per_group, blockIdx.x % p.ctiles);
  const uint32_t part = threadIdx.x % LP, col = threadIdx.x % 32 / LP;
  const int64_t chunk = blockIdx.x / p.ctiles;
  const int64_t t0 = chunk * (int64_t)p.len, t1 = min(t0 + (int64_t)p.len, (int64_t)a.seq.tokens);
  f32x2 h[NS / 2], a2[NS / 2];
  load_pairs<NS, FULL>(a.a + (uint64_t)me.c * N, me.n0, N, a2, kLog2e);
  zero_pairs(h);
  const uint64_t row = ((uint64_t)chunk * a.channels + me.c) * N;
  if (p.carry) load_pairs<NS, FULL>(w.state + row, me.n0, N, h);
  const float bias = a.dt_bias ? a.dt_bias[me.c] : 0.f;
  const bool skip = a.d != nullptr;  // without it no term: 0 times an infinite x would be NaN
  const float dskip = skip ? a.d[me.c] : 0.f;

  const auto begin_state = [&](int64_t seq) {
    zero_pairs(h);
    if (!a.state) return;
    const int64_t slot = a.seq.resumes(seq) ? a.seq.slot(seq) : -1;
    const float* from = nullptr;
    if (w.start && p.carry && a.seq.begin(seq + 1) > t1) from = w.start + row;
    else if (slot >= 0) from = a.state + ((uint64_t)slot * a.channels + me.c) * N;
    if (from) load_pairs<NS, FULL>(from, me.n0, N, h);
  };
  const auto end_state = [&](int64_t seq) {
    const int64_t slot = a.final_state ? a.seq.slot(seq) : -1;
    if (slot >= 0 && me.valid)
      store_pairs<NS, FULL>(a.final_state + ((uint64_t)slot * a.channels + me.c) * N, me.n0, N, h);
  };
  const auto mark = [&](int64_t t) {
    if (a.marks && me.valid)
      store_pairs<NS, FULL>(a.marks + ((uint64_t)(t / kMarkEvery) * a.channels + me.c) * N, me.n0, N, h);
  };
  const auto finish = [&](float o, float xv, float zv) {
    if (skip) o = __fmaf_rn(dskip, xv, o);
    if (GATE) o *= zv * sigmoid(zv);
    return from_f32<T>(o);
  };
  constexpr uint32_t kAll = (1u << K) - 1;

  RowsIn arrays[A];
  arrays[0] = {a.x, a.x_row};
  arrays[1] = {a.dt, a.dt_row};
  if constexpr (GATE) arrays[2] = {a.z, a.z_row};
  T(*const stages)[A][K][Rows::kCols] = rows[threadIdx.x / 32];
  T(&result)[K][Rows::kCols] = results[threadIdx.x / 32];
  RowsCursor<T, LP, A, 1> cursor(arrays, t0, me.warp_c, me.warp_cols);
  const auto fetch = [&](int at, int64_t t, uint32_t live) {
    if (aligned == 2) cursor.copy(stages[at], live);
    else Rows::in(stages[at], arrays, t, live, me.warp_c, me.warp_cols, aligned);
    copies_issued();
  };
  StageBC<T, NP, 2> stage;
  TileMarks m = tile_marks(a.seq, t0, t1), after;
  stage.fetch(a, me.group, t0, m.live);
  fetch(0, t0, m.live);
  stage.put(&bc[0][0][0][0]);
  __syncthreads();
  int buf = 0, at = 0;
  for (int64_t tb = t0; tb < t1; tb += kScanTile, buf ^= 1, m = after) {
    after = tile_marks(a.seq, tb + kScanTile, t1);
    stage.fetch(a, me.group, tb + kScanTile, after.live);
#pragma unroll 1
    for (int k0 = 0; k0 < kScanTile; k0 += K, at ^= 1) {
      const uint32_t live = m.live >> k0 & kAll, start = m.start >> k0 & kAll, end = m.end >> k0 & kAll;
      copies_done();
      fetch(at ^ 1, tb + k0 + K, k0 + K < kScanTile ? m.live >> (k0 + K) : after.live);
      const T(&in)[A][K][Rows::kCols] = stages[at];
      if (live == kAll && !(start & ~1u) && !(end & (kAll >> 1))) {
        if (start & 1) begin_state(tile_seq(m, k0));
        mark(tb + k0);
        float s[kOwn], sx[kOwn], xv[kOwn], o[LP];
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
          xv[j] = to_f32(in[0][j * LP + part][col]);
          s[j] = to_f32(in[1][j * LP + part][col]) + bias;
          if (a.softplus) s[j] = softplus(s[j]);
          sx[j] = s[j] * xv[j];
        }
        f32x2 e[NS / 2], en[NS / 2];
        decay<NS>(from_lane<LP>(s[0], 0), a2, e);
#pragma unroll
        for (int k = 0; k < K; ++k) {  // a token's exponentials are under way while the one before it is added
          const int j = k / LP, q = k % LP;
          if (k + 1 < K) decay<NS>(from_lane<LP>(s[(k + 1) / LP], (k + 1) % LP), a2, en);
          const float(&bk)[2][NP] = bc[buf][k0 + k];
          advance<NS, FULL>(e, from_lane<LP>(sx[j], q), &bk[0][me.n0], me.n0, N, h);
          o[q] = dot<NS>(&bk[1][me.n0], h);
          if (q == LP - 1)
            result[j * LP + part][col] = finish(scatter_sum<LP>(o, part), xv[j], GATE ? to_f32(in[A - 1][j * LP + part][col]) : 0.f);
#pragma unroll
          for (int i = 0; i < NS / 2; ++i) e[i] = en[i];
        }
        if (end >> (K - 1) & 1) end_state(tile_seq(m, k0 + K - 1));
      } else if (live) {
#pragma unroll 1
        for (int k = 0; k < K; ++k) {
          if (!(live >> k & 1)) continue;
          if (start >> k & 1) begin_state(tile_seq(m, k0 + k));
          if (k == 0) mark(tb + k0);
          const float xv = to_f32(in[0][k][col]);
          float s = to_f32(in[1][k][col]) + bias;
          if (a.softplus) s = softplus(s);
          const float(&bk)[2][NP] = bc[buf][k0 + k];
          f32x2 e[NS / 2];
          decay<NS>(s, a2, e);
          advance<NS, FULL>(e, s * xv, &bk[0][me.n0], me.n0, N, h);
          const float o = sum_lanes<LP>(dot<NS>(&bk[1][me.n0], h));
          if (me.first) result[k][col] = finish(o, xv, GATE ? to_f32(in[A - 1][k][col]) : 0.f);
          if (end >> k & 1) end_state(tile_seq(m, k0 + k));
        }
      }
      __syncwarp();
      Rows::out(result, a.y, a.y_row, tb + k0, live, me.warp_c, me.warp_cols, aligned);
    }
    stage.put(&bc[buf ^ 1][0][0][0]);
    __syncthreads();
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
    zero_pairs(h);
    const uint64_t at = ((uint64_t)slot * a.channels + me.c) * N;
    if (a.state && a.seq.resumes(i)) load_pairs<NS, FULL>(a.state + at, me.n0, N, h);
    store_pairs<NS, FULL>(a.final_state + at, me.n0, N, h);
  }
}

// One token of each sequence.  Few sequences: a channel's states over LP lanes, 4
// each, to have blocks for all SMs.
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
  const float xv = to_f32(*cell<T>(a.x, i, a.x_row, cc));
  float s = to_f32(*cell<T>(a.dt, i, a.dt_row, cc));
  const float zv = a.z ? to_f32(*cell<T>(a.z, i, a.z_row, cc)) : 0.f;
  if (a.dt_bias) s += a.dt_bias[cc];
  if (a.softplus) s = softplus(s);
  float o = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (FULL || n0 + j < N) {
      h[j] = __fmaf_rn(ex2(__fmaf_rn(s, a2[j] * kLog2e, kLift)), h[j], s * xv * to_f32(b[n0 + j]));
      o = __fmaf_rn(to_f32(cv[n0 + j]), h[j], o);
    }
  }
  o = sum_lanes<LP>(o);
  if (a.d) o = __fmaf_rn(a.d[cc], xv, o);
  if (a.z) o *= zv * sigmoid(zv);
  if (!valid) return;
  store_states<4, FULL>(st, n0, N, h);
  if (n0 == 0) *cell<T>(a.y, i, a.y_row, c) = from_f32<T>(o);
}

// Many sequences: up to 16 states a lane, as in the scan, and a block's channels
// for kStepTokens of them, whose states are all asked for before the first is
// used, 32 bytes an access.  512 tokens x 4096 channels x 16 states: 57 us, 5.0
// TB/s of states and rows; with 4 states a lane 77 us, the step, the gate and the
// addresses over again in each, and with 16-byte accesses, half a sector each, 67.
constexpr int kStepTokens = 4;
template <class T, int NS, int LP, bool FULL>
__global__ void __launch_bounds__(kScanThreads, kResident) sscan_step_many_kernel(SscanArgs a, uint32_t per_group, uint32_t ctiles) {
  constexpr int NP = NS * LP;
  __shared__ __align__(16) float bc[kStepTokens][2][NP];
  const uint32_t N = a.states;
  const ScanLane<NS, LP> me(a.channels, a.groups, per_group, blockIdx.x % ctiles);
  const int64_t i0 = (int64_t)(blockIdx.x / ctiles) * kStepTokens;
  f32x2 h[kStepTokens][NS / 2], a2[NS / 2];
  float xv[kStepTokens], s[kStepTokens], zv[kStepTokens];
  int64_t at[kStepTokens];
#pragma unroll
  for (int u = 0; u < kStepTokens; ++u) {
    const int64_t i = i0 + u, slot = i < (int64_t)a.seq.n_seq ? a.seq.slot(i) : -1;
    at[u] = slot < 0 ? -1 : (int64_t)(((uint64_t)slot * a.channels + me.c) * N);
    if (at[u] < 0) continue;  // the whole block's
    load_rows<NS, FULL>(a.final_state + at[u], me.n0, N, h[u]);
    xv[u] = to_f32(*cell<T>(a.x, i, a.x_row, me.c));
    s[u] = to_f32(*cell<T>(a.dt, i, a.dt_row, me.c));
    zv[u] = a.z ? to_f32(*cell<T>(a.z, i, a.z_row, me.c)) : 0.f;
  }
  for (uint32_t q = threadIdx.x; q < kStepTokens * 2 * NP; q += kScanThreads) {
    const uint32_t n = q % NP, which = q / NP & 1, u = q / (2 * NP);
    const int64_t i = i0 + u;
    float v = 0.f;
    if (i < (int64_t)a.seq.n_seq && n < N)
      v = to_f32(reinterpret_cast<const T*>(which ? a.c : a.b)[(uint64_t)i * (which ? a.c_stride : a.b_stride) +
                                                              (uint64_t)me.group * (which ? a.c_group : a.b_group) + n]);
    bc[u][which][n] = v;
  }
  load_pairs<NS, FULL>(a.a + (uint64_t)me.c * N, me.n0, N, a2, kLog2e);
  const float bias = a.dt_bias ? a.dt_bias[me.c] : 0.f, dskip = a.d ? a.d[me.c] : 0.f;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kStepTokens; ++u) {
    if (at[u] < 0) continue;
    float step = s[u] + bias;
    if (a.softplus) step = softplus(step);
    f32x2 e[NS / 2];
    decay<NS>(step, a2, e);
    advance<NS, FULL>(e, step * xv[u], &bc[u][0][me.n0], me.n0, N, h[u]);
    float o = sum_lanes<LP>(dot<NS>(&bc[u][1][me.n0], h[u]));
    if (a.d) o = __fmaf_rn(dskip, xv[u], o);
    if (a.z) o *= zv[u] * sigmoid(zv[u]);
    if (!me.valid) continue;
    store_rows<NS, FULL>(a.final_state + at[u], me.n0, N, h[u]);
    if (me.first) *cell<T>(a.y, i0 + u, a.y_row, me.c) = from_f32<T>(o);
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uint64_t>(p) % 16 == 0; }

// The lanes that share a channel: at most 16 states each; at least 4.
constexpr uint32_t padded(uint32_t states) { return states <= 8 ? 8 : states <= 16 ? 16 : states <= 32 ? 32 : 64; }
ScanLanes lanes_of(uint32_t states) {
  const uint32_t np = padded(states);
  return {np <= 16 ? 1u : np / 16, np <= 8 ? 2u : 4u, kResident, np, 8u, 12u};
}

ScanPlan plan_of(const SscanArgs& a) {
  return scan_plan(a.seq.tokens, a.channels, a.groups, a.seq.n_seq, a.seq.seq_ptr != nullptr, lanes_of(a.states));
}

template <class T, int NS, int LP, bool FULL>
cudaError_t go(const SscanArgs& a, const ScanPlan& p, cudaStream_t s) {
  ScanWork w{};
  scan_work(p, a.channels, a.states, true, a.work, &w);
  if (a.state != a.final_state || !a.state) w.start = nullptr;
  const uint64_t grid = p.chunks * p.ctiles;
  if (grid > 0x7fffffffull) return cudaErrorInvalidValue;
  const int aligned = rows_aligned<T, LP>(a, {{a.x, a.x_row}, {a.dt, a.dt_row}, {a.z, a.z_row}, {a.y, a.y_row}});
  if (p.carry) {
    sscan_chunk_kernel<T, NS, LP, FULL><<<(unsigned)grid, kScanThreads, 0, s>>>(a, p, w, aligned);
    const uint64_t cells = (uint64_t)a.channels * a.states;
    sscan_fold_kernel<false><<<(unsigned)((cells + 127) / 128), 128, 0, s>>>(a.a, w, p.chunks, a.channels, a.states);
  }
  if (a.z) sscan_kernel<T, NS, LP, FULL, true><<<(unsigned)grid, kScanThreads, 0, s>>>(a, p, w, aligned);
  else sscan_kernel<T, NS, LP, FULL, false><<<(unsigned)grid, kScanThreads, 0, s>>>(a, p, w, aligned);
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

// Whether the many sequences' kernel fills the SMs with two waves of blocks.
template <int LP>
bool many(const SscanArgs& a, uint32_t& per_group, uint64_t& grid) {
  const uint32_t cpg = a.channels / a.groups;
  per_group = (cpg + kScanThreads / LP - 1) / (kScanThreads / LP);
  grid = (a.seq.n_seq + kStepTokens - 1) / kStepTokens * per_group * a.groups;
  return grid >= 2 * kResident * kSms && grid <= 0x7fffffffull;
}
template <class T, int NS, int LP, bool FULL>
cudaError_t go_many(const SscanArgs& a, uint32_t per_group, uint64_t grid, cudaStream_t s) {
  sscan_step_many_kernel<T, NS, LP, FULL><<<(unsigned)grid, kScanThreads, 0, s>>>(a, per_group, per_group * a.groups);
  return cudaGetLastError();
}

template <class T, int NP, bool FULL>
cudaError_t by_lanes(const SscanArgs& a, const ScanPlan& p, cudaStream_t s) {
  if constexpr (NP <= 16)
    if (p.lanes == 1) return go<T, NP, 1, FULL>(a, p, s);
  if constexpr (NP <= 32)
    if (p.lanes == 2) return go<T, NP / 2, 2, FULL>(a, p, s);
  if constexpr (NP >= 16)
    if (p.lanes == 4) return go<T, NP / 4, 4, FULL>(a, p, s);
  return cudaErrorInvalidValue;
}

template <class T>
cudaError_t by_states(const SscanArgs& a, cudaStream_t s) {
  const uint32_t N = a.states;
  const ScanPlan p = plan_of(a);
  const bool al = aligned16(a.a) && aligned16(a.state) && aligned16(a.final_state) && aligned16(a.marks) && aligned16(a.work);
  if (N == 16 && al) return by_lanes<T, 16, true>(a, p, s);
  if (N == 8 && al) return by_lanes<T, 8, true>(a, p, s);
  if (N == 32 && al) return by_lanes<T, 32, true>(a, p, s);
  if (N == 64 && al) return by_lanes<T, 64, true>(a, p, s);
  if (N <= 8) return by_lanes<T, 8, false>(a, p, s);
  if (N <= 16) return by_lanes<T, 16, false>(a, p, s);
  if (N <= 32) return by_lanes<T, 32, false>(a, p, s);
  return by_lanes<T, 64, false>(a, p, s);
}

template <class T>
cudaError_t step_by_states(const SscanArgs& a, cudaStream_t s) {
  const uint32_t N = a.states;
  const bool al = aligned16(a.a) && aligned16(a.final_state);
  const bool wide = aligned16(a.a) && reinterpret_cast<uint64_t>(a.final_state) % 32 == 0;
  uint32_t per;
  uint64_t grid;
  if (N <= 8 && many<1>(a, per, grid)) return N == 8 && wide ? go_many<T, 8, 1, true>(a, per, grid, s) : go_many<T, 8, 1, false>(a, per, grid, s);
  if (N > 8 && N <= 16 && many<1>(a, per, grid))
    return N == 16 && wide ? go_many<T, 16, 1, true>(a, per, grid, s) : go_many<T, 16, 1, false>(a, per, grid, s);
  if (N > 16 && N <= 32 && many<2>(a, per, grid))
    return N == 32 && wide ? go_many<T, 16, 2, true>(a, per, grid, s) : go_many<T, 16, 2, false>(a, per, grid, s);
  if (N > 32 && many<4>(a, per, grid))
    return N == 64 && wide ? go_many<T, 16, 4, true>(a, per, grid, s) : go_many<T, 16, 4, false>(a, per, grid, s);
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

}  // namespace sparsl
