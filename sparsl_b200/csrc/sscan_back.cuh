// Gradients of the selective scan.  With e_t = exp(s_t A), dy the gradient
// behind the gate, and r_t the gradient that h_t receives from later tokens,
//
//   g_t = r_t + C_t dy_t          r_{t-1} = e_t g_t
//   dx = D dy + s (g . B)         ds = sum_n g (A e h_{t-1} + B x)
//   dA = sum_t g e h_{t-1} s      dB = sum_c g s x       dC = sum_c dy h
//
// The forward pass saved the states before every kMarkEvery-th token.  A block
// of that many tokens is recomputed forwards from its mark with the states kept
// in registers, and then walked backwards.  Its decays are computed once more
// on the way back: the special function unit has the time, the
// registers do not hold them.  Chunks of the token axis run in parallel as in the forward
// pass: the gradient each chunk hands to the one before it is computed first,
// and folded.  dB and dC are summed over a warp's channels and a block's warps
// in shared memory, and over the blocks' partial rows in a fixed order, so that
// results do not change from run to run; so are dA, dD and the step bias's
// gradient over the chunks.
//
// What bounds it: latency.  A state of a cell takes some 24 instructions (3.5 of
// packed arithmetic each way, the sums over channels 3, the cell's own step and
// gates 4, the rest moves, addresses and shared-memory loads), and the 1.7 warps a
// scheduler that its registers allow issue 0.4 of them a clock; no unit is full
// (special functions 30 %, shared memory 53 %).  0.94 ms for 16384 tokens x 2048
// channels x 16 states, against 0.24 for the exponentials, 0.07 for the rows and
// 0.04 for the saved states.
#pragma once

#include <type_traits>

#include "sscan.cuh"

namespace sparsl {

cudaError_t launch_sscan_fold_back(const float* a, const ScanWork& w, uint64_t chunks, uint32_t channels, uint32_t states,
                                   cudaStream_t s);

namespace {

constexpr int kWarps = kScanThreads / 32;
// Blocks an SM holds: at up to 255 registers a thread with 8 states, 128 with 4.
// Three with 8 states: 0.86 ms against 0.94 for this kernel at 16384 tokens x 2048
// channels x 16 states, but the 256 blocks of its whole sequences then fill too little
// of a wave, and the chunks' first pass takes 0.2 ms more than that gains.
constexpr int resident(int states) { return states == 8 ? 2 : 4; }
constexpr int kBlock = (int)kMarkEvery;
static_assert(kBlock == kBatch, "a block is a batch");

struct BackWork {
  ScanWork scan;
  float* da;  // [chunks, channels, states]
  float* dd;  // [chunks, 2, channels]: dD, then the step bias's
  float* bc;  // [channel tiles of a group, tokens, groups, 2, states]
};

__device__ __forceinline__ float gate_grad(float z, float sig) { return sig * __fmaf_rn(z, 1.0f - sig, 1.0f); }

// The gradient that a chunk hands to the state before it, from the end of the
// sequence that reaches into it, or from zero at its own end; in batches of
// eight tokens, the last ones first.
template <class T, int NS, int LP, bool FULL, bool GATE>
__global__ void __launch_bounds__(kScanThreads, 4) sscan_chunk_back_kernel(SscanArgs a, ScanPlan p, ScanWork w, int aligned) {
  constexpr int NP = NS * LP, U = kBatch, kOwn = U / LP, A = GATE ? 3 : 2;
  using Rows = WarpRows<T, LP>;
  __shared__ __align__(16) float sc[2][kScanTile][NP];
  __shared__ __align__(16) T rows[kScanThreads / 32][2][A][U][Rows::kCols];
  const uint32_t N = a.states;
  const ScanLane<NS, LP> me(a.channels, a.groups, p.per_group, blockIdx.x % p.ctiles);
  const uint32_t part = threadIdx.x % LP;
  const int64_t chunk = blockIdx.x / p.ctiles;
  const int64_t t0 = chunk * (int64_t)p.len, t1 = min(t0 + (int64_t)p.len, (int64_t)a.seq.tokens);
  const int64_t seq = a.seq.of(t0);
  const bool any = seq >= 0 && seq < (int64_t)a.seq.n_seq;
  const int64_t begin = any ? a.seq.begin(seq) : 0, end = any ? a.seq.begin(seq + 1) : 0;
  const bool spans = any && begin < t0 && end > t0;
  if (threadIdx.x == 0 && blockIdx.x % p.ctiles == 0) w.cut[chunk] = !spans ? 2 : end <= t1 ? 1 : 0;
  if (!spans) return;
  const int64_t hi = min(end, t1);
  f32x2 r[NS / 2], a2[NS / 2];
  load_pairs<NS, FULL>(a.a + (uint64_t)me.c * N, me.n0, N, a2, kLog2e);
  zero_pairs(r);
  if (end <= t1 && a.dfinal) {
    const int64_t slot = a.seq.slot(seq);
    if (slot >= 0) load_pairs<NS, FULL>(a.dfinal + ((uint64_t)slot * a.channels + me.c) * N, me.n0, N, r);
  }
  const float bias = a.dt_bias ? a.dt_bias[me.c] : 0.f;
  const uint32_t col = threadIdx.x % 32 / LP;
  float sum = 0.f;
  RowsIn arrays[A];
  arrays[0] = {a.dt, a.dt_row};
  arrays[1] = {a.dy, a.dy_row};
  if constexpr (GATE) arrays[2] = {a.z, a.z_row};
  T(*const stages)[A][U][Rows::kCols] = rows[threadIdx.x / 32];
  RowsCursor<T, LP, A, -1> cursor(arrays, hi - U, me.warp_c, me.warp_cols);
  // The bits of tokens t.. that the chunk has.
  const auto above = [&](int64_t t) { return t >= t0 ? ~0u : ~first_bits(t0 - t); };
  const auto fetch = [&](int at, int64_t t) {
    if (aligned == 2) cursor.copy(stages[at], above(t));
    else Rows::in(stages[at], arrays, t, above(t), me.warp_c, me.warp_cols, aligned);
    copies_issued();
  };
  StageBC<T, NP, 1, true> stage;
  stage.fetch(a, me.group, hi - kScanTile, above(hi - kScanTile));
  fetch(0, hi - U);
  stage.put(&sc[0][0][0]);
  __syncthreads();
  int buf = 0, at = 0;
  for (int64_t te = hi; te > t0; te -= kScanTile, buf ^= 1) {  // tokens te - 32 to te - 1, the last first
    stage.fetch(a, me.group, te - 2 * kScanTile, above(te - 2 * kScanTile));
#pragma unroll 1
    for (int k0 = 0; k0 < kScanTile; k0 += U, at ^= 1) {
      const int64_t tb = te - k0 - U;  // the batch's first token
      if (tb + U <= t0) break;
      copies_done();
      fetch(at ^ 1, tb - U);
      const T(&in)[A][U][Rows::kCols] = stages[at];
      const uint32_t live = above(tb);
      float s[kOwn], g[kOwn];
#pragma unroll
      for (int j = 0; j < kOwn; ++j) {
        const int k = j * LP + part;
        s[j] = g[j] = 0.f;  // a token in front of the chunk changes nothing: its decay is 1
        if (live >> k & 1) {
          s[j] = to_f32(in[0][k][col]) + bias;
          if (a.softplus) s[j] = softplus(s[j]);
          sum += s[j];
          g[j] = to_f32(in[1][k][col]);
          if (GATE) {
            const float zv = to_f32(in[A - 1][k][col]);
            g[j] *= zv * sigmoid(zv);
          }
        }
      }
      f32x2 e[NS / 2], en[NS / 2];
      decay<NS>(from_lane<LP>(s[kOwn - 1], LP - 1), a2, e);
#pragma unroll
      for (int k = U - 1; k >= 0; --k) {
        if (k) decay<NS>(from_lane<LP>(s[(k ? k - 1 : 0) / LP], (k ? k - 1 : 0) % LP), a2, en);
        const float gv = from_lane<LP>(g[k / LP], k % LP);
        const f32x2 gg = pair(gv, gv);
        const float* row = &sc[buf][kScanTile - U - k0 + k][me.n0];
#pragma unroll
        for (int i = 0; i < NS / 2; i += 2) {
          const ulonglong2 cc = *reinterpret_cast<const ulonglong2*>(row + 2 * i);
          r[i] = mul2(e[i], fma2(cc.x, gg, r[i]));
          r[i + 1] = mul2(e[i + 1], fma2(cc.y, gg, r[i + 1]));
        }
#pragma unroll
        for (int i = 0; i < NS / 2; ++i) e[i] = en[i];
      }
    }
    stage.put(&sc[buf ^ 1][0][0]);
    __syncthreads();
  }
  sum = sum_lanes<LP>(sum);
  if (!me.valid) return;
  store_pairs<NS, FULL>(w.state + ((uint64_t)chunk * a.channels + me.c) * N, me.n0, N, r);
  if (me.first) w.sum[(uint64_t)chunk * a.channels + me.c] = sum;
}

// Sums over a warp's channels.  For each of four tokens a warp's lanes leave
// their states in 128 NS bytes of shared memory: row by row of channels, quads
// of states at slot ^ turn(row), so that neither the lanes' stores (a row after
// another) nor the sums' loads (a slot's quads of several rows) meet on a bank.
// Adding in shared memory takes a fraction of the instructions that exchanges
// between lanes take.
template <int NS, int LP>
struct WarpSum {
  static constexpr int kRows = 32 / LP, kEach = NS / 4, kSlots = kEach * LP, kQuads = 8 * NS;  // kQuads: of a token
  static constexpr int kShare = 32 / (4 * kSlots) > 0 ? 32 / (4 * kSlots) : 1;                 // lanes per sum
  static constexpr int kItems = 4 * kSlots * kShare;
  static __device__ __forceinline__ uint32_t turn(uint32_t row) {
    if constexpr (NS == 4 || LP > 4) return 0;
    else return (row >> (LP == 1 ? 2 : LP == 2 ? 1 : 0) & 1) * LP;
  }
  // Lane's states of token k (0..3).
  static __device__ __forceinline__ void put(float* v, int k, const f32x2 (&s)[NS / 2]) {
    const uint32_t lane = threadIdx.x & 31, row = lane / LP, part = lane % LP;
    ulonglong2* q = reinterpret_cast<ulonglong2*>(v) + k * kQuads + row * kSlots;
#pragma unroll
    for (int i = 0; i < kEach; ++i) q[(i * LP + part) ^ turn(row)] = make_ulonglong2(s[2 * i], s[2 * i + 1]);
  }
  // The four tokens' sums to out[token * stride + state].
  static __device__ __forceinline__ void add(const float* v, float* out, int stride) {
    const uint32_t lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int it = 0; it < kItems / 32; ++it) {
      const uint32_t item = it * 32 + lane, k = item / (kSlots * kShare), slot = item / kShare % kSlots, share = item % kShare;
      const ulonglong2* q = reinterpret_cast<const ulonglong2*>(v) + k * kQuads;
      f32x2 lo = 0ull, hi = 0ull;
#pragma unroll
      for (int i = 0; i < kRows / kShare; ++i) {
        const uint32_t row = i * kShare + share;
        const ulonglong2 t = q[row * kSlots + (slot ^ turn(row))];
        lo = i ? add2(lo, t.x) : t.x;
        hi = i ? add2(hi, t.y) : t.y;
      }
      float s[4];
      unpair(lo, s[0], s[1]);
      unpair(hi, s[2], s[3]);
#pragma unroll
      for (int o = 1; o < kShare; o <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
      if (share == 0)
        *reinterpret_cast<float4*>(out + k * stride + slot % LP * NS + slot / LP * 4) = make_float4(s[0], s[1], s[2], s[3]);
    }
    __syncwarp();
  }
};

template <class T, int NS, int LP>
struct BackShared {
  float bc[2][kScanTile][2][NS * LP];
  float red[2][kWarps][2][kBlock][NS * LP];  // dB's sums, then dC's
  float sum[kWarps][4][32 * NS];
  float4 cell[kWarps][kBlock][40 / LP];  // step, step times x, gradient behind the gate; rows apart by 8 / LP quads of banks
  float mark[kWarps][2][32 / LP][NS * LP];
  T rows[kWarps][2][4][kBlock][32 / LP];  // x, dt, dy, z
  T results[kWarps][3][kBlock][32 / LP];  // dx, ddt, dz
};

// A block of kBlock tokens at a time, last ones first: forwards from its mark
// with the states kept in registers, then backwards.  EDGES: a sequence begins
// or ends inside the block.
template <class T, int NS, int LP, bool FULL, bool GATE>
__global__ void __launch_bounds__(kScanThreads, resident(NS)) sscan_back_kernel(SscanArgs a, ScanPlan p, BackWork w, int aligned) {
  constexpr int NP = NS * LP, NH = NS / 2, K = kBlock, kOwn = K / LP, kEach = K * 2 * NP / kScanThreads;
  extern __shared__ __align__(16) unsigned char shared_bytes[];
  BackShared<T, NS, LP>& sh = *reinterpret_cast<BackShared<T, NS, LP>*>(shared_bytes);
  const uint32_t N = a.states;
  const ScanLane<NS, LP> me(a.channels, a.groups, p.per_group, blockIdx.x % p.ctiles);
  const uint32_t part = threadIdx.x % LP, warp = threadIdx.x >> 5;
  const int64_t chunk = blockIdx.x / p.ctiles;
  const int64_t t0 = chunk * (int64_t)p.len, t1 = min(t0 + (int64_t)p.len, (int64_t)a.seq.tokens);
  float* sums = &sh.sum[warp][0][0];
  using Rows = WarpRows<T, LP>;
  constexpr int kRows = 40 / LP, A = GATE ? 4 : 3;
  const uint32_t col = threadIdx.x % 32 / LP;
  float4* const cells = &sh.cell[warp][0][col];  // this channel's, of the block's tokens
  f32x2 a2[NH], r[NH], da[NH];
  load_pairs<NS, FULL>(a.a + (uint64_t)me.c * N, me.n0, N, a2, kLog2e);
  zero_pairs(r);
  zero_pairs(da);
  const uint64_t row = ((uint64_t)chunk * a.channels + me.c) * N;
  if (p.carry && me.valid) load_pairs<NS, FULL>(w.scan.state + row, me.n0, N, r);
  const float bias = a.dt_bias ? a.dt_bias[me.c] : 0.f;
  const bool skip = a.d != nullptr;  // without it no term: 0 times an infinite value would be NaN
  const float dskip = skip ? a.d[me.c] : 0.f;
  float dd = 0.f, dbias = 0.f;
  const auto state_row = [&](int64_t seq) {
    const int64_t slot = a.seq.slot(seq);
    return slot < 0 || !me.valid ? -1 : (int64_t)(((uint64_t)slot * a.channels + me.c) * N);
  };
  // The block from t on: the rows of the tokens that `live` names, and the states at its mark.
  RowsIn arrays[A];
  arrays[0] = {a.x, a.x_row};
  arrays[1] = {a.dt, a.dt_row};
  arrays[2] = {a.dy, a.dy_row};
  if constexpr (GATE) arrays[3] = {a.z, a.z_row};
  const int64_t tiles = (t1 - t0 + kScanTile - 1) / kScanTile;
  RowsCursor<T, LP, A, -1> cursor(arrays, t0 + tiles * kScanTile - K, me.warp_c, me.warp_cols);
  const auto fetch = [&](int at, int64_t t, uint32_t live) {
    if (aligned == 2) cursor.copy(sh.rows[warp][at], live);
    else Rows::in(sh.rows[warp][at], arrays, t, live, me.warp_c, me.warp_cols, aligned);
    if (live & 1) {
      const float* from = a.marks + ((uint64_t)(t / K) * a.channels + me.warp_c) * N;
      float* to = &sh.mark[warp][at][0][0];
      if constexpr (FULL) {
#pragma unroll
        for (int i = 0; i < 32 / LP * NP / 4; i += 32) {
          const uint32_t q = i + threadIdx.x % 32;
          if (q < me.warp_cols * (NP / 4)) copy_async<16>(to + 4 * q, from + 4 * q, 16);
        }
      } else {
        for (uint32_t i = threadIdx.x % 32; i < me.warp_cols * N; i += 32) to[i / N * NP + i % N] = from[i];
      }
    }
    copies_issued();
  };
  // Where this thread puts its sums over the block's warps: row t of its channel tile, its own offsets in there.
  float* const part_rows = w.bc + ((uint64_t)me.channel_tile * a.seq.tokens * a.groups + me.group) * 2 * N;
  const uint32_t part_row = a.groups * 2 * N;

  StageBC<T, NP, 2> stage;
  TileMarks m, before;
  if (tiles > 0) {
    m = tile_marks(a.seq, t0 + (tiles - 1) * kScanTile, t1);
    stage.fetch(a, me.group, t0 + (tiles - 1) * kScanTile, m.live);
    stage.put(&sh.bc[0][0][0][0]);
    fetch(0, t0 + tiles * kScanTile - K, m.live >> (kScanTile - K));
  }
  __syncthreads();
  int buf = 0, out = 0, at = 0;
  for (int64_t tile = tiles - 1; tile >= 0; --tile, buf ^= 1, m = before) {
    const int64_t tb = t0 + tile * kScanTile;
    before.live = 0;
    if (tile > 0) {
      before = tile_marks(a.seq, tb - kScanTile, t1);
      stage.fetch(a, me.group, tb - kScanTile, before.live);
    }
#pragma unroll 1
    for (int k0 = kScanTile - K; k0 >= 0; k0 -= K, at ^= 1) {
      constexpr uint32_t kAll = (1u << K) - 1;
      const uint32_t live = m.live >> k0 & kAll, start = m.start >> k0 & kAll, end = m.end >> k0 & kAll;
      const int64_t tk = tb + k0;
      // This lane's own tokens: steps, gates; those that are no tokens change nothing (e = 1).
      float s[kOwn], g[kOwn], xv[kOwn], slope[kOwn], gg[kOwn];
      copies_done();
      fetch(at ^ 1, tk - K, k0 ? m.live >> (k0 - K) : before.live >> (kScanTile - K));
      const T(&in)[4][K][Rows::kCols] = sh.rows[warp][at];
      T(&result)[3][K][Rows::kCols] = sh.results[warp];
#pragma unroll
      for (int j = 0; j < kOwn; ++j) {
        s[j] = g[j] = xv[j] = slope[j] = gg[j] = 0.f;
        if ((live >> (j * LP + part) & 1) && me.valid) {
          const int k = j * LP + part;
          xv[j] = to_f32(in[0][k][col]);
          s[j] = to_f32(in[1][k][col]) + bias;
          slope[j] = 1.f;
          if (a.softplus) s[j] = softplus(s[j], slope[j]);
          g[j] = to_f32(in[2][k][col]);
          if (GATE) {
            const float zv = to_f32(in[3][k][col]), sig = sigmoid(zv);
            gg[j] = g[j] * gate_grad(zv, sig);
            g[j] *= zv * sig;
          }
        }
        cells[(j * LP + part) * kRows] = make_float4(s[j], s[j] * xv[j], g[j], 0.f);
      }
      __syncwarp();
      f32x2 h[NH];
      zero_pairs(h);
      if ((live & 1) && me.valid) load_pairs<NS, FULL>(&sh.mark[warp][at][col][0], me.n0, N, h);
      const float(*const rows)[2][NP] = &sh.bc[buf][k0];
      float(*const red)[K][NP] = sh.red[out][warp];
      const auto walk = [&](auto edges) {
        constexpr bool EDGES = decltype(edges)::value;
        f32x2 hp[K][NH], e[NH], en[NH];
        // This block's sums over tokens, added to the chunk's at its end: one running sum over
        // the thousands of tokens of a chunk loses a decimal place to a sum of sums.
        f32x2 da_block[NH];
        float dd_block = 0.f, dbias_block = 0.f;
        zero_pairs(da_block);
        float o[LP];
        // Forwards.
        float4 now = cells[0], next;
        decay<NS>(now.x, a2, e);
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int j = k / LP, q = k % LP;
          if (k + 1 < K) {
            next = cells[(k + 1) * kRows];
            decay<NS>(next.x, a2, en);
          }
          if (EDGES && k && (start >> k & 1)) {
            zero_pairs(h);
            const int64_t at = a.state ? state_row(tile_seq(m, k0 + k)) : -1;
            if (at >= 0) load_pairs<NS, FULL>(a.state + at, me.n0, N, h);
          }
          const f32x2 xx = pair(now.y, now.y), gv = pair(now.z, now.z);
          f32x2 v[NH], oo = 0ull;
#pragma unroll
          for (int i = 0; i < NH; i += 2) {
            const ulonglong2 bb = *reinterpret_cast<const ulonglong2*>(&rows[k][0][me.n0 + 2 * i]);
            f32x2 add[2] = {mul2(xx, bb.x), mul2(xx, bb.y)};
            if (!FULL) {
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                float lo, hi;
                unpair(add[u], lo, hi);
                const uint32_t n = me.n0 + 2 * (i + u);
                add[u] = pair(n < N ? lo : 0.f, n + 1 < N ? hi : 0.f);
              }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              hp[k][i + u] = h[i + u];
              h[i + u] = fma2(e[i + u], h[i + u], add[u]);
              v[i + u] = mul2(gv, h[i + u]);
            }
            if (GATE) {
              const ulonglong2 cc = *reinterpret_cast<const ulonglong2*>(&rows[k][1][me.n0 + 2 * i]);
              oo = fma2(cc.x, h[i], oo);
              oo = fma2(cc.y, h[i + 1], oo);
            }
          }
          WarpSum<NS, LP>::put(sums, k & 3, v);
          if ((k & 3) == 3) WarpSum<NS, LP>::add(sums, &red[1][0][0] + (k - 3) * NP, NP);
          if (GATE) {
            o[q] = sum2(oo);
            if (q == LP - 1) {
              float pre = scatter_sum<LP>(o, part);
              if (skip) pre = __fmaf_rn(dskip, xv[j], pre);
              result[2][j * LP + part][col] = from_f32<T>(gg[j] * pre);
            }
          }
#pragma unroll
          for (int i = 0; i < NH; ++i) e[i] = en[i];
          now = next;
        }
        // Backwards.
        float gb[LP], ga[LP];
        now = cells[(K - 1) * kRows];
        decay<NS>(now.x, a2, e);
#pragma unroll
        for (int k = K - 1; k >= 0; --k) {
          const int j = k / LP, q = k % LP;
          if (k) {
            next = cells[(k - 1) * kRows];
            decay<NS>(next.x, a2, en);
          }
          if ((EDGES || k == K - 1) && (end >> k & 1)) {
            zero_pairs(r);
            const int64_t at = a.dfinal ? state_row(tile_seq(m, k0 + k)) : -1;
            if (at >= 0) load_pairs<NS, FULL>(a.dfinal + at, me.n0, N, r);
          }
          const f32x2 ss = pair(now.x, now.x), xx = pair(now.y, now.y), gv = pair(now.z, now.z);
          f32x2 v[NH], gb2 = 0ull, ga2 = 0ull;
#pragma unroll
          for (int i = 0; i < NH; i += 2) {
            const ulonglong2 bb = *reinterpret_cast<const ulonglong2*>(&rows[k][0][me.n0 + 2 * i]);
            const ulonglong2 cc = *reinterpret_cast<const ulonglong2*>(&rows[k][1][me.n0 + 2 * i]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const f32x2 gh = fma2(u ? cc.y : cc.x, gv, r[i + u]);
              gb2 = fma2(gh, u ? bb.y : bb.x, gb2);
              r[i + u] = mul2(e[i + u], gh);
              const f32x2 through = mul2(r[i + u], hp[k][i + u]);
              ga2 = fma2(through, a2[i + u], ga2);
              da_block[i + u] = fma2(through, ss, da_block[i + u]);
              v[i + u] = mul2(gh, xx);
            }
          }
          WarpSum<NS, LP>::put(sums, k & 3, v);
          if ((k & 3) == 0) WarpSum<NS, LP>::add(sums, &red[0][0][0] + k * NP, NP);
          gb[q] = sum2(gb2);
          ga[q] = sum2(ga2);
          if (q == 0) {
            const float gbs = scatter_sum<LP>(gb, part), gas = scatter_sum<LP>(ga, part);
            const float ds = (live >> (j * LP + part) & 1) ? __fmaf_rn(gas, 1.0f / kLog2e, xv[j] * gbs) * slope[j] : 0.f;
            dd_block = __fmaf_rn(g[j], xv[j], dd_block);
            dbias_block += ds;
            const float through_b = s[j] * gbs;
            result[0][j * LP + part][col] = from_f32<T>(skip ? __fmaf_rn(dskip, g[j], through_b) : through_b);
            result[1][j * LP + part][col] = from_f32<T>(ds);
          }
          if ((EDGES || k == 0) && (start >> k & 1)) {
            const int64_t at = a.dstate ? state_row(tile_seq(m, k0 + k)) : -1;
            if (at >= 0) store_pairs<NS, FULL>(a.dstate + at, me.n0, N, r);
            zero_pairs(r);  // rows in front of it belong to no sequence, or end one
          }
#pragma unroll
          for (int i = 0; i < NH; ++i) e[i] = en[i];
          now = next;
        }
#pragma unroll
        for (int i = 0; i < NH; ++i) da[i] = add2(da[i], da_block[i]);
        dd += dd_block;
        dbias += dbias_block;
      };
      if (live == kAll && !(start & ~1u) && !(end & (kAll >> 1))) walk(std::false_type{});
      else if (live) walk(std::true_type{});
      __syncwarp();
      Rows::out(result[0], a.dx, a.dx_row, tk, live, me.warp_c, me.warp_cols, aligned);
      Rows::out(result[1], a.ddt, a.ddt_row, tk, live, me.warp_c, me.warp_cols, aligned);
      if (GATE) Rows::out(result[2], a.dz, a.dz_row, tk, live, me.warp_c, me.warp_cols, aligned);
      __syncthreads();
      float* const to = part_rows + (uint64_t)(uint32_t)tk * part_row;
#pragma unroll
      for (int u = 0; u < kEach; ++u) {
        const uint32_t i = u * kScanThreads + threadIdx.x, n = i % NP, k = i / NP % K, which = i / (NP * K);
        if (n >= N || !(live >> k & 1)) continue;
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < kWarps; ++q) v += sh.red[out][q][which][k][n];
        to[(uint64_t)k * part_row + which * N + n] = v;
      }
      out ^= 1;  // the next block of tokens writes the other one while this is read
    }
    if (tile > 0) stage.put(&sh.bc[buf ^ 1][0][0][0]);
    __syncthreads();
  }
  dd = sum_lanes<LP>(dd);
  dbias = sum_lanes<LP>(dbias);
  if (!me.valid) return;
  store_pairs<NS, FULL>(w.da + row, me.n0, N, da);
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
    const int64_t at = state_row(i);
    if (at < 0) continue;
    zero_pairs(r);
    if (a.dfinal) load_pairs<NS, FULL>(a.dfinal + at, me.n0, N, r);
    store_pairs<NS, FULL>(a.dstate + at, me.n0, N, r);
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

// 8 states a lane; 4 where the blocks are too few to fill the SMs.  With 4 (and
// twice the warps) the sums over channels and the rows of B and C take the
// shared memory's bandwidth: 1.46 ms a training step against 1.37 at 16384 tokens
// x 2048 channels x 16 states, but this kernel 41 us against 65 at 1531 x 402 x 11.
ScanLanes lanes_of(uint32_t states) {
  const uint32_t least = states <= 8 ? 1 : states <= 16 ? 2 : states <= 32 ? 4 : 8;
  return {least, least == 8 ? 8 : 2 * least, (uint32_t)resident(8), 8 * least, 16u, 21u};
}

ScanPlan plan_of(uint64_t tokens, uint32_t channels, uint32_t states, uint64_t n_seq, uint32_t groups, bool ragged) {
  return scan_plan(tokens, channels, groups, n_seq, ragged, lanes_of(states));
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

// The chunk pass takes the same chunks with 4 states a lane (8 of 32, 16 of 64):
// its blocks are few.  With 16 states a lane wherever that leaves three blocks an SM
// the gradients' calls took 187 us against 175 (28,600 unequal tokens x 64 channels
// x 16 states), 886 against 877 (10,400 x 4096 x 8), 74 against 71 (700 x 2048 x 8).
constexpr uint32_t chunk_lanes(uint32_t padded) { return padded <= 8 ? 2 : 4; }
ScanPlan chunk_plan(ScanPlan p, uint32_t channels, uint32_t groups, uint32_t padded) {
  p.lanes = chunk_lanes(padded);
  p.per_group = (channels / groups + kScanThreads / p.lanes - 1) / (kScanThreads / p.lanes);
  p.ctiles = p.per_group * groups;
  return p;
}

template <class T, int NS, int LP, bool FULL, bool GATE>
cudaError_t go(const SscanArgs& a, const ScanPlan& p, cudaStream_t s) {
  BackWork w{};
  back_work(p, a.seq.tokens, a.channels, a.states, a.groups, a.work, &w);
  const uint64_t grid = p.chunks * p.ctiles, cells = a.seq.tokens * a.groups * 2 * a.states;
  if (grid > 0x7fffffffull / 8 || cells / 256 >= 0x7fffffffull) return cudaErrorInvalidValue;
  cudaError_t e;
  if (p.carry) {
    constexpr int NP = NS * LP, CL = chunk_lanes(NP);
    const ScanPlan q = chunk_plan(p, a.channels, a.groups, NP);
    sscan_chunk_back_kernel<T, NP / CL, CL, FULL, GATE><<<(unsigned)(q.chunks * q.ctiles), kScanThreads, 0, s>>>(
        a, q, w.scan, rows_aligned<T, CL>(a, {{a.dt, a.dt_row}, {a.dy, a.dy_row}, {a.z, a.z_row}}));
    e = launch_sscan_fold_back(a.a, w.scan, p.chunks, a.channels, a.states, s);
    if (e != cudaSuccess) return e;
  }
  constexpr int bytes = sizeof(BackShared<T, NS, LP>);
  const auto kernel = sscan_back_kernel<T, NS, LP, FULL, GATE>;
  if (bytes > 48 * 1024) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
  }
  const int aligned = rows_aligned<T, LP>(a, {{a.x, a.x_row}, {a.dt, a.dt_row}, {a.dy, a.dy_row}, {a.z, a.z_row},
                                              {a.dx, a.dx_row}, {a.ddt, a.ddt_row}, {a.dz, a.dz_row}});
  kernel<<<(unsigned)grid, kScanThreads, bytes, s>>>(a, p, w, aligned);
  if (cells) sscan_bc_kernel<T><<<(unsigned)((cells + 255) / 256), 256, 0, s>>>(a, w.bc, p.per_group);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const uint64_t as = (uint64_t)a.channels * a.states;
  e = launch_reduce_rows(w.da, p.chunks, as, as, a.da, nullptr, s);
  if (e == cudaSuccess && (a.dd || a.ddt_bias))
    e = launch_reduce_rows(w.dd, p.chunks, 2ull * a.channels, a.channels, a.dd, a.ddt_bias, s);
  return e;
}

template <class T, int NS, int LP>
cudaError_t by_form(const SscanArgs& a, const ScanPlan& p, cudaStream_t s) {
  const bool full = a.states == NS * LP && aligned16(a.a) && aligned16(a.state) && aligned16(a.dstate) &&
                    aligned16(a.dfinal) && aligned16(a.marks) && aligned16(a.work);
  if (full) return a.z ? go<T, NS, LP, true, true>(a, p, s) : go<T, NS, LP, true, false>(a, p, s);
  return a.z ? go<T, NS, LP, false, true>(a, p, s) : go<T, NS, LP, false, false>(a, p, s);
}

template <class T>
cudaError_t by_states(const SscanArgs& a, cudaStream_t s) {
  const ScanPlan p = plan_of(a.seq.tokens, a.channels, a.states, a.seq.n_seq, a.groups, a.seq.seq_ptr != nullptr);
  const bool wide = p.lanes == lanes_of(a.states).least;
  if (a.states <= 8) return wide ? by_form<T, 8, 1>(a, p, s) : by_form<T, 4, 2>(a, p, s);
  if (a.states <= 16) return wide ? by_form<T, 8, 2>(a, p, s) : by_form<T, 4, 4>(a, p, s);
  if (a.states <= 32) return wide ? by_form<T, 8, 4>(a, p, s) : by_form<T, 4, 8>(a, p, s);
  return by_form<T, 8, 8>(a, p, s);
}

}  // namespace

}  // namespace sparsl
