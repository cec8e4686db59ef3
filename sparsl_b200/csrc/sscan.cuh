// What the forward and the backward kernels of the selective scan share: the
// split of the token axis into chunks, the workspace, and a channel's
// arithmetic.
#pragma once

#include <initializer_list>

#include "seq.cuh"

namespace sparsl {

constexpr uint32_t kMarkEvery = 8;  // tokens between two saved states of a training pass
constexpr int kScanThreads = 128;
constexpr int kScanTile = 32;       // tokens whose B and C are staged at a time
constexpr uint32_t kSms = 148;

// The token axis [0, tokens) in chunks of `len` tokens (a multiple of 32),
// whatever sequences they hold.  `carry`: a sequence may span chunks, so the
// states at the chunks' starts are computed first.
struct ScanPlan {
  uint32_t ctiles;     // channel tiles, each within one group
  uint32_t per_group;  // of which each group has this many
  uint32_t lanes;      // that share a channel
  uint64_t len, chunks;
  bool carry;
};

// How many lanes share a channel's states: `least` is what the registers
// demand, up to `most`; the blocks that an SM holds; the states, with those that
// pad them; and how full, in twentieths, whole sequences have to make their waves of
// blocks (`thin`: with lanes of 4 states; above 20: never).
struct ScanLanes {
  uint32_t least, most, resident, states, fill, thin;
};

inline ScanPlan scan_plan(uint64_t tokens, uint32_t channels, uint32_t groups, uint64_t n_seq, bool ragged, ScanLanes l) {
  ScanPlan p;
  const uint32_t cpg = channels / groups;
  const auto tiles = [&](uint32_t lanes) { return (cpg + kScanThreads / lanes - 1) / (kScanThreads / lanes); };
  const uint64_t run = n_seq ? tokens / n_seq : 0, slots = (uint64_t)kSms * l.resident;
  // One wave of blocks over equal chunks, of 64 tokens at least (two where
  // sequences are unequal: chunks whose sequences end in them have little to do in
  // the first pass, and leave their SMs to others); more lanes a channel where
  // that leaves SMs with fewer than three quarters of their blocks.
  for (uint32_t k = l.least; k <= l.most; k *= 2) {
    const uint64_t ct = (uint64_t)groups * tiles(k), some = ragged ? 2 * slots : slots, want = ct >= some ? 1 : some / ct;
    p.lanes = k;
    p.len = (tokens + want - 1) / want;
    p.len = p.len < 64 ? 64 : (p.len + 31) / 32 * 32;
    p.chunks = tokens ? (tokens + p.len - 1) / p.len : 1;
    if (4 * p.chunks * ct >= 3 * slots) break;
  }
  p.carry = p.chunks > 1;
  // Whole sequences instead, in one pass without the states at the chunks'
  // starts, where they fill enough of their waves of blocks.  Measured in us, whole
  // sequences against chunks, bf16 tokens x 2048 channels (share of the waves):
  // Prompts, whose chunks take nearly twice the work, from two fifths on: 16 states,
  // 7 x 2048 tokens (0.38) 357 : 356, 8 x 2048 (0.43) 356 : 381, 8 x 512 96 : 124; 8
  // states, 12 x 1024 (0.32) 200 : 200; 32 states, 6 x 1024 (0.32) 286 : 295; 64 states,
  // 1024 channels, 7 x 1024 (0.38) 486 : 452, 8 x 1024 (0.43) 486 : 513.  With 4 states
  // a lane from three fifths on: 4 x 2048 (0.43) 292 : 205, 6 x 2048 (0.65) 327 : 304,
  // 6 x 512 88 : 100, f32 6 x 1024 162 : 180.
  // Gradients, whose first pass over the chunks is a fifth of it, from four fifths
  // on: 7 x 2048 (0.76) 977 : 948, 8 x 2048 (0.86) 979 : 1070, 12 x 2048 (0.65 of two
  // waves) 1702 : 1513; never with 4 states a lane: 4 x 2048 (0.86) 774 : 582.
  if (!ragged && run && run % 32 == 0)
    for (uint32_t k = l.least; k <= l.most; k *= 2) {
      const uint64_t blocks = n_seq * groups * tiles(k), waves = (blocks + slots - 1) / slots;
      if (20 * blocks < (l.states / k == 4 ? l.thin : l.fill) * waves * slots && run > 64) continue;
      p.lanes = k;
      p.len = run;
      p.chunks = n_seq;
      p.carry = false;
      break;
    }
  p.per_group = tiles(p.lanes);
  p.ctiles = p.per_group * groups;
  return p;
}

// Workspace of a pass with carry: per chunk the state it hands on, the sum of
// its steps, whether a sequence begins in it, and the state its last sequence
// began from (in place, the pool's row may be overwritten before it is read).
struct ScanWork {
  float* state;  // [chunks, channels, states]
  float* start;  // the same, or null
  float* sum;    // [chunks, channels]
  int32_t* cut;  // [chunks]
};
inline uint64_t scan_round(uint64_t v) { return (v + 255) / 256 * 256; }
inline uint64_t scan_work(const ScanPlan& p, uint32_t channels, uint32_t states, bool start, void* base, ScanWork* w) {
  const uint64_t st = scan_round(p.chunks * channels * states * 4), su = scan_round(p.chunks * channels * 4);
  char* b = static_cast<char*>(base);
  uint64_t at = 0;
  if (w) w->state = reinterpret_cast<float*>(b);
  at += st;
  if (w) w->start = start ? reinterpret_cast<float*>(b + at) : nullptr;
  if (start) at += st;
  if (w) w->sum = reinterpret_cast<float*>(b + at);
  at += su;
  if (w) w->cut = reinterpret_cast<int32_t*>(b + at);
  return at + scan_round(p.chunks * 4);
}

// log(1 + e^v): max(v, 0) + log1p(u) with u = e^-|v| in [0, 1], log1p(u) / u by
// its degree-9 Chebyshev interpolant there (relative error 1e-7 in f32, small
// steps included).
__device__ __forceinline__ float softplus_from(float v, float u) {
  float p = -0.0031760570127516985f;
  p = __fmaf_rn(p, u, 0.019542526453733444f);
  p = __fmaf_rn(p, u, -0.056373611092567444f);
  p = __fmaf_rn(p, u, 0.10543623566627502f);
  p = __fmaf_rn(p, u, -0.1526966691017151f);
  p = __fmaf_rn(p, u, 0.1966327428817749f);
  p = __fmaf_rn(p, u, -0.24951615929603577f);
  p = __fmaf_rn(p, u, 0.33329710364341736f);
  p = __fmaf_rn(p, u, -0.49999892711639404f);
  p = __fmaf_rn(p, u, 1.0f);
  return __fmaf_rn(u, p, fmaxf(v, 0.0f));
}
__device__ __forceinline__ float softplus(float v) { return softplus_from(v, ex2(-kLog2e * fabsf(v))); }

// The same and its slope, the sigmoid of v, from one exponential.
__device__ __forceinline__ float softplus(float v, float& slope) {
  const float u = ex2(-kLog2e * fabsf(v)), r = rcp(1.0f + u);
  slope = v >= 0.0f ? r : u * r;
  return softplus_from(v, u);
}

// A channel's value in row t of a token array.
template <class T>
__device__ __forceinline__ T* cell(const void* p, int64_t t, uint32_t row, uint32_t c) {
  const char* q = static_cast<const char*>(p) + ((uint64_t)(uint32_t)t * row + c * (uint32_t)sizeof(T));
  return reinterpret_cast<T*>(const_cast<char*>(q));
}

// NS states of a channel, from index n0 of N; FULL: all exist and every row is
// 16-byte aligned.  States that do not exist stay 0.
template <int NS, bool FULL>
__device__ __forceinline__ void load_states(const float* p, uint32_t n0, uint32_t N, float (&h)[NS]) {
  if constexpr (FULL) {
#pragma unroll
    for (int j = 0; j < NS; j += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + n0 + j);
      h[j] = v.x;
      h[j + 1] = v.y;
      h[j + 2] = v.z;
      h[j + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < NS; ++j) h[j] = n0 + j < N ? p[n0 + j] : 0.f;
  }
}
template <int NS, bool FULL>
__device__ __forceinline__ void store_states(float* p, uint32_t n0, uint32_t N, const float (&h)[NS]) {
  if constexpr (FULL) {
#pragma unroll
    for (int j = 0; j < NS; j += 4)
      *reinterpret_cast<float4*>(p + n0 + j) = make_float4(h[j], h[j + 1], h[j + 2], h[j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < NS; ++j)
      if (n0 + j < N) p[n0 + j] = h[j];
  }
}
template <int NS>
__device__ __forceinline__ void zero_states(float (&h)[NS]) {
#pragma unroll
  for (int j = 0; j < NS; ++j) h[j] = 0.f;
}

// Which of 32 tokens from tb on (below t1) belong to a sequence, begin one and
// end one; lane k keeps the sequence of token tb + k.
struct TileMarks {
  uint32_t live, start, end;
  int64_t seq;
};
__device__ __forceinline__ TileMarks tile_marks(const SeqView& s, int64_t tb, int64_t t1) {
  const int64_t t = tb + (threadIdx.x & 31);
  TileMarks m;
  m.seq = -1;
  bool live = false, start = false, end = false;
  if (t < t1) {
    const int64_t i = s.of(t);
    if (i >= 0 && i < (int64_t)s.n_seq) {
      const int64_t e = s.begin(i + 1);
      live = t < e;
      start = live && t == s.begin(i);
      end = live && t + 1 == e;
      m.seq = i;
    }
  }
  m.live = __ballot_sync(0xffffffffu, live);
  m.start = __ballot_sync(0xffffffffu, start);
  m.end = __ballot_sync(0xffffffffu, end);
  return m;
}
__device__ __forceinline__ int64_t tile_seq(const TileMarks& m, int k) {
  return __shfl_sync(0xffffffffu, (long long)m.seq, k);
}

// A thread's place: LP lanes share a channel, NS states each.
template <int NS, int LP>
struct ScanLane {
  uint32_t group, c, n0, channel_tile, first;
  uint32_t warp_c, warp_cols;  // the warp's first channel, and how many it has
  bool valid;  // the lane's channel exists (else it works on the group's last one and writes nothing)
  __device__ __forceinline__ ScanLane(uint32_t channels, uint32_t groups, uint32_t per_group, uint32_t ct) {
    constexpr uint32_t kWarp = 32 / LP, kBlock = kScanThreads / LP;
    const uint32_t cpg = channels / groups;
    group = ct / per_group;
    channel_tile = ct % per_group;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t cl = channel_tile * kBlock + warp * kWarp + lane / LP;
    valid = cl < cpg;
    c = group * cpg + (valid ? cl : cpg - 1);
    const uint32_t w0 = channel_tile * kBlock + warp * kWarp;
    warp_c = group * cpg + (w0 < cpg ? w0 : cpg - 1);
    warp_cols = w0 >= cpg ? 0 : cpg - w0 < kWarp ? cpg - w0 : kWarp;
    n0 = (lane % LP) * NS;
    first = lane % LP == 0;
  }
};

template <int LP>
__device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
  for (int o = 1; o < LP; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The decays exp(s A) of NS states, two at a time.  The special function unit's
// powers of two are 2e-8 low on the average over [-1, 0) (measured over a million
// arguments each in ten ranges; 3.8e-8 root mean square): a state that remembers a
// thousand tokens would be 2e-5 low.  kLift added to the exponent, in the
// product's own instruction, takes the mean below 1e-8: the error of dA against 64
// bits at 16384 tokens x 2048 channels went from 1.9e-6 to 0.9e-6.
constexpr float kLift = 2.5e-8f;
template <int NS>
__device__ __forceinline__ void decay(float s, const f32x2 (&a2)[NS / 2], f32x2 (&e)[NS / 2]) {
  const f32x2 ss = pair(s, s), lift = pair(kLift, kLift);
#pragma unroll
  for (int j = 0; j < NS / 2; ++j) e[j] = ex2_2(fma2(ss, a2[j], lift));
}
template <int NS, bool FULL>
__device__ __forceinline__ void load_pairs(const float* p, uint32_t n0, uint32_t N, f32x2 (&h)[NS / 2], float scale = 1.f) {
  float v[NS];
  load_states<NS, FULL>(p, n0, N, v);
#pragma unroll
  for (int j = 0; j < NS / 2; ++j) h[j] = pair(v[2 * j] * scale, v[2 * j + 1] * scale);
}
template <int NS, bool FULL>
__device__ __forceinline__ void store_pairs(float* p, uint32_t n0, uint32_t N, const f32x2 (&h)[NS / 2]) {
  float v[NS];
#pragma unroll
  for (int j = 0; j < NS / 2; ++j) unpair(h[j], v[2 * j], v[2 * j + 1]);
  store_states<NS, FULL>(p, n0, N, v);
}
// The same 32 bytes at a time, a whole sector of a lane's row by one instruction
// (FULL, NS a multiple of 8, rows on 32-byte boundaries).
template <int NS, bool FULL>
__device__ __forceinline__ void load_rows(const float* p, uint32_t n0, uint32_t N, f32x2 (&h)[NS / 2]) {
  if constexpr (FULL && NS % 8 == 0) {
#pragma unroll
    for (int j = 0; j < NS / 2; j += 4)
      asm volatile("ld.global.v4.b64 {%0, %1, %2, %3}, [%4];" : "=l"(h[j]), "=l"(h[j + 1]), "=l"(h[j + 2]), "=l"(h[j + 3]) : "l"(p + n0 + 2 * j) : "memory");
  } else {
    load_pairs<NS, FULL>(p, n0, N, h);
  }
}
template <int NS, bool FULL>
__device__ __forceinline__ void store_rows(float* p, uint32_t n0, uint32_t N, const f32x2 (&h)[NS / 2]) {
  if constexpr (FULL && NS % 8 == 0) {
#pragma unroll
    for (int j = 0; j < NS / 2; j += 4)
      asm volatile("st.global.v4.b64 [%0], {%1, %2, %3, %4};" ::"l"(p + n0 + 2 * j), "l"(h[j]), "l"(h[j + 1]), "l"(h[j + 2]), "l"(h[j + 3]) : "memory");
  } else {
    store_pairs<NS, FULL>(p, n0, N, h);
  }
}
template <int M>
__device__ __forceinline__ void zero_pairs(f32x2 (&h)[M]) {
#pragma unroll
  for (int j = 0; j < M; ++j) h[j] = 0ull;
}

// The rows of B, and behind each those of C (R = 2; FROM_C: of C alone), of a tile's tokens: every
// thread fetches some values of the next tile while one is computed, and puts
// them, as f32, into the other of two buffers.
template <class T, int NP, int R, bool FROM_C = false>
struct StageBC {
  static constexpr int kEach = (kScanTile * R * NP + kScanThreads - 1) / kScanThreads;
  T v[kEach];
  uint32_t got;
  __device__ __forceinline__ void fetch(const SscanArgs& a, uint32_t group, int64_t tb, uint32_t live) {
    got = 0;
#pragma unroll
    for (int q = 0; q < kEach; ++q) {
      const uint32_t i = q * kScanThreads + threadIdx.x, n = i % NP, which = i / NP % R, k = i / (NP * R);
      if (k < (uint32_t)kScanTile && (live >> k & 1) && n < a.states) {
        const bool c = FROM_C || which;
        const T* p = reinterpret_cast<const T*>(c ? a.c : a.b);
        v[q] = p[(uint64_t)(tb + k) * (c ? a.c_stride : a.b_stride) + (uint64_t)group * (c ? a.c_group : a.b_group) + n];
        got |= 1u << q;
      }
    }
  }
  __device__ __forceinline__ void put(float* sh) const {
#pragma unroll
    for (int q = 0; q < kEach; ++q) {
      const uint32_t i = q * kScanThreads + threadIdx.x;
      if (i < kScanTile * R * NP) sh[i] = got >> q & 1 ? to_f32(v[q]) : 0.f;
    }
  }
};

template <int LP>
__device__ __forceinline__ float from_lane(float v, int q) {
  if constexpr (LP == 1) return v;
  else return __shfl_sync(0xffffffffu, v, q, LP);
}
// o[q] of LP lanes: lane q gets the sum of their o[q].
template <int LP>
__device__ __forceinline__ float scatter_sum(float (&o)[LP], uint32_t part) {
#pragma unroll
  for (int w = LP / 2; w >= 1; w /= 2) {
    const bool up = part & w;
#pragma unroll
    for (int j = 0; j < w; ++j) {
      const float send = up ? o[j] : o[j + w], keep = up ? o[j + w] : o[j];
      o[j] = keep + __shfl_xor_sync(0xffffffffu, send, w);
    }
  }
  return o[0];
}

__device__ __forceinline__ uint32_t first_bits(int64_t n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; }

// A batch of eight tokens: its rows are copied into shared memory, a warp's
// channels by that warp, while the batch before it is computed, and its results
// leave together.  The copies are asynchronous where every piece of a row is
// aligned: loads into registers would be waited for at the first shared-memory
// load behind them, since a warp has few scoreboards for both.
constexpr int kBatch = 8;

struct RowsIn {
  const void* p;
  uint32_t row;  // bytes
};

template <class T, int LP>
struct WarpRows {
  static constexpr int kCols = 32 / LP, kBytes = kCols * (int)sizeof(T), kPiece = kBytes < 16 ? kBytes : 16, kPieces = kBytes / kPiece;
  static constexpr int kLanes = kBatch * kPieces;  // pieces of one array's batch
  template <int A, int PIECE>
  static __device__ __forceinline__ void pieces(T (*to)[kBatch][kCols], const RowsIn (&from)[A], int64_t t, uint32_t live,
                                                uint32_t c0, uint32_t cols) {
    constexpr uint32_t kN = kBytes / PIECE;
#pragma unroll
    for (int it = 0; it < (int)(A * kBatch * kN + 31) / 32; ++it) {
      const uint32_t i = it * 32 + (threadIdx.x & 31), piece = i % kN, k = i / kN % kBatch, which = i / (kN * kBatch);
      if (which >= A || !(live >> k & 1)) continue;
      RowsIn r = from[0];
#pragma unroll
      for (int q = 1; q < A; ++q)
        if (which == (uint32_t)q) r = from[q];
      const uint32_t first = piece * PIECE, have = cols * (uint32_t)sizeof(T);
      if (have <= first) continue;
      copy_async<PIECE>(reinterpret_cast<char*>(&to[which][k][0]) + first,
                        reinterpret_cast<const char*>(cell<T>(r.p, t + k, r.row, c0)) + first,
                        have - first < PIECE ? have - first : PIECE);
    }
  }
  // Rows t.. of the arrays, from channel c0 on, `cols` of them, those that
  // `live` names.  `aligned`: 2 where whole pieces are, 1 where 4 bytes are.
  template <int A>
  static __device__ __forceinline__ void in(T (*to)[kBatch][kCols], const RowsIn (&from)[A], int64_t t, uint32_t live,
                                            uint32_t c0, uint32_t cols, int aligned) {
    const uint32_t lane = threadIdx.x & 31;
    if (aligned == 2) {
      pieces<A, kPiece>(to, from, t, live, c0, cols);
    } else if (aligned == 1) {
      pieces<A, 4>(to, from, t, live, c0, cols);
    } else {
#pragma unroll
      for (int q = 0; q < A; ++q)
#pragma unroll
        for (int it = 0; it < kBatch / LP; ++it) {
          const uint32_t k = it * LP + lane / kCols, c = lane % kCols;
          if ((live >> k & 1) && c < cols) to[q][k][c] = *cell<T>(from[q].p, t + k, from[q].row, c0 + c);
        }
    }
  }
  // The batch's results: rows t.. of one array.
  static __device__ __forceinline__ void out(const T (&from)[kBatch][kCols], void* to, uint32_t row, int64_t t, uint32_t live,
                                             uint32_t c0, uint32_t cols, int aligned) {
    const uint32_t lane = threadIdx.x & 31;
    if (aligned == 2 && cols == kCols) {
      using Piece = Pack<T, kPiece / (int)sizeof(T)>;
#pragma unroll
      for (int it = 0; it < (kLanes + 31) / 32; ++it) {
        const uint32_t i = it * 32 + lane, piece = i % kPieces, k = i / kPieces;
        if (k < kBatch && (live >> k & 1))
          reinterpret_cast<Piece*>(cell<T>(to, t + k, row, c0))[piece] = reinterpret_cast<const Piece*>(&from[k][0])[piece];
      }
    } else {
#pragma unroll
      for (int it = 0; it < kBatch / LP; ++it) {
        const uint32_t k = it * LP + lane / kCols, c = lane % kCols;
        if ((live >> k & 1) && c < cols) *cell<T>(to, t + k, row, c0 + c) = from[k][c];
      }
    }
  }
};
// The pieces of aligned rows that a lane copies for each batch, batch after batch
// (DIR 1) or back from the last (DIR -1): where they are, kept and moved on, as
// their addresses from scratch took as long as a token's arithmetic.
template <class T, int LP, int A, int DIR>
struct RowsCursor {
  using Rows = WarpRows<T, LP>;
  static constexpr int kN = (A * Rows::kLanes + 31) / 32;
  const char* from[kN];
  uint32_t bytes[kN];  // of the piece that exist; 0: none
  int32_t row[kN];
  __device__ __forceinline__ RowsCursor(const RowsIn (&r)[A], int64_t t, uint32_t c0, uint32_t cols) {
#pragma unroll
    for (int it = 0; it < kN; ++it) {
      const uint32_t i = it * 32 + (threadIdx.x & 31), piece = i % Rows::kPieces, k = i / Rows::kPieces % kBatch;
      // Whole iterations are one array's: known when compiled.
      const uint32_t which = Rows::kLanes % 32 == 0 ? it * 32 / Rows::kLanes : i / Rows::kLanes;
      RowsIn s = r[0];
#pragma unroll
      for (int q = 1; q < A; ++q)
        if (which == (uint32_t)q) s = r[q];
      const uint32_t first = piece * Rows::kPiece, have = cols * (uint32_t)sizeof(T);
      bytes[it] = which >= (uint32_t)A || have <= first ? 0 : have - first < Rows::kPiece ? have - first : Rows::kPiece;
      row[it] = (int32_t)s.row;
      from[it] = static_cast<const char*>(s.p) + ((t + (int64_t)k) * (int64_t)row[it] + (int64_t)c0 * (int64_t)sizeof(T) + first);
    }
  }
  __device__ __forceinline__ void copy(T (*to)[kBatch][Rows::kCols], uint32_t live) {
    char* const base = reinterpret_cast<char*>(&to[0][0][0]) + (threadIdx.x & 31) * Rows::kPiece;
    const uint32_t k0 = (threadIdx.x & 31) / Rows::kPieces;
#pragma unroll
    for (int it = 0; it < kN; ++it) {
      const uint32_t k = (it * (32 / Rows::kPieces) + k0) % kBatch;
      if (bytes[it] && (live >> k & 1)) copy_async<Rows::kPiece>(base + it * 32 * Rows::kPiece, from[it], bytes[it]);
      from[it] += (int64_t)row[it] * (DIR * kBatch);
    }
  }
};

// 2 where the pieces of a warp's channels start on their own size in every row,
// 1 where they start on 4 bytes.
template <class T, int LP>
int rows_aligned(const SscanArgs& a, std::initializer_list<RowsIn> rows) {
  uint64_t bits = (uint64_t)(a.groups > 1 ? a.channels / a.groups : 0) * sizeof(T);
  for (const RowsIn& r : rows)
    if (r.p) bits |= reinterpret_cast<uint64_t>(r.p) | (a.seq.tokens > 1 ? r.row : 0);
  return bits % WarpRows<T, LP>::kPiece == 0 ? 2 : bits % 4 == 0 ? 1 : 0;
}

}  // namespace sparsl
