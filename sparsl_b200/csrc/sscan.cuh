// What the forward and the backward kernels of the selective scan share: the
// split of the token axis into chunks, the workspace, and a channel's
// arithmetic.
#pragma once

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
  uint64_t len, chunks;
  bool carry;
};

// `wanted` blocks fill the GPU: where the channel tiles and the sequences are
// fewer, the token axis is split, which costs the exponentials of the spanning
// sequences once more (for the states at the chunks' starts).
inline ScanPlan scan_plan(uint64_t tokens, uint32_t channels, uint32_t groups, uint64_t n_seq, bool ragged,
                          uint32_t tile_channels, uint32_t wanted) {
  ScanPlan p;
  const uint32_t cpg = channels / groups;
  p.per_group = (cpg + tile_channels - 1) / tile_channels;
  p.ctiles = p.per_group * groups;
  const uint64_t run = n_seq ? tokens / n_seq : 0;
  const uint64_t want = (wanted + p.ctiles - 1) / p.ctiles;
  uint64_t len = (tokens + want - 1) / want;
  len = len < 64 ? 64 : (len + 31) / 32 * 32;
  bool whole = false;  // no sequence spans two chunks
  if (!ragged && run && run % 32 == 0) {
    if (n_seq >= want || run <= 64) {
      len = run;
      whole = true;
    } else {
      // A chunk length that divides the runs, if one of at least half the size does.
      for (uint64_t l = len; 2 * l >= len && l >= 32; l -= 32)
        if (run % l == 0) {
          len = l;
          break;
        }
    }
  }
  p.len = len;
  p.chunks = tokens ? (tokens + len - 1) / len : 1;
  p.carry = !whole && p.chunks > 1;
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
__device__ __forceinline__ float softplus(float v) {
  const float u = ex2(-kLog2e * fabsf(v));
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

}  // namespace sparsl
