// The short causal convolution over each channel's last `width` inputs, its
// gradients, and its form for one token of each sequence.
//
//   u[t, c] = bias[c] + sum_k w[c, k] x[t - (W - 1) + k, c],   y = u or u sigmoid(u)
//
// Taps in front of a sequence come from its state: the W - 1 inputs before its
// first token, or zeros.  All of it is bound by HBM: x read and y written once.
// Measured at 16384 packed tokens x 4096 channels, width 4 with the sigmoid, bf16:
// 55 us, 4.9 TB/s; the two special functions a value alone take 30 us of the 42
// that HBM does.  The gradients of the same size take 418 us in bf16, 315 in f16 and
// 224 in f32, whose bytes take 62 and 125: at 177, 158 and 114 registers a thread an SM
// holds two, three and four blocks, and the times go with that.
#include "seq.cuh"

namespace sparsl {
namespace {

constexpr int kThreads = 128;
constexpr int kRowsAhead = 8;      // rows in flight per thread
constexpr int kRowsAheadBack = 4;  // of x and of dy each
constexpr uint32_t kSms = 148;

// Tokens of a tile: 64 (a partial row of dw and dbias each, in the backward
// pass), fewer where that leaves SMs with fewer than eight blocks.
uint32_t tile_of(uint64_t tokens, uint64_t channels, uint32_t per_block) {
  const uint64_t ctiles = (channels + per_block - 1) / per_block;
  uint32_t tile = 64;
  while (tile > 16 && (tokens + tile - 1) / tile * ctiles < 8 * kSms) tile /= 2;
  return tile;
}

template <class T, int V, int W>
struct Taps {
  float v[W][V];  // v[W - 1] is the newest
  __device__ __forceinline__ void push(const float (&x)[V]) {
#pragma unroll
    for (int k = 0; k + 1 < W; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] = v[k + 1][i];
#pragma unroll
    for (int i = 0; i < V; ++i) v[W - 1][i] = x[i];
  }
};

template <class T, int V, int W>
__device__ __forceinline__ void load_state_row(const ConvArgs& a, int64_t seq, int r, uint32_t c, float (&out)[V]) {
  const T* st = reinterpret_cast<const T*>(a.state);
  const int64_t slot = st && a.seq.resumes(seq) ? a.seq.slot(seq) : -1;
  if (slot < 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = 0.f;
    return;
  }
  load_pack<T, V>(st + ((uint64_t)slot * (W - 1) + r) * a.channels + c, out);
}

// The W - 1 inputs before position `at` of a sequence that begins at `begin`,
// into v[1..W-1] (the next push makes them v[0..W-2]).
template <class T, int V, int W>
__device__ __forceinline__ void load_taps(const ConvArgs& a, int64_t seq, int64_t begin, int64_t at, uint32_t c,
                                          Taps<T, V, W>& w) {
  const T* x = reinterpret_cast<const T*>(a.x);
#pragma unroll
  for (int k = 1; k < W; ++k) {
    const int64_t t = at - W + k;
    if (t >= begin) load_pack<T, V>(x + (uint64_t)t * a.x_stride + c, w.v[k]);
    else load_state_row<T, V, W>(a, seq, (int)(t - begin + W - 1), c, w.v[k]);
  }
}

// The last W - 1 inputs of a sequence into its row of final_state.  Rows
// ascend, so in place every old row is read before it is overwritten.
template <class T, int V, int W>
__device__ __forceinline__ void put_final(const ConvArgs& a, int64_t seq, int64_t begin, int64_t end, uint32_t c) {
  const int64_t slot = a.seq.slot(seq);
  if (slot < 0) return;
  T* out = reinterpret_cast<T*>(a.final_state) + (uint64_t)slot * (W - 1) * a.channels + c;
  const T* x = reinterpret_cast<const T*>(a.x);
#pragma unroll
  for (int r = 0; r + 1 < W; ++r) {
    float v[V];
    const int64_t t = end - (W - 1) + r;
    if (t >= begin) load_pack<T, V>(x + (uint64_t)t * a.x_stride + c, v);
    else load_state_row<T, V, W>(a, seq, (int)(t - begin + W - 1), c, v);
    store_pack<T, V>(out + (uint64_t)r * a.channels, v);
  }
}

template <class T, int V, int W>
__device__ __forceinline__ void load_weights(const ConvArgs& a, uint32_t c, float (&w)[W][V], float (&bias)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = a.bias ? load_param<T>(a.bias, a.params_f32, c + i) : 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) w[k][i] = load_param<T>(a.w, a.params_f32, (uint64_t)(c + i) * W + k);
  }
}

// One thread: V channels of one tile of tokens, every sequence's part of it in
// turn.  A tile owns the sequences that begin in it: it also computes their
// first W - 1 tokens where those reach into the next tile and writes their
// final states, so that only one thread reads and writes a channel of a state
// and the pool may be updated in place.
template <class T, int V, int W, bool SILU>
__global__ void __launch_bounds__(kThreads) conv_kernel(ConvArgs a, uint32_t ctiles, uint32_t tokens_a_tile) {
  const uint32_t ct = blockIdx.x % ctiles;
  const int64_t tile = blockIdx.x / ctiles;
  const int64_t tokens = (int64_t)a.seq.tokens, n = (int64_t)a.seq.n_seq;
  const int64_t t0 = tile * tokens_a_tile;
  const bool last = t0 + tokens_a_tile >= tokens;
  const int64_t t1 = last ? tokens : t0 + tokens_a_tile;
  __shared__ __align__(16) Pack<T, V> ring[kRowsAhead][kThreads];
  int64_t i = a.seq.first_from_warp(t0);
  const uint32_t c = (ct * kThreads + threadIdx.x) * V;
  if (c >= a.channels) return;
  float w[W][V], bias[V];
  load_weights<T, V, W>(a, c, w, bias);
  const T* x = reinterpret_cast<const T*>(a.x) + c;
  T* y = reinterpret_cast<T*>(a.y) + c;

  int64_t at = t0;  // tokens before it are done
  // i - 1 continues into the tile when it ends behind t0.
  for (i = i > 0 ? i - 1 : 0; i < n; ++i) {
    const int64_t begin = a.seq.begin(i);
    if (begin >= t1 && !last) break;
    const int64_t end = max(begin, a.seq.begin(i + 1));
    const bool mine = begin >= t0;
    int64_t from = mine ? max(begin, at) : max(max(begin + (W - 1), t0), at);
    int64_t to = min(end, t1);
    if (mine) to = min(end, max(t1, begin + (W - 1)));
    if (from < to) {
      // Eight rows are always on their way into shared memory, each thread's own
      // columns of them (in registers, eight rows' loads and as many warps do not
      // fit); two-byte columns, which cannot be copied, are loaded when wanted.
      constexpr int R = kRowsAhead;
      constexpr bool kRing = V * sizeof(T) >= 4;
      const T* px = x + (uint64_t)from * a.x_stride;
      T* py = y + (uint64_t)from * a.y_stride;
      const auto ask = [&](int slot, bool any) {
        if constexpr (kRing) {
          if (any) copy_async<V * (int)sizeof(T)>(&ring[slot][threadIdx.x], px, V * (uint32_t)sizeof(T));
          px += a.x_stride;
          copies_issued();
        }
      };
#pragma unroll
      for (int k = 0; k < R; ++k) ask(k, from + k < to);
      Taps<T, V, W> win;
      load_taps<T, V, W>(a, i, begin, from, c, win);
      const auto token = [&](const Pack<T, V>& r) {
        float v[V], u[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = to_f32(r.v[j]);
        win.push(v);
        if constexpr (V % 2 == 0) {
#pragma unroll
          for (int j = 0; j < V; j += 2) {
            f32x2 s = pair(bias[j], bias[j + 1]);
#pragma unroll
            for (int m = 0; m < W; ++m) s = fma2(pair(w[m][j], w[m][j + 1]), pair(win.v[m][j], win.v[m][j + 1]), s);
            unpair(s, u[j], u[j + 1]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            u[j] = bias[j];
#pragma unroll
            for (int m = 0; m < W; ++m) u[j] = __fmaf_rn(w[m][j], win.v[m][j], u[j]);
          }
        }
        if (SILU)
#pragma unroll
          for (int j = 0; j < V; ++j) u[j] = u[j] * sigmoid(u[j]);
        store_pack<T, V>(py, u);
        py += a.y_stride;
      };
      const auto take = [&](int k) {
        if constexpr (kRing) {
          copies_but<R - 1>();
          return ring[k][threadIdx.x];
        } else {
          const Pack<T, V> r = *reinterpret_cast<const Pack<T, V>*>(px);
          px += a.x_stride;
          return r;
        }
      };
      int64_t t = from;
      for (; t + 2 * R <= to; t += R) {
#pragma unroll
        for (int k = 0; k < R; ++k) {
          token(take(k));
          ask(k, true);
        }
      }
      for (; t < to; t += R) {
#pragma unroll
        for (int k = 0; k < R; ++k) {
          if (t + k >= to) break;
          token(take(k));
          ask(k, t + k + R < to);
        }
      }
      at = to;
    }
    if (mine && a.final_state) put_final<T, V, W>(a, i, begin, end, c);
  }
}

// Gradients.  A thread walks a sequence's part [from, to) of its tile and
// W - 1 tokens further: at token t it forms du[t], adds it to the weights'
// sums when t is its own, and then emits dx[t - (W - 1)], whose last term
// du[t] is.  Positions in front of the sequence are its state's rows, so dstate
// and the gradient of the final state come out of the same walk.
template <class T, int V, int W, bool SILU>
__global__ void __launch_bounds__(kThreads) conv_backward_kernel(ConvArgs a, uint32_t ctiles, uint32_t tokens_a_tile) {
  const uint32_t ct = blockIdx.x % ctiles;
  const int64_t tile = blockIdx.x / ctiles;
  const int64_t tokens = (int64_t)a.seq.tokens, n = (int64_t)a.seq.n_seq;
  const int64_t t0 = tile * tokens_a_tile;
  const bool last = t0 + tokens_a_tile >= tokens;
  const int64_t t1 = last ? tokens : t0 + tokens_a_tile;
  int64_t i = a.seq.first_from_warp(t0);
  const uint32_t c = (ct * kThreads + threadIdx.x) * V;
  if (c >= a.channels) return;
  float w[W][V], bias[V], dw[W][V], db[V];
  load_weights<T, V, W>(a, c, w, bias);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    db[j] = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) dw[k][j] = 0.f;
  }
  const T* x = reinterpret_cast<const T*>(a.x) + c;
  const T* dy = reinterpret_cast<const T*>(a.dy) + c;
  T* dx = reinterpret_cast<T*>(a.dx) + c;

  int64_t at = t0;
  for (i = i > 0 ? i - 1 : 0; i < n; ++i) {
    const int64_t begin = a.seq.begin(i);
    if (begin >= t1 && !last) break;
    const int64_t end = max(begin, a.seq.begin(i + 1));
    const bool mine = begin >= t0;
    const int64_t from = max(mine ? begin : t0, at), to = max(from, min(end, t1));
    if (!mine && from >= to) continue;
    const bool states = mine && a.dstate;  // emit the state's rows too
    if (from >= to && !states) continue;
    Taps<T, V, W> win, du;
    load_taps<T, V, W>(a, i, begin, from, c, win);
#pragma unroll
    for (int k = 0; k < W; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) du.v[k][j] = 0.f;
    const int64_t slot = a.dfinal || states ? a.seq.slot(i) : -1;
    const T* df = a.dfinal && slot >= 0 ? reinterpret_cast<const T*>(a.dfinal) + (uint64_t)slot * (W - 1) * a.channels + c
                                        : nullptr;
    T* ds = states && slot >= 0 ? reinterpret_cast<T*>(a.dstate) + (uint64_t)slot * (W - 1) * a.channels + c : nullptr;
    constexpr int K = kRowsAheadBack;
    Pack<T, V> xn[K], dn[K], xr[K], dr[K];
    const int64_t stop = min(to + (W - 1), end);  // tokens behind it have no gradient
    const auto ask = [&](int64_t t) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (t + k < stop) {
          xn[k] = *reinterpret_cast<const Pack<T, V>*>(x + (uint64_t)(t + k) * a.x_stride);
          dn[k] = *reinterpret_cast<const Pack<T, V>*>(dy + (uint64_t)(t + k) * a.dy_stride);
        }
    };
    ask(from);
    for (int64_t tk = from; tk < to + (W - 1); tk += K) {
#pragma unroll
      for (int k = 0; k < K; ++k) xr[k] = xn[k], dr[k] = dn[k];
      ask(tk + K);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int64_t t = tk + k;
        if (t >= to + (W - 1)) break;
        float d[V];
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = 0.f;
        if (t < end) {
          float v[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            v[j] = to_f32(xr[k].v[j]);
            d[j] = to_f32(dr[k].v[j]);
          }
          win.push(v);
          if (SILU) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              float u = bias[j];
#pragma unroll
              for (int m = 0; m < W; ++m) u = __fmaf_rn(w[m][j], win.v[m][j], u);
              const float g = sigmoid(u);
              d[j] *= g * __fmaf_rn(u, 1.0f - g, 1.0f);
            }
          }
          if (t < to) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              db[j] += d[j];
#pragma unroll
              for (int m = 0; m < W; ++m) dw[m][j] = __fmaf_rn(d[j], win.v[m][j], dw[m][j]);
            }
          }
        }
        du.push(d);
        const int64_t s = t - (W - 1);
        float g[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          g[j] = 0.f;
#pragma unroll
          for (int m = 0; m < W; ++m) g[j] = __fmaf_rn(w[W - 1 - m][j], du.v[m][j], g[j]);
        }
        const int64_t fr = s - (end - (W - 1));  // its row in the final state; behind it where seq_ptr does not ascend
        if (df && fr >= 0 && fr < W - 1) {
          float f[V];
          load_pack<T, V>(df + (uint64_t)fr * a.channels, f);
#pragma unroll
          for (int j = 0; j < V; ++j) g[j] += f[j];
        }
        if (s >= from) store_pack<T, V>(dx + (uint64_t)s * a.dx_stride, g);
        else if (ds && s < begin) store_pack<T, V>(ds + (uint64_t)(s - begin + W - 1) * a.channels, g);
      }
    }
    at = max(at, to);
  }
  float* part = a.part + (uint64_t)tile * (W + 1) * a.channels;
#pragma unroll
  for (int j = 0; j < V; ++j) {
#pragma unroll
    for (int k = 0; k < W; ++k) part[(uint64_t)(c + j) * W + k] = dw[k][j];
    part[(uint64_t)a.channels * W + c + j] = db[j];
  }
}

template <class T, int V, int W, bool SILU>
__global__ void __launch_bounds__(kThreads) conv_step_kernel(ConvArgs a, uint32_t ctiles) {
  const uint32_t ct = blockIdx.x % ctiles;
  const int64_t i = blockIdx.x / ctiles;
  const uint32_t c = (ct * kThreads + threadIdx.x) * V;
  if (c >= a.channels) return;
  const int64_t slot = a.seq.slot(i);
  if (slot < 0) return;
  float w[W][V], bias[V], v[W][V], u[V];
  T* st = reinterpret_cast<T*>(a.final_state) + (uint64_t)slot * (W - 1) * a.channels + c;
  load_pack<T, V>(reinterpret_cast<const T*>(a.x) + (uint64_t)i * a.x_stride + c, v[W - 1]);
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) load_pack<T, V>(st + (uint64_t)k * a.channels, v[k]);
  load_weights<T, V, W>(a, c, w, bias);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    u[j] = bias[j];
#pragma unroll
    for (int m = 0; m < W; ++m) u[j] = __fmaf_rn(w[m][j], v[m][j], u[j]);
    if (SILU) u[j] = u[j] * sigmoid(u[j]);
  }
  store_pack<T, V>(reinterpret_cast<T*>(a.y) + (uint64_t)i * a.y_stride + c, u);
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) store_pack<T, V>(st + (uint64_t)k * a.channels, v[k + 1]);
}

enum Form { FORWARD, BACKWARD, STEP };

// Channels of a block in the backward pass whatever the vectors: the tiles, and
// so the workspace, must not depend on alignment.
constexpr uint32_t kBackChannels = kThreads;

template <Form F, class T, int V, int W, bool SILU>
cudaError_t go(const ConvArgs& a, cudaStream_t s) {
  const uint32_t ctiles = (a.channels + kThreads * V - 1) / (kThreads * V);
  const uint32_t tile = F == FORWARD    ? tile_of(a.seq.tokens, a.channels, kThreads * V)
                        : F == BACKWARD ? tile_of(a.seq.tokens, a.channels, kBackChannels)
                                        : 1;
  uint64_t tiles = (a.seq.tokens + tile - 1) / tile;
  if (tiles == 0) tiles = 1;  // sequences without tokens still have final states
  const uint64_t grid = tiles * ctiles;
  if (grid > 0x7fffffffull) return cudaErrorInvalidValue;
  if constexpr (F == FORWARD) conv_kernel<T, V, W, SILU><<<(unsigned)grid, kThreads, 0, s>>>(a, ctiles, tile);
  else if constexpr (F == BACKWARD) conv_backward_kernel<T, V, W, SILU><<<(unsigned)grid, kThreads, 0, s>>>(a, ctiles, tile);
  else conv_step_kernel<T, V, W, SILU><<<(unsigned)grid, kThreads, 0, s>>>(a, ctiles);
  return cudaGetLastError();
}

template <Form F, class T, int V, int W>
cudaError_t by_silu(const ConvArgs& a, cudaStream_t s) {
  return a.silu ? go<F, T, V, W, true>(a, s) : go<F, T, V, W, false>(a, s);
}
template <Form F, class T, int V>
cudaError_t by_width(const ConvArgs& a, cudaStream_t s) {
  switch (a.width) {
    case 2: return by_silu<F, T, V, 2>(a, s);
    case 3: return by_silu<F, T, V, 3>(a, s);
    case 4: return by_silu<F, T, V, 4>(a, s);
    default: return cudaErrorInvalidValue;
  }
}
// Vectors of channels where every row starts on a vector's boundary, single
// channels otherwise.
template <Form F, class T>
cudaError_t by_vector(const ConvArgs& a, cudaStream_t s) {
  constexpr int V = 8 / sizeof(T);  // 16-byte vectors' weights and taps leave too few warps: 79 us against 55 at 16384 x 4096 bf16
  uint64_t m = a.channels | a.x_stride | a.y_stride | a.dy_stride | a.dx_stride;
  uint64_t p = 0;
  for (const void* q : {a.x, (const void*)a.y, a.state, (const void*)a.final_state, a.dy, (const void*)a.dx,
                        (const void*)a.dstate, a.dfinal})
    p |= reinterpret_cast<uint64_t>(q);
  if (m % V == 0 && p % (V * sizeof(T)) == 0) return by_width<F, T, V>(a, s);
  return by_width<F, T, 1>(a, s);
}
template <Form F>
cudaError_t by_type(const ConvArgs& a, cudaStream_t s) {
  switch (a.type) {
    case SEQ_F32: return by_vector<F, float>(a, s);
    case SEQ_F16: return by_vector<F, __half>(a, s);
    default: return by_vector<F, __nv_bfloat16>(a, s);
  }
}

// Sums over the rows of part[rows, cols], each column's in one fixed order:
// columns below `split` into out, the rest into more (null: not wanted).
__global__ void __launch_bounds__(1024) reduce_rows_kernel(const float* part, uint64_t rows, uint64_t cols,
                                                          uint64_t split, float* out, float* more) {
  __shared__ float sh[32][32];
  const uint32_t lane = threadIdx.x % 32, g = threadIdx.x / 32;
  const uint64_t c = (uint64_t)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < cols)
    for (uint64_t r = g; r < rows; r += 32) s += part[r * cols + c];
  sh[g][lane] = s;
  __syncthreads();
  if (g == 0 && c < cols) {
#pragma unroll
    for (int k = 1; k < 32; ++k) s += sh[k][lane];
    if (c < split) {
      if (out) out[c] = s;
    }
    else if (more) more[c - split] = s;
  }
}

}  // namespace

cudaError_t launch_reduce_rows(const float* part, uint64_t rows, uint64_t cols, uint64_t split, float* out, float* more,
                               cudaStream_t s) {
  if (cols == 0) return cudaSuccess;
  reduce_rows_kernel<<<(unsigned)((cols + 31) / 32), 1024, 0, s>>>(part, rows, cols, split, out, more);
  return cudaGetLastError();
}

namespace {
uint64_t back_tiles(uint64_t tokens, uint64_t channels) {
  const uint32_t tile = tile_of(tokens, channels, kBackChannels);
  const uint64_t tiles = (tokens + tile - 1) / tile;
  return tiles ? tiles : 1;
}
}  // namespace

size_t conv_backward_bytes(uint64_t tokens, uint64_t channels, uint32_t width) {
  return back_tiles(tokens, channels) * (width + 1) * channels * 4;
}

cudaError_t launch_conv(const ConvArgs& a, cudaStream_t s) { return by_type<FORWARD>(a, s); }
cudaError_t launch_conv_step(const ConvArgs& a, cudaStream_t s) { return by_type<STEP>(a, s); }
cudaError_t launch_conv_backward(const ConvArgs& a, cudaStream_t s) {
  cudaError_t e = by_type<BACKWARD>(a, s);
  if (e != cudaSuccess) return e;
  // A partial row holds dw's channels * width sums, then dbias's.
  const uint64_t split = (uint64_t)a.channels * a.width;
  return launch_reduce_rows(a.part, back_tiles(a.seq.tokens, a.channels), split + a.channels, split, a.dw, a.dbias, s);
}

}  // namespace sparsl
