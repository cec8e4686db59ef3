// Layer norm over the channels of each row, and its gradients.
//
//   hat = (x - mean) rstd,   y = hat w + bias,   rstd = 1 / sqrt(var + eps)
//   dx  = rstd (w dy - mean(w dy) - hat mean(w dy hat))
//   dw  = sum over rows of dy hat,   dbias = sum over rows of dy
//
// Bound by HBM: forward x read and y written once, backward x and dy read and
// dx written once.  A group of threads keeps a row in registers (64 values a
// thread at most), so the variance is the mean of squared deviations, not a
// difference of sums; longer rows are read again for each of the steps.  In
// the backward pass a block walks many rows, its threads keeping the sums of dw
// and dbias for their own channels in registers, and the blocks' partial rows
// are added in a fixed order.  Measured at 16384 x 2048 bf16: forward 36 us (3.7
// TB/s), backward 48 us (4.2 TB/s) and 8 us for the partial rows; at 4099 x 5003
// f32, rows that no 16-byte access fits, 45 and 62 us (3.6 and 3.9 TB/s).  The
// gradients of rows over 8192 values read x and dy twice in one kernel and once in
// another, value by value: 479 us at 8192 x 12288 bf16, whose bytes take 94.
#include "seq.cuh"

namespace sparsl {
namespace {

constexpr uint32_t kSms = 148;

// Sums of v over the B threads that share a row; `turn` alternates from sum to
// sum, so that one barrier does.
template <int B, int M>
__device__ __forceinline__ void row_sum(float (&v)[M], float (*sh)[32 * M], int& turn) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int m = 0; m < M; ++m) v[m] += __shfl_xor_sync(0xffffffffu, v[m], o);
  if constexpr (B > 32) {
    constexpr int kW = B / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float* s = sh[turn];
    turn ^= 1;
    if (lane == 0)
#pragma unroll
      for (int m = 0; m < M; ++m) s[warp * M + m] = v[m];
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) {
      v[m] = lane < kW ? s[lane * M + m] : 0.f;
#pragma unroll
      for (int o = kW / 2; o; o >>= 1) v[m] += __shfl_xor_sync(0xffffffffu, v[m], o);
      v[m] = __shfl_sync(0xffffffffu, v[m], 0);
    }
  }
}

// B threads per row (several rows side by side in a block of 128 where B is
// smaller), V values per access, I accesses per thread.  A block walks the rows
// with weight and bias in registers, the next row asked for while one is done:
// with a block per row the parameters' traffic from L2 was twice the rows'
// (85 us against 50 at 16384 x 2048 bf16, which norm_rows_kernel now takes in 36).
template <class T, int V, int B, int I>
__global__ void __launch_bounds__(B < 128 ? 128 : B) norm_kernel(NormArgs a) {
  __shared__ float sh[2][32];
  constexpr int kSide = B < 128 ? 128 / B : 1;
  const uint32_t tid = threadIdx.x % B;
  const uint64_t step = (uint64_t)gridDim.x * kSide;
  uint64_t row = (uint64_t)blockIdx.x * kSide + threadIdx.x / B;
  float w[I][V], bias[I][V];
  Pack<T, V> next[I];
  const auto ask = [&](uint64_t r) {
    const T* x = reinterpret_cast<const T*>(a.x) + r * a.x_stride;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const uint32_t c = (i * B + tid) * V;
      if (c < a.channels) next[i] = *reinterpret_cast<const Pack<T, V>*>(x + c);
    }
  };
  if (row < a.rows) ask(row);
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t c = (i * B + tid) * V + j;
      w[i][j] = a.w && c < a.channels ? load_param<T>(a.w, a.params_f32, c) : 1.f;
      bias[i][j] = a.bias && c < a.channels ? load_param<T>(a.bias, a.params_f32, c) : 0.f;
    }
  const float channels = (float)a.channels;
  int turn = 0;
  for (; row < a.rows; row += step) {
    float v[I][V], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] = (i * B + tid) * V < a.channels ? to_f32(next[i].v[j]) : 0.f;
        s[0] += v[i][j];
      }
    if (row + step < a.rows) ask(row + step);
    row_sum<B>(s, sh, turn);
    const float mean = s[0] / channels;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] -= mean;
        if ((i * B + tid) * V < a.channels) s[0] = __fmaf_rn(v[i][j], v[i][j], s[0]);
      }
    row_sum<B>(s, sh, turn);
    const float rstd = 1.0f / sqrtf(s[0] / channels + a.eps);
    if (tid == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = reinterpret_cast<T*>(a.y) + row * a.y_stride;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const uint32_t c = (i * B + tid) * V;
      if (c >= a.channels) continue;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = __fmaf_rn(v[i][j] * rstd, w[i][j], bias[i][j]);
      store_pack<T, V>(y + c, o);
    }
  }
}

// The rows a thread works on next, its own values of them.  Whole accesses of 16
// bytes are copied into shared memory while a row is computed, STAGES rows ahead
// (loads into registers are waited for at the first exchange between lanes); a
// thread reads what it copied itself, so no barrier is needed.  Single values,
// whose copies would be as many instructions again, wait in registers.
template <class T, int V, int B, int I, int ARRAYS, int STAGES>
struct RowsAhead {
  static constexpr bool kAsync = V > 1;
  static constexpr int kStages = kAsync ? STAGES : 1;
  static constexpr int kBytes = kAsync ? STAGES * ARRAYS * I * (int)sizeof(Pack<T, V>) : 0;  // per thread
  Pack<T, V>* sh;  // [stage][array][access][thread]
  Pack<T, V> held[kAsync ? 1 : ARRAYS][kAsync ? 1 : I];
  uint32_t threads, tid;
  uint64_t channels;
  __device__ __forceinline__ RowsAhead(void* p, uint32_t tid_, uint64_t channels_)
      : sh(static_cast<Pack<T, V>*>(p) + threadIdx.x), threads(blockDim.x), tid(tid_), channels(channels_) {}
  __device__ __forceinline__ Pack<T, V>* at(int stage, int array, int i) const {
    return sh + ((stage * ARRAYS + array) * I + i) * threads;
  }
  __device__ __forceinline__ void ask(int stage, int array, const T* row) {
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const uint32_t c = (i * B + tid) * V;
      if (c >= channels) continue;
      if constexpr (kAsync) copy_async<V * (int)sizeof(T)>(at(stage, array, i), row + c, V * (uint32_t)sizeof(T));
      else held[array][i] = *reinterpret_cast<const Pack<T, V>*>(row + c);
    }
  }
  __device__ __forceinline__ Pack<T, V> get(int stage, int array, int i) const {
    if constexpr (kAsync) return *at(stage, array, i);
    else return held[array][i];
  }
};

// Many rows: up to 64 values per thread, so that a row's two sums cost little
// beside it, a warp per row where that holds one (no barrier then), and the
// parameters, which 64 values' registers have no room for, in shared memory.
template <class T, int V, int B, int I, int STAGES>
__global__ void __launch_bounds__(256) norm_rows_kernel(NormArgs a) {
  extern __shared__ __align__(16) float params[];  // weight, then bias, each padded to whole accesses; the rows ahead
  __shared__ float sh[2][32];
  constexpr int kSide = 256 / B;
  const uint32_t tid = threadIdx.x % B, padded = (uint32_t)((a.channels + 3) / 4 * 4);
  const uint64_t step = (uint64_t)gridDim.x * kSide;
  uint64_t row = (uint64_t)blockIdx.x * kSide + threadIdx.x / B;
  const T* x = reinterpret_cast<const T*>(a.x);
  using Ahead = RowsAhead<T, V, B, I, 1, STAGES>;
  Ahead ahead(params + 2 * padded, tid, a.channels);
#pragma unroll
  for (int k = 0; k < Ahead::kStages; ++k) {
    if (row + k * step < a.rows) ahead.ask(k, 0, x + (row + k * step) * a.x_stride);
    copies_issued();
  }
  for (uint32_t c = threadIdx.x; c < padded; c += 256) {
    params[c] = a.w && c < a.channels ? load_param<T>(a.w, a.params_f32, c) : 1.f;
    params[padded + c] = a.bias && c < a.channels ? load_param<T>(a.bias, a.params_f32, c) : 0.f;
  }
  __syncthreads();
  const float channels = (float)a.channels;
  int turn = 0, stage = 0;
  for (; row < a.rows; row += step, stage = stage + 1 == Ahead::kStages ? 0 : stage + 1) {
    copies_but<Ahead::kStages - 1>();
    float v[I][V], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const bool in = (i * B + tid) * V < a.channels;
      Pack<T, V> r;
      if (in) r = ahead.get(stage, 0, i);
      float part = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] = in ? to_f32(r.v[j]) : 0.f;
        part += v[i][j];
      }
      s[0] += part;
    }
    const uint64_t far = row + Ahead::kStages * step;
    if (far < a.rows) ahead.ask(stage, 0, x + far * a.x_stride);
    copies_issued();
    row_sum<B>(s, sh, turn);
    const float mean = s[0] / channels;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const bool in = (i * B + tid) * V < a.channels;
      float part = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] -= mean;
        part = __fmaf_rn(v[i][j], v[i][j], part);
      }
      if (in) s[0] += part;
    }
    row_sum<B>(s, sh, turn);
    const float rstd = 1.0f / sqrtf(s[0] / channels + a.eps);
    if (tid == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = reinterpret_cast<T*>(a.y) + row * a.y_stride;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const uint32_t c = (i * B + tid) * V;
      if (c >= a.channels) continue;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = __fmaf_rn(v[i][j] * rstd, params[c + j], params[padded + c + j]);
      store_pack<T, V>(y + c, o);
    }
  }
}

// Rows longer than the registers hold: 1024 threads, x read three times (the
// second and third from the caches).
template <class T>
__global__ void __launch_bounds__(1024) norm_long_kernel(NormArgs a) {
  __shared__ float sh[2][32];
  int turn = 0;
  const uint64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
  float s[1] = {0.f};
  for (uint64_t c = threadIdx.x; c < a.channels; c += 1024) s[0] += to_f32(x[c]);
  row_sum<1024>(s, sh, turn);
  const float mean = s[0] / (float)a.channels;
  s[0] = 0.f;
  for (uint64_t c = threadIdx.x; c < a.channels; c += 1024) {
    const float d = to_f32(x[c]) - mean;
    s[0] = __fmaf_rn(d, d, s[0]);
  }
  row_sum<1024>(s, sh, turn);
  const float rstd = 1.0f / sqrtf(s[0] / (float)a.channels + a.eps);
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
  T* y = reinterpret_cast<T*>(a.y) + row * a.y_stride;
  for (uint64_t c = threadIdx.x; c < a.channels; c += 1024) {
    float o = (to_f32(x[c]) - mean) * rstd;
    if (a.w) o = o * load_param<T>(a.w, a.params_f32, c);
    if (a.bias) o += load_param<T>(a.bias, a.params_f32, c);
    y[c] = from_f32<T>(o);
  }
}

template <class T, int V, int B, int I, int STAGES>
__global__ void __launch_bounds__(B) norm_backward_kernel(NormArgs a) {
  extern __shared__ __align__(16) float rows_ahead[];
  __shared__ float sh[2][64];
  const uint32_t tid = threadIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* dy = reinterpret_cast<const T*>(a.dy);
  using Ahead = RowsAhead<T, V, B, I, 2, STAGES>;
  Ahead ahead(rows_ahead, tid, a.channels);
  const uint64_t step = gridDim.x;
  const auto ask = [&](int stage, uint64_t row) {
    if (row < a.rows) {
      ahead.ask(stage, 0, x + row * a.x_stride);
      ahead.ask(stage, 1, dy + row * a.dy_stride);
    }
    copies_issued();
  };
#pragma unroll
  for (int k = 0; k < Ahead::kStages; ++k) ask(k, blockIdx.x + k * step);
  float mean_n = 0.f, rstd_n = 0.f;
  if (blockIdx.x < a.rows) mean_n = a.mean[blockIdx.x], rstd_n = a.rstd[blockIdx.x];
  float w[I][V], dw[I][V], db[I][V];
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t c = (i * B + tid) * V + j;
      w[i][j] = c < a.channels ? (a.w ? load_param<T>(a.w, a.params_f32, c) : 1.f) : 0.f;
      dw[i][j] = db[i][j] = 0.f;
    }
  const float scale = 1.0f / (float)a.channels;
  int turn = 0, stage = 0;
  for (uint64_t row = blockIdx.x; row < a.rows; row += step, stage = stage + 1 == Ahead::kStages ? 0 : stage + 1) {
    const float mean = mean_n, rstd = rstd_n;
    if (row + step < a.rows) mean_n = a.mean[row + step], rstd_n = a.rstd[row + step];
    copies_but<Ahead::kStages - 1>();
    float h[I][V], g[I][V], s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const bool in = (i * B + tid) * V < a.channels;
      Pack<T, V> xr, dr;
      if (in) {
        xr = ahead.get(stage, 0, i);
        dr = ahead.get(stage, 1, i);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        h[i][j] = in ? (to_f32(xr.v[j]) - mean) * rstd : 0.f;
        g[i][j] = in ? to_f32(dr.v[j]) : 0.f;
        db[i][j] += g[i][j];
        dw[i][j] = __fmaf_rn(g[i][j], h[i][j], dw[i][j]);
        g[i][j] *= w[i][j];
        s[0] += g[i][j];
        s[1] = __fmaf_rn(g[i][j], h[i][j], s[1]);
      }
    }
    ask(stage, row + Ahead::kStages * step);
    row_sum<B>(s, sh, turn);
    const float m0 = s[0] * scale, m1 = s[1] * scale;
    T* dx = reinterpret_cast<T*>(a.dx) + row * a.dx_stride;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const uint32_t c = (i * B + tid) * V;
      if (c >= a.channels) continue;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = rstd * (g[i][j] - m0 - h[i][j] * m1);
      store_pack<T, V>(dx + c, o);
    }
  }
  float* part = a.part + (uint64_t)blockIdx.x * 2 * a.channels;
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t c = (i * B + tid) * V + j;
      if (c < a.channels) {
        part[c] = dw[i][j];
        part[a.channels + c] = db[i][j];
      }
    }
}

template <class T>
__global__ void __launch_bounds__(1024) norm_long_dx_kernel(NormArgs a) {
  __shared__ float sh[2][64];
  int turn = 0;
  const uint64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
  const T* dy = reinterpret_cast<const T*>(a.dy) + row * a.dy_stride;
  const float mean = a.mean[row], rstd = a.rstd[row];
  float s[2] = {0.f, 0.f};
  for (uint64_t c = threadIdx.x; c < a.channels; c += 1024) {
    const float g = to_f32(dy[c]) * (a.w ? load_param<T>(a.w, a.params_f32, c) : 1.f);
    s[0] += g;
    s[1] = __fmaf_rn(g, (to_f32(x[c]) - mean) * rstd, s[1]);
  }
  row_sum<1024>(s, sh, turn);
  const float scale = 1.0f / (float)a.channels;
  T* dx = reinterpret_cast<T*>(a.dx) + row * a.dx_stride;
  for (uint64_t c = threadIdx.x; c < a.channels; c += 1024) {
    const float g = to_f32(dy[c]) * (a.w ? load_param<T>(a.w, a.params_f32, c) : 1.f);
    dx[c] = from_f32<T>(rstd * (g - s[0] * scale - (to_f32(x[c]) - mean) * rstd * (s[1] * scale)));
  }
}

// Partial column sums for long rows: a block takes 256 columns of a share of the rows.
template <class T>
__global__ void __launch_bounds__(256) norm_long_params_kernel(NormArgs a, uint32_t shares) {
  const uint64_t c = (uint64_t)(blockIdx.x / shares) * 256 + threadIdx.x;
  if (c >= a.channels) return;
  const uint32_t share = blockIdx.x % shares;
  float dw = 0.f, db = 0.f;
  for (uint64_t row = share; row < a.rows; row += shares) {
    const float g = to_f32(reinterpret_cast<const T*>(a.dy)[row * a.dy_stride + c]);
    const float h = (to_f32(reinterpret_cast<const T*>(a.x)[row * a.x_stride + c]) - a.mean[row]) * a.rstd[row];
    db += g;
    dw = __fmaf_rn(g, h, dw);
  }
  float* part = a.part + (uint64_t)share * 2 * a.channels;
  part[c] = dw;
  part[a.channels + c] = db;
}

// Partial rows of dw and dbias: a block each.
uint64_t back_parts(uint64_t rows) {
  const uint64_t most = 4 * kSms;
  return rows < most ? (rows ? rows : 1) : most;
}

template <class T, int V, int B, int I>
cudaError_t go(const NormArgs& a, cudaStream_t s) {
  constexpr uint64_t kSide = B < 128 ? 128 / B : 1;
  const uint64_t blocks = (a.rows + kSide - 1) / kSide, most = (uint64_t)kSms * (B < 128 ? 12 : B >= 1024 ? 2 : 1536 / B);
  norm_kernel<T, V, B, I><<<(unsigned)(blocks < most ? blocks : most), B < 128 ? 128 : B, 0, s>>>(a);
  return cudaGetLastError();
}

// `most` is what the kernel may ever take: the setting is the kernel's, not the
// launch's, and another thread's call must not find it lowered.
template <class K>
cudaError_t allow(K kernel, int most) {
  return most > 40 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most) : cudaSuccess;
}

template <class T, int V, int B, int VALUES>
cudaError_t go_rows(const NormArgs& a, cudaStream_t s) {
  constexpr int kSide = 256 / B, kStages = 2;
  constexpr int kAhead = 256 * RowsAhead<T, V, B, VALUES / V, 1, kStages>::kBytes;
  const int bytes = (int)((a.channels + 3) / 4 * 4 * 8) + kAhead;
  const auto kernel = norm_rows_kernel<T, V, B, VALUES / V, kStages>;
  const cudaError_t e = allow(kernel, B * VALUES * 8 + kAhead);
  if (e != cudaSuccess) return e;
  const uint64_t blocks = (a.rows + kSide - 1) / kSide, fit = 220 * 1024 / bytes, regs = VALUES >= 64 ? 2 : VALUES >= 24 ? 3 : 5;
  const uint64_t most = (uint64_t)kSms * (fit < regs ? (fit ? fit : 1) : regs);
  kernel<<<(unsigned)(blocks < most ? blocks : most), 256, bytes, s>>>(a);
  return cudaGetLastError();
}

// Many rows of up to 8192 values in 16-byte accesses: norm_rows_kernel, 16 to 64
// values per thread (36 us against 50 at 16384 x 2048 bf16; single values are
// better kept in registers, 45 us against 62 at 4099 x 5003 f32).  Otherwise 8 values per thread, 16 where 1024 threads of 8 do not hold a row;
// rows over 16384 values are read again for each of the steps.
template <class T, int V>
cudaError_t forward(const NormArgs& a, cudaStream_t s) {
  constexpr int I = 8 / V;
  const uint64_t c = a.channels;
  if (V > 1 && a.rows >= 16 * kSms) {
    if (c <= 512) return go_rows<T, V, 32, 16>(a, s);
    if (c <= 1024) return go_rows<T, V, 32, 32>(a, s);
    if (c <= 2048) return go_rows<T, V, 32, 64>(a, s);
    if (c <= 4096) return go_rows<T, V, 256, 16>(a, s);
    if (c <= 6144) return go_rows<T, V, 256, 24>(a, s);
    if (c <= 8192) return go_rows<T, V, 256, 32>(a, s);
  }
  if (c <= 256) return go<T, V, 32, I>(a, s);
  if (c <= 1024) return go<T, V, 128, I>(a, s);
  if (c <= 2048) return go<T, V, 256, I>(a, s);
  if (c <= 4096) return go<T, V, 512, I>(a, s);
  if (V == 1 && c <= 6144) return go<T, V, 512, 12 / V + (12 % V ? 1 : 0)>(a, s);
  if (c <= 8192) return go<T, V, 1024, I>(a, s);
  if (c <= 16384) return go<T, V, 1024, 2 * I>(a, s);
  if (a.rows > 0x7fffffffull) return cudaErrorInvalidValue;
  norm_long_kernel<T><<<(unsigned)a.rows, 1024, 0, s>>>(a);
  return cudaGetLastError();
}

template <class T, int V, int B, int I>
cudaError_t go_back(const NormArgs& a, cudaStream_t s) {
  // Two rows ahead; one where that leaves an SM a single block.
  constexpr int kThree = RowsAhead<T, V, B, I, 2, 3>::kBytes * B, kStages = kThree <= 72 * 1024 ? 3 : 2;
  const int bytes = RowsAhead<T, V, B, I, 2, kStages>::kBytes * B;
  const auto kernel = norm_backward_kernel<T, V, B, I, kStages>;
  const cudaError_t e = allow(kernel, bytes);
  if (e != cudaSuccess) return e;
  kernel<<<(unsigned)back_parts(a.rows), B, bytes, s>>>(a);
  return cudaGetLastError();
}

// 16 values per thread (8 in rows of up to 512, 12 in those of up to 6144): a
// row's sums cost half of what they do with 8.  Longer rows' dx and sums take a
// kernel each.
template <class T, int V>
cudaError_t backward(const NormArgs& a, cudaStream_t s) {
  constexpr int I = 8 / V;
  const uint64_t c = a.channels;
  if (c <= 512) return go_back<T, V, 64, I>(a, s);
  if (c <= 1024) return go_back<T, V, 64, 2 * I>(a, s);
  if (c <= 2048) return go_back<T, V, 128, 2 * I>(a, s);
  if (c <= 4096) return go_back<T, V, 256, 2 * I>(a, s);
  if (c <= 6144) return go_back<T, V, 512, 12 / V + (12 % V ? 1 : 0)>(a, s);
  if (c <= 8192) return go_back<T, V, 512, 2 * I>(a, s);
  if (a.rows > 0x7fffffffull) return cudaErrorInvalidValue;
  norm_long_dx_kernel<T><<<(unsigned)a.rows, 1024, 0, s>>>(a);
  const uint64_t shares = back_parts(a.rows), blocks = (c + 255) / 256 * shares;
  if (blocks > 0x7fffffffull) return cudaErrorInvalidValue;
  norm_long_params_kernel<T><<<(unsigned)blocks, 256, 0, s>>>(a, (uint32_t)shares);
  return cudaGetLastError();
}

template <class T, bool BACK>
cudaError_t by_vector(const NormArgs& a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  uint64_t m = a.channels | a.x_stride | a.y_stride | a.dy_stride | a.dx_stride, p = 0;
  for (const void* q : {a.x, (const void*)a.y, a.dy, (const void*)a.dx}) p |= reinterpret_cast<uint64_t>(q);
  const bool wide = m % V == 0 && p % 16 == 0;
  if constexpr (BACK) return wide ? backward<T, V>(a, s) : backward<T, 1>(a, s);
  else return wide ? forward<T, V>(a, s) : forward<T, 1>(a, s);
}

template <bool BACK>
cudaError_t by_type(const NormArgs& a, cudaStream_t s) {
  switch (a.type) {
    case SEQ_F32: return by_vector<float, BACK>(a, s);
    case SEQ_F16: return by_vector<__half, BACK>(a, s);
    default: return by_vector<__nv_bfloat16, BACK>(a, s);
  }
}

}  // namespace

size_t norm_backward_bytes(uint64_t rows, uint64_t channels) { return back_parts(rows) * 2 * channels * 4; }
cudaError_t launch_norm(const NormArgs& a, cudaStream_t s) { return a.rows && a.channels ? by_type<false>(a, s) : cudaSuccess; }
cudaError_t launch_norm_backward(const NormArgs& a, cudaStream_t s) {
  if (!a.channels) return cudaSuccess;
  if (!a.rows) {  // no rows: the parameters' gradients are sums of nothing
    cudaError_t e = a.dw ? cudaMemsetAsync(a.dw, 0, a.channels * 4, s) : cudaSuccess;
    if (e == cudaSuccess && a.dbias) e = cudaMemsetAsync(a.dbias, 0, a.channels * 4, s);
    return e;
  }
  cudaError_t e = by_type<true>(a, s);
  if (e != cudaSuccess || (!a.dw && !a.dbias)) return e;
  return launch_reduce_rows(a.part, back_parts(a.rows), 2 * a.channels, a.channels, a.dw, a.dbias, s);
}

}  // namespace sparsl
