// Layer norm over the channels of each row, and its gradients.
//
//   hat = (x - mean) rstd,   y = hat w + bias,   rstd = 1 / sqrt(var + eps)
//   dx  = rstd (w dy - mean(w dy) - hat mean(w dy hat))
//   dw  = sum over rows of dy hat,   dbias = sum over rows of dy
//
// Bound by HBM: forward x read and y written once, backward x and dy read and
// dx written once.  A group of threads keeps a row in registers (32 values a
// thread at most), so the variance is the mean of squared deviations, not a
// difference of sums; longer rows are read again for each of the steps.  In
// the backward pass a block walks many rows, its threads keeping the sums of dw
// and dbias for their own channels in registers, and the blocks' partial rows
// are added in a fixed order.
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
// (85 us against 34 at 16384 x 2048 bf16).
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

template <class T, int V, int B, int I>
__global__ void __launch_bounds__(B) norm_backward_kernel(NormArgs a) {
  __shared__ float sh[2][64];
  const uint32_t tid = threadIdx.x;
  float w[I][V], dw[I][V], db[I][V];
  Pack<T, V> xn[I], dn[I];
  float mean_n = 0.f, rstd_n = 0.f;
  const auto ask = [&](uint64_t row) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
    const T* dy = reinterpret_cast<const T*>(a.dy) + row * a.dy_stride;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const uint32_t c = (i * B + tid) * V;
      if (c < a.channels) {
        xn[i] = *reinterpret_cast<const Pack<T, V>*>(x + c);
        dn[i] = *reinterpret_cast<const Pack<T, V>*>(dy + c);
      }
    }
    mean_n = a.mean[row];
    rstd_n = a.rstd[row];
  };
  if (blockIdx.x < a.rows) ask(blockIdx.x);
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t c = (i * B + tid) * V + j;
      w[i][j] = c < a.channels ? (a.w ? load_param<T>(a.w, a.params_f32, c) : 1.f) : 0.f;
      dw[i][j] = db[i][j] = 0.f;
    }
  const float scale = 1.0f / (float)a.channels;
  int turn = 0;
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float mean = mean_n, rstd = rstd_n;
    float h[I][V], g[I][V], s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const bool in = (i * B + tid) * V < a.channels;
        h[i][j] = in ? (to_f32(xn[i].v[j]) - mean) * rstd : 0.f;
        g[i][j] = in ? to_f32(dn[i].v[j]) : 0.f;
        db[i][j] += g[i][j];
        dw[i][j] = __fmaf_rn(g[i][j], h[i][j], dw[i][j]);
        g[i][j] *= w[i][j];
        s[0] += g[i][j];
        s[1] = __fmaf_rn(g[i][j], h[i][j], s[1]);
      }
    if (row + gridDim.x < a.rows) ask(row + gridDim.x);
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

// 8 values of a row per thread, 16 where 1024 threads of 8 do not hold it: rows
// up to 16384 values; longer ones are read again for each of the steps.
template <class T, int V>
cudaError_t forward(const NormArgs& a, cudaStream_t s) {
  constexpr int I = 8 / V;
  const uint64_t c = a.channels;
  if (c <= 256) return go<T, V, 32, I>(a, s);
  if (c <= 1024) return go<T, V, 128, I>(a, s);
  if (c <= 2048) return go<T, V, 256, I>(a, s);
  if (c <= 4096) return go<T, V, 512, I>(a, s);
  if (c <= 6144) return go<T, V, 512, 12 / V + (12 % V ? 1 : 0)>(a, s);
  if (c <= 8192) return go<T, V, 1024, I>(a, s);
  if (c <= 16384) return go<T, V, 1024, 2 * I>(a, s);
  if (a.rows > 0x7fffffffull) return cudaErrorInvalidValue;
  norm_long_kernel<T><<<(unsigned)a.rows, 1024, 0, s>>>(a);
  return cudaGetLastError();
}

template <class T, int V, int B, int I>
cudaError_t go_back(const NormArgs& a, cudaStream_t s) {
  norm_backward_kernel<T, V, B, I><<<(unsigned)back_parts(a.rows), B, 0, s>>>(a);
  return cudaGetLastError();
}

// 8 values per thread up to rows of 4096, 12 and 16 up to 6144 and 8192; longer
// rows' dx and sums take a kernel each.
template <class T, int V>
cudaError_t backward(const NormArgs& a, cudaStream_t s) {
  constexpr int I = 8 / V;
  const uint64_t c = a.channels;
  if (c <= 512) return go_back<T, V, 64, I>(a, s);
  if (c <= 1024) return go_back<T, V, 128, I>(a, s);
  if (c <= 2048) return go_back<T, V, 256, I>(a, s);
  if (c <= 4096) return go_back<T, V, 512, I>(a, s);
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
