// Sequence operators: the short causal convolution, the selective state space
// scan and layer norm over token arrays [tokens, channels].
//
// Tokens of all sequences lie one after another; sequence i holds the tokens
// [seq_ptr[i], seq_ptr[i + 1]), or n_seq equal runs without seq_ptr.  Every
// kernel clamps what it reads from seq_ptr to [0, tokens] and treats a slot
// outside [0, n_slots) as none, so no content of those device arrays leads an
// access out of the buffers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace sparsl {

struct SeqView {
  uint64_t tokens;
  uint64_t n_seq;
  uint64_t run;            // tokens of each sequence when seq_ptr is null
  const int32_t* seq_ptr;  // n_seq + 1, or null
  const int32_t* slots;    // n_seq, or null: sequence i keeps its state in row i
  const uint8_t* resume;   // n_seq, or null: all continue from their state
  uint64_t n_slots;

  __device__ __forceinline__ int64_t begin(int64_t i) const {
    if (!seq_ptr) return i * (int64_t)run;
    const int64_t v = __ldg(seq_ptr + i);
    return v < 0 ? 0 : (v > (int64_t)tokens ? (int64_t)tokens : v);
  }
  // The last sequence that begins at or before token t (-1: none).
  __device__ __forceinline__ int64_t of(int64_t t) const {
    if (!seq_ptr) {
      const int64_t i = run ? t / (int64_t)run : (int64_t)n_seq;
      return i < (int64_t)n_seq ? i : (int64_t)n_seq;
    }
    int64_t lo = 0, hi = (int64_t)n_seq + 1;  // the first entry above t lies in [lo, hi]
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (begin(mid) <= t) lo = mid + 1; else hi = mid;
    }
    return lo - 1;
  }
  // The first sequence that begins at or behind token t (n_seq: none).
  __device__ __forceinline__ int64_t first_from(int64_t t) const {
    if (!seq_ptr) {
      if (!run) return t > 0 ? (int64_t)n_seq : 0;
      const int64_t i = (t + (int64_t)run - 1) / (int64_t)run;
      return i < (int64_t)n_seq ? i : (int64_t)n_seq;
    }
    int64_t lo = 0, hi = (int64_t)n_seq;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (begin(mid) < t) lo = mid + 1; else hi = mid;
    }
    return lo;
  }
  // The same by a whole warp: 32 probes at a time instead of one.
  __device__ __forceinline__ int64_t first_from_warp(int64_t t) const {
    if (!seq_ptr) return first_from(t);
    const uint32_t lane = threadIdx.x & 31;
    int64_t lo = 0, len = (int64_t)n_seq;  // the answer lies in [lo, lo + len]
    while (len > 32) {
      const int64_t each = (len + 31) / 32, at = lo + lane * each;
      const uint32_t n = __popc(__ballot_sync(0xffffffffu, at < lo + len && begin(at) < t));
      if (n == 0) return lo;
      const int64_t end = lo + len;
      lo += (n - 1) * each + 1;
      len = lo + each - 1 < end ? each - 1 : end - lo;
    }
    return lo + __popc(__ballot_sync(0xffffffffu, lane < len && begin(lo + lane) < t));
  }
  // The state row of sequence i, or -1.
  __device__ __forceinline__ int64_t slot(int64_t i) const {
    const int64_t s = slots ? (int64_t)__ldg(slots + i) : i;
    return s >= 0 && s < (int64_t)n_slots ? s : -1;
  }
  __device__ __forceinline__ bool resumes(int64_t i) const { return !resume || __ldg(resume + i) != 0; }
};

enum SeqType : int { SEQ_F32 = 0, SEQ_F16 = 1, SEQ_BF16 = 2 };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A parameter (weight, bias) is f32 or has the tokens' type.
template <class T>
__device__ __forceinline__ float load_param(const void* p, bool f32, uint64_t i) {
  return f32 ? __ldg(reinterpret_cast<const float*>(p) + i) : to_f32(reinterpret_cast<const T*>(p)[i]);
}

// V values of type T as one access where V * sizeof(T) is 4, 8 or 16 bytes.
template <class T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};
template <class T, int V>
__device__ __forceinline__ void load_pack(const T* p, float (&out)[V]) {
  const Pack<T, V> k = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = to_f32(k.v[i]);
}
template <class T, int V>
__device__ __forceinline__ void store_pack(T* p, const float (&in)[V]) {
  Pack<T, V> k;
#pragma unroll
  for (int i = 0; i < V; ++i) k.v[i] = from_f32<T>(in[i]);
  *reinterpret_cast<Pack<T, V>*>(p) = k;
}

// Copies into shared memory that nothing waits for before copies_done() (or,
// with the last N groups still under way, copies_but<N>()).
template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from, uint32_t bytes) {
  const uint32_t s = (uint32_t)__cvta_generic_to_shared(to);
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s), "l"(from), "r"(bytes) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(s), "l"(from), "n"(BYTES), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void copies_done() {
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();
}

constexpr float kLog2e = 1.4426950408889634f;

// 2^v and 1/v by the special function unit (relative error below 2^-22 and
// 2^-23): the sums they enter are rounded at 2^-24 a step, and the outputs
// they reach at most at that of f32.  Results below 2^-126 are zero: a state that
// one token takes that far down is gone.
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// Two f32 side by side: one instruction for both, each rounded by itself.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(f32x2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 ex2_2(f32x2 v) {
  float lo, hi;
  unpair(v, lo, hi);
  return pair(ex2(lo), ex2(hi));
}
__device__ __forceinline__ float sum2(f32x2 v) {
  float lo, hi;
  unpair(v, lo, hi);
  return lo + hi;
}

__device__ __forceinline__ float sigmoid(float v) { return rcp(1.0f + ex2(-kLog2e * v)); }

// Column sums of part[rows, cols]: columns below `split` into out, the rest into more (may be null).
cudaError_t launch_reduce_rows(const float* part, uint64_t rows, uint64_t cols, uint64_t split, float* out, float* more,
                               cudaStream_t s);

// ---- the short causal convolution (conv.cu) ----
struct ConvArgs {
  SeqView seq;
  int type;
  uint32_t channels, width;
  bool silu, params_f32;
  const void* x;
  uint64_t x_stride;
  const void* w;     // [channels, width]
  const void* bias;  // [channels] or null
  void* y;
  uint64_t y_stride;
  const void* state;  // [n_slots, width - 1, channels] or null
  void* final_state;
  // backward
  const void* dy;
  uint64_t dy_stride;
  void* dx;
  uint64_t dx_stride;
  float* dw;
  float* dbias;
  void* dstate;
  const void* dfinal;
  float* part;
};
size_t conv_backward_bytes(uint64_t tokens, uint64_t channels, uint32_t width);
cudaError_t launch_conv(const ConvArgs& a, cudaStream_t s);
cudaError_t launch_conv_backward(const ConvArgs& a, cudaStream_t s);
cudaError_t launch_conv_step(const ConvArgs& a, cudaStream_t s);

// ---- the selective scan (sscan.cu) ----
struct SscanArgs {
  SeqView seq;
  int type;
  uint32_t channels, states, groups;
  bool softplus;
  const void *x, *dt, *z, *b, *c;
  uint64_t x_stride, dt_stride, z_stride, b_stride, c_stride, b_group, c_group;
  const float *a, *d, *dt_bias;
  void* y;
  uint64_t y_stride;
  const float* state;  // [n_slots, channels, states] or null
  float* final_state;
  float* marks;  // states before every kMarkEvery-th token, or null
  void* work;
  // backward
  const void* dy;
  uint64_t dy_stride;
  void *dx, *ddt, *dz, *db, *dc;
  uint64_t dx_stride, ddt_stride, dz_stride, db_stride, dc_stride, db_group, dc_group;
  float *da, *dd, *ddt_bias;
  float* dstate;
  const float* dfinal;
  // Row strides in bytes (the launch fills them in): a row's address is one 32 x 32 -> 64 bit product.
  uint32_t x_row, dt_row, z_row, y_row, dy_row, dx_row, ddt_row, dz_row;
};
constexpr uint64_t kMostStride = (1u << 29) - 1;  // elements from token to token: 4-byte rows of it still count in 31 bits
constexpr uint32_t kMaxStates = 64;
size_t sscan_bytes(uint64_t tokens, uint64_t channels, uint32_t states, uint64_t n_seq, uint32_t groups);
size_t sscan_backward_bytes(uint64_t tokens, uint64_t channels, uint32_t states, uint64_t n_seq, uint32_t groups);
size_t sscan_mark_bytes(uint64_t tokens, uint64_t channels, uint32_t states);
// How a pass is laid out, for tests: lanes a channel, chunks of the token axis and
// their tokens, whether states are handed on between them, and the lanes a channel
// of the pass in front that computes those (0: none).
struct ScanLayout {
  uint64_t lanes, chunks, len, carry, chunk_lanes;
};
ScanLayout sscan_layout(uint64_t tokens, uint32_t channels, uint32_t states, uint64_t n_seq, uint32_t groups, bool ragged);
ScanLayout sscan_backward_layout(uint64_t tokens, uint32_t channels, uint32_t states, uint64_t n_seq, uint32_t groups, bool ragged);
cudaError_t launch_sscan(const SscanArgs& a, cudaStream_t s);
cudaError_t launch_sscan_backward(const SscanArgs& a, cudaStream_t s);
cudaError_t launch_sscan_step(const SscanArgs& a, cudaStream_t s);

// By the tokens' type.
cudaError_t launch_sscan_f32(const SscanArgs& a, cudaStream_t s);
cudaError_t launch_sscan_f16(const SscanArgs& a, cudaStream_t s);
cudaError_t launch_sscan_bf16(const SscanArgs& a, cudaStream_t s);
cudaError_t launch_sscan_step_f32(const SscanArgs& a, cudaStream_t s);
cudaError_t launch_sscan_step_f16(const SscanArgs& a, cudaStream_t s);
cudaError_t launch_sscan_step_bf16(const SscanArgs& a, cudaStream_t s);
cudaError_t launch_sscan_backward_f32(const SscanArgs& a, cudaStream_t s);
cudaError_t launch_sscan_backward_f16(const SscanArgs& a, cudaStream_t s);
cudaError_t launch_sscan_backward_bf16(const SscanArgs& a, cudaStream_t s);

// ---- layer norm (norm.cu) ----
struct NormArgs {
  int type;
  bool params_f32;
  uint64_t rows, channels;
  const void* x;
  uint64_t x_stride;
  const void *w, *bias;
  float eps;
  void* y;
  uint64_t y_stride;
  float *mean, *rstd;
  const void* dy;
  uint64_t dy_stride;
  void* dx;
  uint64_t dx_stride;
  float *dw, *dbias;
  float* part;
};
size_t norm_backward_bytes(uint64_t rows, uint64_t channels);
cudaError_t launch_norm(const NormArgs& a, cudaStream_t s);
cudaError_t launch_norm_backward(const NormArgs& a, cudaStream_t s);

}  // namespace sparsl
