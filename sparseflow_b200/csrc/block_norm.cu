// What stands between two blocks of a transformer, in one pass over its rows (all in 32 bits, each output rounded once):
//   z = y                       or   norm(y) * post_weight (+ post_bias)
//   r = x + scale * gate * z    (no y: r = x)
//   h = norm(r) * weight (+ bias)
//   norm(v) = v / sqrt(mean(v^2) + eps)                       (rms)
//           = (v - mean(v)) / sqrt(mean((v - mean(v))^2) + eps)   (layer)
// h is the norm of the unrounded r.  HBM-bound: x and y are read once, r and h written once; a block owns a row and keeps it in
// registers between the reductions (one for an rms norm, two for a layer norm, each: the mean first, then the centered
// squares, so that a large mean costs no digits).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "launch.h"
#include "sm100_ptx.cuh"

namespace sfb200 {
namespace {

struct NormParams {
  const void *x, *y, *weight, *bias, *post_weight, *post_bias, *gate;
  void *r, *h;
  int64_t ld_x, ld_y, ld_r, ld_h, ld_gate;
  int rows, cols, rows_per_gate, gate_step;      // gate_step: 1 a value per column, 0 one value for the row
  float scale, eps, post_eps, inv_cols;
  int layer;
};

template <class T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V consecutive values: V = 8 through 16-byte accesses, V = 1 one by one
template <class T, int V>
struct alignas(V == 8 ? 16 : sizeof(T)) Pack {
  T v[V];
};
template <class T, int V>
__device__ __forceinline__ void load_f(const void* base, int64_t at, float* f) {
  const Pack<T, V> k = *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(base) + at);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_f<T>(k.v[i]);
}
template <class T, int V>
__device__ __forceinline__ void store_f(void* base, int64_t at, const float* f) {
  Pack<T, V> k;
#pragma unroll
  for (int i = 0; i < V; ++i) k.v[i] = from_f<T>(f[i]);
  *reinterpret_cast<Pack<T, V>*>(static_cast<T*>(base) + at) = k;
}

__device__ __forceinline__ float block_sum(float v, float* part) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (warps == 1) return v;
  __syncthreads();                      // the parts of the sum before are read
  if (lane == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < warps ? part[lane] : 0.f;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// f[NV][V]: the thread's values of the row (zero behind its end) -> normalised, weighted
template <class YT, int V, int NV>
__device__ __forceinline__ void normalise(float (&f)[NV][V], const NormParams& p, const void* weight, const void* bias, float eps, float* part) {
  float s = 0.f;
  if (p.layer) {
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < V; ++i) s += f[n][i];
    const float mean = block_sum(s, part) * p.inv_cols;
    s = 0.f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const bool in = (n * blockDim.x + threadIdx.x) * V < static_cast<unsigned>(p.cols);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        f[n][i] = in ? f[n][i] - mean : 0.f;
        s = fmaf(f[n][i], f[n][i], s);
      }
    }
  } else {
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < V; ++i) s = fmaf(f[n][i], f[n][i], s);
  }
  const float inv = rsqrtf(block_sum(s, part) * p.inv_cols + eps);
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const unsigned c = (n * blockDim.x + threadIdx.x) * V;
    if (c < static_cast<unsigned>(p.cols)) {
      float w[V], b[V];
      load_f<YT, V>(weight, c, w);
      if (bias != nullptr) load_f<YT, V>(bias, c, b);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        f[n][i] = f[n][i] * inv * w[i];
        if (bias != nullptr) f[n][i] += b[i];
      }
    }
  }
}

// XT: type of x and r; YT: type of y, h, weights and gate
template <class XT, class YT, int V, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT) block_norm_kernel(const NormParams p) {
  __shared__ float part[32];
  dependency_wait();
  dependency_trigger();
  const int64_t row = blockIdx.x;
  const unsigned cols = static_cast<unsigned>(p.cols);
  float f[NV][V], z[NV][V];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const unsigned c = (n * blockDim.x + threadIdx.x) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) f[n][i] = z[n][i] = 0.f;
    if (c < cols) {
      load_f<XT, V>(p.x, row * p.ld_x + c, f[n]);
      if (p.y != nullptr) load_f<YT, V>(p.y, row * p.ld_y + c, z[n]);
    }
  }
  if (p.y != nullptr) {
    if (p.post_weight != nullptr) normalise<YT, V, NV>(z, p, p.post_weight, p.post_bias, p.post_eps, part);
    const int64_t gate_row = p.gate != nullptr ? row / p.rows_per_gate * p.ld_gate : 0;
    const float row_gate = p.gate != nullptr && p.gate_step == 0 ? to_f<YT>(static_cast<const YT*>(p.gate)[gate_row]) : 1.f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const unsigned c = (n * blockDim.x + threadIdx.x) * V;
      if (c < cols) {
        float g[V];
        const bool per_col = p.gate != nullptr && p.gate_step != 0;
        if (per_col) load_f<YT, V>(p.gate, gate_row + c, g);
#pragma unroll
        for (int i = 0; i < V; ++i) f[n][i] = fmaf(p.scale * (per_col ? g[i] : row_gate), z[n][i], f[n][i]);
        if (p.r != nullptr) store_f<XT, V>(p.r, row * p.ld_r + c, f[n]);
      }
    }
  }
  if (p.h == nullptr) return;
  normalise<YT, V, NV>(f, p, p.weight, p.bias, p.eps, part);
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const unsigned c = (n * blockDim.x + threadIdx.x) * V;
    if (c < cols) store_f<YT, V>(p.h, row * p.ld_h + c, f[n]);
  }
}

template <class XT, class YT, int V, int NV>
int launch_nv(const NormParams& p, int threads, cudaStream_t stream) {
  if (threads <= 256) return launch_dependent(block_norm_kernel<XT, YT, V, NV, 256>, p.rows, threads, 0, 0, stream, p);
  return launch_dependent(block_norm_kernel<XT, YT, V, NV, 1024>, p.rows, threads, 0, 0, stream, p);
}
template <class XT, class YT>
int launch_types(const NormParams& p, bool vec, cudaStream_t stream) {
  const int per = vec ? 8 : 1, pieces = (p.cols + per - 1) / per;
  auto threads = [&](int nv) { return ((pieces + nv - 1) / nv + 31) / 32 * 32; };
  if (vec) {
    if (pieces <= 512) return launch_nv<XT, YT, 8, 1>(p, threads(1), stream);
    if (pieces <= 2048) return launch_nv<XT, YT, 8, 2>(p, threads(2), stream);
    return kErrInvalid;
  }
  if (pieces <= 1024) return launch_nv<XT, YT, 1, 4>(p, threads(4), stream);
  if (pieces <= 16384) return launch_nv<XT, YT, 1, 16>(p, threads(16), stream);
  return kErrInvalid;
}

}  // namespace

int launch_block_norm(const NormArgs& a, cudaStream_t stream) {
  if (a.rows < 0 || a.cols < 1 || a.cols > kNormMaxCols) return kErrInvalid;
  if (!a.x || (!a.r && !a.h) || (a.h && !a.weight) || (a.y && !a.r) || (!a.y && (a.r || a.gate || a.post_weight))) return kErrInvalid;
  if (a.ld_x < a.cols || (a.y && a.ld_y < a.cols) || (a.r && a.ld_r < a.cols) || (a.h && a.ld_h < a.cols)) return kErrInvalid;
  if (a.gate && (a.gate_rows < 1 || a.rows % a.gate_rows != 0 || (a.gate_cols != 1 && a.gate_cols != a.cols))) return kErrInvalid;
  if (a.x_type < 0 || a.x_type > 2 || a.y_type < 0 || a.y_type > 2 || (a.x_type != a.y_type && a.x_type != 2)) return kErrInvalid;
  if (a.rows == 0) return kOk;
  NormParams p{};
  p.x = a.x; p.y = a.y; p.weight = a.weight; p.bias = a.bias; p.post_weight = a.post_weight; p.post_bias = a.post_bias;
  p.gate = a.gate; p.r = a.r; p.h = a.h;
  p.ld_x = a.ld_x; p.ld_y = a.ld_y; p.ld_r = a.ld_r; p.ld_h = a.ld_h; p.ld_gate = a.ld_gate;
  p.rows = a.rows; p.cols = a.cols;
  p.rows_per_gate = a.gate ? a.rows / a.gate_rows : 1;
  p.gate_step = a.gate_cols == 1 ? 0 : 1;
  p.scale = a.scale; p.eps = a.eps; p.post_eps = a.post_eps;
  p.inv_cols = 1.0f / static_cast<float>(a.cols);
  p.layer = a.layer;
  const bool gate_vec = a.gate && p.gate_step;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.r) |
                          reinterpret_cast<uintptr_t>(a.h) | reinterpret_cast<uintptr_t>(a.weight) | reinterpret_cast<uintptr_t>(a.bias) |
                          reinterpret_cast<uintptr_t>(a.post_weight) | reinterpret_cast<uintptr_t>(a.post_bias) |
                          (gate_vec ? reinterpret_cast<uintptr_t>(a.gate) : 0);
  const int64_t pitches = a.cols | a.ld_x | (a.y ? a.ld_y : 0) | (a.r ? a.ld_r : 0) | (a.h ? a.ld_h : 0) | (gate_vec ? a.ld_gate : 0);
  const bool vec = pitches % 8 == 0 && bases % 16 == 0;
  if (a.x_type == 2) {
    if (a.y_type == 2) return launch_types<float, float>(p, vec, stream);
    if (a.y_type == kBF16) return launch_types<float, __nv_bfloat16>(p, vec, stream);
    return launch_types<float, __half>(p, vec, stream);
  }
  if (a.x_type == kBF16) return launch_types<__nv_bfloat16, __nv_bfloat16>(p, vec, stream);
  return launch_types<__half, __half>(p, vec, stream);
}

}  // namespace sfb200
