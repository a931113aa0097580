// What stands between two blocks of a transformer, in one pass over its rows (all in 32 bits, each output rounded once):
//   z = y                       or   norm(y) * post_weight (+ post_bias)
//   r = x + scale * gate * z    (no y: r = x)
//   h = norm(r) * weight (+ bias)
//   norm(v) = v / sqrt(mean(v^2) + eps)                       (rms)
//           = (v - mean(v)) / sqrt(mean((v - mean(v))^2) + eps)   (layer)
// h is the norm of the unrounded r.  HBM-bound: x and y are read once, r and h written once.  A block owns a row and keeps it in registers between the
// reductions: one for an rms norm, two for a layer norm (the mean first, then the centered squares, so that a large mean costs no
// digits).  x and y wait there in their own type, so that three blocks of a wide row fit an SM and one's loads run under another's reductions.
//
// Eight values per access: 16-byte pieces of the tensors, also where a row begins inside one (odd widths): a thread owns
// the columns of a whole piece, 8j - m .. with m the row's offset, reads it with the neighbour's values in it (inside the tensor) and drops those; the
// pieces at the ends of a row are stored value by value, and weights, which begin at column 0, are shifted by m from two pieces.
// Value by value throughout where the tensors' rows do not lie alike in their pieces.
// Measured: 4096 x 8192 (f32 stream, bf16, norm on both sides) 73 us replayed (5.5 TB/s; streaming stores and 256-byte prefetches: the same), 16384 x 2048 bf16 58 us (4.6 TB/s; issue-bound: 50 instructions
// a piece), 8192 x 4097 layer norms 122 us, 24 x 4096 2.7 us (latency).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <atomic>

#include "device_state.h"
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

// Sum over the row's threads (WARP: a warp).  `turn` alternates between two sets of parts, so that one barrier does; the parts are added by
// every thread, in order, four per load: cheaper than a second round of shuffles.  PADDED: the parts of no warp are zero.
template <bool WARP, bool PADDED>
__device__ __forceinline__ float row_sum(float v, float (*part)[32], int& turn) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if (WARP) return v;
  const int warps = blockDim.x >> 5;
  float* mine = part[turn];
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) mine[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < warps; w += 4) {
    const float4 q = *reinterpret_cast<const float4*>(mine + w);
    if (PADDED) v += (q.x + q.y) + (q.z + q.w);
    else v += q.x + (w + 1 < warps ? q.y : 0.f) + (w + 2 < warps ? q.z : 0.f) + (w + 3 < warps ? q.w : 0.f);
  }
  return v;
}

// V values of a row from column c (c may lie before the row, c + V behind it): those of the row, zero for the others.  `room`: values of the tensor
// from there to its end.
template <class T, int V, bool SHIFT>
__device__ __forceinline__ Pack<T, V> load_piece(const void* base, int64_t at, int64_t room) {
  Pack<T, V> k;
  if (!SHIFT || room >= V) {
    k = *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(base) + at);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) k.v[i] = i < room ? static_cast<const T*>(base)[at + i] : from_f<T>(0.f);
  }
  return k;
}
template <class T, int V, bool SHIFT>
__device__ __forceinline__ void store_piece(void* base, int64_t at, int c, int cols, const float* f) {
  if (!SHIFT || (c >= 0 && c + V <= cols)) {
    store_f<T, V>(base, at, f);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i >= 0 && c + i < cols) static_cast<T*>(base)[at + i] = from_f<T>(f[i]);
  }
}
// V values of a vector over the columns (whole pieces from column 0, if `pieces`) from column c = 8j - m
template <class T, int V, bool SHIFT>
__device__ __forceinline__ void load_vector(const void* base, int64_t first, int c, int cols, int m, bool pieces, float* f) {
  const T* v = static_cast<const T*>(base) + first;
  if (!SHIFT || (V == 8 && pieces && m == 0 && c + V <= cols)) {
    load_f<T, V>(v, c, f);
  } else if (V == 8 && sizeof(T) == 2 && pieces && c >= 0 && c + m + 8 <= cols) {
    const uint4 a = *reinterpret_cast<const uint4*>(v + c + m - 8), b = *reinterpret_cast<const uint4*>(v + c + m);
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};      // columns c + m - 8 ..: c is 8 - m values on, the same for the whole block
    const int off = 8 - m;
    if (off & 4) {
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (off & 2) {
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    if (off & 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint16_t bits = static_cast<uint16_t>(w[i / 2] >> (16 * (i % 2)));
      T t;
      memcpy(&t, &bits, sizeof(T) == 2 ? 2 : 0);
      f[i] = to_f<T>(t);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = c + i >= 0 && c + i < cols ? to_f<T>(v[c + i]) : 0.f;
  }
}

// Asynchronous copy of `bytes` (0 .. 16, the rest zero) to shared memory
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
template <class T, int V, bool SHIFT>
__device__ __forceinline__ void copy_piece(uint32_t dst, const T* src, int64_t room) {
#pragma unroll
  for (int b = 0; b < V * static_cast<int>(sizeof(T)); b += 16) {
    if (!SHIFT) {
      copy16(dst + b, reinterpret_cast<const uint8_t*>(src) + b, 16);
    } else {
      const int64_t left = room * static_cast<int64_t>(sizeof(T)) - b;
      const int bytes = left >= 16 ? 16 : left > 0 ? static_cast<int>(left) : 0;
      copy16(dst + b, reinterpret_cast<const uint8_t*>(src) + (bytes > 0 ? b : 0), bytes);
    }
  }
}

// XT: type of x and r; YT: type of y, h, weights and gate.  WARP: a warp per row, eight rows per block; otherwise a block per row.
// RING: blocks stay; while a row is reduced, asynchronous copies bring the next one into shared memory, every thread its own pieces, so
// that nobody waits for anybody.  With SHIFT the block's rows are eight apart or a multiple of it: one m, and the vectors are shifted once, into
// shared memory too (`vectors` of them, in the order post_bias, post_weight, weight, bias, gate where all rows share it).
template <class XT, class YT, int V, int NV, bool SHIFT, bool LAYER, bool WARP, bool RING, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) block_norm_kernel(const NormParams p) {
  __shared__ __align__(16) float part[2][32];
  extern __shared__ __align__(16) uint8_t ring[];
  if (RING)      // the parts of no warp; the first barrier of a sum comes before they are read
    for (int i = threadIdx.x; i < 64; i += blockDim.x)
      if ((i & 31) >= static_cast<int>(blockDim.x >> 5)) part[i >> 5][i & 31] = 0.f;
  dependency_wait();
  dependency_trigger();
  int row_i = WARP ? static_cast<int>(blockIdx.x * 8 + (threadIdx.x >> 5)) : static_cast<int>(blockIdx.x);
  if (row_i >= p.rows) return;
  const int m = SHIFT ? static_cast<int>(row_i * p.ld_x & 7) : 0;
  const int c0 = static_cast<int>(WARP ? threadIdx.x & 31 : threadIdx.x) * V - m, step = (WARP ? 32 : static_cast<int>(blockDim.x)) * V;
  auto outside = [&](int c, int i) { return c + i < 0 || c + i >= p.cols; };
  int turn = 0;
  Pack<XT, V>* x_slot = reinterpret_cast<Pack<XT, V>*>(ring) + threadIdx.x;                          // [NV][threads]
  Pack<YT, V>* y_slot = reinterpret_cast<Pack<YT, V>*>(ring + NV * blockDim.x * sizeof(Pack<XT, V>)) + threadIdx.x;
  Pack<YT, V>* vectors = y_slot + NV * blockDim.x;                                                   // [vector][NV][threads]
  auto fetch = [&](int r) {
    const int64_t row = r, behind = p.rows - 1 - row;
    if (r < p.rows) {
      const XT* x = static_cast<const XT*>(p.x) + row * p.ld_x + c0;
      const YT* y = static_cast<const YT*>(p.y) + row * p.ld_y + c0;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int c = c0 + n * step;
        if (c >= p.cols) continue;
        copy_piece<XT, V, SHIFT>(smem_u32(x_slot + n * blockDim.x), x + n * step, behind * p.ld_x + p.cols - c);
        if (p.y != nullptr) copy_piece<YT, V, SHIFT>(smem_u32(y_slot + n * blockDim.x), y + n * step, behind * p.ld_y + p.cols - c);
      }
    }
  };
  const bool one_gate = p.gate != nullptr && p.gate_step != 0 && p.rows_per_gate >= p.rows;
  auto vector = [&](const void* base, int64_t first, int which, int n, int c, bool pieces, float* f) {
    if (RING && SHIFT && which >= 0) {
      const Pack<YT, V> k = vectors[(which * NV + n) * blockDim.x];
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = to_f<YT>(k.v[i]);
    } else {
      load_vector<YT, V, SHIFT>(base, first, c, p.cols, m, pieces, f);
    }
  };
  if (RING) {
    fetch(row_i);
    if (SHIFT) {
      const void* all[5] = {p.post_bias, p.post_weight, p.weight, p.bias, one_gate ? p.gate : nullptr};
#pragma unroll
      for (int k = 0; k < 5; ++k)
        if (all[k] != nullptr)
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            float f[V];
            load_vector<YT, V, SHIFT>(all[k], 0, c0 + n * step, p.cols, m, true, f);
            Pack<YT, V> v;
#pragma unroll
            for (int i = 0; i < V; ++i) v.v[i] = from_f<YT>(f[i]);      // as they were: the type's own values
            vectors[(k * NV + n) * blockDim.x] = v;
          }
    }
  }
  for (;;) {
    const int64_t row = row_i;
    bool fetched = !RING;
    // the next row may replace this one in shared memory once it is in registers: behind the first sum over the row
    auto fetch_next = [&]() {
      if (!fetched) fetch(row_i + static_cast<int>(gridDim.x));
      fetched = true;
    };
    Pack<XT, V> xv[NV];
    Pack<YT, V> yv[NV];
    if (RING) asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = c0 + n * step;
      if (c < p.cols) {
        const int64_t behind = p.rows - 1 - row;
        xv[n] = RING ? x_slot[n * blockDim.x] : load_piece<XT, V, SHIFT>(p.x, row * p.ld_x + c, behind * p.ld_x + p.cols - c);
        if (p.y != nullptr) yv[n] = RING ? y_slot[n * blockDim.x] : load_piece<YT, V, SHIFT>(p.y, row * p.ld_y + c, behind * p.ld_y + p.cols - c);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          xv[n].v[i] = from_f<XT>(0.f);
          yv[n].v[i] = from_f<YT>(0.f);
        }
      }
      if (SHIFT && (c < 0 || c + V > p.cols)) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (outside(c, i)) {
            xv[n].v[i] = from_f<XT>(0.f);
            yv[n].v[i] = from_f<YT>(0.f);
          }
      }
    }
    // 1 / sqrt(mean of squares + eps) of values that are zero outside the row; layer: of the centered values, `mean` theirs
    auto inverse_norm = [&](auto value, float eps, float& mean) {
      float s = 0.f;
      if (LAYER) {
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
          for (int i = 0; i < V; ++i) s += value(n, i);
        mean = row_sum<WARP, RING>(s, part, turn) * p.inv_cols;
        fetch_next();
        s = 0.f;
      }
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int c = c0 + n * step;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float d = value(n, i);
          if (LAYER) d = (SHIFT ? outside(c, i) : c >= p.cols) ? 0.f : d - mean;
          s = fmaf(d, d, s);
        }
      }
      s = row_sum<WARP, RING>(s, part, turn);
      fetch_next();
      return rsqrtf(s * p.inv_cols + eps);
    };
    float f[NV][V];
    if (p.y != nullptr) {
      float z_mean = 0.f, z_inv = 1.f;
      if (p.post_weight != nullptr) z_inv = inverse_norm([&](int n, int i) { return to_f<YT>(yv[n].v[i]); }, p.post_eps, z_mean);
      const int64_t gate_row = p.gate != nullptr ? static_cast<int64_t>(row_i / p.rows_per_gate) * p.ld_gate : 0;
      const bool per_col = p.gate != nullptr && p.gate_step != 0;
      const float row_gate = p.scale * (p.gate != nullptr && !per_col ? to_f<YT>(static_cast<const YT*>(p.gate)[gate_row]) : 1.f);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int c = c0 + n * step;
        if (c < p.cols) {
          // f = x + factor * (z - mean) + offset: factor = scale * gate * inverse norm * post weight, offset = scale * gate * post bias
          float factor[V], w[V];
#pragma unroll
          for (int i = 0; i < V; ++i) f[n][i] = to_f<XT>(xv[n].v[i]);
          if (per_col) {
            vector(p.gate, gate_row, one_gate ? 4 : -1, n, c, gate_row % 8 == 0, factor);
            if (p.post_bias != nullptr) {
              vector(p.post_bias, 0, 0, n, c, true, w);
#pragma unroll
              for (int i = 0; i < V; ++i) f[n][i] = fmaf(p.scale * factor[i], w[i], f[n][i]);
            }
            if (p.post_weight != nullptr) {
              vector(p.post_weight, 0, 1, n, c, true, w);
#pragma unroll
              for (int i = 0; i < V; ++i) factor[i] *= w[i];
            }
          } else {
            if (p.post_bias != nullptr) {
              vector(p.post_bias, 0, 0, n, c, true, w);
#pragma unroll
              for (int i = 0; i < V; ++i) f[n][i] = fmaf(row_gate, w[i], f[n][i]);
            }
            if (p.post_weight != nullptr) {
              vector(p.post_weight, 0, 1, n, c, true, factor);
            } else {
#pragma unroll
              for (int i = 0; i < V; ++i) factor[i] = 1.f;
            }
          }
          const float common = (per_col ? p.scale : row_gate) * z_inv;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float z = to_f<YT>(yv[n].v[i]);
            f[n][i] = fmaf((LAYER ? z - z_mean : z) * common, factor[i], f[n][i]);
          }
          store_piece<XT, V, SHIFT>(p.r, row * p.ld_r + c, c, p.cols, f[n]);
          if (SHIFT && (c < 0 || c + V > p.cols)) {
#pragma unroll
            for (int i = 0; i < V; ++i)
              if (outside(c, i)) f[n][i] = 0.f;
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) f[n][i] = 0.f;
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < V; ++i) f[n][i] = to_f<XT>(xv[n].v[i]);
    }
    if (p.h != nullptr) {
      float mean = 0.f;
      const float inv = inverse_norm([&](int n, int i) { return f[n][i]; }, p.eps, mean);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int c = c0 + n * step;
        if (c < p.cols) {
          float w[V];
          vector(p.weight, 0, 2, n, c, true, w);
#pragma unroll
          for (int i = 0; i < V; ++i) f[n][i] = ((LAYER ? f[n][i] - mean : f[n][i]) * inv) * w[i];
          if (p.bias != nullptr) {
            vector(p.bias, 0, 3, n, c, true, w);
#pragma unroll
            for (int i = 0; i < V; ++i) f[n][i] += w[i];
          }
          store_piece<YT, V, SHIFT>(p.h, row * p.ld_h + c, c, p.cols, f[n]);
        }
      }
    } else if (RING) {
      __syncthreads();
      fetch_next();
    }
    if (!RING) break;
    row_i += static_cast<int>(gridDim.x);
    if (row_i >= p.rows) break;
  }
}

// Rows per SM and pieces of a row from which blocks stay: with a row or two each there is nothing to fetch ahead, and eight or more short rows per SM cover each
// other (16384 x 1024 f32 38 us, with the ring 44; 3000 x 1001 8.6 and 10.6; 4096 x 8192 f32 83 and 73, 8192 x 4097 layer norms 160 and 122).
constexpr int kRingRows = 4, kRingPieces = 257, kRingSizes = 17;

template <class Kernel>
int launch_ring(Kernel kernel, const NormParams& p, int threads, int smem, bool shift, int num_sms, std::atomic<int>* known, cudaStream_t stream) {
  // blocks per SM, asked for once per device, block size and shared-memory size (they change rarely)
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return kErrCuda;
  std::atomic<int>& slot = known[dev * kRingSizes + threads / 32];
  int per_sm = slot.load(std::memory_order_relaxed);
  if (per_sm / 16 != smem / 16) {
    int n = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess || n < 1)
      return kErrCuda;
    per_sm = smem / 16 * 16 + (n < 15 ? n : 15);
    slot.store(per_sm, std::memory_order_relaxed);
  }
  int grid = num_sms * (per_sm % 16);
  if (shift) grid = grid / 8 * 8;      // one m per block
  return launch_dependent(kernel, grid < p.rows ? grid : p.rows, threads, smem, 0, stream, p);
}

template <class XT, class YT, bool SHIFT, bool LAYER>
int launch_pieces(const NormParams& p, int num_sms, cudaStream_t stream) {
  const int pieces = (p.cols + (SHIFT ? 14 : 7)) / 8;      // a row may begin at the last value of a piece
  auto threads = [&](int nv) { return ((pieces + nv - 1) / nv + 31) / 32 * 32; };
  const int groups = (p.rows + 7) / 8;
  if (pieces <= 32) return launch_dependent(block_norm_kernel<XT, YT, 8, 1, SHIFT, LAYER, true, false, 256, 5>, groups, 256, 0, 0, stream, p);
  if (pieces <= 64) return launch_dependent(block_norm_kernel<XT, YT, 8, 2, SHIFT, LAYER, true, false, 256, 4>, groups, 256, 0, 0, stream, p);
  // a row or less per SM is latency: a piece per thread (24 rows of 1024 1.74 us, with two 2.36; of 4096 2.26 and 2.66; of 8192, where the sums of
  // 32 warps are added, 4.2 and 3.7)
  if (p.rows <= num_sms && pieces <= 640)
    return launch_dependent(block_norm_kernel<XT, YT, 8, 1, SHIFT, LAYER, false, false, 640, 1>, p.rows, threads(1), 0, 0, stream, p);
  const int nv = pieces <= 1024 ? 2 : 4;
  const int smem = threads(nv) * nv * 8 * static_cast<int>(sizeof(XT) + sizeof(YT) * (SHIFT ? 6 : 1));
  if (p.rows >= kRingRows * num_sms && pieces >= kRingPieces && smem <= 110 * 1024) {
    static std::atomic<int> known[3][kMaxDevices * kRingSizes];
    if (pieces <= 512) return launch_ring(block_norm_kernel<XT, YT, 8, 2, SHIFT, LAYER, false, true, 256, 4>, p, threads(2), smem, SHIFT, num_sms, known[0], stream);
    if (pieces <= 1024) return launch_ring(block_norm_kernel<XT, YT, 8, 2, SHIFT, LAYER, false, true, 512, 2>, p, threads(2), smem, SHIFT, num_sms, known[1], stream);
    return launch_ring(block_norm_kernel<XT, YT, 8, 4, SHIFT, LAYER, false, true, 512, 1>, p, threads(4), smem, SHIFT, num_sms, known[2], stream);
  }
  if (pieces <= 512) return launch_dependent(block_norm_kernel<XT, YT, 8, 2, SHIFT, LAYER, false, false, 256, 4>, p.rows, threads(2), 0, 0, stream, p);
  if (pieces <= 1024) return launch_dependent(block_norm_kernel<XT, YT, 8, 2, SHIFT, LAYER, false, false, 512, 2>, p.rows, threads(2), 0, 0, stream, p);
  return launch_dependent(block_norm_kernel<XT, YT, 8, 4, SHIFT, LAYER, false, false, 512, 1>, p.rows, threads(4), 0, 0, stream, p);
}
template <class XT, class YT, bool LAYER>
int launch_layer(const NormParams& p, bool vec, bool shift, int num_sms, cudaStream_t stream) {
  if (vec) return launch_pieces<XT, YT, false, LAYER>(p, num_sms, stream);
  if (shift && p.cols <= 16370) return launch_pieces<XT, YT, true, LAYER>(p, num_sms, stream);
  if (p.cols <= 1024) return launch_dependent(block_norm_kernel<XT, YT, 1, 4, false, LAYER, false, false, 256, 1>, p.rows, (p.cols + 127) / 128 * 32, 0, 0, stream, p);
  return launch_dependent(block_norm_kernel<XT, YT, 1, 16, false, LAYER, false, false, 1024, 1>, p.rows, (p.cols + 511) / 512 * 32, 0, 0, stream, p);
}
template <class XT, class YT>
int launch_types(const NormParams& p, bool vec, bool shift, int num_sms, cudaStream_t stream) {
  return p.layer ? launch_layer<XT, YT, true>(p, vec, shift, num_sms, stream) : launch_layer<XT, YT, false>(p, vec, shift, num_sms, stream);
}

}  // namespace

int launch_block_norm(const NormArgs& a, cudaStream_t stream) {
  if (a.rows < 0 || a.rows > 0x7fffffff - 4096 || a.cols < 1 || a.cols > kNormMaxCols) return kErrInvalid;
  if (a.rows == 0) return kOk;
  if (!a.x || (!a.r && !a.h) || (a.h && !a.weight) || (a.y && !a.r) || (!a.y && (a.r || a.gate || a.post_weight))) return kErrInvalid;
  if (a.ld_x < a.cols || (a.y && a.ld_y < a.cols) || (a.r && a.ld_r < a.cols) || (a.h && a.ld_h < a.cols)) return kErrInvalid;
  if (a.gate && (a.gate_rows < 1 || a.rows % a.gate_rows != 0 || (a.gate_cols != 1 && a.gate_cols != a.cols))) return kErrInvalid;
  if (a.x_type < 0 || a.x_type > 2 || a.y_type < 0 || a.y_type > 2 || (a.x_type != a.y_type && a.x_type != 2)) return kErrInvalid;
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
  // rows of all tensors alike in their pieces: same pitch modulo 8, 16-byte aligned (32 where the values are float)
  const int64_t pitch = a.ld_x & 7;
  const bool shift = (!a.y || (a.ld_y & 7) == pitch) && (!a.r || (a.ld_r & 7) == pitch) && (!a.h || (a.ld_h & 7) == pitch) &&
                     bases % 16 == 0 && ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.r)) % (a.x_type == 2 ? 32 : 16)) == 0 &&
                     (a.y_type != 2 || bases % 32 == 0) && (!gate_vec || reinterpret_cast<uintptr_t>(a.gate) % 16 == 0);
  if (a.x_type == 2) {
    if (a.y_type == 2) return launch_types<float, float>(p, vec, shift, a.num_sms, stream);
    if (a.y_type == kBF16) return launch_types<float, __nv_bfloat16>(p, vec, shift, a.num_sms, stream);
    return launch_types<float, __half>(p, vec, shift, a.num_sms, stream);
  }
  if (a.x_type == kBF16) return launch_types<__nv_bfloat16, __nv_bfloat16>(p, vec, shift, a.num_sms, stream);
  return launch_types<__half, __half>(p, vec, shift, a.num_sms, stream);
}

}  // namespace sfb200
