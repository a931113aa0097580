// Weighted sum of the experts' rows of every token:
//   out[t] = residual[t] + sum_j weights[t, j] * y[slots[t, j]]     (a slot outside 0 .. y_rows-1 adds nothing),
// in 32 bits, in the order of j, rounded once: no atomics, the same bits on every run.
// HBM-bound: top_k + 1 (+ 1) rows of 16-bit values per token.  A thread owns eight columns of a token and has the rows of four
// slots in flight at once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "launch.h"
#include "row_divider.h"
#include "sm100_ptx.cuh"

namespace sfb200 {
namespace {

struct CombineParams {
  const uint16_t* y;
  const int* slots;
  const float* weights;
  const uint16_t* residual;
  uint16_t* out;
  int64_t ld_y, ld_res, ld_out;
  int y_rows, top_k, cols;
  uint32_t pieces, row_pieces;      // of this launch; per token
  RowDivider div;
};

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// V columns per thread: 8 (16-byte accesses) or 1
template <int V>
struct Piece {
  uint32_t w[V == 8 ? 4 : 1];
};
template <int V>
__device__ __forceinline__ Piece<V> load_piece(const uint16_t* p) {
  Piece<V> r;
  if (V == 8) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    r.w[0] = v.x;
    if (V == 8) { r.w[V == 8 ? 1 : 0] = v.y; r.w[V == 8 ? 2 : 0] = v.z; r.w[V == 8 ? 3 : 0] = v.w; }
  } else {
    r.w[0] = *p;
  }
  return r;
}

template <bool BF16, int V>
__global__ void __launch_bounds__(256) combine_kernel(const CombineParams p) {
  constexpr int W = V == 8 ? 4 : 1;
  dependency_wait();
  dependency_trigger();
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= p.pieces) return;
  const uint32_t t = static_cast<uint32_t>(i * p.div.mul >> p.div.shift);
  const int c = static_cast<int>(i - t * p.row_pieces) * V;
  float2 acc[W];
#pragma unroll
  for (int w = 0; w < W; ++w) acc[w] = make_float2(0.f, 0.f);
  const int* slots = p.slots + static_cast<size_t>(t) * p.top_k;
  const float* weights = p.weights + static_cast<size_t>(t) * p.top_k;
  Piece<V> res{};
  if (p.residual != nullptr) res = load_piece<V>(p.residual + t * p.ld_res + c);
  for (int j0 = 0; j0 < p.top_k; j0 += 4) {
    Piece<V> v[4];
    float f[4];
    bool some[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int s = j0 + j < p.top_k ? slots[j0 + j] : -1;
      some[j] = s >= 0 && s < p.y_rows;
      if (some[j]) {
        v[j] = load_piece<V>(p.y + s * p.ld_y + c);
        f[j] = weights[j0 + j];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (some[j]) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float2 u = unpack2<BF16>(v[j].w[w]);
          acc[w].x = fmaf(f[j], u.x, acc[w].x);
          acc[w].y = fmaf(f[j], u.y, acc[w].y);
        }
      }
  }
  if (p.residual != nullptr) {
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float2 u = unpack2<BF16>(res.w[w]);
      acc[w].x += u.x;
      acc[w].y += u.y;
    }
  }
  uint16_t* out = p.out + t * p.ld_out + c;
  if (V == 8) {
    *reinterpret_cast<uint4*>(out) = make_uint4(pack2<BF16>(acc[0].x, acc[0].y), pack2<BF16>(acc[W > 1 ? 1 : 0].x, acc[W > 1 ? 1 : 0].y),
                                                pack2<BF16>(acc[W > 2 ? 2 : 0].x, acc[W > 2 ? 2 : 0].y),
                                                pack2<BF16>(acc[W > 3 ? 3 : 0].x, acc[W > 3 ? 3 : 0].y));
  } else {
    *out = static_cast<uint16_t>(pack2<BF16>(acc[0].x, 0.f));
  }
}

}  // namespace

int launch_moe_combine(const CombineArgs& a, cudaStream_t stream) {
  if (a.tokens < 0 || a.cols < 1 || a.top_k < 1 || a.y_rows < 0) return kErrInvalid;
  if (a.fmt != kF16 && a.fmt != kBF16) return kErrInvalid;
  if (a.tokens == 0) return kOk;
  if (!a.slots || !a.weights || !a.out || (!a.y && a.y_rows > 0)) return kErrInvalid;
  if (a.ld_y < a.cols || a.ld_out < a.cols || (a.residual && a.ld_res < a.cols)) return kErrInvalid;
  const bool vec = a.cols % 8 == 0 && a.ld_y % 8 == 0 && a.ld_out % 8 == 0 && (!a.residual || a.ld_res % 8 == 0) &&
                   ((reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.residual)) & 15) == 0;
  CombineParams p{};
  p.y = static_cast<const uint16_t*>(a.y);
  p.ld_y = a.ld_y;
  p.ld_res = a.ld_res;
  p.ld_out = a.ld_out;
  p.y_rows = a.y_rows;
  p.top_k = a.top_k;
  p.cols = a.cols;
  p.row_pieces = static_cast<uint32_t>(vec ? a.cols / 8 : a.cols);
  if (p.row_pieces > (1u << 28)) return kErrInvalid;
  p.div = row_divider(p.row_pieces);
  const int most = static_cast<int>(((1ull << 31) - 1) / p.row_pieces);      // tokens of a launch
  for (int t0 = 0, n; t0 < a.tokens; t0 += n) {
    n = a.tokens - t0 < most ? a.tokens - t0 : most;
    p.slots = a.slots + static_cast<size_t>(t0) * a.top_k;
    p.weights = a.weights + static_cast<size_t>(t0) * a.top_k;
    p.residual = a.residual ? static_cast<const uint16_t*>(a.residual) + t0 * a.ld_res : nullptr;
    p.out = static_cast<uint16_t*>(a.out) + t0 * a.ld_out;
    p.pieces = static_cast<uint32_t>(n) * p.row_pieces;
    const int grid = static_cast<int>((p.pieces + 255) / 256);
    auto kernel = vec ? (a.fmt == kBF16 ? combine_kernel<true, 8> : combine_kernel<false, 8>)
                      : (a.fmt == kBF16 ? combine_kernel<true, 1> : combine_kernel<false, 1>);
    const int rc = launch_dependent(kernel, grid, 256, 0, 0, stream, p);
    if (rc != kOk) return rc;
  }
  return kOk;
}

}  // namespace sfb200
