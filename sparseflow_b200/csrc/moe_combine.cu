// Weighted sum of the experts' rows of every token:
//   out[t] = residual[t] + sum_j weights[t, j] * y[slots[t, j]]     (a slot outside 0 .. y_rows-1 adds nothing),
// in 32 bits, in the order of j, rounded once: no atomics, the same bits on every run.
// HBM-bound: top_k + 1 (+ 1) rows of 16-bit values per token.  A thread owns a 16-byte piece of the result and has the rows of four
// slots in flight at once.  Rows that begin inside a piece (odd widths) are read as the two pieces that hold the eight values, shifted
// into place; at the ends of a row, value by value.  Measured: 4096 tokens, 8 rows of
// 2048 and a residual 29.6 us (5.6 TB/s); 2000 tokens, 8 rows of 8191 101 us, value by value it was 138 us.
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
  int64_t y_size, res_size;         // elements from the base to the end
  int64_t y_at, res_at, out_at;     // the first element's place: the tensor's offset in its 16 bytes and this launch's first token
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

struct Piece {
  uint32_t w[4];
};
// Eight values from element `at` of a 16-byte aligned tensor of `size` elements; those of columns outside 0 .. cols-1 are not read (zero).
// SHIFT = false: whole pieces.
template <bool SHIFT>
__device__ __forceinline__ Piece load_piece(const uint16_t* base, int64_t at, int64_t size, int c, int cols) {
  Piece r;
  if (!SHIFT) {
    const uint4 v = *reinterpret_cast<const uint4*>(base + at);
    r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
    return r;
  }
  const int d = static_cast<int>(at & 7);
  const int64_t first = at - d;
  if (first >= 0 && first + (d ? 16 : 8) <= size) {
    const uint4 a = *reinterpret_cast<const uint4*>(base + first);
    uint4 b = make_uint4(0, 0, 0, 0);
    if (d) b = *reinterpret_cast<const uint4*>(base + first + 8);
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (d & 4) {
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (d & 2) {
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = d & 1 ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
    return r;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r.w[i] = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (c + 2 * i + h >= 0 && c + 2 * i + h < cols) r.w[i] |= static_cast<uint32_t>(base[at + 2 * i + h]) << (16 * h);
  }
  return r;
}

template <bool BF16, bool SHIFT>
__global__ void __launch_bounds__(256) combine_kernel(const CombineParams p) {
  dependency_wait();
  dependency_trigger();
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= p.pieces) return;
  const uint32_t t = static_cast<uint32_t>(i * p.div.mul >> p.div.shift);
  const int c = static_cast<int>(i - t * p.row_pieces) * 8 - (SHIFT ? static_cast<int>(t * p.ld_out + p.out_at & 7) : 0);
  if (SHIFT && c >= p.cols) return;
  float2 acc[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) acc[w] = make_float2(0.f, 0.f);
  const int* slots = p.slots + static_cast<size_t>(t) * p.top_k;
  const float* weights = p.weights + static_cast<size_t>(t) * p.top_k;
  Piece res{};
  if (p.residual != nullptr) res = load_piece<SHIFT>(p.residual, p.res_at + t * p.ld_res + c, p.res_size, c, p.cols);
  for (int j0 = 0; j0 < p.top_k; j0 += 4) {
    Piece v[4];
    float f[4];
    bool some[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int s = j0 + j < p.top_k ? slots[j0 + j] : -1;
      some[j] = s >= 0 && s < p.y_rows;
      if (some[j]) {
        v[j] = load_piece<SHIFT>(p.y, p.y_at + s * p.ld_y + c, p.y_size, c, p.cols);
        f[j] = weights[j0 + j];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (some[j]) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float2 u = unpack2<BF16>(v[j].w[w]);
          acc[w].x = fmaf(f[j], u.x, acc[w].x);
          acc[w].y = fmaf(f[j], u.y, acc[w].y);
        }
      }
  }
  if (p.residual != nullptr) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float2 u = unpack2<BF16>(res.w[w]);
      acc[w].x += u.x;
      acc[w].y += u.y;
    }
  }
  uint16_t* out = p.out + p.out_at + t * p.ld_out + c;
  uint32_t o[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) o[w] = pack2<BF16>(acc[w].x, acc[w].y);
  if (!SHIFT || (c >= 0 && c + 8 <= p.cols)) {
    *reinterpret_cast<uint4*>(out) = make_uint4(o[0], o[1], o[2], o[3]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k >= 0 && c + k < p.cols) out[k] = static_cast<uint16_t>(o[k / 2] >> (16 * (k % 2)));
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
  if ((reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.residual)) & 1) return kErrInvalid;
  CombineParams p{};
  // The kernel counts elements from a 16-byte boundary.  One that lies in front of a tensor's first element is inside the piece that holds it; values
  // of that piece which are not the tensor's are dropped.
  auto place = [](const void* b) { return static_cast<int64_t>(reinterpret_cast<uintptr_t>(b) & 15) / 2; };
  const int64_t y_at = place(a.y), res_at = place(a.residual), out_at = place(a.out);
  p.y = static_cast<const uint16_t*>(a.y) - y_at;
  p.y_at = y_at;
  p.residual = static_cast<const uint16_t*>(a.residual) - (a.residual ? res_at : 0);
  p.out = static_cast<uint16_t*>(a.out) - out_at;
  p.ld_y = a.ld_y;
  p.ld_res = a.ld_res;
  p.ld_out = a.ld_out;
  p.y_rows = a.y_rows;
  p.top_k = a.top_k;
  p.cols = a.cols;
  p.y_size = y_at + static_cast<int64_t>(a.y_rows - 1) * a.ld_y + a.cols;
  p.res_size = res_at + static_cast<int64_t>(a.tokens - 1) * a.ld_res + a.cols;
  p.row_pieces = static_cast<uint32_t>((a.cols + (vec ? 7 : 14)) / 8);      // a row may begin at the last value of a piece
  if (p.row_pieces > (1u << 28)) return kErrInvalid;
  p.div = row_divider(p.row_pieces);
  const int most = static_cast<int>(((1ull << 31) - 1) / p.row_pieces);      // tokens of a launch
  for (int t0 = 0, n; t0 < a.tokens; t0 += n) {
    n = a.tokens - t0 < most ? a.tokens - t0 : most;
    p.slots = a.slots + static_cast<size_t>(t0) * a.top_k;
    p.weights = a.weights + static_cast<size_t>(t0) * a.top_k;
    p.res_at = res_at + t0 * a.ld_res;
    p.out_at = out_at + t0 * a.ld_out;
    p.pieces = static_cast<uint32_t>(n) * p.row_pieces;
    const int grid = static_cast<int>((p.pieces + 255) / 256);
    auto kernel = vec ? (a.fmt == kBF16 ? combine_kernel<true, false> : combine_kernel<false, false>)
                      : (a.fmt == kBF16 ? combine_kernel<true, true> : combine_kernel<false, true>);
    const int rc = launch_dependent(kernel, grid, 256, 0, 0, stream, p);
    if (rc != kOk) return rc;
  }
  return kOk;
}

}  // namespace sfb200
