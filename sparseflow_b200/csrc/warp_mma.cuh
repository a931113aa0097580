// Warp-level matrix products m16n8k16 / m16n8k8 of 16-bit operands with 32-bit sums, and the splitting of a 32-bit value into two
// 16-bit ones.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace sfb200 {

template <bool BF16>
__device__ __forceinline__ void mma_k16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool BF16>
__device__ __forceinline__ float2 unpack16x2(uint32_t v) {
  if (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16x2(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// (a, b) = hi + lo: hi the nearest 16-bit values, lo those of what is left (nothing where hi is infinite)
template <bool BF16>
__device__ __forceinline__ void split16x2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack16x2<BF16>(a, b);
  const float2 h = unpack16x2<BF16>(hi);
  lo = pack16x2<BF16>(isinf(h.x) ? 0.f : a - h.x, isinf(h.y) ? 0.f : b - h.y);
}

}  // namespace sfb200
