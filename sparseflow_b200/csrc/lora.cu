// Low-rank adapters of many requests at once:  out[t] = y[t] + s_g * (x[t] . A_g^T) . B_g^T   for every row t of group g
// (A_g [r, K], B_g [N, r]); a row of no group keeps y[t].  The rows of a group are listed by the grouping (moe_route.cu), so one
// launch serves any mix of adapters.
//
// Two launches.  lora_down: u = s_g * x . A_g^T, [place in the grouping, r], 32-bit, K split over the warps of a block and summed in
// shared memory in a fixed order.  lora_up: out = y + u . B_g^T.  Both run on warp-level matrix instructions with fragments loaded straight from
// global memory: the order of the summed index is free as long as both operands use the same one, so lane q of a row's four
// lanes takes 8 consecutive values (one 16-byte load), the first four of which stand for k = 2q, 2q+1, 2q+8, 2q+9 of one
// instruction and the other four of the next; the columns of B_g are dealt the same way, so that a lane ends up with eight consecutive
// outputs of a row.
//
// Rounding: u is needed as a 16-bit operand; a single rounding of it would put an error of half a step of the 16-bit type on the added
// term, so it enters as hi + lo (two instructions; what is lost is a quarter step squared).  f16: the row of u is scaled by
// a power of two so that its largest magnitude is in [1, 2), and the sum is scaled back, so no u over- or underflows.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "launch.h"
#include "sm100_ptx.cuh"
#include "warp_mma.cuh"

namespace sfb200 {
namespace {

struct LoraParams {
  const uint16_t *y, *x, *a, *b;
  const float* scales;      // [groups]
  uint16_t* out;
  const int *offsets, *rows, *slots;
  float* u;                 // [n, r]
  int64_t ld_y, ld_x, ld_out;
  int n, groups, K, N, tile, tiles, copy_blocks;      // n: rows; tile: rows per tile; tiles: upper bound of their number
};

// Tile number -> its group and rows [first, first + count); false: no such tile.  Executed by whole warps.
__device__ bool find_tile(const LoraParams& p, int tile, int& group, int& first, int& count) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int g0 = 0; g0 < p.groups; g0 += 32) {
    const int g = g0 + lane;
    int begin = 0, size = 0;
    if (g < p.groups) {
      begin = p.offsets[g];
      size = p.offsets[g + 1] - begin;
    }
    const int own = (size + p.tile - 1) / p.tile;
    int end = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, end, d);
      if (lane >= d) end += v;
    }
    end += before;
    const unsigned hit = __ballot_sync(0xffffffffu, tile < end);
    if (hit) {
      const int l = __ffs(hit) - 1;
      const int start = __shfl_sync(0xffffffffu, end - own, l);
      begin = __shfl_sync(0xffffffffu, begin, l);
      size = __shfl_sync(0xffffffffu, size, l);
      const int at = (tile - start) * p.tile;
      group = g0 + l;
      first = begin + at;
      count = size - at < p.tile ? size - at : p.tile;
      return true;
    }
    before = __shfl_sync(0xffffffffu, end, 31);
  }
  return false;
}

__device__ __forceinline__ uint4 load16(const uint16_t* p, bool ok) {
  return ok ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
}

constexpr int kDownWarps = 8;

// MF: 16-row fragments of a tile; NF: 8-column fragments of the rank
template <bool BF16, int MF, int NF>
__global__ void __launch_bounds__(kDownWarps * 32) lora_down_kernel(const LoraParams p) {
  extern __shared__ float red[];      // [warps][16 * MF][8 * NF]
  dependency_wait();
  dependency_trigger();
  int group, first, count;
  if (!find_tile(p, blockIdx.x, group, first, count)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  constexpr int R = 8 * NF;
  const uint16_t* xr[MF][2];
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = m * 16 + h * 8 + g;
      xr[m][h] = p.x + p.rows[first + (i < count ? i : 0)] * p.ld_x + 8 * q;      // rows behind the tile: its first row, not stored
    }
  const uint16_t* ar = p.a + (static_cast<size_t>(group) * R + g) * p.K + 8 * q;
  float acc[MF][NF][4];
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][f][i] = 0.f;
#pragma unroll 2
  for (int k0 = warp * 32; k0 < p.K; k0 += kDownWarps * 32) {
    const bool ok = k0 + 8 * q < p.K;
    uint4 xv[MF][2], av[NF];
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      xv[m][0] = load16(xr[m][0] + k0, ok);
      xv[m][1] = load16(xr[m][1] + k0, ok);
    }
#pragma unroll
    for (int f = 0; f < NF; ++f) av[f] = load16(ar + static_cast<size_t>(8 * f) * p.K + k0, ok);
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int m = 0; m < MF; ++m) {
        mma_k16<BF16>(acc[m][f], xv[m][0].x, xv[m][1].x, xv[m][0].y, xv[m][1].y, av[f].x, av[f].y);
        mma_k16<BF16>(acc[m][f], xv[m][0].z, xv[m][1].z, xv[m][0].w, xv[m][1].w, av[f].z, av[f].w);
      }
  }
  float* mine = red + warp * (16 * MF * R);
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float2*>(mine + (m * 16 + h * 8 + g) * R + 8 * f + 2 * q) = make_float2(acc[m][f][2 * h], acc[m][f][2 * h + 1]);
  __syncthreads();
  const float s = p.scales[group];
  for (int i = threadIdx.x; i < count * R; i += kDownWarps * 32) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kDownWarps; ++w) v += red[w * (16 * MF * R) + i];
    p.u[static_cast<size_t>(first) * R + i] = v * s;
  }
}

// Rows of no group, by copy: blocks behind the tiles, one row per warp and step.
__device__ void copy_rows(const LoraParams& p, int block) {
  if (p.out == p.y) return;
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  for (int t = block * warps + (threadIdx.x >> 5); t < p.n; t += p.copy_blocks * warps) {
    if (p.slots[t] >= 0) continue;
    for (int c = lane * 8; c < p.N; c += 256)
      *reinterpret_cast<uint4*>(p.out + t * p.ld_out + c) = *reinterpret_cast<const uint4*>(p.y + t * p.ld_y + c);
  }
}

// Eight (R >= 32), four (16) or two (8) values of the rank per lane and step, as the operand of MMA k-steps.
template <int R>
struct RankStep {
  static constexpr int LANE = R >= 32 ? 8 : R / 4;      // values per lane and chunk
  static constexpr int CHUNK = 4 * LANE;                // rank values per chunk: 32, 16 or 8
  static constexpr int CHUNKS = R / CHUNK;
  static constexpr int WORDS = LANE / 2;
};

constexpr int kUpWarps = 4;

// ROW_WARPS warps take 16 rows each (tile = 16 * ROW_WARPS), the others further columns; COLS columns per block.
template <bool BF16, int NF, int ROW_WARPS>
__global__ void __launch_bounds__(kUpWarps * 32) lora_up_kernel(const LoraParams p, int cols_per_block) {
  constexpr int R = 8 * NF;
  using S = RankStep<R>;
  dependency_wait();
  dependency_trigger();
  if (static_cast<int>(blockIdx.y) >= p.tiles) {
    copy_rows(p, (blockIdx.y - p.tiles) * gridDim.x + blockIdx.x);
    return;
  }
  int group, first, count;
  if (!find_tile(p, blockIdx.y, group, first, count)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int rw = warp % ROW_WARPS, cw = warp / ROW_WARPS;
  constexpr int COL_WARPS = kUpWarps / ROW_WARPS;
  const int i0 = rw * 16 + g, i1 = i0 + 8;
  if (rw * 16 >= count) return;
  // the rows' u as operand words, hi and lo, of rows i0 and i1
  uint32_t hi[2][S::CHUNKS][S::WORDS], lo[2][S::CHUNKS][S::WORDS];
  float back[2] = {1.f, 1.f};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = h ? i1 : i0;
    float v[S::CHUNKS][S::LANE];
    float most = 0.f;
#pragma unroll
    for (int c = 0; c < S::CHUNKS; ++c)
#pragma unroll
      for (int j = 0; j < S::LANE; j += 2) {
        const float2 w = i < count ? *reinterpret_cast<const float2*>(p.u + static_cast<size_t>(first + i) * R + c * S::CHUNK + q * S::LANE + j)
                                   : make_float2(0.f, 0.f);
        v[c][j] = w.x;
        v[c][j + 1] = w.y;
        most = fmaxf(most, fmaxf(fabsf(w.x), fabsf(w.y)));
      }
    float to = 1.f;
    if (!BF16) {
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int e = static_cast<int>(__float_as_uint(most) >> 23);      // 0 for zero and subnormal, 255 for inf and NaN
      if (e >= 2 && e <= 252) {
        back[h] = __uint_as_float(static_cast<uint32_t>(e) << 23);
        to = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
      }
    }
#pragma unroll
    for (int c = 0; c < S::CHUNKS; ++c)
#pragma unroll
      for (int j = 0; j < S::WORDS; ++j) split16x2<BF16>(v[c][2 * j] * to, v[c][2 * j + 1] * to, hi[h][c][j], lo[h][c][j]);
  }
  const int64_t row0 = i0 < count ? p.rows[first + i0] : -1, row1 = i1 < count ? p.rows[first + i1] : -1;
  const int col_end = min(p.N, static_cast<int>(blockIdx.x + 1) * cols_per_block);
  for (int c0 = blockIdx.x * cols_per_block + cw * 32; c0 < col_end; c0 += COL_WARPS * 32) {
    // this lane's eight output columns: c0 + 8q ..; fragment f holds columns 8q' + 2f, +1 of lane q', so row n = 2q' + i of
    // the operand is column 8 * (n / 2) + 2f + n % 2
    const int col = c0 + 8 * q;
    const bool in = col < p.N;
    const uint4 y0 = load16(p.y + row0 * p.ld_y + col, in && row0 >= 0), y1 = load16(p.y + row1 * p.ld_y + col, in && row1 >= 0);
    float acc[4][4];
#pragma unroll
    for (int f = 0; f < 4; ++f) {
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[f][i] = 0.f;
      const int bc = c0 + 8 * (g >> 1) + 2 * f + (g & 1);
      const bool ok = bc < p.N;
      const uint16_t* br = p.b + (static_cast<size_t>(group) * p.N + (ok ? bc : 0)) * R + q * S::LANE;
#pragma unroll
      for (int c = 0; c < S::CHUNKS; ++c) {
        uint32_t w[4] = {0, 0, 0, 0};
        const uint16_t* src = br + c * S::CHUNK;
        if (ok) {
          if (S::LANE == 8) {
            const uint4 v = *reinterpret_cast<const uint4*>(src);
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
          } else if (S::LANE == 4) {
            const uint2 v = *reinterpret_cast<const uint2*>(src);
            w[0] = v.x; w[1] = v.y;
          } else {
            w[0] = *reinterpret_cast<const uint32_t*>(src);
          }
        }
#pragma unroll
        for (int j = 0; j < S::WORDS; j += 2) {
          const bool two = j + 1 < S::WORDS;      // R = 8: the upper half of the instruction's k is zero
          const int j1 = two ? j + 1 : j;
          mma_k16<BF16>(acc[f], hi[0][c][j], hi[1][c][j], two ? hi[0][c][j1] : 0u, two ? hi[1][c][j1] : 0u, w[j], two ? w[j1] : 0u);
          mma_k16<BF16>(acc[f], lo[0][c][j], lo[1][c][j], two ? lo[0][c][j1] : 0u, two ? lo[1][c][j1] : 0u, w[j], two ? w[j1] : 0u);
        }
      }
    }
    if (!in) continue;
    auto emit = [&](int64_t row, const uint4& yv, int h) {
      if (row < 0) return;
      const uint32_t yw[4] = {yv.x, yv.y, yv.z, yv.w};
      uint32_t o[4];
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const float2 v = unpack16x2<BF16>(yw[f]);
        o[f] = pack16x2<BF16>(fmaf(acc[f][2 * h], back[h], v.x), fmaf(acc[f][2 * h + 1], back[h], v.y));
      }
      *reinterpret_cast<uint4*>(p.out + row * p.ld_out + col) = make_uint4(o[0], o[1], o[2], o[3]);
    };
    emit(row0, y0, 0);
    emit(row1, y1, 1);
  }
}

template <bool BF16, int MF, int NF>
int launch_down(const LoraParams& p, cudaStream_t stream) {
  constexpr int smem = kDownWarps * 16 * MF * 8 * NF * 4;
  if (smem > 48 * 1024) {
    static bool set[16] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 16 || !set[dev]) {
      if (cudaFuncSetAttribute(lora_down_kernel<BF16, MF, NF>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return kErrCuda;
      if (dev < 16) set[dev] = true;
    }
  }
  return launch_dependent(lora_down_kernel<BF16, MF, NF>, p.tiles, kDownWarps * 32, smem, 0, stream, p);
}

template <bool BF16, int NF>
int launch_rank(LoraParams p, cudaStream_t stream) {
  auto set_tile = [&](int tile) {
    p.tile = tile;
    p.tiles = (p.n + tile - 1) / tile + (p.groups < p.n ? p.groups : p.n);
  };
  // few rows: 16-row tiles
  const bool small = p.n <= 512;
  set_tile(small ? 16 : 32);
  int rc = small ? launch_down<BF16, 1, NF>(p, stream) : launch_down<BF16, 2, NF>(p, stream);
  if (rc != kOk) return rc;
  set_tile(small ? 16 : 64);
  if (p.tiles > 65000) return kErrInvalid;
  const int cols = small ? 256 : 128, gx = (p.N + cols - 1) / cols;
  p.copy_blocks = p.out == p.y ? 0 : gx * (small ? 1 : 2);
  const dim3 grid(gx, p.tiles + p.copy_blocks / gx, 1);
  if (small) return launch_dependent(lora_up_kernel<BF16, NF, 1>, grid, kUpWarps * 32, 0, 0, stream, p, cols);
  return launch_dependent(lora_up_kernel<BF16, NF, 4>, grid, kUpWarps * 32, 0, 0, stream, p, cols);
}

template <bool BF16>
int launch_type(const LoraParams& p, int rank, cudaStream_t stream) {
  switch (rank) {
    case 8: return launch_rank<BF16, 1>(p, stream);
    case 16: return launch_rank<BF16, 2>(p, stream);
    case 32: return launch_rank<BF16, 4>(p, stream);
    case 64: return launch_rank<BF16, 8>(p, stream);
    case 128: return launch_rank<BF16, 16>(p, stream);
    default: return kErrInvalid;
  }
}

}  // namespace

int launch_lora_add(const LoraArgs& a, cudaStream_t stream) {
  if (a.n < 0 || a.groups < 1 || a.groups > 1024 || a.K < 8 || a.K % 8 != 0 || a.N < 8 || a.N % 8 != 0) return kErrInvalid;
  if (a.fmt != kF16 && a.fmt != kBF16) return kErrInvalid;
  if (a.n == 0) return kOk;
  if (!a.y || !a.x || !a.a || !a.b || !a.scales || !a.out || !a.offsets || !a.rows || !a.slots || !a.workspace) return kErrInvalid;
  if (a.ld_x < a.K || a.ld_y < a.N || a.ld_out < a.N || (a.ld_x | a.ld_y | a.ld_out) % 8 != 0) return kErrInvalid;
  if ((reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.a) | reinterpret_cast<uintptr_t>(a.b) |
       reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.workspace)) & 15)
    return kErrInvalid;
  LoraParams p{};
  p.y = static_cast<const uint16_t*>(a.y);
  p.x = static_cast<const uint16_t*>(a.x);
  p.a = static_cast<const uint16_t*>(a.a);
  p.b = static_cast<const uint16_t*>(a.b);
  p.scales = a.scales;
  p.out = static_cast<uint16_t*>(a.out);
  p.offsets = a.offsets;
  p.rows = a.rows;
  p.slots = a.slots;
  p.u = static_cast<float*>(a.workspace);
  p.ld_y = a.ld_y;
  p.ld_x = a.ld_x;
  p.ld_out = a.ld_out;
  p.n = a.n;
  p.groups = a.groups;
  p.K = a.K;
  p.N = a.N;
  return a.fmt == kBF16 ? launch_type<true>(p, a.rank, stream) : launch_type<false>(p, a.rank, stream);
}

}  // namespace sfb200
