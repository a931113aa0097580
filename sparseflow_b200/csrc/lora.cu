// Low-rank adapters of many requests at once:  out[t] = y[t] + s_g * (x[t] . A_g^T) . B_g^T   for every row t of group g
// (A_g [r, K], B_g [N, r]); a row of no group keeps y[t].  The rows of a group are listed by the grouping (moe_route.cu), so one
// launch serves any mix of adapters.
//
// Two launches.  lora_down: u = s_g * x . A_g^T in 32 bits, K cut over a cluster of blocks whose partial sums are added, in order, through
// distributed shared memory; u is left as the operand of the second product.  lora_up: out = y + u . B_g^T.  The work is bytes (x, y,
// out once: 7.9 GFLOP on 229 MB at 4097 rows, 4096 -> 64 -> 11008), so what counts is loads in flight and few re-reads of the adapters:
//   * many rows per adapter: tiles of 128 rows; lora_down streams x and A_g through a ring of four 64-wide stages in shared memory,
//     lora_up (128 rows, 64 from rank 64) y and B_g through a ring of four 32-column stages, the rows' u staying in registers;
//   * few rows per adapter: tiles of 16 rows, operands straight from global memory.  The order of the summed index is free as long as both
//     operands use the same one, so lane q of a row's four lanes takes 8 consecutive values (one 16-byte load), the first four
//     of which stand for k = 2q, 2q+1, 2q+8, 2q+9 of one instruction and the other four of the next.
// lora_up deals the columns of B_g the same way, so that a lane ends up with eight consecutive outputs of a row, and begins to read everything but
// u before it waits for lora_down: all of that was complete before lora_down began (launch.h).
//
// Measured: 48 rows, 48 of 64 adapters, rank 16, 4096 -> 4096 8.0 us replayed (latency: two launches); 4097 rows, 8 adapters, rank 64,
// 4096 -> 11008 68-70 us among other calls, 76 replayed in a row (lora_down 18, lora_up 46 when profiled one by one: tensor pipe 20 and 42 % of cycles, DRAM 21 and 38 %: latency of the loads
// in front of each tile, and the issue of hi and lo products, about 14 us).
//
// Tiles of 128 or 16 rows are chosen by the rows per resident adapter, not per used one: the host does not know which are used.  A long prompt of one
// request beside a bank of many runs the 16-row form, which reads its adapter once per 16 rows.
//
// Rounding: u is needed as a 16-bit operand; a single rounding of it would put an error of half a step of the 16-bit type on the added
// term, so it enters as hi + lo (two instructions; what is lost is a quarter step squared).  f16: the row of u is scaled by
// a power of two so that its largest magnitude is in [1, 2), and the sum is scaled back, so no u over- or underflows.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "device_state.h"
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
  uint32_t *hi, *lo;        // u as 16-bit pairs, [n, r / 2] each
  float* back;              // [n]: what the sums of a row of u are multiplied with
  int64_t ld_y, ld_x, ld_out;
  int n, groups, K, N, tile, tiles, copy_blocks;      // n: rows; tile: rows per tile; tiles: upper bound of their number
  int splits, slice;                                  // slices of K (blocks of a cluster), of `slice` values
  int tiles_first;                                    // lora_up's grid: tiles along x, columns along y (more tiles than y takes)
};

// Tile number -> its group and rows [first, first + count); false: no such tile (and first = number of tiles).  Executed by whole warps.
// Held inside 0 .. n whatever is in memory.
__device__ bool find_tile(const LoraParams& p, int tile, int& group, int& first, int& count) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int g0 = 0; g0 < p.groups; g0 += 32) {
    const int g = g0 + lane;
    int begin = 0, size = 0;
    if (g < p.groups) {
      begin = min(max(p.offsets[g], 0), p.n);
      size = min(max(p.offsets[g + 1], begin), p.n) - begin;
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
  first = before;
  return false;
}

// Row of a place for reading x; one that is no row of the batch (no grouping makes such) reads another and is not stored.
__device__ __forceinline__ int row_read(const LoraParams& p, int place) { return min(max(p.rows[place], 0), p.n - 1); }
// Row of a place for y and out, -1 for none.
__device__ __forceinline__ int row_written(const LoraParams& p, int place) {
  const int row = p.rows[place];
  return row < p.n ? row : -1;
}

__device__ __forceinline__ uint4 load16(const uint16_t* p, bool ok) {
  return ok ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ float2 load_cluster_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// The blocks of a cluster hold partial sums part[rows][R] of the same `count` rows in shared memory; each block finishes its share of the rows: the
// sum over the blocks in order, scaled, as hi and lo operand words.
template <bool BF16, int R>
__device__ void finish_rows(const LoraParams& p, const float* part, int first, int count, float scale, int threads) {
  constexpr int TPR = R / 2 < 32 ? R / 2 : 32, PAIRS = R / 2 / TPR;      // threads per row; pairs per thread
  const int rank = blockIdx.x % p.splits, each = (count + p.splits - 1) / p.splits;
  const int begin = rank * each, end = min(count, begin + each);
  const uint32_t base = smem_u32(part);
  cluster_sync_all();
  for (int r0 = begin; r0 < end; r0 += threads / TPR) {
    const int row = r0 + threadIdx.x / TPR, l = threadIdx.x % TPR;
    const bool in = row < end;
    float2 v[PAIRS];
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      v[i] = make_float2(0.f, 0.f);
      if (in)
        for (int src = 0; src < p.splits; ++src) {
          const float2 w = load_cluster_f2(mapa_u32(base + (row * R + 2 * (l + i * TPR)) * 4, src));
          v[i].x += w.x;
          v[i].y += w.y;
        }
      v[i].x *= scale;
      v[i].y *= scale;
      most = fmaxf(most, fmaxf(fabsf(v[i].x), fabsf(v[i].y)));
    }
    float to = 1.f, back = 1.f;
    if (!BF16) {
#pragma unroll
      for (int d = TPR / 2; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
      const int e = static_cast<int>(__float_as_uint(most) >> 23);      // 0 for zero and subnormal, 255 for inf and NaN
      if (e >= 2 && e <= 252) {
        back = __uint_as_float(static_cast<uint32_t>(e) << 23);
        to = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
      }
    }
    if (in) {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        uint32_t hi, lo;
        split16x2<BF16>(v[i].x * to, v[i].y * to, hi, lo);
        const size_t at = static_cast<size_t>(first + row) * (R / 2) + l + i * TPR;
        p.hi[at] = hi;
        p.lo[at] = lo;
      }
      if (l == 0) p.back[first + row] = back;
    }
  }
  cluster_sync_all();      // no block leaves while another reads its partial sums
}

constexpr int kDownWarps = 8;

// MF: 16-row fragments of a tile; NF: 8-column fragments of the rank
template <bool BF16, int MF, int NF>
__global__ void __launch_bounds__(kDownWarps * 32) lora_down_kernel(const LoraParams p) {
  extern __shared__ __align__(16) float red[];      // [warps][16 * MF][8 * NF]
  dependency_wait();
  dependency_trigger();
  int group, first, count;
  if (!find_tile(p, blockIdx.x / p.splits, group, first, count)) return;      // the same for all blocks of a cluster
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  constexpr int R = 8 * NF;
  const uint16_t* xr[MF][2];
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = m * 16 + h * 8 + g;
      xr[m][h] = p.x + row_read(p, first + (i < count ? i : 0)) * p.ld_x + 8 * q;      // rows behind the tile: its first row, not stored
    }
  const uint16_t* ar = p.a + (static_cast<size_t>(group) * R + g) * p.K + 8 * q;
  float acc[MF][NF][4];
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][f][i] = 0.f;
  const int k_begin = static_cast<int>(blockIdx.x % p.splits) * p.slice, k_end = min(p.K, k_begin + p.slice);
#pragma unroll 2
  for (int k0 = k_begin + warp * 32; k0 < k_end; k0 += kDownWarps * 32) {
    const bool ok = k0 + 8 * q < k_end;
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
  for (int i = threadIdx.x; i < count * R; i += kDownWarps * 32) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kDownWarps; ++w) v += red[w * (16 * MF * R) + i];
    red[i] = v;      // the first warp's part, read by this thread only
  }
  finish_rows<BF16, R>(p, red, first, count, p.scales[group], kDownWarps * 32);
}

// ---- many rows per adapter: 128 rows x R, K in 64-wide stages through shared memory (rows of 128 bytes, 16-byte pieces exchanged by row % 8)
constexpr int kTileRows = 128, kStageK = 64, kStages = 4;

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

template <bool BF16, int NF>
__global__ void __launch_bounds__(256, 2) lora_down_tile_kernel(const LoraParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int R = 8 * NF, RB = R < 16 ? 16 : R;      // rows of the A_g operand in shared memory: whole 16-row reads
  constexpr int STAGE = (kTileRows + RB) * 128;
  dependency_wait();
  dependency_trigger();
  int group, first, count;
  if (!find_tile(p, blockIdx.x / p.splits, group, first, count)) return;      // the same for all blocks of a cluster
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = smem_u32(smem);
  const int k_begin = static_cast<int>(blockIdx.x % p.splits) * p.slice, k_end = min(p.K, k_begin + p.slice);
  const int stages = (k_end - k_begin + kStageK - 1) / kStageK;
  // thread: 16-byte piece i % 8 of rows i / 8 + 32 j
  const int piece = threadIdx.x & 7, r0 = threadIdx.x >> 3;
  const uint16_t* xr[kTileRows / 32];
#pragma unroll
  for (int j = 0; j < kTileRows / 32; ++j) {
    const int i = r0 + 32 * j;
    xr[j] = p.x + row_read(p, first + (i < count ? i : 0)) * p.ld_x + 8 * piece;      // rows behind the tile: its first row, not stored
  }
  const uint16_t* ar = p.a + (static_cast<size_t>(group) * R + r0) * p.K + 8 * piece;
  const uint32_t dst = r0 * 128 + ((piece ^ (r0 & 7)) << 4);
  auto fetch = [&](int st) {
    if (st < stages) {
      const int k = k_begin + st * kStageK;
      const bool ok = k + 8 * piece < k_end;
      const int at = ok ? k : 0;
      const uint32_t to = base + (st % kStages) * STAGE + dst;
#pragma unroll
      for (int j = 0; j < kTileRows / 32; ++j) copy16(to + j * 32 * 128, xr[j] + at, ok);
#pragma unroll
      for (int j = 0; j < (RB + 31) / 32; ++j)
        if (r0 + 32 * j < RB) copy16(to + (kTileRows + 32 * j) * 128, r0 + 32 * j < R ? ar + static_cast<size_t>(32 * j) * p.K + at : p.a, ok && r0 + 32 * j < R);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  float acc[NF][4];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[f][i] = 0.f;
#pragma unroll
  for (int st = 0; st < kStages - 1; ++st) fetch(st);
  // ldmatrix row of this lane: x rows warp * 16 + lane % 16, k half lane / 16; A_g rows (lane % 8) + 8 * (lane / 16), k half (lane / 8) % 2
  const int am = warp * 16 + (lane & 15), bn = (lane & 7) + 8 * (lane >> 4);
  const int ak = lane >> 4, bk = (lane >> 3) & 1;
  for (int st = 0; st < stages; ++st) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncthreads();
    fetch(st + kStages - 1);
    const uint32_t xs = base + (st % kStages) * STAGE, as = xs + kTileRows * 128;
#pragma unroll
    for (int kk = 0; kk < kStageK / 16; ++kk) {
      uint32_t xa[4];
      load_matrices(xa, xs + am * 128 + (((2 * kk + ak) ^ (am & 7)) << 4));
#pragma unroll
      for (int f = 0; f < (NF + 1) / 2; ++f) {
        uint32_t b[4];
        const int row = 16 * f + bn;
        load_matrices(b, as + row * 128 + (((2 * kk + bk) ^ (row & 7)) << 4));
        mma_k16<BF16>(acc[2 * f], xa[0], xa[1], xa[2], xa[3], b[0], b[1]);
        if (2 * f + 1 < NF) mma_k16<BF16>(acc[2 * f + 1 < NF ? 2 * f + 1 : 0], xa[0], xa[1], xa[2], xa[3], b[2], b[3]);
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();      // the ring becomes the partial sums
  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = warp * 16 + h * 8 + (lane >> 2);
#pragma unroll
    for (int f = 0; f < NF; ++f) *reinterpret_cast<float2*>(part + i * R + 8 * f + 2 * (lane & 3)) = make_float2(acc[f][2 * h], acc[f][2 * h + 1]);
  }
  finish_rows<BF16, R>(p, part, first, count, p.scales[group], 256);
}

// Rows of no group, by copy: blocks behind the tiles, 32 rows of the block's columns each, a warp eight rows, all its loads first.
__device__ void copy_rows(const LoraParams& p, int block, int c_begin, int c_end) {
  const int lane = threadIdx.x & 31, t0 = block * 32 + (threadIdx.x >> 5) * 8;
  bool none[8];
  unsigned any = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    none[i] = t0 + i < p.n && p.slots[t0 + i < p.n ? t0 + i : 0] < 0;
    any |= none[i];
  }
  if (!any) return;
  for (int c = c_begin + lane * 8; c < c_end; c += 256) {
    uint4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = load16(p.y + (t0 + i) * p.ld_y + c, none[i]);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (none[i]) *reinterpret_cast<uint4*>(p.out + (t0 + i) * p.ld_out + c) = v[i];
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

constexpr int kUpWarps = 4, kUpCols = 32, kUpStages = 4;

// The u of a row (place in the grouping) as operand words of this lane.
template <int R>
__device__ __forceinline__ void load_u(const uint32_t* words, int64_t place, bool ok, uint32_t (&w)[RankStep<R>::CHUNKS][RankStep<R>::WORDS]) {
  using S = RankStep<R>;
  const uint32_t* src = words + place * (R / 2) + (threadIdx.x & 3) * S::WORDS;
#pragma unroll
  for (int c = 0; c < S::CHUNKS; ++c, src += S::CHUNK / 2) {
    if (S::WORDS == 4) {
      const uint4 v = ok ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
      w[c][0] = v.x; w[c][1 % S::WORDS] = v.y; w[c][2 % S::WORDS] = v.z; w[c][3 % S::WORDS] = v.w;
    } else if (S::WORDS == 2) {
      const uint2 v = ok ? *reinterpret_cast<const uint2*>(src) : make_uint2(0, 0);
      w[c][0] = v.x; w[c][1 % S::WORDS] = v.y;
    } else {
      w[c][0] = ok ? *src : 0u;
    }
  }
}
// acc[m][f] += u . B^T of 16 * MF rows x 32 columns over chunk c of the rank, hi then lo; the 4 * MF sums are independent of each other, so
// that the latency of an instruction is covered.  Words j, j + 1 of a chunk are the two halves of an instruction's k (R = 8: the upper half is zero).
template <bool BF16, int R, int MF>
__device__ __forceinline__ void add_products(float (&acc)[MF][4][4], const uint32_t (&hi)[MF][2][RankStep<R>::CHUNKS][RankStep<R>::WORDS],
                                             const uint32_t (&lo)[MF][2][RankStep<R>::CHUNKS][RankStep<R>::WORDS],
                                             const uint32_t (&b)[4][RankStep<R>::WORDS], int c) {
  using S = RankStep<R>;
  constexpr bool two = S::WORDS > 1;
#pragma unroll
  for (int j = 0; j < S::WORDS; j += 2) {
    const int j1 = two ? j + 1 : j;
#pragma unroll
    for (int part = 0; part < 2; ++part)
#pragma unroll
      for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int m = 0; m < MF; ++m) {
          const auto& u = part ? lo[m] : hi[m];
          mma_k16<BF16>(acc[m][f], u[0][c][j], u[1][c][j], two ? u[0][c][j1] : 0u, two ? u[1][c][j1] : 0u, b[f][j], two ? b[f][j1] : 0u);
        }
  }
}
template <bool BF16>
__device__ __forceinline__ uint4 add_to(const uint4& y, const float (&acc)[4][4], int h, float back) {
  const uint32_t yw[4] = {y.x, y.y, y.z, y.w};
  uint32_t w[4];
#pragma unroll
  for (int f = 0; f < 4; ++f) {
    const float2 v = unpack16x2<BF16>(yw[f]);
    w[f] = pack16x2<BF16>(fmaf(acc[f][2 * h], back, v.x), fmaf(acc[f][2 * h + 1], back, v.y));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// A lane's eight output columns of a 32-column step are c0 + 8q ..; fragment f holds columns 8q' + 2f, +1 of lane q', so row n = 2q' + i of the
// operand B is column 8 * (n / 2) + 2f + n % 2.
__device__ __forceinline__ int operand_column(int f) {
  const int g = (threadIdx.x & 31) >> 2;
  return 8 * (g >> 1) + 2 * f + (g & 1);
}

// Few rows per adapter: 16 rows per block, the warps side by side on the columns.
template <bool BF16, int NF>
__global__ void __launch_bounds__(kUpWarps * 32) lora_up_kernel(const LoraParams p, int cols_per_block) {
  constexpr int R = 8 * NF;
  using S = RankStep<R>;
  const int tile = p.tiles_first ? blockIdx.x : blockIdx.y;
  const int c_begin = (p.tiles_first ? blockIdx.y : blockIdx.x) * cols_per_block, c_end = min(p.N, c_begin + cols_per_block);
  if (tile >= p.tiles) {
    dependency_wait();
    dependency_trigger();
    copy_rows(p, tile - p.tiles, c_begin, c_end);
    return;
  }
  int group = 0, first = 0, count = 0;
  if (!find_tile(p, tile, group, first, count)) {
    dependency_wait();
    dependency_trigger();
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  int64_t row[2];      // of y and out; -1 behind the tile
#pragma unroll
  for (int h = 0; h < 2; ++h) row[h] = h * 8 + g < count ? row_written(p, first + h * 8 + g) : -1;
  uint4 yv[2];
  uint32_t bw[S::CHUNKS][4][S::WORDS];
  auto fetch = [&](int c0) {
    const int col = c0 + 8 * q;
#pragma unroll
    for (int h = 0; h < 2; ++h) yv[h] = load16(p.y + row[h] * p.ld_y + col, col < c_end && row[h] >= 0);
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const int bc = c0 + operand_column(f);
      uint32_t w[S::CHUNKS][S::WORDS];
      load_u<R>(reinterpret_cast<const uint32_t*>(p.b), static_cast<int64_t>(group) * p.N + bc, bc < c_end, w);
#pragma unroll
      for (int c = 0; c < S::CHUNKS; ++c)
#pragma unroll
        for (int j = 0; j < S::WORDS; ++j) bw[c][f][j] = w[c][j];
    }
  };
  int c0 = c_begin + warp * 32;
  if (c0 < c_end) fetch(c0);
  dependency_wait();
  dependency_trigger();
  uint32_t hi[1][2][S::CHUNKS][S::WORDS], lo[1][2][S::CHUNKS][S::WORDS];
  float back[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = h * 8 + g;
    load_u<R>(p.hi, first + i, i < count, hi[0][h]);
    load_u<R>(p.lo, first + i, i < count, lo[0][h]);
    back[h] = !BF16 && i < count ? p.back[first + i] : 1.f;
  }
#pragma unroll 1
  for (; c0 < c_end; c0 += kUpWarps * 32) {
    float acc[1][4][4];
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[0][f][i] = 0.f;
#pragma unroll
    for (int c = 0; c < S::CHUNKS; ++c) add_products<BF16, R, 1>(acc, hi, lo, bw[c], c);
    const uint4 o0 = add_to<BF16>(yv[0], acc[0], 0, back[0]), o1 = add_to<BF16>(yv[1], acc[0], 1, back[1]);
    const int col = c0 + 8 * q, next = c0 + kUpWarps * 32;
    if (next < c_end) fetch(next);      // other elements than the ones stored below, also where out is y
    if (col < c_end && row[0] >= 0) *reinterpret_cast<uint4*>(p.out + row[0] * p.ld_out + col) = o0;
    if (col < c_end && row[1] >= 0) *reinterpret_cast<uint4*>(p.out + row[1] * p.ld_out + col) = o1;
  }
}

// Many rows per adapter: tiles of 64 * MF rows, 16 * MF per warp, `cols` columns per block in steps of kUpCols.
template <bool BF16, int NF, int MF>
__global__ void __launch_bounds__(kUpWarps * 32) lora_up_tile_kernel(const LoraParams p, int cols) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int R = 8 * NF, B_BYTES = kUpCols * R * 2, Y_BYTES = kUpWarps * 32 * MF * 2 * 16, STAGE = B_BYTES + Y_BYTES;
  using S = RankStep<R>;
  const int tile = p.tiles_first ? blockIdx.x : blockIdx.y;
  const int c_begin = (p.tiles_first ? blockIdx.y : blockIdx.x) * cols, c_end = min(p.N, c_begin + cols);
  if (tile >= p.tiles) {
    dependency_wait();
    dependency_trigger();
    copy_rows(p, tile - p.tiles, c_begin, c_end);
    return;
  }
  int group = 0, first = 0, count = 0;
  if (!find_tile(p, tile, group, first, count)) {
    dependency_wait();
    dependency_trigger();
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const uint32_t base = smem_u32(smem);
  const int steps = (c_end - c_begin + kUpCols - 1) / kUpCols;
  const uint16_t* y_row[MF][2];      // behind the tile: null
  uint16_t* out_row[MF][2];
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = warp * 16 * MF + m * 16 + h * 8 + g;
      const int64_t row = i < count ? row_written(p, first + i) : -1;
      y_row[m][h] = row >= 0 ? p.y + row * p.ld_y + 8 * q : nullptr;
      out_row[m][h] = p.out + row * p.ld_out + 8 * q;
    }
  // Stage: 32 columns of B_g (rows of R values; from rank 64 the 64-byte halves of odd rows are exchanged, so that eight lanes read
  // eight different banks), then each thread's own pieces of y.
  const uint16_t* b_src = p.b + static_cast<size_t>(group) * p.N * R;
  auto fetch = [&](int st) {
    if (st < steps) {
      const int c0 = c_begin + st * kUpCols;
      const uint32_t to = base + (st % kUpStages) * STAGE;
      constexpr int PIECES = B_BYTES / 16, ROW = R / 8;      // 16-byte pieces of the stage, of a row
#pragma unroll
      for (int j = 0; j < (PIECES + kUpWarps * 32 - 1) / (kUpWarps * 32); ++j) {
        const int i = threadIdx.x + j * kUpWarps * 32, n = i / ROW;
        const int dst = R >= 64 ? i ^ ((n & 1) << 2) : i;
        if (i < PIECES) copy16(to + dst * 16, b_src + (c0 + n < c_end ? static_cast<size_t>(c0) * R + i * 8 : 0), c0 + n < c_end);
      }
#pragma unroll
      for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (c0 + 8 * q < c_end && y_row[m][h] != nullptr) copy16(to + B_BYTES + ((m * 2 + h) * kUpWarps * 32 + threadIdx.x) * 16, y_row[m][h] + c0, true);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int st = 0; st < kUpStages - 1; ++st) fetch(st);
  dependency_wait();
  dependency_trigger();
  uint32_t hi[MF][2][S::CHUNKS][S::WORDS], lo[MF][2][S::CHUNKS][S::WORDS];
  float back[MF][2];
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = warp * 16 * MF + m * 16 + h * 8 + g;
      load_u<R>(p.hi, first + i, i < count, hi[m][h]);
      load_u<R>(p.lo, first + i, i < count, lo[m][h]);
      back[m][h] = !BF16 && i < count ? p.back[first + i] : 1.f;
    }
#pragma unroll 1
  for (int st = 0; st < steps; ++st) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kUpStages - 2) : "memory");
    __syncthreads();
    fetch(st + kUpStages - 1);
    if (warp * 16 * MF >= count) continue;      // a warp behind the tile's rows only copies
    const uint8_t* stage = smem + (st % kUpStages) * STAGE;
    float acc[MF][4][4];
#pragma unroll
    for (int m = 0; m < MF; ++m)
#pragma unroll
      for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][f][i] = 0.f;
#pragma unroll
    for (int c = 0; c < S::CHUNKS; ++c) {
      uint32_t b[4][S::WORDS];
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const int n = operand_column(f);
        const uint8_t* src = stage + n * R * 2 + (R >= 64 ? (((c * 4 + q) ^ ((n & 1) << 2)) << 4) : c * S::CHUNK * 2 + q * S::LANE * 2);
        if (S::WORDS == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(src);
          b[f][0] = v.x; b[f][1 % S::WORDS] = v.y; b[f][2 % S::WORDS] = v.z; b[f][3 % S::WORDS] = v.w;
        } else if (S::WORDS == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(src);
          b[f][0] = v.x; b[f][1 % S::WORDS] = v.y;
        } else {
          b[f][0] = *reinterpret_cast<const uint32_t*>(src);
        }
      }
      add_products<BF16, R, MF>(acc, hi, lo, b, c);
    }
    const int col = c_begin + st * kUpCols;
#pragma unroll
    for (int m = 0; m < MF; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (col + 8 * q < c_end && y_row[m][h] != nullptr) {
          const uint4 y = *reinterpret_cast<const uint4*>(stage + B_BYTES + ((m * 2 + h) * kUpWarps * 32 + threadIdx.x) * 16);
          *reinterpret_cast<uint4*>(out_row[m][h] + col) = add_to<BF16>(y, acc[m], h, back[m][h]);
        }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <class Kernel>
int allow_smem(Kernel kernel, int bytes, bool (&set)[kMaxDevices]) {
  if (bytes <= 48 * 1024) return kOk;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return kErrCuda;
  if (set[dev]) return kOk;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return kErrCuda;
  set[dev] = true;
  return kOk;
}

// Tiles and slices of K.  Many rows per adapter (48 on average): 128-row tiles, K cut into slices of 256 at least; few: 16-row tiles, K cut into slices
// of 512 at least; two, four or eight slices while there are at most eight blocks per SM.
struct LoraPlan {
  bool tiled;
  int tile, tiles, splits, slice;
};
LoraPlan plan_lora(int n, int groups, int K, int num_sms) {
  LoraPlan l;
  l.tiled = n >= 48 * groups;
  l.tile = l.tiled ? kTileRows : 16;
  l.tiles = (n + l.tile - 1) / l.tile + (groups < n ? groups : n);
  const int unit = l.tiled ? 4 * kStageK : 512, units = (K + unit - 1) / unit, want = (l.tiled ? 4 : 8) * num_sms;
  l.splits = 1;
  while (l.splits < (l.tiled ? 4 : 8) && 2 * l.splits <= units && 2 * l.splits * l.tiles <= want) l.splits *= 2;
  l.slice = (units + l.splits - 1) / l.splits * unit;
  return l;
}

template <bool BF16, int NF>
int launch_rank(LoraParams p, int num_sms, cudaStream_t stream) {
  constexpr int R = 8 * NF;
  const LoraPlan l = plan_lora(p.n, p.groups, p.K, num_sms);
  p.tile = l.tile;
  p.tiles = l.tiles;
  p.splits = l.splits;
  p.slice = l.slice;
  int rc;
  if (l.tiled) {
    constexpr int smem = kStages * (kTileRows + (R < 16 ? 16 : R)) * 128;
    static_assert(smem >= kTileRows * R * 4, "the partial sums fit the ring");
    static bool set[kMaxDevices] = {};
    if ((rc = allow_smem(lora_down_tile_kernel<BF16, NF>, smem, set)) != kOk) return rc;
    rc = launch_dependent(lora_down_tile_kernel<BF16, NF>, p.tiles * p.splits, 256, smem, p.splits, stream, p);
  } else {
    constexpr int smem = kDownWarps * 16 * R * 4;
    static bool set[kMaxDevices] = {};
    if ((rc = allow_smem(lora_down_kernel<BF16, 1, NF>, smem, set)) != kOk) return rc;
    rc = launch_dependent(lora_down_kernel<BF16, 1, NF>, p.tiles * p.splits, kDownWarps * 32, smem, p.splits, stream, p);
  }
  if (rc != kOk) return rc;
  constexpr int MF = R >= 64 ? 1 : 2;
  if (l.tiled) {
    p.tile = 64 * MF;
    p.tiles = (p.n + p.tile - 1) / p.tile + (p.groups < p.n ? p.groups : p.n);
  }
  p.copy_blocks = p.out == p.y ? 0 : (p.n + 31) / 32;
  int cols = 128;
  if (l.tiled) {
    // about six blocks of work per SM: a block begins with a chain of loads (its tile, its rows, their u) of about 2 us
    const double tiles = static_cast<double>(p.n) / p.tile + 0.5 * (p.groups < p.n ? p.groups : p.n);
    cols = static_cast<int>(tiles * p.N / (6 * num_sms));
    cols = cols < 128 ? 128 : (cols + 63) / 64 * 64;
  }
  const int across = (p.N + cols - 1) / cols, along = p.tiles + p.copy_blocks;
  p.tiles_first = along > 65535;
  if (p.tiles_first && across > 65535) return kErrInvalid;
  const dim3 grid(p.tiles_first ? along : across, p.tiles_first ? across : along, 1);
  if (!l.tiled) return launch_dependent(lora_up_kernel<BF16, NF>, grid, kUpWarps * 32, 0, 0, stream, p, cols);
  constexpr int smem = kUpStages * (kUpCols * R * 2 + kUpWarps * 32 * MF * 2 * 16);
  static bool set[kMaxDevices] = {};
  if ((rc = allow_smem(lora_up_tile_kernel<BF16, NF, MF>, smem, set)) != kOk) return rc;
  return launch_dependent(lora_up_tile_kernel<BF16, NF, MF>, grid, kUpWarps * 32, smem, 0, stream, p, cols);
}

template <bool BF16>
int launch_type(const LoraParams& p, int rank, int num_sms, cudaStream_t stream) {
  switch (rank) {
    case 8: return launch_rank<BF16, 1>(p, num_sms, stream);
    case 16: return launch_rank<BF16, 2>(p, num_sms, stream);
    case 32: return launch_rank<BF16, 4>(p, num_sms, stream);
    case 64: return launch_rank<BF16, 8>(p, num_sms, stream);
    case 128: return launch_rank<BF16, 16>(p, num_sms, stream);
    default: return kErrInvalid;
  }
}

}  // namespace

size_t lora_workspace_bytes(int n, int rank) { return (static_cast<size_t>(rank) + 1) * n * sizeof(float); }

int launch_lora_add(const LoraArgs& a, cudaStream_t stream) {
  if (a.n < 0 || a.n > 0x7fffffff - 4096 || a.groups < 1 || a.groups > 1024 || a.K < 8 || a.K % 8 != 0 || a.N < 8 || a.N % 8 != 0) return kErrInvalid;
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
  p.hi = static_cast<uint32_t*>(a.workspace);
  p.lo = p.hi + static_cast<size_t>(a.n) * (a.rank / 2);
  p.back = reinterpret_cast<float*>(p.lo + static_cast<size_t>(a.n) * (a.rank / 2));
  p.ld_y = a.ld_y;
  p.ld_x = a.ld_x;
  p.ld_out = a.ld_out;
  p.n = a.n;
  p.groups = a.groups;
  p.K = a.K;
  p.N = a.N;
  return a.fmt == kBF16 ? launch_type<true>(p, a.rank, a.num_sms, stream) : launch_type<false>(p, a.rank, a.num_sms, stream);
}

}  // namespace sfb200
