// Shared by the grouped sparse GEMM kernels: tables of tiles built on the device, and the drain of an accumulator whose token count
// is known at run time.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "device_state.h"
#include "kernels.h"
#include "sm100_pair.cuh"
#include "sm100_ptx.cuh"

namespace sfb200 {

constexpr int kMaxExperts = 1024;

struct GroupedParams {
  const uint32_t* meta;   // [experts][row_tiles][k_tiles][128][4]
  const void* bias;       // store: [experts, n_out]; SiLU.mul: gate rows, [experts, n_out / 2]; or null
  const void* bias_up;    // SiLU.mul: up rows, or null
  const int* offsets;     // [experts + 1]
  const int* rows;        // [total]: row of x for every place, or null (x is in the order of the places)
  void* y;
  int* status;
  int experts, n_out, K, ldy, total, x_rows;
  int row_tiles;          // metadata tiles of 128 rows per expert
  int k_tiles128;
  int m_blks;             // row tiles of the kernel per expert
  int fmt, act;
};

inline GroupedParams grouped_params(const GroupedGemmArgs& a) {
  GroupedParams p{};
  p.meta = static_cast<const uint32_t*>(a.meta);
  p.bias = a.bias;
  p.bias_up = a.bias_up;
  p.offsets = a.offsets;
  p.rows = a.rows;
  p.x_rows = a.x_rows;
  p.y = a.y;
  p.status = a.status;
  p.experts = a.experts;
  p.n_out = a.n_out;
  p.K = a.K;
  p.ldy = a.ldy;
  p.total = a.total;
  p.row_tiles = (a.n_out + 127) / 128;
  p.k_tiles128 = (a.K + 127) / 128;
  p.m_blks = p.row_tiles;
  p.fmt = a.fmt;
  p.act = a.act;
  return p;
}

// Token tiles of an expert with n tokens, at most bn each.
__device__ __forceinline__ int token_tiles(int n, int bn) { return (n + bn - 1) / bn; }

// One warp: first_tile[e] = tiles of the experts before e, first_row[e] = offsets[e], held inside 0 .. total whatever is in memory.
__device__ __forceinline__ void build_tile_table(const GroupedParams& p, int bn, int* first_tile, int* first_row) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int e0 = 0; e0 < p.experts; e0 += 32) {
    const int e = e0 + lane;
    int begin = 0, end = 0;
    if (e < p.experts) {
      begin = min(max(p.offsets[e], 0), p.total);
      end = min(max(p.offsets[e + 1], begin), p.total);
    }
    const int own = token_tiles(end - begin, bn) * p.m_blks;
    int sum = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += v;
    }
    if (e < p.experts) {
      first_tile[e] = before + sum - own;
      first_row[e] = begin;
      if (e == p.experts - 1) {
        first_tile[p.experts] = before + sum;
        first_row[p.experts] = end;
      }
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
}

struct GroupedTile {
  int e;          // expert; the caller starts at 0 and asks for growing tile numbers
  int m_blk;      // row tile of the expert
  int tok0;       // first row of x and y
  int count;      // tokens, 1 .. bn
};
__device__ __forceinline__ void locate_tile(const GroupedParams& p, int bn, const int* first_tile, const int* first_row, int tile, GroupedTile& t) {
  while (tile >= first_tile[t.e + 1]) ++t.e;
  const int n = first_row[t.e + 1] - first_row[t.e];      // offsets ascend: the next expert begins where this one ends
  const int tiles = token_tiles(n, bn);
  const int r = tile - first_tile[t.e];
  t.m_blk = r / tiles;
  const int b = r - t.m_blk * tiles;
  // equal token tiles, in multiples of 8 so that their outputs stay whole
  const int each = ((n + tiles - 1) / tiles + 7) & ~7;
  t.tok0 = first_row[t.e] + b * each;
  const int left = n - b * each;
  t.count = left < each ? left : each;
}

// Four rows of a token operand into 4 x 128 bytes of a swizzled tile, by one copy (box of one row).  The pair form credits the bytes to
// the barrier of the pair's even CTA.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* m, int x, const int (&r)[4], uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_gather4_pair(uint32_t dst, const CUtensorMap* m, int x, const int (&r)[4], uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4, %5, %6}], "
      "[%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(leader_bar)
      : "memory");
}
// The four rows of x that copy number `at` fetches: places first + 4 * at .. of a run of `count`.
__device__ __forceinline__ void gather_rows_of(const GroupedParams& p, int first, int count, int at, int (&r)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    int i = 4 * at + j;
    if (i >= count) i = count - 1;
    r[j] = count > 0 ? min(max(p.rows[first + i], 0), p.x_rows - 1) : 0;
  }
}

// 16-token chunks [c_begin, c_end) of a warp's 32 accumulator lanes (rows row_w ..): load, convert, transpose through the staging
// tile (two buffers from `stage0`), store whole rows of the output.  `release` runs when the last chunk is in registers.
template <int EPI, class Release>
__device__ __forceinline__ void drain_tile(const GroupedParams& p, const GroupedTile& t, int row_w, uint32_t t_acc, int c_begin, int c_end,
                                           uint32_t stage0, int buf_mask, uint64_t policy, Release release) {
  constexpr int D_ROW_BYTES = EPI == kEpiSwiGLU ? 32 : 64;
  constexpr int D_BUF_BYTES = 16 * D_ROW_BYTES;
  const int lane = threadIdx.x & 31, g = lane >> 2;
  const int mt = lane >> 3, rr = lane & 7;
  const uint32_t st_off = static_cast<uint32_t>((rr + 8 * (mt >> 1)) * D_ROW_BYTES + 16 * (mt & 1));
  const int out_cols = EPI == kEpiSwiGLU ? p.n_out / 2 : p.n_out;
  const int out_x = EPI == kEpiSwiGLU ? row_w / 2 : row_w;
  float b0 = 0.f, b1 = 0.f, b2 = 0.f, b3 = 0.f;      // bias of rows g, g + 8, 16 + g, 24 + g
  if (EPI == kEpiStore && p.bias != nullptr) {
    const uint16_t* bias = static_cast<const uint16_t*>(p.bias) + static_cast<size_t>(t.e) * p.n_out;
    if (row_w + g < p.n_out) b0 = bias_at(bias, row_w + g, p.fmt);
    if (row_w + g + 8 < p.n_out) b1 = bias_at(bias, row_w + g + 8, p.fmt);
    if (row_w + g + 16 < p.n_out) b2 = bias_at(bias, row_w + g + 16, p.fmt);
    if (row_w + g + 24 < p.n_out) b3 = bias_at(bias, row_w + g + 24, p.fmt);
  }
  const bool gate_up_bias = EPI == kEpiSwiGLU && (p.bias != nullptr || p.bias_up != nullptr);
  if (gate_up_bias) {
    const size_t at = static_cast<size_t>(t.e) * out_cols;
    load_gate_up_bias(p.bias == nullptr ? nullptr : static_cast<const uint16_t*>(p.bias) + at,
                      p.bias_up == nullptr ? nullptr : static_cast<const uint16_t*>(p.bias_up) + at, row_w, g, p.n_out, p.fmt, b0, b1, b2, b3);
  }
  auto store_chunk = [&](const uint32_t* a, const uint32_t* b, int c) {
    const uint32_t stage = stage0 + (c & buf_mask) * D_BUF_BYTES;
    __syncwarp();
    // which conversion runs is tested once per chunk, not once per value: the drain is a chain of dependent instructions
    if (EPI == kEpiSwiGLU) {
      auto emit = [&](auto f, const int fmt) {
        stmatrix_x4_trans(stage + st_off, pack16(f(0, b0, b2), f(1, b0, b2), fmt), pack16(f(2, b1, b3), f(3, b1, b3), fmt),
                          pack16(f(4, b0, b2), f(5, b0, b2), fmt), pack16(f(6, b1, b3), f(7, b1, b3), fmt));
      };
      if (gate_up_bias) emit([&](int i, float bg, float bu) { return silu_mul_bias(a[i], b[i], bg, bu); }, p.fmt);
      else if (p.fmt == kBF16) emit([&](int i, float, float) { return silu_mul(a[i], b[i]); }, kBF16);
      else emit([&](int i, float, float) { return silu_mul(a[i], b[i]); }, kF16);
    } else {
      auto emit = [&](auto f, const int fmt) {
        stmatrix_x4_trans(stage + st_off, pack16(f(a[0], b0), f(a[1], b0), fmt), pack16(f(a[2], b1), f(a[3], b1), fmt),
                          pack16(f(a[4], b0), f(a[5], b0), fmt), pack16(f(a[6], b1), f(a[7], b1), fmt));
        stmatrix_x4_trans(stage + st_off + 32, pack16(f(b[0], b2), f(b[1], b2), fmt), pack16(f(b[2], b3), f(b[3], b3), fmt),
                          pack16(f(b[4], b2), f(b[5], b2), fmt), pack16(f(b[6], b3), f(b[7], b3), fmt));
      };
      auto plain = [](uint32_t v, float bias) { return __uint_as_float(v) + bias; };
      if (p.act == kActNone && p.fmt == kBF16) emit(plain, kBF16);
      else if (p.act == kActNone) emit(plain, kF16);
      else emit([&](uint32_t v, float bias) { return act_fn(__uint_as_float(v) + bias, p.act); }, p.fmt);
    }
    __syncwarp();
    constexpr int UNITS = D_ROW_BYTES / 16, ROUNDS = UNITS / 2, TOKENS = 32 / UNITS;
    const int tk = lane / UNITS, part = lane % UNITS, col = out_x + part * 8;
    uint16_t* dst = static_cast<uint16_t*>(p.y) + static_cast<size_t>(t.tok0 + c * 16 + tk) * p.ldy + col;
    const uint32_t src = stage + tk * D_ROW_BYTES + part * 16;
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j) {
      if (c * 16 + tk + j * TOKENS < t.count && col < out_cols) {
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(src + j * TOKENS * D_ROW_BYTES));
        asm volatile("st.global.L2::cache_hint.v4.b32 [%0], {%1, %2, %3, %4}, %5;" ::"l"(dst + static_cast<size_t>(j * TOKENS) * p.ldy), "r"(v.x),
                     "r"(v.y), "r"(v.z), "r"(v.w), "l"(policy)
                     : "memory");
      }
    }
  };
  uint32_t ra[8], rb[8], sa[8], sb[8];
  auto load_chunk = [&](int c, uint32_t(&lo)[8], uint32_t(&hi)[8]) {
    tmem_ld_16x256b_x2(t_acc + 16 * c, lo);
    tmem_ld_16x256b_x2(t_acc + 16 * c + (static_cast<uint32_t>(16) << 16), hi);
  };
  if (c_begin >= c_end) {
    release();
    return;
  }
  load_chunk(c_begin, ra, rb);
#pragma unroll 1
  for (int c = c_begin; c < c_end; c += 2) {
    tmem_ld_wait();
    if (c + 1 < c_end) load_chunk(c + 1, sa, sb);
    else release();
    store_chunk(ra, rb, c);
    if (c + 1 < c_end) {
      tmem_ld_wait();
      if (c + 2 < c_end) load_chunk(c + 2, ra, rb);
      else release();
      store_chunk(sa, sb, c + 1);
    }
  }
}

}  // namespace sfb200
