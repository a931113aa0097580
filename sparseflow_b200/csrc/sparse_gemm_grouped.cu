// 2:4-sparse matrix products grouped by expert with ragged sizes (sm_100a):
//   y[p] = act(W_e . x[p] + bias_e)                              for offsets[e] <= p < offsets[e + 1]
//   h[p] = silu(Wg_e . x[p] + bg_e) * (Wu_e . x[p] + bu_e)       with gate and up rows interleaved by 16
// on the operand formats of sparse_gemm_sm100.cu, the experts' weights one after the other.
//
// The sizes are known on the device only (the router wrote them), so nothing here waits for the host: the grid is what fits the
// GPU, every block turns offsets[] into a table of tile numbers and walks the tiles with a stride.  A tile is 128 rows of one
// expert's weight times up to BN of its tokens; the tokens of an expert are cut into equal tiles, and the
// instruction's token count is the tile's own (a multiple of 16), so an expert with three tokens pays for 16.
// Row tiles are the slow index inside an expert: blocks next to each other share a weight tile.
// The token box of a copy may reach behind the expert's last token: those columns belong to other experts or lie outside the tensor
// (zero), and are not stored.  Likewise rows behind the last row tile of an expert.
//
// One persistent CTA per SM, 6 warps: warp 0 = TMA producer, warp 1 = MMA issuer and tensor-memory owner, warps 2..5 = drain
// (tensor memory -> registers -> 16-token staging tile -> 16-byte stores, rolled over 16-column chunks).
// Rounding: one rounding of the result.  The sums over K are 32-bit in tensor memory; the tensor cores add with an error of 2.1e-6 of the
// result's norm at K 4096 and 6.0e-6 at 11008 (32-bit FMA chains 0.4e-6 and 0.7e-6), which moves 1 to 3 of a thousand bf16 results to a neighbouring value and
// leaves their error against 64 bits as it was (1.64e-3 of the norm, the rounding's own).  SiLU through the fast exponential and division: of 88064
// results of the first call below none differed from those of a 64-bit SiLU on the same sums.
// Bound by HBM: every chosen expert's weights once.  Measured: one token of 2 experts, 22016 x 4096 37 us (5.4 TB/s); 64 tokens of 6 of
// 64 experts, 2048 x 1408 36 us (5.8 TB/s); ncu: DRAM 61 and 68 % of peak cycles, tensor pipe 3 %.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "grouped.cuh"
#include "kernels.h"
#include "launch.h"
#include "sm100_pair.cuh"
#include "sm100_ptx.cuh"
#include "tensor_map.h"

namespace sfb200 {
namespace {

template <int BN_, int STAGES_, int EPI_, bool GATHER_>
struct GCfg {
  static constexpr int BN = BN_, STAGES = STAGES_, EPI = EPI_;
  static constexpr bool GATHER = GATHER_;      // token rows fetched four by four through p.rows
  static constexpr int GATHER_WARPS = GATHER ? 4 : 0, THREADS = 192 + 32 * GATHER_WARPS;
  static constexpr int BK = 128;
  static constexpr int A_BYTES = 128 * 64 * 2;
  static constexpr int B_SUB_BYTES = BN * 128;
  static constexpr int B_BYTES = 2 * B_SUB_BYTES;
  static constexpr int E_BYTES = 2048;
  static constexpr int ACC = 2;
  static constexpr int TMEM_USED = ACC * BN + 4 * STAGES;
  static constexpr int TMEM_COLS = TMEM_USED <= 64 ? 64 : TMEM_USED <= 128 ? 128 : TMEM_USED <= 256 ? 256 : 512;
  static constexpr int D_ROW_BYTES = EPI == kEpiSwiGLU ? 32 : 64;
  static constexpr int D_BYTES = 4 * 2 * 16 * D_ROW_BYTES;      // four warps, two buffers of 16 tokens
  static constexpr int OFF_A = 0;
  static constexpr int OFF_B = OFF_A + STAGES * A_BYTES;
  static constexpr int OFF_E = OFF_B + STAGES * B_BYTES;
  static constexpr int OFF_D = OFF_E + STAGES * E_BYTES;
  static constexpr int OFF_BAR = OFF_D + D_BYTES;
  static constexpr int OFF_TABLE = OFF_BAR + 256;
  static constexpr int SMEM_BYTES = OFF_TABLE + 1024;      // + the tables of tiles, sized at launch, + alignment slack
  static_assert(BN % 16 == 0 && BN >= 32 && BN <= 128, "BN");
  static_assert(8 * (2 * STAGES + 4) + 8 <= 256, "barriers");
};

template <class C>
__global__ void __launch_bounds__(C::THREADS, 1)
grouped_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GroupedParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  const uint32_t bar_full = smem_u32(bars);
  const uint32_t bar_empty = bar_full + 8 * C::STAGES;
  const uint32_t bar_accf = bar_empty + 8 * C::STAGES;
  const uint32_t bar_acce = bar_accf + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_BAR + 8 * (2 * C::STAGES + 4));
  volatile int* err = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* first_tile = reinterpret_cast<int*>(smem + C::OFF_TABLE);      // [experts + 1]
  int* first_row = first_tile + p.experts + 1;                        // [experts + 1]

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int k_iters = (p.K + C::BK - 1) / C::BK;

  if (threadIdx.x == 0) {
    *err = 0;
    for (int s = 0; s < C::STAGES; ++s) {
      // one arrival announces the bytes; every gathering warp arrives too, also where it has no row to fetch: a warp that only watched
      // the stages go by could fall two phases behind and wait for a parity that does not come again
      mbar_init(bar_full + 8 * s, 1 + C::GATHER_WARPS);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(bar_accf + 8 * a, 1);
      mbar_init(bar_acce + 8 * a, 4);
    }
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish();
  }
  dependency_wait();
  dependency_trigger();
  if (warp == 0) build_tile_table(p, C::BN, first_tile, first_row);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int num_tiles = first_tile[p.experts];

  if (warp == 0) {
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      GroupedTile t;
      t.e = 0;
      for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
        locate_tile(p, C::BN, first_tile, first_row, tile, t);
        const uint32_t* meta = p.meta + (static_cast<size_t>(t.e) * p.row_tiles + t.m_blk) * p.k_tiles128 * 512;
        const uint32_t b_bytes = C::GATHER ? static_cast<uint32_t>((t.count + 3) / 4) * 1024u : C::B_BYTES;
        for (int kt = 0; kt < k_iters; ++kt) {
          ok = mbar_wait(bar_empty + 8 * s, ph ^ 1, err, p.status, 1);
          if (!ok) break;
          const uint32_t full = bar_full + 8 * s;
          mbar_arrive_expect_tx(full, C::A_BYTES + C::E_BYTES + b_bytes);
          tma_load_2d(sbase + C::OFF_A + s * C::A_BYTES, &tmA, kt * 64, t.e * p.n_out + t.m_blk * 128, full);
          bulk_load_1d(sbase + C::OFF_E + s * C::E_BYTES, meta + static_cast<size_t>(kt) * 512, C::E_BYTES, full);
          if (!C::GATHER) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              tma_load_2d(sbase + C::OFF_B + s * C::B_BYTES + j * C::B_SUB_BYTES, &tmB, kt * C::BK + j * 64, t.tok0, full);
          }
          if (++s == C::STAGES) { s = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      int s = 0, as = 0;
      uint32_t ph = 0, aph = 0;
      bool ok = true;
      GroupedTile t;
      t.e = 0;
      for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
        locate_tile(p, C::BN, first_tile, first_row, tile, t);
        const uint32_t idesc = make_idesc_f16(128, (t.count + 15) & ~15, p.fmt, true);
        ok = mbar_wait(bar_acce + 8 * as, aph ^ 1, err, p.status, 3);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + as * C::BN;
        for (int kt = 0; kt < k_iters; ++kt) {
          ok = mbar_wait(bar_full + 8 * s, ph, err, p.status, 2);
          if (!ok) break;
          tc_fence_after();
          const uint32_t e_cols = C::ACC * C::BN + 4 * s;
          tc_cp_128x128b(tmem_base + e_cols, make_smem_desc(sbase + C::OFF_E + s * C::E_BYTES, 0, 128, kSwNone));
          const uint32_t a_addr = sbase + C::OFF_A + s * C::A_BYTES;
          const uint32_t b_addr = sbase + C::OFF_B + s * C::B_BYTES;
#pragma unroll
          for (int kb = 0; kb < 4; ++kb)
            tc_mma_sp_f16(d_tmem, make_smem_desc(a_addr + kb * 32, 16, 1024, kSw128),
                          make_smem_desc(b_addr + (kb >> 1) * C::B_SUB_BYTES + (kb & 1) * 64, 16, 1024, kSw128),
                          tmem_base + e_cols + (kb & ~1), idesc | (kb & 1), (kt > 0 || kb > 0) ? 1u : 0u);
          tc_commit(bar_empty + 8 * s);
          if (++s == C::STAGES) { s = 0; ph ^= 1; }
        }
        if (!ok) break;
        tc_commit(bar_accf + 8 * as);
        if (++as == C::ACC) { as = 0; aph ^= 1; }
      }
    }
  } else if (C::GATHER && warp >= 6) {
    // token rows, four by four
    const int at = lane * C::GATHER_WARPS + warp - 6;
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    GroupedTile t;
    t.e = 0;
    for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
      locate_tile(p, C::BN, first_tile, first_row, tile, t);
      int rows[4];
      gather_rows_of(p, t.tok0, t.count, at, rows);
      for (int kt = 0; kt < k_iters; ++kt) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * s, ph ^ 1, err, p.status, 5));
        if (!ok) break;
        if (4 * at < t.count) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
            tma_gather4(sbase + C::OFF_B + s * C::B_BYTES + j * C::B_SUB_BYTES + at * 512, &tmB, kt * C::BK + j * 64, rows, bar_full + 8 * s);
        }
        if (lane == 0) mbar_arrive(bar_full + 8 * s);
        if (++s == C::STAGES) { s = 0; ph ^= 1; }
      }
    }
  } else {
    const int q = warp & 3;
    const uint64_t pol = l2_policy_evict_first();
    int as = 0;
    uint32_t aph = 0;
    bool ok = true;
    GroupedTile t;
    t.e = 0;
    for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
      locate_tile(p, C::BN, first_tile, first_row, tile, t);
      ok = __all_sync(0xffffffffu, mbar_wait(bar_accf + 8 * as, aph, err, p.status, 4));
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + as * C::BN;
      drain_tile<C::EPI>(p, t, t.m_blk * 128 + q * 32, t_acc, 0, (t.count + 15) / 16,
                         sbase + C::OFF_D + (warp - 2) * 2 * 16 * C::D_ROW_BYTES, 1, pol, [&]() {
                           tc_fence_before();
                           __syncwarp();
                           if (lane == 0) mbar_arrive(bar_acce + 8 * as);
                         });
      if (++as == C::ACC) { as = 0; aph ^= 1; }
    }
  }

  __syncwarp();
  if (*err) {
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

template <class C>
int launch_cfg(const GroupedGemmArgs& a, cudaStream_t stream) {
  const int smem = C::SMEM_BYTES + (2 * (a.experts + 1) * 4 + 15) / 16 * 16;
  if (smem > 232448) return kErrInvalid;
  static bool attr_set[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return kErrCuda;
  if (!attr_set[dev]) {
    if (cudaFuncSetAttribute(grouped_gemm_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448) != cudaSuccess) return kErrCuda;
    attr_set[dev] = true;
  }
  CUtensorMap tmA, tmB;
  const uint64_t kc = static_cast<uint64_t>(a.K) / 2;
  if (!make_map_2d(&tmA, a.values, static_cast<uint64_t>(a.experts) * a.n_out, kc, kc * 2, 128, 64, CU_TENSOR_MAP_SWIZZLE_128B, a.fmt))
    return kErrTensorMap;
  if (!make_map_2d(&tmB, a.x, a.x_rows, a.K, static_cast<uint64_t>(a.ldx) * 2, C::GATHER ? 1 : C::BN, 64, CU_TENSOR_MAP_SWIZZLE_128B, a.fmt)) return kErrTensorMap;
  const GroupedParams p = grouped_params(a);
  return launch_dependent(grouped_gemm_kernel<C>, a.num_sms, C::THREADS, smem, 0, stream, tmA, tmB, p);
}

template <int EPI, bool GATHER>
int dispatch(const GroupedGemmArgs& a, int variant, cudaStream_t stream) {
  if (variant == 32) return launch_cfg<GCfg<32, 7, EPI, GATHER>>(a, stream);
  if (variant == 64) return launch_cfg<GCfg<64, 6, EPI, GATHER>>(a, stream);
  return launch_grouped_gemm_pair(a, variant, stream);
}

// dst[i] = src[rows[i]] (a row outside 0 .. src_rows-1: zeros)
__global__ void __launch_bounds__(256) gather_rows_kernel(const uint16_t* src, int64_t ld, int src_rows, const int* rows, int n, int pieces, uint16_t* dst) {
  dependency_wait();
  dependency_trigger();
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int r = rows[i];
    const bool ok = r >= 0 && r < src_rows;
    for (int c = threadIdx.x; c < pieces; c += 256) {
      const uint4 v = ok ? *reinterpret_cast<const uint4*>(src + r * ld + c * 8) : make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(dst + (static_cast<size_t>(i) * pieces + c) * 8) = v;
    }
  }
}

// Estimated time in us of a variant (32, 64: single-CTA tiles of that many tokens; 1128, 1240, 2128, 2240: pair tiles of 256 or 512
// rows) from the average tokens per expert: launch + passes over the SMs or pairs x (128-wide K steps x step time + drain), or the weights at
// 6.2 TB/s, and a sixth of the shorter of the two.  Sizes are ragged: an expert takes half a tile more than its tokens fill, once they fill
// three quarters of one.  Constants fitted to 200 settings under steady load, every variant timed on each (1000-22016 rows, K 512-11008, 4-128 experts,
// 1-1000 tokens per expert; relative error 0.1).  The choice by it averages 1.02 of the fastest variant (gathered rows: 1.03), worst 1.27.
double grouped_cost(int variant, bool gather, int total, int experts, int n_out, int K, int num_sms) {
  struct Step { double base, per_token, drain, tail, launch; };
  struct Form { int variant, rows, tokens; Step plain, gather; };
  static const Form forms[] = {
      {32, 128, 32, {0.0, 0.008, 0.21, 0.02, 3.6}, {0.248, 0.0044, 0.52, 0.80, 0.0}},
      {64, 128, 64, {0.2325, 0.0005, 0.58, 0.20, 1.6}, {0.218, 0.0066, 0.58, 0.0, 0.0}},
      {1128, 256, 128, {0.219, 0.0005, 1.35, 0.92, 2.6}, {0.0, 0.0045, 0.62, 0.0, 5.3}},
      {1240, 256, 240, {0.265, 0.0009, 1.46, 0.93, 3.5}, {0.315, 0.0015, 1.35, 0.47, 0.0}},
      {2128, 512, 128, {0.329, 0.0015, 3.87, 0.97, 0.0}, {0.3325, 0.0018, 2.98, 0.89, 1.1}},
      {2240, 512, 240, {0.359, 0.0026, 4.08, 0.78, 0.0}, {0.375, 0.0028, 3.86, 0.72, 0.0}}};
  for (const Form& f : forms) {
    if (f.variant != variant) continue;
    const Step& s = gather ? f.gather : f.plain;
    const double avg = total > experts ? static_cast<double>(total) / experts : 1.0;
    const double active = total < experts ? total : experts;
    const double cuts = avg <= 0.75 * f.tokens ? 1.0 : avg / f.tokens + 0.5;
    const double tiles = active * ((n_out + f.rows - 1) / f.rows) * cuts, units = f.rows == 128 ? num_sms : num_sms / 2;
    const double passes = tiles > units ? tiles / units + s.tail : 1.0;
    const double work = passes * (((K + 127) / 128) * (s.base + s.per_token * (avg / cuts)) + s.drain);
    const double hbm = active * n_out * (K * 1.125) / 6.2e6;
    return s.launch + (work > hbm ? work + 0.15 * hbm : hbm + 0.15 * work);
  }
  return 1e30;
}

}  // namespace

// What a call runs: the variant estimated fastest; with `gather`, 10000 more where copying the rows into the order of the experts and
// multiplying the copy is estimated faster than fetching four rows per copy instruction inside the product (such fetches take about 35 cycles each
// whatever they bring, which bounds tiles with many tokens: 22016 x 4096, 8 experts of 512 tokens 510 us, contiguous 352 us).
int plan_grouped(int total, int experts, int n_out, int K, bool gather, int num_sms) {
  static const int variants[] = {32, 64, 1128, 1240, 2128, 2240};
  int best = 0;
  double cost = 1e300;
  // the tables of tiles, 8 bytes per expert, stand beside the ring in shared memory: 2128 leaves 1.8 KB for them, the other forms hold kMaxExperts
  auto fits = [&](int v) { return v != 2128 || experts <= 220; };
  for (int v : variants) {
    if (!fits(v)) continue;
    const double c = grouped_cost(v, gather, total, experts, n_out, K, num_sms);
    if (c < cost) { cost = c; best = v; }
  }
  if (!gather) return best;
  const double copy = 3.0 + static_cast<double>(total) * K * 4.0 / 7.4e6;
  for (int v : variants) {
    if (!fits(v)) continue;
    const double c = copy + grouped_cost(v, false, total, experts, n_out, K, num_sms);
    if (c < cost) { cost = c; best = 10000 + v; }
  }
  return best;
}

int launch_grouped_gemm(const GroupedGemmArgs& a, cudaStream_t stream) {
  if (a.experts < 1 || a.experts > kMaxExperts || a.total < 0 || a.K <= 0 || a.K % 64 != 0 || a.n_out <= 0 || a.n_out % 8 != 0) return kErrInvalid;
  if (a.fmt != kF16 && a.fmt != kBF16) return kErrInvalid;
  if (a.total == 0) return kOk;
  if (!a.x || !a.values || !a.meta || !a.y || !a.offsets || a.x_rows < 1) return kErrInvalid;
  const int out_cols = a.epi == kEpiSwiGLU ? a.n_out / 2 : a.n_out;
  if (a.ldx < a.K || a.ldx % 8 != 0 || a.ldy < out_cols || a.ldy % 8 != 0) return kErrInvalid;
  if ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.values) | reinterpret_cast<uintptr_t>(a.meta) |
       reinterpret_cast<uintptr_t>(a.y)) & 15)
    return kErrInvalid;
  // coordinates of the copies and tile numbers are 32-bit
  if (static_cast<int64_t>(a.experts) * a.n_out > 0x7fffffffll - 256) return kErrInvalid;
  if (static_cast<int64_t>((a.n_out + 127) / 128) * (a.total / 16 + a.experts) > 0x7fffffffll) return kErrInvalid;
  if (a.epi == kEpiSwiGLU && a.n_out % 32 != 0) return kErrInvalid;
  GroupedGemmArgs b = a;
  int variant = a.variant ? a.variant : plan_grouped(a.total, a.experts, a.n_out, a.K, a.rows != nullptr, a.num_sms);
  if (variant >= 10000) {
    variant -= 10000;
    if (!a.rows || !a.scratch || (reinterpret_cast<uintptr_t>(a.scratch) & 15)) return kErrInvalid;
    const int rc = launch_dependent(gather_rows_kernel, a.total < 16 * a.num_sms ? a.total : 16 * a.num_sms, 256, 0, 0, stream,
                                    static_cast<const uint16_t*>(a.x), static_cast<int64_t>(a.ldx), a.x_rows, a.rows, a.total, a.K / 8,
                                    static_cast<uint16_t*>(a.scratch));
    if (rc != kOk) return rc;
    b.x = a.scratch;
    b.ldx = a.K;
    b.x_rows = a.total;
    b.rows = nullptr;
  }
  if (a.epi == kEpiSwiGLU) return b.rows ? dispatch<kEpiSwiGLU, true>(b, variant, stream) : dispatch<kEpiSwiGLU, false>(b, variant, stream);
  return b.rows ? dispatch<kEpiStore, true>(b, variant, stream) : dispatch<kEpiStore, false>(b, variant, stream);
}

}  // namespace sfb200
