// Grouped 2:4-sparse products (sparse_gemm_grouped.cu) on CTA pairs, for many tokens per expert: 256 or 512 weight rows x up to 240 tokens
// per tile with tcgen05.mma.sp.cta_group::2, the structure of sparse_gemm_sm100_2cta.cu with what the ragged sizes change:
//   * tiles come from the device's offsets; an expert's tokens are cut into equal tiles, the token tile being the fast index (pairs next to
//     each other share a weight tile) and the instruction's token count that of the tile;
//   * each CTA of the pair fetches half of the token tile, in boxes of 32 or 40 rows, or four rows per lane of several gathering warps
//     through the grouping, where that is estimated cheaper than a permuted copy in front (plan_grouped);
//   * two accumulator sets (256-row tiles): the drain of a tile hides behind the K loop of the next.
// Bound by the tiles first: a token tile ends at 240, so an expert of 250 tokens runs every weight tile through shared memory twice, with half-filled
// instructions; the last pass over the pairs is partly empty; a K loop of few steps leaves the drain's share large.  Clocks under steady load come on
// top.  Measured: 4096 tokens, 4 of 32 experts, 2816 x 2048 (16 K steps per tile): 94 us alone at full clock (tensor pipe 53 % of cycles, L2 59 %), under load
// 122 us, with the tokens gathered 130-142 us; 1001 tokens, 2 of 8 experts, 4096 x 11008 (about 300 tiles on 74 pairs): 127 us alone (DRAM 47 %, tensor pipe
// 38 %), under load 140-152 us.
#include <cuda.h>
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

template <int BN_, int STAGES_, int BOX_, int RS_, int EPI_, bool GATHER_>
struct PCfg {
  static constexpr int EPI = EPI_, RS = RS_;                   // RS: 128-row sets per CTA
  static constexpr bool GATHER = GATHER_;
  static constexpr int BN = BN_, HALF = BN / 2, BOX = BOX_;      // tokens per tile, per CTA, per copy
  static constexpr int BK = 128, STAGES = STAGES_;
  static constexpr int A_SUB_BYTES = 128 * 64 * 2, A_BYTES = RS * A_SUB_BYTES;
  static constexpr int B_SUB_BYTES = HALF * 128;
  static constexpr int B_BYTES = 2 * B_SUB_BYTES;
  static constexpr int E_SUB_BYTES = 2048, E_BYTES = RS * E_SUB_BYTES;
  static constexpr int ACC_BUFS = RS == 1 ? 2 : 1;             // accumulator sets of RS * BN columns
  static constexpr int E_COL0 = 2 * BN;
  static constexpr int EPI_WARPS = RS_ == 1 ? 8 : 16, GATHER_WARPS = GATHER ? (RS_ == 1 ? 8 : 4) : 0, THREADS = 64 + 32 * (EPI_WARPS + GATHER_WARPS);
  static constexpr int D_ROW_BYTES = EPI == kEpiSwiGLU ? 32 : 64;
  static constexpr int D_BUFS = 1, D_WARP_BYTES = D_BUFS * 16 * D_ROW_BYTES;
  static constexpr int OFF_A = 0;
  static constexpr int OFF_B = OFF_A + STAGES * A_BYTES;
  static constexpr int OFF_E = OFF_B + STAGES * B_BYTES;
  static constexpr int OFF_D = OFF_E + STAGES * E_BYTES;
  static constexpr int OFF_BAR = OFF_D + EPI_WARPS * D_WARP_BYTES;
  static constexpr int OFF_TABLE = OFF_BAR + 256;
  static constexpr int SMEM_BYTES = OFF_TABLE + 1024;      // + the tables of tiles, sized at launch, + alignment slack
  static_assert(HALF % BOX == 0 && BOX % 8 == 0 && HALF <= 128, "token halves: whole boxes, at most four rows per lane");
  static_assert(E_COL0 + 4 * RS * STAGES <= 512, "tensor memory");
};

template <class C>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(C::THREADS, 1)
grouped_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmE,
                         const GroupedParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  const uint32_t bar_full = smem_u32(bars);                 // used in the even CTA only
  const uint32_t bar_empty = bar_full + 8 * C::STAGES;      // both CTAs
  const uint32_t bar_accf = bar_empty + 8 * C::STAGES;      // both CTAs, one per accumulator set
  const uint32_t bar_acce = bar_accf + 16;                  // even CTA only, one per accumulator set
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_BAR + 8 * (2 * C::STAGES + 4));
  volatile int* err = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* first_tile = reinterpret_cast<int*>(smem + C::OFF_TABLE);
  int* first_row = first_tile + p.experts + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const bool leader = rank == 0;
  const int pair_id = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int k_iters = (p.K + C::BK - 1) / C::BK;

  if (threadIdx.x == 0) {
    *err = 0;
    for (int s = 0; s < C::STAGES; ++s) {
      // one arrival announces the bytes; every gathering warp arrives too, also where it has no row to fetch: a warp that only watched
      // the stages go by could fall two phases behind and wait for a parity that does not come again
      mbar_init(bar_full + 8 * s, 1 + 2 * C::GATHER_WARPS);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_accf + 8 * b, 1);
      mbar_init(bar_acce + 8 * b, 2 * C::EPI_WARPS);
    }
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmE);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  dependency_wait();
  dependency_trigger();
  if (warp == 0) build_tile_table(p, C::BN, first_tile, first_row);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // both CTAs' barriers are initialised before anything remote touches them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int num_tiles = first_tile[p.experts];

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    if (elect_one()) {
      const uint32_t leader_full0 = mapa_u32(bar_full, 0);
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      GroupedTile t;
      t.e = 0;
      for (int tile = pair_id; tile < num_tiles && ok; tile += num_pairs) {
        locate_tile(p, C::BN, first_tile, first_row, tile, t);
        const int half = ((t.count + 15) & ~15) / 2;                       // rows of the operand in each CTA
        const int in0 = t.count < half ? t.count : half, in1 = t.count - in0;      // of which hold a token
        const int mine = leader ? in0 : in1, tok = t.tok0 + rank * half;
        int e_x[C::RS], a_y[C::RS];
#pragma unroll
        for (int rs = 0; rs < C::RS; ++rs) {
          // 128-row tile of the expert's weight; one that lies wholly behind its rows loads the last tile again: not stored
          const int row_tile = min((t.m_blk * 2 + rank) * C::RS + rs, p.row_tiles - 1);
          e_x[rs] = (t.e * p.row_tiles + row_tile) * p.k_tiles128 * 256;
          a_y[rs] = t.e * p.n_out + row_tile * 128;
        }
        const int boxes = (mine + C::BOX - 1) / C::BOX;
        const uint32_t bytes =
            C::GATHER ? static_cast<uint32_t>((in0 + 3) / 4 + (in1 + 3) / 4) * 1024u
                      : static_cast<uint32_t>((in0 + C::BOX - 1) / C::BOX + (in1 + C::BOX - 1) / C::BOX) * (C::BOX * 256u);
        for (int kt = 0; kt < k_iters; ++kt) {
          ok = mbar_wait(bar_empty + 8 * s, ph ^ 1, err, p.status, 1);
          if (!ok) break;
          const uint32_t full = leader_full0 + 8 * s;
          const uint32_t b_dst = sbase + C::OFF_B + s * C::B_BYTES;
          if (leader) mbar_arrive_expect_tx(bar_full + 8 * s, 2 * (C::A_BYTES + C::E_BYTES) + bytes);      // of both CTAs
#pragma unroll
          for (int rs = 0; rs < C::RS; ++rs) {
            tma_load_2d_pair(sbase + C::OFF_A + s * C::A_BYTES + rs * C::A_SUB_BYTES, &tmA, kt * 64, a_y[rs], full);
            tma_load_1d_pair(sbase + C::OFF_E + s * C::E_BYTES + rs * C::E_SUB_BYTES, &tmE, e_x[rs] + kt * 256, full);
          }
          if (!C::GATHER) {
            for (int b = 0; b < boxes; ++b)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                tma_load_2d_pair(b_dst + j * C::B_SUB_BYTES + b * C::BOX * 128, &tmB, kt * C::BK + j * 64, tok + b * C::BOX, full);
          }
          if (++s == C::STAGES) { s = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (even CTA only)
    if (leader && elect_one()) {
      int s = 0;
      uint32_t ph = 0, it = 0;
      bool ok = true;
      GroupedTile t;
      t.e = 0;
      for (int tile = pair_id; tile < num_tiles && ok; tile += num_pairs, ++it) {
        locate_tile(p, C::BN, first_tile, first_row, tile, t);
        const uint32_t idesc = make_idesc_f16(256, (t.count + 15) & ~15, p.fmt, true);
        const uint32_t as = C::ACC_BUFS == 2 ? it & 1u : 0u, use = C::ACC_BUFS == 2 ? it >> 1 : it;
        const uint32_t d_tmem = tmem_base + as * C::BN;
        ok = mbar_wait(bar_acce + 8 * as, (use & 1u) ^ 1u, err, p.status, 3);
        if (!ok) break;
        tc_fence_after();
        for (int kt = 0; kt < k_iters; ++kt) {
          ok = mbar_wait(bar_full + 8 * s, ph, err, p.status, 2);
          if (!ok) break;
          tc_fence_after();
          const uint32_t e_cols = C::E_COL0 + 4 * C::RS * s;
#pragma unroll
          for (int rs = 0; rs < C::RS; ++rs)
            tc_cp_128x128b_pair(tmem_base + e_cols + 4 * rs,
                                make_smem_desc(sbase + C::OFF_E + s * C::E_BYTES + rs * C::E_SUB_BYTES, 0, 128, kSwNone));
          const uint32_t a_addr = sbase + C::OFF_A + s * C::A_BYTES;
          const uint32_t b_addr = sbase + C::OFF_B + s * C::B_BYTES;
#pragma unroll
          for (int kb = 0; kb < 4; ++kb) {
            const uint64_t bdesc = make_smem_desc(b_addr + (kb >> 1) * C::B_SUB_BYTES + (kb & 1) * 64, 16, 1024, kSw128);
#pragma unroll
            for (int rs = 0; rs < C::RS; ++rs)
              tc_mma_sp_f16_pair(d_tmem + rs * C::BN, make_smem_desc(a_addr + rs * C::A_SUB_BYTES + kb * 32, 16, 1024, kSw128), bdesc,
                                 tmem_base + e_cols + 4 * rs + (kb & ~1), idesc | (kb & 1), (kt > 0 || kb > 0) ? 1u : 0u);
          }
          tc_commit_pair(bar_empty + 8 * s);
          if (++s == C::STAGES) { s = 0; ph ^= 1; }
        }
        if (!ok) break;
        tc_commit_pair(bar_accf + 8 * as);
      }
    }
  } else if (C::GATHER && warp >= 2 + C::EPI_WARPS) {
    // ------------------------------------------------------------ token rows through the grouping, four by four (both CTAs)
    // (a warp issues its lanes' copies one by one, 25-40 cycles each: hence several warps)
    const int at = lane * C::GATHER_WARPS + warp - 2 - C::EPI_WARPS;
    const uint32_t leader_full0 = mapa_u32(bar_full, 0);
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    GroupedTile t;
    t.e = 0;
    for (int tile = pair_id; tile < num_tiles && ok; tile += num_pairs) {
      locate_tile(p, C::BN, first_tile, first_row, tile, t);
      const int half = ((t.count + 15) & ~15) / 2;
      const int in0 = t.count < half ? t.count : half;
      const int mine = leader ? in0 : t.count - in0;
      int rows[4];
      gather_rows_of(p, t.tok0 + rank * half, mine, at, rows);
      for (int kt = 0; kt < k_iters; ++kt) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * s, ph ^ 1, err, p.status, 5));
        if (!ok) break;
        if (4 * at < mine) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
            tma_gather4_pair(sbase + C::OFF_B + s * C::B_BYTES + j * C::B_SUB_BYTES + at * 512, &tmB, kt * C::BK + j * 64, rows, leader_full0 + 8 * s);
        }
        if (lane == 0) mbar_arrive_remote(leader_full0 + 8 * s);
        if (++s == C::STAGES) { s = 0; ph ^= 1; }
      }
    }
  } else {
    // ------------------------------------------------------------ drain (both CTAs)
    constexpr int PARTS = C::EPI_WARPS / 4 / C::RS;      // warps that share an accumulator's lanes
    const int q = warp & 3, rs = ((warp - 2) >> 2) / PARTS, part = ((warp - 2) >> 2) % PARTS;
    const uint32_t leader_acce0 = mapa_u32(bar_acce, 0);
    const uint64_t pol = l2_policy_evict_first();
    const uint32_t stage0 = sbase + C::OFF_D + (warp - 2) * C::D_WARP_BYTES;
    bool ok = true;
    uint32_t it = 0;
    GroupedTile t;
    t.e = 0;
    for (int tile = pair_id; tile < num_tiles && ok; tile += num_pairs, ++it) {
      locate_tile(p, C::BN, first_tile, first_row, tile, t);
      const uint32_t as = C::ACC_BUFS == 2 ? it & 1u : 0u, use = C::ACC_BUFS == 2 ? it >> 1 : it;
      ok = __all_sync(0xffffffffu, mbar_wait(bar_accf + 8 * as, use & 1u, err, p.status, 4));
      if (!ok) break;
      tc_fence_after();
      const int chunks = (t.count + 15) / 16;
      drain_tile<C::EPI>(p, t, ((t.m_blk * 2 + rank) * C::RS + rs) * 128 + q * 32,
                         tmem_base + (static_cast<uint32_t>(q * 32) << 16) + (as + rs) * C::BN,
                         chunks * part / PARTS, chunks * (part + 1) / PARTS, stage0, C::D_BUFS - 1, pol, [&]() {
                           tc_fence_before();
                           __syncwarp();
                           if (lane == 0) mbar_arrive_remote(leader_acce0 + 8 * as);
                         });
    }
  }

  // ------------------------------------------------------------ teardown
  __syncwarp();
  if (*err) {
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // the peer may still be signalling this CTA's barriers until here
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
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
    if (cudaFuncSetAttribute(grouped_gemm_pair_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448) != cudaSuccess) return kErrCuda;
    attr_set[dev] = true;
  }
  CUtensorMap tmA, tmB, tmE;
  const uint64_t kc = static_cast<uint64_t>(a.K) / 2;
  if (!make_map_2d(&tmA, a.values, static_cast<uint64_t>(a.experts) * a.n_out, kc, kc * 2, 128, 64, CU_TENSOR_MAP_SWIZZLE_128B, a.fmt))
    return kErrTensorMap;
  if (!make_map_2d(&tmB, a.x, a.x_rows, a.K, static_cast<uint64_t>(a.ldx) * 2, C::GATHER ? 1 : C::BOX, 64, CU_TENSOR_MAP_SWIZZLE_128B, a.fmt))
    return kErrTensorMap;
  if (!make_map_1d_u64(&tmE, a.meta, a.experts * meta_bytes(a.n_out, a.K) / 8, 256)) return kErrTensorMap;
  GroupedParams p = grouped_params(a);
  p.m_blks = (a.n_out + 256 * C::RS - 1) / (256 * C::RS);
  return launch_dependent(grouped_gemm_pair_kernel<C>, a.num_sms / 2 * 2, C::THREADS, smem, 0, stream, tmA, tmB, tmE, p);
}

template <int BN, int STAGES, int BOX, int RS>
int dispatch_epi(const GroupedGemmArgs& a, cudaStream_t stream) {
  if (a.epi == kEpiSwiGLU)
    return a.rows ? launch_cfg<PCfg<BN, STAGES, BOX, RS, kEpiSwiGLU, true>>(a, stream) : launch_cfg<PCfg<BN, STAGES, BOX, RS, kEpiSwiGLU, false>>(a, stream);
  return a.rows ? launch_cfg<PCfg<BN, STAGES, BOX, RS, kEpiStore, true>>(a, stream) : launch_cfg<PCfg<BN, STAGES, BOX, RS, kEpiStore, false>>(a, stream);
}

}  // namespace

int launch_grouped_gemm_pair(const GroupedGemmArgs& a, int variant, cudaStream_t stream) {
  // the metadata of all experts is one tensor with 32-bit coordinates
  if (a.experts * (meta_bytes(a.n_out, a.K) / 8) > 0x7fffffffull) return kErrInvalid;
  switch (variant) {      // rows per tile: 256 (1...) or 512 (2...), tokens; shorter token tiles leave room for more stages
    case 1128: return dispatch_epi<128, 6, 32, 1>(a, stream);
    case 1240: return dispatch_epi<240, 4, 40, 1>(a, stream);
    case 2128: return dispatch_epi<128, 4, 32, 2>(a, stream);
    case 2240: return dispatch_epi<240, 3, 40, 2>(a, stream);
    default: return kErrInvalid;
  }
}

}  // namespace sfb200
