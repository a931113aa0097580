// Grouping of rows, and the router of a mixture of experts.
//
// Grouping: entries 0 .. n-1 carry the id of a group (or none); offsets[g] counts the entries of the groups before g, and the
// entries of a group keep their order, so that the place of an entry is
//   slots[i] = offsets[id_i] + |{i' < i : id_i' = id_i}|,   rows[slots[i]] = i / per_row.
// Integer counts only: the same result on every run.
//
// Router: p = softmax(l_t); the top_k largest logits of a token, ties to the lowest expert (-0 and +0 are one), with their p (or p over the sum of the
// chosen).  An expert whose logit is -inf or NaN is never chosen; a token with fewer than top_k others gets expert -1, weight 0
// there, and belongs to no group (rows of padding: all logits -inf).  +inf counts as the largest finite number.
//
// One warp works on one token: a lane keeps the logits of experts lane, lane + 32, ... as unsigned keys that order like the
// numbers, and top_k rounds take the largest key and, among equals, the lowest expert (two warp reductions a round).
// Work is latency: 16 bytes a chosen entry and one pass over the logits are 1 us of HBM time at 8192 x 128.  Blocks own runs
// of consecutive tokens; with one block everything is a single launch, otherwise a second launch adds up the
// blocks' counts (at most kMaxBlocks x groups) and places the entries.  Measured (replayed): 32 tokens x 64 experts, top 6, 6.0-6.3 us in one launch;
// 8192 x 128, top 8, 17.7 us in two.  There a block has 64 tokens and 32 warps: two tokens per warp, both at once.  Profiled one by one (cold caches):
// group_kernel 15.9 us, issue slots 52 % busy over the blocks' life (750 instructions a token), the rest waits for the logits and for the
// reductions; place_kernel 10.1 us, issue slots 26 % busy: loads of the counts and ids, and a barrier after each step.  Grouping alone: 48 entries 2.8 us,
// 4097 6.3, 16384 8.1.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "kernels.h"
#include "launch.h"
#include "sm100_ptx.cuh"

namespace sfb200 {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxBlocks = 128, kMaxGroups = 1024;
constexpr int kMaxEntries = 0x7fffffff - 4096;      // the strides of the loops stay inside 32 bits

struct GroupParams {
  const int* ids;      // [n]: the caller's, or the experts that the router wrote
  int n;               // entries
  int groups;
  int per_row;         // entries per row
  int chunk;           // entries per block
  int* counts;         // [blocks][groups], two launches only
  int* offsets;        // [groups + 1]
  int* rows;           // [n]
  int* slots;          // [n]
};
struct RouteParams {
  const void* logits;
  int64_t ld;
  int tokens, experts, top_k, dtype, renorm, tokens_per_block;
  float* weights;      // [tokens, top_k]
  int* chosen;         // [tokens, top_k]
};

__device__ __forceinline__ int entry_group(const GroupParams& p, int i, int end) {
  if (i >= end) return -1;
  const int id = p.ids[i];
  return id >= 0 && id < p.groups ? id : -1;
}

// The chunk's entries per group into hist[groups].
__device__ void count_chunk(const GroupParams& p, int begin, int end, int* hist) {
  for (int g = threadIdx.x; g < p.groups; g += static_cast<int>(blockDim.x)) hist[g] = 0;
  __syncthreads();
  for (int i0 = begin; i0 < end; i0 += static_cast<int>(blockDim.x)) {
    const int g = entry_group(p, i0 + threadIdx.x, end);
    const unsigned same = __match_any_sync(0xffffffffu, g);
    if (g >= 0 && __ffs(same) - 1 == (threadIdx.x & 31)) atomicAdd(&hist[g], __popc(same));
  }
  __syncthreads();
}

// total[g] -> exclusive prefix sums in base[g]; returns the sum of all.  groups <= 1024: two per thread.
__device__ int scan_groups(int groups, const int* total, int* base) {
  __shared__ int warp_sum[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g0 = 2 * threadIdx.x;
  const int a = g0 < groups ? total[g0] : 0, b = g0 + 1 < groups ? total[g0 + 1] : 0;
  int v = a + b;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += u;
  }
  if (lane == 31) warp_sum[warp] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const int s = warp_sum[w];
    if (w < warp) before += s;
    all += s;
  }
  const int first = before + v - a - b;
  if (g0 < groups) base[g0] = first;
  if (g0 + 1 < groups) base[g0 + 1] = first + a;
  __syncthreads();
  return all;
}

// Places the chunk's entries: base[g] is the place of the chunk's first entry of group g; wcnt is scratch.
__device__ void place_chunk(const GroupParams& p, int begin, int end, int* base, uint16_t* wcnt) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i0 = begin; i0 < end; i0 += kThreads) {
    for (int j = threadIdx.x; j < kWarps * p.groups; j += kThreads) wcnt[j] = 0;
    __syncthreads();
    const int i = i0 + threadIdx.x, g = entry_group(p, i, end);
    const unsigned same = __match_any_sync(0xffffffffu, g);
    const int rank = __popc(same & ((1u << lane) - 1u));
    if (g >= 0 && rank == 0) wcnt[warp * p.groups + g] = static_cast<uint16_t>(__popc(same));
    __syncthreads();
    for (int e = threadIdx.x; e < p.groups; e += kThreads) {      // counts of the warps before, at most kThreads
      int run = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const int c = wcnt[w * p.groups + e];
        wcnt[w * p.groups + e] = static_cast<uint16_t>(run);
        run += c;
      }
    }
    __syncthreads();
    if (i < end) {
      int at = -1;
      if (g >= 0) {
        at = base[g] + wcnt[warp * p.groups + g] + rank;
        p.rows[at] = i / p.per_row;
      }
      p.slots[i] = at;
    }
    __syncthreads();
    if (g >= 0) {      // the last warp that has an entry of this group carries its base on
      if (rank == 0) atomicAdd(&base[g], __popc(same));
    }
    __syncthreads();
  }
}

__device__ __forceinline__ uint32_t order_key(float v) {
  if (!(v > -INFINITY)) return 0;                 // -inf and NaN: never chosen
  if (v == 0.f) v = 0.f;                          // -0 and +0 are equal: a tie, one key for both
  const uint32_t u = __float_as_uint(fminf(v, FLT_MAX));
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// NL: logits per lane.  NT tokens at a time: the rounds of one token are a chain of reductions, those of two cover each other.
template <int NL, int NT>
__device__ void route_tokens(const RouteParams& r, int t_begin, int t_end) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int warps = blockDim.x >> 5;
  for (int t0 = t_begin + warp; t0 < t_end; t0 += NT * warps) {
    uint32_t key[NT][NL];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int t = t0 + n * warps, e = i * 32 + lane;
        float v = -INFINITY;
        if (t < t_end && e < r.experts) {
          const int64_t at = t * r.ld + e;
          if (r.dtype == 2) v = static_cast<const float*>(r.logits)[at];
          else if (r.dtype == kBF16) v = __bfloat162float(static_cast<const __nv_bfloat16*>(r.logits)[at]);
          else v = __half2float(static_cast<const __half*>(r.logits)[at]);
        }
        key[n][i] = order_key(v);
      }
    float largest[NT], everyone[NT], mine[NT];      // lane j keeps the j-th choice
    int expert[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      largest[n] = everyone[n] = mine[n] = 0.f;
      expert[n] = -1;
    }
    for (int j = 0; j < r.top_k; ++j) {
      uint32_t top[NT];
      unsigned e[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint32_t k = 0;
        e[n] = 0x7fffffffu;
#pragma unroll
        for (int i = 0; i < NL; ++i)
          if (key[n][i] > k) { k = key[n][i]; e[n] = i * 32 + lane; }
        top[n] = __reduce_max_sync(0xffffffffu, k);
        if (k != top[n]) e[n] = 0x7fffffffu;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (top[n] == 0) continue;      // nothing left to choose (the whole warp)
        const int chosen = static_cast<int>(__reduce_min_sync(0xffffffffu, e[n]));
        const float v = key_value(top[n]);
        if (j == 0) {
          largest[n] = v;
          if (!r.renorm) {
#pragma unroll
            for (int i = 0; i < NL; ++i)
              if (key[n][i] != 0) everyone[n] += expf(key_value(key[n][i]) - v);
            everyone[n] = warp_sum(everyone[n]);
          }
        }
        if (lane == j) { expert[n] = chosen; mine[n] = expf(v - largest[n]); }
#pragma unroll
        for (int i = 0; i < NL; ++i)
          if (i * 32 + lane == chosen) key[n][i] = 0;
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int t = t0 + n * warps;
      if (r.renorm) everyone[n] = warp_sum(mine[n]);
      if (t < t_end && lane < r.top_k) {
        const int64_t at = static_cast<int64_t>(t) * r.top_k + lane;
        r.weights[at] = expert[n] >= 0 ? mine[n] / everyone[n] : 0.f;
        r.chosen[at] = expert[n];
      }
    }
  }
}

// NL = 0: the ids are the caller's.  ONE: a single block does everything; otherwise this launch leaves the blocks' counts, and its blocks
// are twice as large where the logits of two tokens leave the registers: the choice of a token is latency, and 128 blocks have an SM each.
template <int NL, bool ONE>
constexpr int group_threads() { return !ONE && NL <= 8 ? 1024 : kThreads; }
template <int NL, bool ONE>
__global__ void __launch_bounds__(group_threads<NL, ONE>()) group_kernel(const RouteParams r, const GroupParams p) {
  __shared__ int base[kMaxGroups], hist[kMaxGroups];
  __shared__ uint16_t wcnt[ONE ? kWarps * kMaxGroups : 1];
  dependency_wait();
  dependency_trigger();
  const int64_t begin64 = static_cast<int64_t>(blockIdx.x) * p.chunk;
  const int begin = static_cast<int>(begin64 < p.n ? begin64 : p.n);
  const int end = begin64 + p.chunk < p.n ? begin + p.chunk : p.n;
  if (NL > 0) {
    const int t0 = blockIdx.x * r.tokens_per_block;
    const int t1 = r.tokens - t0 > r.tokens_per_block ? t0 + r.tokens_per_block : r.tokens;
    route_tokens<NL == 0 ? 1 : NL, NL == 32 ? 1 : 2>(r, t0, t1);
    __syncthreads();
  }
  count_chunk(p, begin, end, hist);
  if (ONE) {
    const int all = scan_groups(p.groups, hist, base);
    for (int g = threadIdx.x; g < p.groups; g += kThreads) p.offsets[g] = base[g];
    if (threadIdx.x == 0) p.offsets[p.groups] = all;
    for (int i = all + threadIdx.x; i < p.n; i += kThreads) p.rows[i] = -1;
    __syncthreads();
    place_chunk(p, begin, end, base, wcnt);
  } else {
    for (int g = threadIdx.x; g < p.groups; g += static_cast<int>(blockDim.x)) p.counts[static_cast<size_t>(blockIdx.x) * p.groups + g] = hist[g];
  }
}

__global__ void __launch_bounds__(kThreads) place_kernel(const GroupParams p) {
  __shared__ int base[kMaxGroups], total[kMaxGroups], pre[kMaxGroups];
  __shared__ uint16_t wcnt[kWarps * kMaxGroups];
  dependency_wait();
  dependency_trigger();
  const int me = blockIdx.x, blocks = gridDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // a warp adds up the counts of every 16th block, eight blocks' loads at once: one trip to L2 where a thread per group took sixteen
  for (int g = threadIdx.x; g < p.groups; g += kThreads) total[g] = pre[g] = 0;
  __syncthreads();
  for (int g = lane; g < p.groups; g += 32) {
    int sum = 0, below = 0;
#pragma unroll
    for (int j = 0; j < kMaxBlocks / kWarps; ++j) {
      const int b = warp + j * kWarps;
      const int c = b < blocks ? p.counts[static_cast<size_t>(b) * p.groups + g] : 0;
      sum += c;
      below += b < me ? c : 0;
    }
    if (sum) atomicAdd(&total[g], sum);
    if (below) atomicAdd(&pre[g], below);
  }
  __syncthreads();
  const int all = scan_groups(p.groups, total, base);
  if (me == 0) {
    for (int g = threadIdx.x; g < p.groups; g += kThreads) p.offsets[g] = base[g];
    if (threadIdx.x == 0) p.offsets[p.groups] = all;
    __syncthreads();
  }
  for (int g = threadIdx.x; g < p.groups; g += kThreads) base[g] += pre[g];
  __syncthreads();
  const int64_t begin64 = static_cast<int64_t>(me) * p.chunk;
  const int begin = static_cast<int>(begin64 < p.n ? begin64 : p.n);
  const int end = begin64 + p.chunk < p.n ? begin + p.chunk : p.n;
  for (int i = (begin > all ? begin : all) + threadIdx.x; i < end; i += kThreads) p.rows[i] = -1;      // behind the last group
  place_chunk(p, begin, end, base, wcnt);
}

template <int NL>
int launch_group(const RouteParams& r, const GroupParams& p, int blocks, cudaStream_t stream) {
  if (blocks == 1) return launch_dependent(group_kernel<NL, true>, 1, kThreads, 0, 0, stream, r, p);
  const int rc = launch_dependent(group_kernel<NL, false>, blocks, group_threads<NL, false>(), 0, 0, stream, r, p);
  if (rc != kOk) return rc;
  return launch_dependent(place_kernel, blocks, kThreads, 0, 0, stream, p);
}

}  // namespace

size_t group_workspace_bytes(int groups) { return static_cast<size_t>(kMaxBlocks) * groups * sizeof(int); }

int launch_group_rows(const GroupArgs& a, cudaStream_t stream) {
  if (a.n < 0 || a.n > kMaxEntries || a.groups < 1 || a.groups > kMaxGroups || a.per_row < 1 || !a.offsets) return kErrInvalid;
  if (a.n > 0 && (!a.ids || !a.rows || !a.slots)) return kErrInvalid;
  GroupParams p{a.ids, a.n, a.groups, a.per_row, 0, static_cast<int*>(a.workspace), a.offsets, a.rows, a.slots};
  // one block to 4096 entries: eight rounds of 512 cost less than a second launch
  const int blocks = a.n <= 4096 ? 1 : kMaxBlocks;
  if (blocks > 1 && !a.workspace) return kErrInvalid;
  p.chunk = blocks == 1 ? a.n : (a.n + blocks - 1) / blocks;
  return launch_group<0>(RouteParams{}, p, blocks, stream);
}

int launch_moe_route(const RouteArgs& a, cudaStream_t stream) {
  if (a.tokens < 0 || a.experts < 1 || a.experts > kMaxGroups || a.top_k < 1 || a.top_k > 32 || a.top_k > a.experts) return kErrInvalid;
  if (a.dtype < 0 || a.dtype > 2 || a.ld < a.experts || !a.offsets) return kErrInvalid;
  if (a.tokens > 0 && (!a.logits || !a.weights || !a.chosen || !a.rows || !a.slots)) return kErrInvalid;
  if (static_cast<int64_t>(a.tokens) * a.top_k > kMaxEntries) return kErrInvalid;
  const int n = a.tokens * a.top_k;
  // to 32 tokens one block (two tokens a warp) costs less than a second launch (6.2 us; 64 tokens 9.8 us, in two launches 6.6); beyond, 16 tokens a
  // block or more
  int per_block = a.tokens;
  if (a.tokens > 32) {
    per_block = (a.tokens + kMaxBlocks - 1) / kMaxBlocks;
    if (per_block < kWarps) per_block = kWarps;
  }
  const int blocks = a.tokens > 0 ? (a.tokens + per_block - 1) / per_block : 1;
  if (blocks > 1 && !a.workspace) return kErrInvalid;
  const RouteParams r{a.logits, a.ld, a.tokens, a.experts, a.top_k, a.dtype, a.renorm, per_block, a.weights, a.chosen};
  const GroupParams p{a.chosen, n, a.experts, a.top_k, per_block * a.top_k, static_cast<int*>(a.workspace), a.offsets, a.rows, a.slots};
  if (a.experts <= 32) return launch_group<1>(r, p, blocks, stream);
  if (a.experts <= 64) return launch_group<2>(r, p, blocks, stream);
  if (a.experts <= 128) return launch_group<4>(r, p, blocks, stream);
  if (a.experts <= 256) return launch_group<8>(r, p, blocks, stream);
  return launch_group<32>(r, p, blocks, stream);
}

}  // namespace sfb200
