// C-ABI entry points of the operators around the gated FFN (group 1b of include/sparseflow_b200.h).
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/sparseflow_b200.h"
#include "device_state.h"
#include "kernels.h"

using namespace sfb200;

extern "C" {

size_t sfb200_group_workspace_bytes(int groups) { return groups > 0 ? group_workspace_bytes(groups) : 0; }

int sfb200_group_rows(const int* ids, int n, int groups, int per_row, int* offsets, int* rows, int* slots, void* workspace, void* stream) {
  int err = kOk;
  if (!device_state(&err)) return err;
  return launch_group_rows(GroupArgs{ids, n, groups, per_row, offsets, rows, slots, workspace}, static_cast<cudaStream_t>(stream));
}

int sfb200_moe_route(const void* logits, int64_t ld, int tokens, int experts, int top_k, int dtype, int renormalize, float* weights, int* chosen,
                     int* offsets, int* rows, int* slots, void* workspace, void* stream) {
  int err = kOk;
  if (!device_state(&err)) return err;
  return launch_moe_route(RouteArgs{logits, ld, tokens, experts, top_k, dtype, renormalize, weights, chosen, offsets, rows, slots, workspace},
                          static_cast<cudaStream_t>(stream));
}

static int grouped(const void* x, int ldx, int x_rows, const int* rows, void* scratch, const void* values, const void* meta, void* y, int ldy,
                   int total, int experts, int N, int K, int dtype, const void* bias, const void* bias_up, int act, int epi, const int* offsets,
                   void* stream) {
  int err = kOk;
  DeviceState* s = device_state(&err);
  if (!s) return err;
  GroupedGemmArgs a{};
  a.x = x;
  a.values = values;
  a.meta = meta;
  a.bias = bias;
  a.bias_up = bias_up;
  a.offsets = offsets;
  a.rows = rows;
  a.scratch = scratch;
  a.variant = s->force_grouped;
  a.y = y;
  a.status = s->status;
  a.x_rows = x_rows;
  a.total = total;
  a.experts = experts;
  a.n_out = N;
  a.K = K;
  a.ldx = ldx;
  a.ldy = ldy;
  a.fmt = dtype;
  a.epi = epi;
  a.act = act;
  a.num_sms = s->num_sms;
  return launch_grouped_gemm(a, static_cast<cudaStream_t>(stream));
}

size_t sfb200_grouped_scratch_bytes(int total, int experts, int N, int K) {
  int err = kOk;
  DeviceState* s = device_state(&err);
  if (!s || total <= 0 || experts <= 0 || N <= 0 || K <= 0) return 0;
  const int variant = s->force_grouped ? s->force_grouped : plan_grouped(total, experts, N, K, true, s->num_sms);
  return variant >= 10000 ? static_cast<size_t>(total) * K * 2 : 0;
}

/* Which form a grouped product over `total` places runs on a GPU with num_sms SMs: 32 / 64 single-CTA tiles of that many tokens; 1128, 1240 /
 * 2128, 2240 CTA-pair tiles of 256 / 512 rows; 10000 more: rows copied into the order of the experts first.  Host-only. */
SFB200_API int sfb200_debug_plan_grouped(int total, int experts, int N, int K, int gather, int num_sms) {
  if (total <= 0 || experts <= 0 || N <= 0 || K <= 0 || num_sms <= 0) return 0;
  return plan_grouped(total, experts, N, K, gather != 0, num_sms);
}

/* Test hook: force the form of grouped products (0 = automatic). */
SFB200_API int sfb200_debug_force_grouped(int variant) {
  int err = kOk;
  DeviceState* s = device_state(&err);
  if (!s) return err;
  s->force_grouped = variant;
  return kOk;
}

int sfb200_grouped_sparse_gemm(const void* x, int ldx, int x_rows, const int* rows, void* scratch, const void* values, const void* meta, void* y,
                               int ldy, int total, int experts, int N, int K, int dtype, const void* bias, int act, const int* offsets, void* stream) {
  return grouped(x, ldx, x_rows, rows, scratch, values, meta, y, ldy, total, experts, N, K, dtype, bias, nullptr, act, kEpiStore, offsets, stream);
}

int sfb200_grouped_sparse_gemm_swiglu(const void* x, int ldx, int x_rows, const int* rows, void* scratch, const void* values_gu, const void* meta_gu,
                                      void* h, int ldh, int total, int experts, int I, int K, int dtype, const void* gate_bias, const void* up_bias,
                                      const int* offsets, void* stream) {
  if (I <= 0 || I > 0x3fffffff) return kErrInvalid;
  return grouped(x, ldx, x_rows, rows, scratch, values_gu, meta_gu, h, ldh, total, experts, 2 * I, K, dtype, gate_bias, up_bias, kActNone, kEpiSwiGLU,
                 offsets, stream);
}

int sfb200_moe_combine(const void* y, int64_t ld_y, int y_rows, const int* slots, const float* weights, const void* residual, int64_t ld_res,
                       void* out, int64_t ld_out, int tokens, int top_k, int cols, int dtype, void* stream) {
  int err = kOk;
  if (!device_state(&err)) return err;
  return launch_moe_combine(CombineArgs{y, ld_y, y_rows, slots, weights, residual, ld_res, out, ld_out, tokens, top_k, cols, dtype},
                            static_cast<cudaStream_t>(stream));
}

int sfb200_block_norm(const void* x, int64_t ld_x, const void* y, int64_t ld_y, const void* weight, const void* bias, const void* post_weight,
                      const void* post_bias, const void* gate, int64_t ld_gate, int gate_rows, int gate_cols, void* r, int64_t ld_r, void* h,
                      int64_t ld_h, int rows, int cols, int x_type, int y_type, float scale, float eps, float post_eps, int layer, void* stream) {
  int err = kOk;
  DeviceState* s = device_state(&err);
  if (!s) return err;
  NormArgs a{};
  a.x = x; a.y = y; a.weight = weight; a.bias = bias; a.post_weight = post_weight; a.post_bias = post_bias; a.gate = gate;
  a.r = r; a.h = h;
  a.ld_x = ld_x; a.ld_y = ld_y; a.ld_r = ld_r; a.ld_h = ld_h; a.ld_gate = ld_gate;
  a.rows = rows; a.cols = cols; a.gate_rows = gate_rows; a.gate_cols = gate_cols;
  a.x_type = x_type; a.y_type = y_type;
  a.num_sms = s->num_sms;
  a.scale = scale; a.eps = eps; a.post_eps = post_eps; a.layer = layer;
  return launch_block_norm(a, static_cast<cudaStream_t>(stream));
}

size_t sfb200_lora_workspace_bytes(int n, int rank) { return n > 0 && rank > 0 ? lora_workspace_bytes(n, rank) : 0; }

int sfb200_lora_add(const void* y, int64_t ld_y, const void* x, int64_t ld_x, const void* a, const void* b, const float* scales, void* out,
                    int64_t ld_out, int n, int groups, int rank, int K, int N, int dtype, const int* offsets, const int* rows, const int* slots,
                    void* workspace, void* stream) {
  int err = kOk;
  DeviceState* s = device_state(&err);
  if (!s) return err;
  LoraArgs l{};
  l.y = y; l.x = x; l.a = a; l.b = b; l.scales = scales; l.out = out;
  l.offsets = offsets; l.rows = rows; l.slots = slots; l.workspace = workspace;
  l.ld_y = ld_y; l.ld_x = ld_x; l.ld_out = ld_out;
  l.n = n; l.groups = groups; l.rank = rank; l.K = K; l.N = N; l.fmt = dtype; l.num_sms = s->num_sms;
  return launch_lora_add(l, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
