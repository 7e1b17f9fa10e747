// extern "C" entry points for tuning and serving over the frozen experts: the
// router's training step, low-rank adapters, activation checkpoints (declared in
// include/xk_moe.h). Arguments are checked here, before any launch.
#include "common.h"

namespace xk {

int64_t balance_workspace_bytes(int64_t M, int64_t E);
int launch_balance_loss(const void* logits, int dtype, int64_t M, int64_t E, const int32_t* ids, int64_t k,
                        const uint8_t* mask, float* loss, int32_t* counts, int32_t* tokens, void* workspace,
                        hipStream_t stream);
int launch_router_backward(const void* logits, int dtype, int64_t M, int64_t E, const int32_t* ids, int64_t k,
                           const uint8_t* mask, const int32_t* counts, const int32_t* tokens, const float* grad_loss,
                           const float* grad_weights, int renorm, void* grad, hipStream_t stream);
int lora_max_rank();
int64_t lora_workspace_bytes(int64_t M, int64_t K, int64_t L, int64_t r);
int64_t lora_backward_workspace_bytes(int64_t M, int64_t K, int64_t N, int64_t L, int64_t r, int dtype);
int launch_lora(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, const void* a, const void* b, int64_t L,
                int64_t N, int64_t r, const int32_t* ids, const float* scaling, const void* base, int64_t ldbase,
                void* out, float* hidden, void* ws, hipStream_t stream);
int launch_lora_backward(const void* dy, int dtype, int64_t lddy, const void* x, int64_t ldx, const uint8_t* x_scales,
                         int64_t M, int64_t K, const void* a, const void* b, int64_t L, int64_t N, int64_t r,
                         const int32_t* ids, const float* scaling, const float* hidden, void* dx, void* da, void* db,
                         void* ws, hipStream_t stream);
int launch_act_checkpoint(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, uint8_t* values,
                          uint8_t* scales, hipStream_t stream);
int launch_act_restore(const uint8_t* values, const uint8_t* scales, int64_t M, int64_t K, int dtype, void* out,
                       hipStream_t stream);

namespace {

// Sizes past these do not occur and keep every product below in 64 bits.
constexpr int64_t kMaxRows = int64_t(1) << 30, kMaxCols = int64_t(1) << 24;
constexpr int kMaxAdapters = 1024;
// of adapters: what the launches' grids hold at any rank and type
constexpr int64_t kMaxLoraRows = int64_t(1) << 29, kMaxLoraCols = 1000000;

bool any_dtype(int dt) { return dt == XK_DT_BF16 || dt == XK_DT_FP32 || dt == XK_DT_FP16; }

int check_router(const char* op, int dtype, int64_t M, int64_t E, int64_t k) {
  XK_REQUIRE(any_dtype(dtype), "%s: dtype code %d is not bf16, fp32 or fp16", op, dtype);
  XK_REQUIRE(M >= 0 && M < kMaxRows && E >= 1 && E <= kMaxCols, "%s: bad sizes M=%lld E=%lld", op, (long long)M,
             (long long)E);
  XK_REQUIRE(k >= 1 && k <= E, "%s: top_k=%lld outside [1, E=%lld]", op, (long long)k, (long long)E);
  XK_REQUIRE(M * k < (int64_t(1) << 31), "%s: M*top_k=%lld does not fit the counts", op, (long long)(M * k));
  return XK_OK;
}

int check_lora(const char* op, int dtype, int64_t M, int64_t K, int64_t N, int64_t L, int64_t r) {
  XK_REQUIRE(dtype == XK_DT_BF16 || dtype == XK_DT_FP32, "%s: dtype code %d is neither bf16 nor fp32", op, dtype);
  XK_REQUIRE(M >= 0 && M < kMaxLoraRows && K >= 1 && K <= kMaxLoraCols && N >= 1 && N <= kMaxLoraCols,
             "%s: bad sizes M=%lld K=%lld N=%lld", op, (long long)M, (long long)K, (long long)N);
  XK_REQUIRE(L >= 1 && L <= kMaxAdapters, "%s: %lld adapters, outside [1, %d]", op, (long long)L, kMaxAdapters);
  XK_REQUIRE(r >= 1 && r <= lora_max_rank(), "%s: rank %lld outside [1, %d]", op, (long long)r, lora_max_rank());
  return XK_OK;
}

int check_workspace(const char* op, const void* ws, int64_t bytes, int64_t need) {
  if (need == 0) return XK_OK;
  if (ws == nullptr || bytes < need)
    return set_error(XK_ERR_WORKSPACE, "%s: workspace %lld B < %lld B", op, (long long)bytes, (long long)need);
  XK_REQUIRE(reinterpret_cast<uintptr_t>(ws) % 16 == 0, "%s: workspace is not 16-byte aligned", op);
  return XK_OK;
}

}  // namespace
}  // namespace xk

using namespace xk;

extern "C" {

// (the size queries give 0 for sizes that the calls refuse)
int64_t xk_moe_balance_loss_workspace_bytes(int64_t M, int64_t E) {
  return check_router("balance_loss", XK_DT_FP32, M, E, 1) ? 0 : balance_workspace_bytes(M, E);
}

int xk_moe_balance_loss(const void* gating_output, int32_t dtype, int64_t M, int64_t E, const int32_t* topk_ids,
                        int64_t top_k, const uint8_t* mask, float* loss, int32_t* counts, int32_t* tokens,
                        void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  clear_error();
  if (int rc = check_router("balance_loss", dtype, M, E, top_k)) return rc;
  XK_REQUIRE(M == 0 || (gating_output && topk_ids), "balance_loss: null input pointer");
  XK_REQUIRE(loss && counts && tokens, "balance_loss: null output pointer");
  if (int rc = check_workspace("balance_loss", workspace, workspace_bytes, balance_workspace_bytes(M, E))) return rc;
  return launch_balance_loss(gating_output, dtype, M, E, topk_ids, top_k, mask, loss, counts, tokens, workspace,
                             stream);
}

int xk_moe_router_backward(const void* gating_output, int32_t dtype, int64_t M, int64_t E, const int32_t* topk_ids,
                           int64_t top_k, const uint8_t* mask, const float* grad_loss, const int32_t* counts,
                           const int32_t* tokens, const float* grad_weights, int32_t renormalize, void* grad_gating,
                           hipStream_t stream) {
  clear_error();
  if (int rc = check_router("router_backward", dtype, M, E, top_k)) return rc;
  XK_REQUIRE(M == 0 || grad_loss || grad_weights, "router_backward: neither grad_loss nor grad_weights");
  XK_REQUIRE(!grad_loss || counts, "router_backward: grad_loss needs the counts");
  if (M == 0) return XK_OK;
  XK_REQUIRE(gating_output && topk_ids && grad_gating, "router_backward: null pointer");
  return launch_router_backward(gating_output, dtype, M, E, topk_ids, top_k, mask, counts, tokens, grad_loss,
                                grad_weights, renormalize != 0, grad_gating, stream);
}

int64_t xk_lora_projection_workspace_bytes(int64_t M, int64_t K, int64_t L, int64_t r) {
  return check_lora("lora_projection", XK_DT_BF16, M, K, 1, L, r) ? 0 : lora_workspace_bytes(M, K, L, r);
}

int xk_lora_projection(const void* x, int32_t dtype, int64_t ldx, int64_t M, int64_t K, const void* lora_a,
                       const void* lora_b, int64_t L, int64_t N, int64_t r, const int32_t* adapter_ids,
                       const float* scaling, const void* base, int64_t ldbase, void* out, float* hidden,
                       void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  clear_error();
  if (int rc = check_lora("lora_projection", dtype, M, K, N, L, r)) return rc;
  if (M == 0) return XK_OK;
  XK_REQUIRE(x && lora_a && lora_b && adapter_ids && out, "lora_projection: null pointer");
  XK_REQUIRE(M == 1 || (ldx >= K && (base == nullptr || ldbase >= N)), "lora_projection: rows overlap (ldx, ldbase)");
  XK_REQUIRE(base != out || ldbase == N, "lora_projection: out is base, but rows are not N apart");
  if (int rc = check_workspace("lora_projection", workspace, workspace_bytes, lora_workspace_bytes(M, K, L, r)))
    return rc;
  return launch_lora(x, dtype, ldx, M, K, lora_a, lora_b, L, N, r, adapter_ids, scaling, base, ldbase, out, hidden,
                     workspace, stream);
}

int64_t xk_lora_projection_backward_workspace_bytes(int64_t M, int64_t K, int64_t N, int64_t L, int64_t r,
                                                    int32_t dtype) {
  return check_lora("lora_projection_backward", dtype, M, K, N, L, r)
             ? 0
             : lora_backward_workspace_bytes(M, K, N, L, r, dtype);
}

int xk_lora_projection_backward(const void* grad_out, int32_t dtype, int64_t ldg, const void* x, int64_t ldx,
                                const uint8_t* x_scales, int64_t M, int64_t K, const void* lora_a,
                                const void* lora_b, int64_t L, int64_t N, int64_t r, const int32_t* adapter_ids,
                                const float* scaling, const float* hidden, void* grad_x, void* grad_a, void* grad_b,
                                void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  clear_error();
  if (int rc = check_lora("lora_projection_backward", dtype, M, K, N, L, r)) return rc;
  XK_REQUIRE(lora_a && lora_b && grad_a && grad_b, "lora_projection_backward: null pointer");
  XK_REQUIRE(M == 0 || (grad_out && x && adapter_ids && hidden && grad_x), "lora_projection_backward: null pointer");
  XK_REQUIRE(M <= 1 || (ldx >= K && ldg >= N), "lora_projection_backward: rows overlap (ldx, ldg)");
  XK_REQUIRE(x_scales == nullptr || M <= 1 || ldx == K, "lora_projection_backward: 8-bit rows are K apart");
  if (int rc = check_workspace("lora_projection_backward", workspace, workspace_bytes,
                               lora_backward_workspace_bytes(M, K, N, L, r, dtype)))
    return rc;
  return launch_lora_backward(grad_out, dtype, ldg, x, ldx, x_scales, M, K, lora_a, lora_b, L, N, r, adapter_ids,
                              scaling, hidden, grad_x, grad_a, grad_b, workspace, stream);
}

int xk_act_checkpoint(const void* x, int32_t dtype, int64_t ldx, int64_t M, int64_t K, uint8_t* values,
                      uint8_t* scales, hipStream_t stream) {
  clear_error();
  XK_REQUIRE(any_dtype(dtype), "act_checkpoint: dtype code %d is not bf16, fp32 or fp16", dtype);
  XK_REQUIRE(M >= 0 && M < kMaxRows && K >= 1 && K <= kMaxCols, "act_checkpoint: bad sizes M=%lld K=%lld",
             (long long)M, (long long)K);
  if (M == 0) return XK_OK;
  XK_REQUIRE(x && values && scales, "act_checkpoint: null pointer");
  XK_REQUIRE(M == 1 || ldx >= K, "act_checkpoint: rows overlap (ldx)");
  return launch_act_checkpoint(x, dtype, ldx, M, K, values, scales, stream);
}

int xk_act_restore(const uint8_t* values, const uint8_t* scales, int64_t M, int64_t K, int32_t dtype, void* out,
                   hipStream_t stream) {
  clear_error();
  XK_REQUIRE(any_dtype(dtype), "act_restore: dtype code %d is not bf16, fp32 or fp16", dtype);
  XK_REQUIRE(M >= 0 && M < kMaxRows && K >= 1 && K <= kMaxCols, "act_restore: bad sizes M=%lld K=%lld", (long long)M,
             (long long)K);
  if (M == 0) return XK_OK;
  XK_REQUIRE(values && scales && out, "act_restore: null pointer");
  return launch_act_restore(values, scales, M, K, dtype, out, stream);
}

}  // extern "C"
