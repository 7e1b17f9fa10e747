// extern "C" entry points of the dense block beside the experts: the gated feed-forward
// block and its gradients, MXFP4 quantisation and products (declared in
// include/xk_moe.h). Arguments are checked here, before any launch.
#include "mx4.h"

namespace xk {

int64_t gated_ffn_workspace_bytes(int64_t M, int64_t H, int64_t I);
int64_t gated_ffn_backward_workspace_bytes(int64_t M, int64_t H, int64_t I, int recompute);
int launch_gated_ffn(const void* x, int dtype, int64_t ldx, int64_t M, int64_t H, const void* w13, const void* w2,
                     int64_t I, float limit, void* out, void* gate_up, void* ws, hipStream_t stream);
int launch_gated_ffn_backward(const void* dy, int dtype, int64_t ldg, const void* x, int64_t ldx, int64_t M, int64_t H,
                              const void* w13, const void* w2, int64_t I, const void* gate_up, float limit, void* dx,
                              void* dw13, void* dw2, void* ws, hipStream_t stream);
int launch_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, int dtype, void* out,
                            hipStream_t stream);
int64_t mxfp4_linear_workspace_bytes(int64_t M, int64_t K, int64_t N);
int launch_mxfp4_linear(const void* x, int dtype, int64_t ldx, const uint8_t* x_scales, int64_t M, int64_t K,
                        const uint8_t* codes, const uint8_t* scales, int64_t N, const void* bias, void* out,
                        int out_dtype, void* workspace, hipStream_t stream);

namespace {

// What the kernels' 32-bit offsets within a tile (256 rows) and the launches' grids hold.
constexpr int64_t kMaxRows = int64_t(1) << 29, kMaxCols = 1000000, kMaxApart = 2000000;
constexpr int64_t kMaxTiles = int64_t(1) << 30, kMaxValues = int64_t(1) << 33;

bool any_dtype(int dt) { return dt == XK_DT_BF16 || dt == XK_DT_FP32 || dt == XK_DT_FP16; }
bool at(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// tiles of 64 x 64, more than any kernel here takes
bool fits(int64_t rows, int64_t cols) { return cdiv(rows, 64) * cdiv(cols, 64) <= kMaxTiles; }

int check_workspace(const char* op, const void* ws, int64_t bytes, int64_t need) {
  if (need == 0) return XK_OK;
  if (ws == nullptr || bytes < need)
    return set_error(XK_ERR_WORKSPACE, "%s: workspace %lld B < %lld B", op, (long long)bytes, (long long)need);
  XK_REQUIRE(at(ws, 256), "%s: workspace is not 256-byte aligned", op);
  return XK_OK;
}

int check_ffn(const char* op, int dtype, int64_t M, int64_t H, int64_t I) {
  XK_REQUIRE(dtype == XK_DT_BF16 || dtype == XK_DT_FP16, "%s: dtype code %d is neither bf16 nor fp16", op, dtype);
  XK_REQUIRE(M >= 0 && M < kMaxRows && H >= 1 && H <= kMaxCols && I >= 1 && I <= kMaxCols / 2,
             "%s: bad sizes M=%lld hidden=%lld ispp=%lld", op, (long long)M, (long long)H, (long long)I);
  XK_REQUIRE(fits(M, H) && fits(M, I) && fits(2 * I, H), "%s: more tiles than a launch holds", op);
  return XK_OK;
}

// values that are quantised or restored: the kernels number groups of 4 and more in 32 bits
int check_values(const char* op, int64_t M, int64_t K) {
  XK_REQUIRE(M >= 0 && M < (int64_t(1) << 33) && K >= 1 && K <= (int64_t(1) << 22), "%s: bad sizes M=%lld K=%lld", op,
             (long long)M, (long long)K);
  XK_REQUIRE(M * cdiv(K, 32) * 32 < kMaxValues, "%s: %lld x %lld values, 2^33 or more", op, (long long)M, (long long)K);
  return XK_OK;
}

// rows of n values ld apart that start at 16 bytes, where the width lets them
int check_rows(const char* op, const char* name, const void* p, int64_t rows, int64_t n, int64_t ld) {
  XK_REQUIRE(rows <= 1 || ld >= n, "%s: rows of %s overlap", op, name);
  XK_REQUIRE(rows <= 1 || ld <= kMaxApart, "%s: rows of %s lie more than %lld apart", op, name, (long long)kMaxApart);
  XK_REQUIRE(at(p, 16) && (rows <= 1 || n % 8 != 0 || ld % 8 == 0), "%s: rows of %s do not start at 16 bytes", op, name);
  return XK_OK;
}

}  // namespace
}  // namespace xk

using namespace xk;

extern "C" {

// (the size queries give 0 for sizes that the calls refuse)
int64_t xk_gated_ffn_workspace_bytes(int64_t M, int64_t hidden, int64_t ispp) {
  return check_ffn("gated_ffn", XK_DT_BF16, M, hidden, ispp) ? 0 : gated_ffn_workspace_bytes(M, hidden, ispp);
}

int xk_gated_ffn(const void* x, int32_t dtype, int64_t ldx, int64_t M, int64_t hidden, const void* w13, const void* w2,
                 int64_t ispp, float swiglu_limit, void* out, void* gate_up, void* workspace, int64_t workspace_bytes,
                 hipStream_t stream) {
  clear_error();
  if (int rc = check_ffn("gated_ffn", dtype, M, hidden, ispp)) return rc;
  if (M == 0) return XK_OK;
  XK_REQUIRE(x && w13 && w2 && out, "gated_ffn: null pointer");
  if (int rc = check_rows("gated_ffn", "x", x, M, hidden, ldx)) return rc;
  XK_REQUIRE(at(w13, 16) && at(w2, 16), "gated_ffn: w13 or w2 is not 16-byte aligned");
  if (int rc = check_workspace("gated_ffn", workspace, workspace_bytes, gated_ffn_workspace_bytes(M, hidden, ispp)))
    return rc;
  return launch_gated_ffn(x, dtype, M == 1 ? hidden : ldx, M, hidden, w13, w2, ispp, swiglu_limit, out, gate_up,
                          workspace, stream);
}

int64_t xk_gated_ffn_backward_workspace_bytes(int64_t M, int64_t hidden, int64_t ispp, int32_t recompute) {
  return check_ffn("gated_ffn_backward", XK_DT_BF16, M, hidden, ispp)
             ? 0
             : gated_ffn_backward_workspace_bytes(M, hidden, ispp, recompute);
}

int xk_gated_ffn_backward(const void* grad_out, int32_t dtype, int64_t ldg, const void* x, int64_t ldx, int64_t M,
                          int64_t hidden, const void* w13, const void* w2, int64_t ispp, const void* gate_up,
                          float swiglu_limit, void* grad_x, void* grad_w13, void* grad_w2, void* workspace,
                          int64_t workspace_bytes, hipStream_t stream) {
  clear_error();
  if (int rc = check_ffn("gated_ffn_backward", dtype, M, hidden, ispp)) return rc;
  XK_REQUIRE(w13 && w2 && grad_w13 && grad_w2, "gated_ffn_backward: null pointer");
  XK_REQUIRE(M == 0 || (grad_out && x && grad_x), "gated_ffn_backward: null pointer");
  if (int rc = check_rows("gated_ffn_backward", "grad_out", grad_out, M, hidden, ldg)) return rc;
  if (int rc = check_rows("gated_ffn_backward", "x", x, M, hidden, ldx)) return rc;
  XK_REQUIRE(at(w13, 16) && at(w2, 16), "gated_ffn_backward: w13 or w2 is not 16-byte aligned");
  if (int rc = check_workspace("gated_ffn_backward", workspace, workspace_bytes,
                               gated_ffn_backward_workspace_bytes(M, hidden, ispp, gate_up == nullptr)))
    return rc;
  return launch_gated_ffn_backward(grad_out, dtype, M <= 1 ? hidden : ldg, x, M <= 1 ? hidden : ldx, M, hidden, w13,
                                   w2, ispp, gate_up, swiglu_limit, grad_x, grad_w13, grad_w2, workspace, stream);
}

int xk_mxfp4_quantize(const void* x, int32_t dtype, int64_t ldx, int64_t M, int64_t K, uint8_t* codes,
                      uint8_t* scales, hipStream_t stream) {
  clear_error();
  XK_REQUIRE(any_dtype(dtype), "mxfp4_quantize: dtype code %d is not bf16, fp32 or fp16", dtype);
  if (int rc = check_values("mxfp4_quantize", M, K)) return rc;
  if (M == 0) return XK_OK;
  XK_REQUIRE(x && codes && scales, "mxfp4_quantize: null pointer");
  XK_REQUIRE(M == 1 || ldx >= K, "mxfp4_quantize: rows overlap (ldx)");
  return launch_mxfp4_quantize(x, dtype, ldx, M, K, codes, scales, cdiv(K, 32), ScaleRows{}, stream);
}

int xk_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, int32_t dtype, void* out,
                        hipStream_t stream) {
  clear_error();
  XK_REQUIRE(any_dtype(dtype), "mxfp4_dequantize: dtype code %d is not bf16, fp32 or fp16", dtype);
  if (int rc = check_values("mxfp4_dequantize", M, K)) return rc;
  if (M == 0) return XK_OK;
  XK_REQUIRE(codes && scales && out, "mxfp4_dequantize: null pointer");
  return launch_mxfp4_dequantize(codes, scales, M, K, dtype, out, stream);
}

static int check_linear(int64_t M, int64_t K, int64_t N) {
  XK_REQUIRE(M >= 0 && M < kMaxRows && K >= 1 && K <= kMaxCols && N >= 1 && N <= kMaxCols,
             "mxfp4_linear: bad sizes M=%lld K=%lld N=%lld", (long long)M, (long long)K, (long long)N);
  XK_REQUIRE(fits(M, N), "mxfp4_linear: more tiles than a launch holds");
  return check_values("mxfp4_linear", M, K);
}

int64_t xk_mxfp4_linear_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  return check_linear(M, K, N) ? 0 : mxfp4_linear_workspace_bytes(M, K, N);
}

int xk_mxfp4_linear(const void* x, int32_t dtype, int64_t ldx, const uint8_t* x_scales, int64_t M, int64_t K,
                    const uint8_t* w_codes, const uint8_t* w_scales, int64_t N, const void* bias, void* out,
                    int32_t out_dtype, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  clear_error();
  XK_REQUIRE(x_scales != nullptr || any_dtype(dtype), "mxfp4_linear: dtype code %d is not bf16, fp32 or fp16", dtype);
  XK_REQUIRE(any_dtype(out_dtype), "mxfp4_linear: output dtype code %d is not bf16, fp32 or fp16", out_dtype);
  if (int rc = check_linear(M, K, N)) return rc;
  if (M == 0) return XK_OK;
  XK_REQUIRE(x && w_codes && w_scales && out, "mxfp4_linear: null pointer");
  XK_REQUIRE(x_scales != nullptr || M == 1 || ldx >= K, "mxfp4_linear: rows overlap (ldx)");
  XK_REQUIRE(at(w_codes, 16) && (x_scales == nullptr || at(x, 16)), "mxfp4_linear: codes are not 16-byte aligned");
  XK_REQUIRE(at(w_scales, 4) && at(x_scales, 4), "mxfp4_linear: scales are not 4-byte aligned");
  if (int rc = check_workspace("mxfp4_linear", workspace, workspace_bytes, mxfp4_linear_workspace_bytes(M, K, N)))
    return rc;
  return launch_mxfp4_linear(x, dtype, ldx, x_scales, M, K, w_codes, w_scales, N, bias, out, out_dtype, workspace,
                             stream);
}

}  // extern "C"
