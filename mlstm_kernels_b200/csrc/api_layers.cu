// extern "C" entry points of the operators around a recurrence: argument validation and dispatch.
#include "launch.cuh"

namespace mlstm {

static bool kernel_dtype(int t) { return t == MLSTM_F32 || t == MLSTM_BF16 || t == MLSTM_F16; }
static bool scratch_aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace mlstm

using namespace mlstm;

extern "C" {

size_t mlstm_b200_layer_norm_bw_workspace_bytes(long long rows, int NH, int D) {
  return rows > 0 && NH > 0 && D > 0 ? layer_norm_bw_bytes(rows, NH, D) : 0;
}

int mlstm_b200_layer_norm_fw(const void* x, const long long* x_strides, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                             long long n0, long long n1, int NH, int D, int dtype, int param_dtype, float eps, void* stream) {
  if (!kernel_dtype(dtype) || !kernel_dtype(param_dtype)) return MLSTM_ERR_DTYPE;
  if (!x || !x_strides || !y || (mean == nullptr) != (rstd == nullptr)) return MLSTM_ERR_NULL;
  return launch_layer_norm_fw(x, x_strides, weight, bias, y, mean, rstd, n0, n1, NH, D, dtype, param_dtype, eps, static_cast<cudaStream_t>(stream));
}

int mlstm_b200_layer_norm_bw(const void* x, const long long* x_strides, const void* weight, const float* mean, const float* rstd, const void* dy,
                             const long long* dy_strides, void* dx, const long long* dx_strides, void* dw, void* db, void* workspace,
                             size_t workspace_bytes, long long n0, long long n1, int NH, int D, int dtype, int param_dtype, void* stream) {
  if (!kernel_dtype(dtype) || !kernel_dtype(param_dtype)) return MLSTM_ERR_DTYPE;
  if (n0 <= 0 || n1 <= 0 || NH <= 0 || D <= 0) return MLSTM_ERR_SHAPE;
  if (!x || !x_strides || !mean || !rstd || !dy || !dy_strides || !dx || !dx_strides) return MLSTM_ERR_NULL;
  if (dw || db) {
    if (!workspace) return MLSTM_ERR_NULL;
    if (!scratch_aligned(workspace)) return MLSTM_ERR_ALIGN;
    if (workspace_bytes < layer_norm_bw_bytes(n0 * n1, NH, D)) return MLSTM_ERR_WORKSPACE;
  }
  return launch_layer_norm_bw(x, x_strides, weight, mean, rstd, dy, dy_strides, dx, dx_strides, dw, db, static_cast<float*>(workspace), n0, n1, NH, D,
                              dtype, param_dtype, static_cast<cudaStream_t>(stream));
}

size_t mlstm_b200_short_conv_bw_workspace_bytes(int B, int S, int D, int W) {
  return B > 0 && S > 0 && D > 0 && W >= 2 && W <= 4 ? short_conv_bw_bytes(B, S, D, W) : 0;
}

int mlstm_b200_short_conv_fw(const void* x, const long long* x_strides, const void* x_initial, const void* weight, const void* bias, void* y,
                             void* x_last, int B, int S, int D, int W, int silu, int dtype, int w_dtype, void* stream) {
  if (!kernel_dtype(dtype) || !kernel_dtype(w_dtype)) return MLSTM_ERR_DTYPE;
  if (!x || !x_strides || !weight || !y) return MLSTM_ERR_NULL;
  return launch_short_conv_fw(x, x_strides, x_initial, weight, bias, y, x_last, B, S, D, W, silu != 0, dtype, w_dtype, static_cast<cudaStream_t>(stream));
}

int mlstm_b200_short_conv_bw(const void* x, const long long* x_strides, const void* x_initial, const void* weight, const void* bias, const void* dy,
                             const long long* dy_strides, const void* dx_last, void* dx, void* dx_initial, void* dw, void* db, void* workspace,
                             size_t workspace_bytes, int B, int S, int D, int W, int silu, int dtype, int w_dtype, void* stream) {
  if (!kernel_dtype(dtype) || !kernel_dtype(w_dtype)) return MLSTM_ERR_DTYPE;
  if (B <= 0 || S <= 0 || D <= 0 || W < 2 || W > 4) return MLSTM_ERR_SHAPE;
  if (!x || !x_strides || !weight || !dy || !dy_strides || !dx) return MLSTM_ERR_NULL;
  if (dw || db) {
    if (!workspace) return MLSTM_ERR_NULL;
    if (!scratch_aligned(workspace)) return MLSTM_ERR_ALIGN;
    if (workspace_bytes < short_conv_bw_bytes(B, S, D, W)) return MLSTM_ERR_WORKSPACE;
  }
  return launch_short_conv_bw(x, x_strides, x_initial, weight, bias, dy, dy_strides, dx_last, dx, dx_initial, dw, db, static_cast<float*>(workspace), B, S,
                              D, W, silu != 0, dtype, w_dtype, static_cast<cudaStream_t>(stream));
}

int mlstm_b200_short_conv_step(const void* x, const void* state, const void* weight, const void* bias, void* y, void* state_new, int B, int D, int W,
                               int silu, int dtype, int w_dtype, void* stream) {
  if (!kernel_dtype(dtype) || !kernel_dtype(w_dtype)) return MLSTM_ERR_DTYPE;
  if (!x || !state || !weight || !y || !state_new) return MLSTM_ERR_NULL;
  return launch_short_conv_step(x, state, weight, bias, y, state_new, B, D, W, silu != 0, dtype, w_dtype, static_cast<cudaStream_t>(stream));
}

size_t mlstm_b200_ssm_checkpoint_bytes(int B, int S, int D, int N) { return ssm_sizes_ok(B, S, D, N, 1) ? ssm_ckpt_bytes(B, S, D, N) : 0; }
size_t mlstm_b200_ssm_workspace_bytes(int B, int S, int D, int N, int G, int backward) {
  return !ssm_sizes_ok(B, S, D, N, G) ? 0 : backward ? ssm_bw_bytes(B, S, D, N, G) : ssm_fw_bytes(B, S, D, N, G);
}

int mlstm_b200_ssm_scan_fw(const void* x, const void* dt, const float* a, const void* b, const void* c, const float* skip, const void* z,
                           const float* dt_bias, const float* h_initial, const long long* strides, void* y, float* h_last, void* checkpoints,
                           void* workspace, size_t workspace_bytes, int B, int S, int D, int N, int G, int softplus, int dtype, void* stream) {
  if (!kernel_dtype(dtype)) return MLSTM_ERR_DTYPE;
  if (!ssm_sizes_ok(B, S, D, N, G)) return MLSTM_ERR_SHAPE;
  if (!x || !dt || !a || !b || !c || !strides || !y) return MLSTM_ERR_NULL;
  const size_t need = ssm_fw_bytes(B, S, D, N, G);
  if (need > 0 && !workspace) return MLSTM_ERR_NULL;
  if (!scratch_aligned(workspace) || !scratch_aligned(checkpoints)) return MLSTM_ERR_ALIGN;
  if (workspace_bytes < need) return MLSTM_ERR_WORKSPACE;
  return launch_ssm_fw(SsmIn{x, dt, z, b, c, a, skip, dt_bias, h_initial}, strides, y, h_last, static_cast<float*>(checkpoints), workspace, B, S, D, N, G,
                       softplus != 0, dtype, static_cast<cudaStream_t>(stream));
}

int mlstm_b200_ssm_scan_bw(const void* x, const void* dt, const float* a, const void* b, const void* c, const float* skip, const void* z,
                           const float* dt_bias, const long long* strides, const void* checkpoints, const void* dy, const long long* dy_strides,
                           const float* dh_last, void* dx, void* ddt, float* da, void* db, void* dc, float* dskip, void* dz, float* ddt_bias,
                           float* dh_initial, void* workspace, size_t workspace_bytes, int B, int S, int D, int N, int G, int softplus, int dtype,
                           void* stream) {
  if (!kernel_dtype(dtype)) return MLSTM_ERR_DTYPE;
  if (!ssm_sizes_ok(B, S, D, N, G)) return MLSTM_ERR_SHAPE;
  if (!x || !dt || !a || !b || !c || !strides || !checkpoints || !dy || !dy_strides || !dx || !ddt || !da || !db || !dc || !workspace) return MLSTM_ERR_NULL;
  if ((z != nullptr) != (dz != nullptr)) return MLSTM_ERR_NULL;
  if (!scratch_aligned(workspace) || !scratch_aligned(checkpoints)) return MLSTM_ERR_ALIGN;
  if (workspace_bytes < ssm_bw_bytes(B, S, D, N, G)) return MLSTM_ERR_WORKSPACE;
  return launch_ssm_bw(SsmIn{x, dt, z, b, c, a, skip, dt_bias, nullptr}, strides, dy, dy_strides, dh_last, static_cast<const float*>(checkpoints), dx, ddt,
                       dz, db, dc, da, dskip, ddt_bias, dh_initial, workspace, B, S, D, N, G, softplus != 0, dtype, static_cast<cudaStream_t>(stream));
}

int mlstm_b200_ssm_step(const void* x, const void* dt, const float* a, const void* b, const void* c, const float* skip, const void* z,
                        const float* dt_bias, const float* h, void* y, float* h_new, int B, int D, int N, int G, int softplus, int dtype, void* stream) {
  if (!kernel_dtype(dtype)) return MLSTM_ERR_DTYPE;
  if (!x || !dt || !a || !b || !c || !h || !y || !h_new) return MLSTM_ERR_NULL;
  return launch_ssm_step(x, dt, z, b, c, a, skip, dt_bias, h, y, h_new, B, D, N, G, softplus != 0, dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
