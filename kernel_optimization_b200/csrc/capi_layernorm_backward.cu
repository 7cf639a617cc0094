// C-ABI launchers of the LayerNorm backward pass: the workspace query and FP32 rows.
#include "layernorm_backward_launch.h"

using namespace ko::ln_backward;

extern "C" {

int ko_layernorm_backward_workspace(int dtype, int64_t rows, int32_t cols, size_t *bytes) {
    KO_REQUIRE(bytes != nullptr, KO_ERR_INVALID_ARG, "layernorm backward: NULL bytes");
    *bytes = 0;
    KO_REQUIRE(dtype >= KO_DTYPE_F32 && dtype <= KO_DTYPE_BF16, KO_ERR_INVALID_ARG, "layernorm backward: unknown dtype %d", dtype);
    if (int st = check_shape(rows, cols)) return st;
    if (rows == 0 || cols == 0) return KO_OK;
    ko::DeviceInfo info;
    if (int st = ko::current_device_info(&info)) return st;
    *bytes = workspace_for(dtype, rows, cols, info);
    return KO_OK;
}

int ko_layernorm_backward_f32(const float *dy, const float *x, float *dx, int64_t rows, int32_t cols, float eps, const float *gamma,
                              const float *residual, float *dgamma, float *dbeta, int ddof, void *workspace,
                              size_t workspace_bytes, void *stream) {
    return dispatch<float>(KO_DTYPE_F32, dy, x, dx, rows, cols, eps, gamma, residual, dgamma, dbeta, ddof, workspace, workspace_bytes, stream);
}

}  // extern "C"
