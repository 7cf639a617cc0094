// C-ABI launcher of the LayerNorm backward pass for F16 rows.
#include "layernorm_backward_launch.h"

extern "C" int ko_layernorm_backward_f16(const uint16_t *dy, const uint16_t *x, uint16_t *dx, int64_t rows, int32_t cols, float eps,
                              const uint16_t *gamma, const uint16_t *residual, float *dgamma, float *dbeta, int ddof,
                              void *workspace, size_t workspace_bytes, void *stream) {
    using T = __half;
    return ko::ln_backward::dispatch<T>(KO_DTYPE_F16, reinterpret_cast<const T *>(dy), reinterpret_cast<const T *>(x), reinterpret_cast<T *>(dx), rows, cols,
                       eps, reinterpret_cast<const T *>(gamma), reinterpret_cast<const T *>(residual), dgamma, dbeta, ddof, workspace,
                       workspace_bytes, stream);
}
