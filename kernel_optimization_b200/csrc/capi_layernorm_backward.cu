// C-ABI launchers of the LayerNorm backward pass.
#include "row_launch.h"

#include <algorithm>

#include "../nn_operators/layernorm/layernorm_backward.h"

namespace {

// How a call is cut up; the same for the workspace query and the call itself.
struct Plan {
    bool vec;           // 16-byte accesses
    int row_chunks;     // blocks along the rows = partial rows
    size_t terms_bytes; // row terms, rounded up to 16 bytes
    size_t bytes;       // whole workspace
};

Plan plan_for(int dtype, int64_t rows, int cols, bool aligned, const ko::DeviceInfo &info) {
    Plan p{};
    const int per_vec = dtype == KO_DTYPE_F32 ? 4 : 8;
    p.vec = aligned && cols % per_vec == 0;
    // Row chunks for eight blocks of 256 threads per SM whichever access width is used, so that the workspace does not
    // depend on the pointers; a chunk has at least 8 rows, one for each of the block's warps.
    const int64_t strips = (cols + 32 * per_vec - 1) / (32 * per_vec);
    const int64_t wanted = std::max<int64_t>(1, 8LL * info.sm_count / strips);
    p.row_chunks = (int)std::min<int64_t>(std::min<int64_t>(wanted, (rows + 7) / 8), 65535);
    p.terms_bytes = (size_t)rows * sizeof(ko::LayerNormRowTerms);
    p.bytes = p.terms_bytes + (size_t)p.row_chunks * 2 * (size_t)cols * sizeof(float);
    return p;
}

int check_shape(int64_t rows, int32_t cols) {
    KO_REQUIRE(rows >= 0 && cols >= 0, KO_ERR_INVALID_ARG, "layernorm backward: negative shape [%lld, %d]", (long long)rows, cols);
    KO_REQUIRE(cols <= (1 << 30), KO_ERR_SHAPE, "layernorm backward: %d columns, at most 2^30", cols);
    return KO_OK;
}

template <typename T, int E>
int launch(const ko::LayerNormBackwardArgs<T> &a, const Plan &plan, const ko::DeviceInfo &info, ko::LayerNormRowTerms *terms,
           float *dgamma, float *dbeta, cudaStream_t s) {
    const unsigned blocks = ko::clamp_grid(a.rows, 8LL * info.sm_count);
    if (int st = ko::launch_overlapped(ko::layernorm_backward_terms_kernel<T, E>, blocks, 256u, 0, s, a, terms)) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.cols + 32 * E - 1) / (32 * E)), (unsigned)plan.row_chunks, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    KO_CUDA(cudaLaunchKernelEx(&cfg, ko::layernorm_backward_apply_kernel<T, E>, a, (const ko::LayerNormRowTerms *)terms));
    if (a.partials == nullptr) return KO_OK;
    return ko::launch_overlapped(ko::layernorm_backward_fold_kernel<>, (unsigned)((a.cols + 31) / 32), 256u, 0, s, a.partials,
                                 plan.row_chunks, a.cols, dgamma, dbeta);
}

template <typename T>
int dispatch(int dtype, const T *dy, const T *x, T *dx, int64_t rows, int32_t cols, float eps, const T *gamma, const T *residual,
             float *dgamma, float *dbeta, int ddof, void *workspace, size_t workspace_bytes, void *stream) {
    if (int st = check_shape(rows, cols)) return st;
    KO_REQUIRE(ddof == 0 || ddof == 1, KO_ERR_INVALID_ARG, "layernorm backward: ddof must be 0 or 1, got %d", ddof);
    if (cols == 0) return KO_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (rows == 0) {  // sums over no rows
        if (dgamma) KO_CUDA(cudaMemsetAsync(dgamma, 0, (size_t)cols * sizeof(float), s));
        if (dbeta) KO_CUDA(cudaMemsetAsync(dbeta, 0, (size_t)cols * sizeof(float), s));
        return KO_OK;
    }
    KO_REQUIRE(dy != nullptr && x != nullptr && dx != nullptr, KO_ERR_INVALID_ARG, "layernorm backward: NULL pointer");
    KO_REQUIRE(dgamma == nullptr || dgamma != dbeta, KO_ERR_INVALID_ARG, "layernorm backward: dgamma and dbeta must not be the same buffer");
    ko::DeviceInfo info;
    if (int st = ko::current_device_info(&info)) return st;
    const bool aligned = ko::aligned16(dy) && ko::aligned16(x) && ko::aligned16(dx) && (!gamma || ko::aligned16(gamma)) &&
                         (!residual || ko::aligned16(residual));
    const Plan plan = plan_for(dtype, rows, cols, aligned, info);
    KO_REQUIRE(workspace != nullptr && workspace_bytes >= plan.bytes, KO_ERR_INVALID_ARG,
               "layernorm backward: the workspace needs %zu bytes, got %zu", plan.bytes, workspace ? workspace_bytes : (size_t)0);
    KO_REQUIRE(ko::aligned16(workspace), KO_ERR_ALIGN, "layernorm backward: the workspace must be 16-byte aligned");
    auto *terms = static_cast<ko::LayerNormRowTerms *>(workspace);
    float *partials = dgamma || dbeta ? reinterpret_cast<float *>(static_cast<char *>(workspace) + plan.terms_bytes) : nullptr;
    const ko::LayerNormBackwardArgs<T> a{dy, x, dx, rows, cols, eps, gamma, residual, partials, ddof};
    if (plan.vec) return launch<T, ko::RowIo<T>::kPerVec>(a, plan, info, terms, dgamma, dbeta, s);
    return launch<T, 1>(a, plan, info, terms, dgamma, dbeta, s);
}

}  // namespace

extern "C" {

int ko_layernorm_backward_workspace(int dtype, int64_t rows, int32_t cols, size_t *bytes) {
    KO_REQUIRE(bytes != nullptr, KO_ERR_INVALID_ARG, "layernorm backward: NULL bytes");
    *bytes = 0;
    KO_REQUIRE(dtype >= KO_DTYPE_F32 && dtype <= KO_DTYPE_BF16, KO_ERR_INVALID_ARG, "layernorm backward: unknown dtype %d", dtype);
    if (int st = check_shape(rows, cols)) return st;
    if (rows == 0 || cols == 0) return KO_OK;
    ko::DeviceInfo info;
    if (int st = ko::current_device_info(&info)) return st;
    *bytes = plan_for(dtype, rows, cols, true, info).bytes;
    return KO_OK;
}

int ko_layernorm_backward_f32(const float *dy, const float *x, float *dx, int64_t rows, int32_t cols, float eps, const float *gamma,
                              const float *residual, float *dgamma, float *dbeta, int ddof, void *workspace,
                              size_t workspace_bytes, void *stream) {
    return dispatch<float>(KO_DTYPE_F32, dy, x, dx, rows, cols, eps, gamma, residual, dgamma, dbeta, ddof, workspace, workspace_bytes, stream);
}

int ko_layernorm_backward_f16(const uint16_t *dy, const uint16_t *x, uint16_t *dx, int64_t rows, int32_t cols, float eps,
                              const uint16_t *gamma, const uint16_t *residual, float *dgamma, float *dbeta, int ddof,
                              void *workspace, size_t workspace_bytes, void *stream) {
    using T = __half;
    return dispatch<T>(KO_DTYPE_F16, reinterpret_cast<const T *>(dy), reinterpret_cast<const T *>(x), reinterpret_cast<T *>(dx), rows, cols,
                       eps, reinterpret_cast<const T *>(gamma), reinterpret_cast<const T *>(residual), dgamma, dbeta, ddof, workspace,
                       workspace_bytes, stream);
}

int ko_layernorm_backward_bf16(const uint16_t *dy, const uint16_t *x, uint16_t *dx, int64_t rows, int32_t cols, float eps,
                               const uint16_t *gamma, const uint16_t *residual, float *dgamma, float *dbeta, int ddof,
                               void *workspace, size_t workspace_bytes, void *stream) {
    using T = __nv_bfloat16;
    return dispatch<T>(KO_DTYPE_BF16, reinterpret_cast<const T *>(dy), reinterpret_cast<const T *>(x), reinterpret_cast<T *>(dx), rows, cols,
                       eps, reinterpret_cast<const T *>(gamma), reinterpret_cast<const T *>(residual), dgamma, dbeta, ddof, workspace,
                       workspace_bytes, stream);
}

}  // extern "C"
