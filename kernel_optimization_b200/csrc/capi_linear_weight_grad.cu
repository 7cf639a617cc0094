// C-ABI launchers of the linear layer's gradients with respect to its weight and bias.
#include "linear_launch.h"
#include "../../include/ko_b200_tuning.h"

namespace {

int dispatch(int in_fmt, int out_fmt, int64_t M, int64_t N, int64_t K, const void *dY, const void *X, const void *C,
                              void *dW, float *dbias, void *workspace, size_t workspace_bytes, void *stream, const ko::PinnedPlan &pin) {
    const char *name = "linear backward weight";
    if (int st = ko::check_linear(name, in_fmt, out_fmt, 0, M, N, K)) return st;
    if (N == 0) return KO_OK;
    KO_REQUIRE(N % 8 == 0 && K % 8 == 0, KO_ERR_SHAPE, "%s: N = %lld and K = %lld must be multiples of 8 (16-byte row pitch)", name, (long long)N,
               (long long)K);
    KO_REQUIRE(K == 0 || dW != nullptr, KO_ERR_INVALID_ARG, "%s: NULL dW", name);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const size_t out_bytes = (size_t)N * (size_t)K * (out_fmt ? 2 : 4);
    if (M == 0) {  // sums over no tokens
        if (out_bytes && C == nullptr) KO_CUDA(cudaMemsetAsync(dW, 0, out_bytes, s));
        if (out_bytes && C != nullptr && C != dW) KO_CUDA(cudaMemcpyAsync(dW, C, out_bytes, cudaMemcpyDeviceToDevice, s));
        if (dbias) KO_CUDA(cudaMemsetAsync(dbias, 0, (size_t)N * sizeof(float), s));
        return KO_OK;
    }
    KO_REQUIRE(dY != nullptr && (K == 0 || X != nullptr), KO_ERR_INVALID_ARG, "%s: NULL pointer", name);
    KO_REQUIRE(ko::aligned16(dY) && ko::aligned16(X), KO_ERR_ALIGN, "%s: dY and X must be 16-byte aligned", name);
    KO_REQUIRE(ko::aligned_to(dW, out_fmt ? 2 : 4) && ko::aligned_to(C, out_fmt ? 2 : 4) && ko::aligned_to(dbias, 4), KO_ERR_ALIGN,
               "%s: an operand is not aligned to its element", name);
    KO_REQUIRE(K == 0 || (dW != dY && dW != X && (const void *)dbias != dW), KO_ERR_INVALID_ARG, "%s: outputs must not alias the inputs or each other", name);
    KO_REQUIRE(dbias == nullptr || ((const void *)dbias != dY && (K == 0 || ((const void *)dbias != X && (const void *)dbias != C))), KO_ERR_INVALID_ARG,
               "%s: dbias must not alias an input", name);
    ko::DeviceInfo info;
    if (int st = ko::current_device_info(&info)) return st;
    ko::LinearParams p = {};
    p.M = (int)N; p.N = (int)K; p.K = (int)M;  // the product's shape
    p.D = dW; p.fmt = in_fmt; p.out_fmt = out_fmt; p.b_row_major = 1;
    p.extra = C;
    p.dbias = dbias;
    if (K == 0) {  // no dW, only the column sums
        if (dbias == nullptr) return KO_OK;
        const uint16_t *dy = static_cast<const uint16_t *>(dY);
        const unsigned blocks = (unsigned)((N + 63) / 64);
        if (in_fmt) ko::column_sum_kernel<true><<<blocks, 256, 0, s>>>(dy, (long long)M, (int)N, dbias);
        else ko::column_sum_kernel<false><<<blocks, 256, 0, s>>>(dy, (long long)M, (int)N, dbias);
        KO_CUDA(cudaGetLastError());
        return KO_OK;
    }
    return out_fmt ? ko::run_product<ko::LinearMode::kWeightGrad, true>(p, dY, X, workspace, workspace_bytes, s, info, name, pin)
                   : ko::run_product<ko::LinearMode::kWeightGrad, false>(p, dY, X, workspace, workspace_bytes, s, info, name, pin);
}

}  // namespace

extern "C" {

int ko_linear_backward_weight_workspace(int64_t M, int64_t N, int64_t K, size_t *bytes) {
    KO_REQUIRE(bytes != nullptr, KO_ERR_INVALID_ARG, "linear backward weight: NULL bytes");
    *bytes = 0;
    if (int st = ko::check_linear("linear backward weight", 0, 0, 0, M, N, K)) return st;
    if (M == 0 || N == 0) return KO_OK;
    ko::DeviceInfo info;
    if (int st = ko::current_device_info(&info)) return st;
    *bytes = ko::product_workspace(N, K, M, info.sm_count, true);
    return KO_OK;
}

int ko_linear_backward_weight(int in_fmt, int out_fmt, int64_t M, int64_t N, int64_t K, const void *dY, const void *X, const void *C,
                              void *dW, float *dbias, void *workspace, size_t workspace_bytes, void *stream) {
    return dispatch(in_fmt, out_fmt, M, N, K, dY, X, C, dW, dbias, workspace, workspace_bytes, stream, {});
}

int ko_linear_backward_weight_tuned(int in_fmt, int out_fmt, int64_t M, int64_t N, int64_t K, const void *dY, const void *X, const void *C,
                                    void *dW, float *dbias, void *workspace, size_t workspace_bytes, int tile, int slices, void *stream) {
    KO_REQUIRE(tile == 0 || tile == 128 || tile == 256 || tile == 2048, KO_ERR_INVALID_ARG, "linear backward weight: tile code %d not in {128,256,2048}", tile);
    KO_REQUIRE(slices == 0 || tile != 0, KO_ERR_INVALID_ARG, "linear backward weight: slices need a tile code");
    return dispatch(in_fmt, out_fmt, M, N, K, dY, X, C, dW, dbias, workspace, workspace_bytes, stream, {tile, slices});
}

}  // extern "C"
