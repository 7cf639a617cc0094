// C-ABI launchers of the linear layer's gradient with respect to its input.
#include "linear_launch.h"
#include "../../include/ko_b200_tuning.h"

namespace {

int dispatch(int in_fmt, int out_fmt, int activation, int64_t M, int64_t N, int64_t K, const void *dY, const void *W,
                             const void *Z, void *dX, void *workspace, size_t workspace_bytes, void *stream, const ko::PinnedPlan &pin) {
    const char *name = "linear backward input";
    if (int st = ko::check_linear(name, in_fmt, out_fmt, activation, M, N, K)) return st;
    if (M == 0 || K == 0) return KO_OK;
    KO_REQUIRE(N >= 8 && N % 8 == 0 && K % 8 == 0, KO_ERR_SHAPE, "%s: N = %lld and K = %lld must be positive multiples of 8 (16-byte row pitch)",
               name, (long long)N, (long long)K);
    KO_REQUIRE(dY != nullptr && W != nullptr && dX != nullptr, KO_ERR_INVALID_ARG, "%s: NULL pointer", name);
    KO_REQUIRE(activation == ko::kActNone || Z != nullptr, KO_ERR_INVALID_ARG, "%s: an activation's slope needs the pre-activation Z", name);
    KO_REQUIRE(ko::aligned16(dY) && ko::aligned16(W), KO_ERR_ALIGN, "%s: dY and W must be 16-byte aligned", name);
    KO_REQUIRE(ko::aligned_to(dX, out_fmt ? 2 : 4) && ko::aligned_to(Z, 2), KO_ERR_ALIGN, "%s: an operand is not aligned to its element", name);
    KO_REQUIRE(dX != dY && dX != W && (out_fmt || dX != Z), KO_ERR_INVALID_ARG, "%s: dX must not alias dY, W or a Z of another type", name);
    ko::DeviceInfo info;
    if (int st = ko::current_device_info(&info)) return st;
    ko::LinearParams p = {};
    p.M = (int)M; p.N = (int)K; p.K = (int)N;  // the product's shape
    p.D = dX; p.fmt = in_fmt; p.out_fmt = out_fmt; p.b_row_major = 1;
    p.extra = activation == ko::kActNone ? nullptr : Z;
    p.activation = activation;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return out_fmt ? ko::run_product<ko::LinearMode::kInputGrad, true>(p, dY, W, workspace, workspace_bytes, s, info, name, pin)
                   : ko::run_product<ko::LinearMode::kInputGrad, false>(p, dY, W, workspace, workspace_bytes, s, info, name, pin);
}

}  // namespace

extern "C" {

int ko_linear_backward_input_workspace(int64_t M, int64_t N, int64_t K, size_t *bytes) {
    KO_REQUIRE(bytes != nullptr, KO_ERR_INVALID_ARG, "linear backward input: NULL bytes");
    *bytes = 0;
    if (int st = ko::check_linear("linear backward input", 0, 0, 0, M, N, K)) return st;
    if (M == 0 || N == 0 || K == 0) return KO_OK;
    ko::DeviceInfo info;
    if (int st = ko::current_device_info(&info)) return st;
    *bytes = ko::product_workspace(M, K, N, info.sm_count);
    return KO_OK;
}

int ko_linear_backward_input(int in_fmt, int out_fmt, int activation, int64_t M, int64_t N, int64_t K, const void *dY, const void *W,
                             const void *Z, void *dX, void *workspace, size_t workspace_bytes, void *stream) {
    return dispatch(in_fmt, out_fmt, activation, M, N, K, dY, W, Z, dX, workspace, workspace_bytes, stream, {});
}

int ko_linear_backward_input_tuned(int in_fmt, int out_fmt, int activation, int64_t M, int64_t N, int64_t K, const void *dY, const void *W,
                                   const void *Z, void *dX, void *workspace, size_t workspace_bytes, int tile, int slices, void *stream) {
    return dispatch(in_fmt, out_fmt, activation, M, N, K, dY, W, Z, dX, workspace, workspace_bytes, stream, {tile, slices});
}

}  // extern "C"
