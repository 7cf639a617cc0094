// C-ABI launchers of the linear layer's forward pass.
#include "linear_launch.h"

#include "../nn_operators/linear/linear_few_tokens.h"

namespace ko {

int check_linear(const char *name, int in_fmt, int out_fmt, int activation, int64_t M, int64_t N, int64_t K) {
    KO_REQUIRE(in_fmt == 0 || in_fmt == 1, KO_ERR_INVALID_ARG, "%s: in_fmt must be 0 (f16) or 1 (bf16)", name);
    KO_REQUIRE(out_fmt == 0 || out_fmt == in_fmt + 1, KO_ERR_INVALID_ARG, "%s: out_fmt must be 0 (f32) or the input type's %d", name, in_fmt + 1);
    KO_REQUIRE(activation >= 0 && activation < kActCount, KO_ERR_INVALID_ARG, "%s: unknown activation %d", name, activation);
    KO_REQUIRE(M >= 0 && N >= 0 && K >= 0, KO_ERR_INVALID_ARG, "%s: negative shape {%lld,%lld,%lld}", name, (long long)M, (long long)N, (long long)K);
    KO_REQUIRE(M <= 0x7fffff00 && N <= 0x7fffff00 && K <= 0x7fffff00, KO_ERR_SHAPE, "%s: a dimension exceeds 2^31-256", name);
    return KO_OK;
}

}  // namespace ko

namespace {

// how the few-token kernel is launched: blocks of 16 * slabs rows of W, `cluster` of them sharing one stretch's K
struct FewTokensPlan {
    int slabs, cluster;
};
FewTokensPlan plan_few_tokens(int64_t M, int64_t N, int64_t K, int sms) {
    FewTokensPlan plan{M <= 8 ? 1 : 2, 1};
    const int64_t blocks = (N + 16 * plan.slabs - 1) / (16 * plan.slabs);
    // more blocks until the device is full, as long as every warp keeps at least one piece of K
    while (plan.cluster < 8 && blocks * plan.cluster < 2LL * sms && (int64_t)plan.cluster * 8 * 128 < K) plan.cluster *= 2;
    return plan;
}

template <bool kBf16, bool kOut16, int kTiles, int kSlabs, int kChunks>
int launch_few_tokens(const ko::FewTokensParams &q, int cluster, cudaStream_t s) {
    const long long blocks = ((long long)q.p.N + 16 * kSlabs - 1) / (16 * kSlabs) * cluster;
    KO_REQUIRE(blocks <= 0x7fffffffLL, KO_ERR_SHAPE, "linear: %lld blocks exceed the grid limit", blocks);
    return ko::launch_clustered_overlapped(ko::linear_few_tokens_kernel<kBf16, kOut16, kTiles, kSlabs, kChunks, 8>, (unsigned)blocks, 256u,
                                           (unsigned)cluster, 0, s, q);
}
template <bool kBf16, bool kOut16>
int few_tokens(const ko::FewTokensParams &q, const ko::DeviceInfo &info, cudaStream_t s) {
    const FewTokensPlan plan = plan_few_tokens(q.p.M, q.p.N, q.p.K, info.sm_count);
    if (q.p.M <= 8) return launch_few_tokens<kBf16, kOut16, 1, 1, 4>(q, plan.cluster, s);
    if (q.p.M <= 16) return launch_few_tokens<kBf16, kOut16, 2, 2, 2>(q, plan.cluster, s);
    return launch_few_tokens<kBf16, kOut16, 4, 2, 2>(q, plan.cluster, s);
}

}  // namespace

extern "C" {

int ko_linear_workspace(int64_t M, int64_t N, int64_t K, size_t *bytes) {
    KO_REQUIRE(bytes != nullptr, KO_ERR_INVALID_ARG, "linear: NULL bytes");
    *bytes = 0;
    if (int st = ko::check_linear("linear", 0, 0, 0, M, N, K)) return st;
    if (M <= ko::kFewTokens || N == 0 || K == 0) return KO_OK;
    ko::DeviceInfo info;
    if (int st = ko::current_device_info(&info)) return st;
    *bytes = ko::product_workspace(M, N, K, info.sm_count);
    return KO_OK;
}

int ko_linear(int in_fmt, int out_fmt, int activation, int64_t M, int64_t N, int64_t K, const void *X, const void *W, const void *bias,
              const void *residual, void *Y, void *Z, void *workspace, size_t workspace_bytes, void *stream) {
    if (int st = ko::check_linear("linear", in_fmt, out_fmt, activation, M, N, K)) return st;
    if (M == 0 || N == 0) return KO_OK;
    KO_REQUIRE(K >= 8 && K % 8 == 0, KO_ERR_SHAPE, "linear: K = %lld must be a positive multiple of 8 (16-byte row pitch)", (long long)K);
    KO_REQUIRE(X != nullptr && W != nullptr && Y != nullptr, KO_ERR_INVALID_ARG, "linear: NULL pointer");
    KO_REQUIRE(ko::aligned16(X) && ko::aligned16(W), KO_ERR_ALIGN, "linear: X and W must be 16-byte aligned");
    KO_REQUIRE(ko::aligned_to(Y, out_fmt ? 2 : 4) && ko::aligned_to(residual, out_fmt ? 2 : 4) && ko::aligned_to(bias, 2) && ko::aligned_to(Z, 2),
               KO_ERR_ALIGN, "linear: an operand is not aligned to its element");
    KO_REQUIRE(Y != X && Y != W && Z != X && Z != W && Y != Z, KO_ERR_INVALID_ARG, "linear: outputs must not alias the inputs or each other");
    KO_REQUIRE(Z == nullptr || Z != residual, KO_ERR_INVALID_ARG, "linear: Z must not be the residual");
    ko::DeviceInfo info;
    if (int st = ko::current_device_info(&info)) return st;
    ko::LinearParams p = {};
    p.M = (int)M; p.N = (int)N; p.K = (int)K;
    p.D = Y; p.fmt = in_fmt; p.out_fmt = out_fmt; p.b_row_major = 0;
    p.bias = bias; p.extra = residual; p.pre = Z; p.activation = activation;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (M <= ko::kFewTokens) {
        const ko::FewTokensParams q{p, X, W};
        if (in_fmt) return out_fmt ? few_tokens<true, true>(q, info, s) : few_tokens<true, false>(q, info, s);
        return out_fmt ? few_tokens<false, true>(q, info, s) : few_tokens<false, false>(q, info, s);
    }
    return out_fmt ? ko::run_product<ko::LinearMode::kForward, true>(p, X, W, workspace, workspace_bytes, s, info, "linear")
                   : ko::run_product<ko::LinearMode::kForward, false>(p, X, W, workspace, workspace_bytes, s, info, "linear");
}

}  // extern "C"
