// C-ABI launchers of the linear layer's forward pass.
#include "linear_launch.h"
#include "../../include/ko_b200_tuning.h"

#include "../nn_operators/linear/linear_few_tokens.h"

namespace ko {

int check_linear(const char *name, int in_fmt, int out_fmt, int activation, int64_t M, int64_t N, int64_t K) {
    KO_REQUIRE(in_fmt == 0 || in_fmt == 1, KO_ERR_INVALID_ARG, "%s: in_fmt must be 0 (f16) or 1 (bf16)", name);
    KO_REQUIRE(out_fmt == 0 || out_fmt == in_fmt + 1, KO_ERR_INVALID_ARG, "%s: out_fmt must be 0 (f32) or the input type's %d", name, in_fmt + 1);
    KO_REQUIRE(activation >= 0 && activation < kActCount, KO_ERR_INVALID_ARG, "%s: unknown activation %d", name, activation);
    KO_REQUIRE(M >= 0 && N >= 0 && K >= 0, KO_ERR_INVALID_ARG, "%s: negative shape {%lld,%lld,%lld}", name, (long long)M, (long long)N, (long long)K);
    // room for a last step past the end in 32-bit counters
    KO_REQUIRE(M <= 0x7fff0000 && N <= 0x7fff0000 && K <= 0x7fff0000, KO_ERR_SHAPE, "%s: a dimension exceeds 2^31-65536", name);
    return KO_OK;
}

}  // namespace ko

namespace {

template <bool kBf16, bool kOut16, bool kPromote, int kTiles, int kSlabs, int kWarps>
int launch_few_tokens_as(const ko::FewTokensParams &q, const ko::DeviceInfo &info, cudaStream_t s) {
    constexpr int kChunks = 4;
    const long long groups = ((long long)q.p.N + 16 * kSlabs - 1) / (16 * kSlabs);
    // Blocks share a stretch of W rows, each with its part of K, while that leaves at most four blocks per SM and every warp
    // a piece of K.  Measured (us, 1 / 2 / 4 / 8 blocks): 16 x 4096 x 4096 13.0 / 10.6 / 13.5 / 23.4, 16 x 2000 x 8192 19.4 /
    // 14.1 / 10.6 / 13.8, 4 x 1024 x 8192 17.1 / 10.7 / 7.5 / 5.8, 8 x 14336 x 4096 25.5 / 30.5 / 34.7 / 61.0.
    unsigned cluster = 1;
    while (cluster < 8 && groups * cluster * 2 <= 4LL * info.sm_count && (long long)cluster * 2 * kWarps * 32 * kChunks <= q.p.K) cluster *= 2;
    KO_REQUIRE(groups * cluster <= 0x7fffffffLL, KO_ERR_SHAPE, "linear: %lld blocks exceed the grid limit", groups * cluster);
    return ko::launch_clustered_overlapped(ko::linear_few_tokens_kernel<kBf16, kOut16, kPromote, kTiles, kSlabs, kChunks, kWarps>,
                                           (unsigned)(groups * cluster), 32u * kWarps, cluster, 0, s, q);
}
// a warp's accumulators take as much of K of a 16-bit result as a tile's (less where blocks share it)
template <bool kBf16, bool kOut16, int kTiles, int kSlabs, int kWarps>
int launch_few_tokens(const ko::FewTokensParams &q, const ko::DeviceInfo &info, cudaStream_t s) {
    if (!kOut16 || q.p.K > ko::blocks_in_one_accumulator(true) * 64 * kWarps)
        return launch_few_tokens_as<kBf16, kOut16, true, kTiles, kSlabs, kWarps>(q, info, s);
    return launch_few_tokens_as<kBf16, kOut16, !kOut16, kTiles, kSlabs, kWarps>(q, info, s);
}
// Up to 16 tokens, and whenever K is short, 16 rows of W a block and eight warps; beyond, 32 rows, so that a token's
// fragments serve two slabs, and four warps (32 x 4096 x 4096: 11.8 against 14.8 us, 20 x 2000 x 8192 11.3 against 15.1;
// but 32 x 4096 x 1024: 8.4 against 6.0).
template <bool kBf16, bool kOut16>
int few_tokens(const ko::FewTokensParams &q, const ko::DeviceInfo &info, cudaStream_t s) {
    if (q.p.M <= 8) return launch_few_tokens<kBf16, kOut16, 1, 1, 8>(q, info, s);
    if (q.p.M <= 16) return launch_few_tokens<kBf16, kOut16, 2, 1, 8>(q, info, s);
    if (q.p.K <= 1024) return launch_few_tokens<kBf16, kOut16, 4, 1, 8>(q, info, s);
    return launch_few_tokens<kBf16, kOut16, 4, 2, 4>(q, info, s);
}

int linear_dispatch(int in_fmt, int out_fmt, int activation, int64_t M, int64_t N, int64_t K, const void *X, const void *W, const void *bias,
              const void *residual, void *Y, void *Z, void *workspace, size_t workspace_bytes, void *stream, const ko::PinnedPlan &pin) {
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
    if (M <= ko::kFewTokens && pin.tile == 0) {
        const ko::FewTokensParams q{p, X, W};
        if (in_fmt) return out_fmt ? few_tokens<true, true>(q, info, s) : few_tokens<true, false>(q, info, s);
        return out_fmt ? few_tokens<false, true>(q, info, s) : few_tokens<false, false>(q, info, s);
    }
    return out_fmt ? ko::run_product<ko::LinearMode::kForward, true>(p, X, W, workspace, workspace_bytes, s, info, "linear", pin)
                   : ko::run_product<ko::LinearMode::kForward, false>(p, X, W, workspace, workspace_bytes, s, info, "linear", pin);
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
    return linear_dispatch(in_fmt, out_fmt, activation, M, N, K, X, W, bias, residual, Y, Z, workspace, workspace_bytes, stream, {});
}

int ko_linear_tuned(int in_fmt, int out_fmt, int activation, int64_t M, int64_t N, int64_t K, const void *X, const void *W, const void *bias,
                    const void *residual, void *Y, void *Z, void *workspace, size_t workspace_bytes, int tile, int slices, void *stream) {
    KO_REQUIRE(tile == 0 || tile == 128 || tile == 256 || tile == 2048, KO_ERR_INVALID_ARG, "linear: tile code %d not in {128,256,2048}", tile);
    KO_REQUIRE(slices == 0 || tile != 0, KO_ERR_INVALID_ARG, "linear: slices need a tile code");
    return linear_dispatch(in_fmt, out_fmt, activation, M, N, K, X, W, bias, residual, Y, Z, workspace, workspace_bytes, stream, {tile, slices});
}

}  // extern "C"
