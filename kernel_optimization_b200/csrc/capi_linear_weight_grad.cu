// C-ABI launchers of the linear layer's gradients with respect to its weight and bias.
#include "linear_launch.h"
#include "../../include/ko_b200_tuning.h"

namespace {

// beside: right behind the product's launch, which keeps the order with earlier work (see column_sum_kernel); else in its turn
template <bool kBf16>
int column_sums(bool beside, const void *in, int64_t rows, int cols, float *out, cudaStream_t s) {
    const unsigned strips = (unsigned)((cols + 63) / 64);
    const uint16_t *dy = static_cast<const uint16_t *>(in);
    unsigned cluster = 1;
    while (cluster < 8 && rows > 256LL * cluster) cluster *= 2;  // about 256 rows a block, one round of its loads
    if (beside)
        return ko::launch_clustered_overlapped(ko::column_sum_kernel<kBf16, 8>, strips * cluster, 256u, cluster, (size_t)0, s, dy, (long long)rows, cols,
                                               out);
    // With the device to itself: 16384 rows of 4096 / 2048 columns take 24 / 15 us in blocks of 8 warps and 33 / 31 in blocks of 32,
    // which pay while there are few of them (32768 x 512 beside a product: 18 against 13 us).
    if (strips * cluster >= 128 || rows <= 2048)
        return ko::launch_clustered(ko::column_sum_kernel<kBf16, 8>, strips * cluster, 256u, cluster, s, dy, (long long)rows, cols, out);
    return ko::launch_clustered(ko::column_sum_kernel<kBf16, 32>, strips * cluster, 1024u, cluster, s, dy, (long long)rows, cols, out);
}

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
    ko::DeviceInfo info;
    if (int st = ko::current_device_info(&info)) return st;
    ko::LinearParams p = {};
    p.M = (int)N; p.N = (int)K; p.K = (int)M;  // the product's shape
    p.D = dW; p.fmt = in_fmt; p.out_fmt = out_fmt; p.b_row_major = 1;
    p.extra = C;
    // The column sums go beside the product, unless dY is large: then their reads throw out of the L2 what the product would
    // read again, and it is quicker to let them go first.  Measured with / without dbias (us): 16384 x 1024 x 4096 102 / 100,
    // 16384 x 768 x 768 29.3 / 27.6, 777 x 1000 x 520 10.5 / 10.0; 16384 x 4096 x 1024 126 beside, 121 ahead / 101.
    // Ahead as well where the product promotes its sums, which takes all of an SM's registers.
    const bool large = (size_t)M * (size_t)N * 2 > ((size_t)48 << 20);
    const auto sums = [&](bool now, bool as_beside) -> int {
        if (dbias == nullptr || !now) return KO_OK;
        return in_fmt ? column_sums<true>(as_beside, dY, M, (int)N, dbias, s) : column_sums<false>(as_beside, dY, M, (int)N, dbias, s);
    };
    if (K == 0) return sums(true, false);
    const auto first = [&](bool promoted) { return sums(large || promoted, false); };
    const auto beside = [&](bool promoted) { return sums(!large && !promoted, true); };
    return out_fmt ? ko::run_product<ko::LinearMode::kWeightGrad, true>(p, dY, X, workspace, workspace_bytes, s, info, name, pin, first, beside)
                   : ko::run_product<ko::LinearMode::kWeightGrad, false>(p, dY, X, workspace, workspace_bytes, s, info, name, pin, first, beside);
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
    *bytes = ko::product_workspace(N, K, M, info.sm_count);
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
