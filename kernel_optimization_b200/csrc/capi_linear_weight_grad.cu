// C-ABI launchers of the linear layer's gradients with respect to its weight and bias.
#include "linear_launch.h"
#include "../../include/ko_b200_tuning.h"

namespace {

// blocks along the tokens of the column sum: eight blocks of 256 threads per SM, at least 64 tokens each
int column_chunks(int64_t tokens, int64_t cols, int sms) {
    const int64_t strips = (cols + 255) / 256;
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(8LL * sms / strips, (tokens + 63) / 64), 65535));
}
size_t column_bytes(int64_t tokens, int64_t cols, int sms) {
    const int chunks = column_chunks(tokens, cols, sms);
    return chunks > 1 ? (size_t)chunks * (size_t)cols * sizeof(float) : 0;
}
size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

template <bool kBf16>
int column_sum(const void *in, int64_t rows, int cols, float *partials, float *out, int sms, cudaStream_t s) {
    const int chunks = column_chunks(rows, cols, sms);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((cols + 255) / 256), (unsigned)chunks, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    KO_CUDA(cudaLaunchKernelEx(&cfg, ko::column_sum_kernel<kBf16>, static_cast<const uint16_t *>(in), (long long)rows, cols,
                               chunks > 1 ? partials : out));
    if (chunks == 1) return KO_OK;
    return ko::launch_overlapped(ko::column_fold_kernel<>, (unsigned)((cols + 31) / 32), 256u, (size_t)0, s, (const float *)partials, chunks, cols, out);
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
    KO_REQUIRE(dW != dY && dW != X && (dbias == nullptr || (const void *)dbias != dW), KO_ERR_INVALID_ARG, "%s: outputs must not alias the inputs or each other", name);
    ko::DeviceInfo info;
    if (int st = ko::current_device_info(&info)) return st;
    size_t product_bytes = round16(ko::product_workspace(N, K, M, info.sm_count));
    if (pin.slices > 1)  // the bias gradient's part lies behind the product's
        product_bytes = std::max(product_bytes, (size_t)((N + 127) / 128) * ((K + pin.tile - 1) / pin.tile) * pin.slices * 128 * pin.tile * sizeof(float));
    const size_t sum_bytes = column_bytes(M, N, info.sm_count);
    const size_t need = product_bytes + sum_bytes;
    KO_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), KO_ERR_INVALID_ARG, "%s: the workspace needs %zu bytes, got %zu", name,
               need, workspace ? workspace_bytes : (size_t)0);
    KO_REQUIRE(ko::aligned16(workspace), KO_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", name);
    if (dbias) {
        float *partials = reinterpret_cast<float *>(static_cast<char *>(workspace) + product_bytes);
        if (int st = in_fmt ? column_sum<true>(dY, M, (int)N, partials, dbias, info.sm_count, s) : column_sum<false>(dY, M, (int)N, partials, dbias, info.sm_count, s))
            return st;
    }
    if (K == 0) return KO_OK;
    ko::LinearParams p = {};
    p.M = (int)N; p.N = (int)K; p.K = (int)M;  // the product's shape
    p.D = dW; p.fmt = in_fmt; p.out_fmt = out_fmt; p.b_row_major = 1;
    p.extra = C;
    return out_fmt ? ko::run_product<ko::LinearMode::kWeightGrad, true>(p, dY, X, workspace, product_bytes, s, info, name, pin)
                   : ko::run_product<ko::LinearMode::kWeightGrad, false>(p, dY, X, workspace, product_bytes, s, info, name, pin);
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
    *bytes = round16(ko::product_workspace(N, K, M, info.sm_count)) + column_bytes(M, N, info.sm_count);
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
