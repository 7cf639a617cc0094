// Host side of the LayerNorm backward pass, shared by the element types' translation units.
#pragma once

#include "row_launch.h"

#include <algorithm>

#include "../nn_operators/layernorm/layernorm_backward.h"

namespace ko {
namespace ln_backward {

// How a call is cut up.
struct Plan {
    int row_chunks;      // blocks along the rows = partial rows
    size_t terms_bytes;  // row terms (two-kernel form), a multiple of 16 bytes
    size_t bytes;        // whole workspace
};

// columns the resident kernels hold at most: 16 warps, 16 columns a thread
constexpr int kResidentColumns = 8192;

inline Plan plan_for(int dtype, int64_t rows, int cols, bool vec, const ko::DeviceInfo &info) {
    Plan p{};
    if (cols <= kResidentColumns) {
        p.row_chunks = (int)std::min<int64_t>(rows, 2LL * info.sm_count);  // at most two blocks per SM
    } else {
        // row chunks for eight blocks of 256 threads per SM; a chunk has at least 8 rows, one for each of the block's warps
        const int64_t width = vec ? (dtype == KO_DTYPE_F32 ? 128 : 256) : 32;
        const int64_t strips = (cols + width - 1) / width;
        const int64_t wanted = std::max<int64_t>(1, 8LL * info.sm_count / strips);
        p.row_chunks = (int)std::min<int64_t>(std::min<int64_t>(wanted, (rows + 7) / 8), 65535);
        p.terms_bytes = (size_t)rows * sizeof(ko::LayerNormRowTerms);
    }
    p.bytes = p.terms_bytes + (size_t)p.row_chunks * 2 * (size_t)cols * sizeof(float);
    return p;
}

inline bool can_use_vectors(int dtype, int cols) { return cols % (dtype == KO_DTYPE_F32 ? 4 : 8) == 0; }

// room for either access width: which one runs depends on the pointers' alignment
inline size_t workspace_for(int dtype, int64_t rows, int cols, const ko::DeviceInfo &info) {
    const size_t single = plan_for(dtype, rows, cols, false, info).bytes;
    return can_use_vectors(dtype, cols) ? std::max(single, plan_for(dtype, rows, cols, true, info).bytes) : single;
}

inline int check_shape(int64_t rows, int32_t cols) {
    KO_REQUIRE(rows >= 0 && cols >= 0, KO_ERR_INVALID_ARG, "layernorm backward: negative shape [%lld, %d]", (long long)rows, cols);
    KO_REQUIRE(cols <= (1 << 30), KO_ERR_SHAPE, "layernorm backward: %d columns, at most 2^30", cols);
    return KO_OK;
}

template <typename T>
int launch_fold(const ko::LayerNormBackwardArgs<T> &a, int partial_rows, float *dgamma, float *dbeta, cudaStream_t s) {
    if (a.partials == nullptr) return KO_OK;
    return ko::launch_overlapped(ko::layernorm_backward_fold_kernel<>, (unsigned)((a.cols + 31) / 32), 1024u, 0, s, a.partials, partial_rows, a.cols,
                                 dgamma, dbeta);
}

// rows beyond what a block's registers hold: the rows' terms first, then dx and the column sums
template <typename T, int E>
int launch_two_pass(const ko::LayerNormBackwardArgs<T> &a, const Plan &plan, const ko::DeviceInfo &info, ko::LayerNormRowTerms *terms,
                    cudaStream_t s) {
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
    return KO_OK;
}

template <typename T, int E, int kVecs, int kLanes>
int launch_resident(const ko::LayerNormBackwardArgs<T> &a, const ko::DeviceInfo &info, int *partial_rows, cudaStream_t s) {
    constexpr int kWarps = backward_warps(kLanes), kRows = 32 * kWarps / kLanes, kBlocks = backward_blocks_per_sm(kLanes);
    auto kernel = ko::layernorm_backward_resident_kernel<T, E, kVecs, kLanes>;
    const unsigned blocks = ko::clamp_grid((a.rows + kRows - 1) / kRows, (long long)kBlocks * info.sm_count);
    size_t smem = kRows > 1 ? 2 * sizeof(float) * kLanes * kVecs * E : 0;
    int stages = 0;
    unsigned *status = nullptr;
    if (E > 1) {
        // the SM's shared memory, shared by its blocks; 3 KB of each share cover static shared memory and the system's 1 KB
        const size_t share = ((size_t)info.max_smem_optin + 1024) / kBlocks - 3072;
        const size_t stage = (size_t)kRows * backward_pitch<T, E, kVecs, kLanes>(a.cols) * (a.residual ? 3 : 2);
        stages = (int)std::min<size_t>(share / stage, kBackwardMaxStages);
        KO_REQUIRE(stages >= 2, KO_ERR_SHAPE, "layernorm backward: %d columns leave no room for two stages", a.cols);  // 8192 FP32 columns do
        smem = std::max(smem, stages * stage);
        if (int st = ko::device_status_word(1, &status)) return st;
    }
    *partial_rows = (int)blocks;
    if (int st = ko::ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), smem)) return st;
    return ko::launch_overlapped(kernel, blocks, 32u * kWarps, smem, s, a, stages, status);
}

// the smallest form that holds the row
template <typename T, int E>
int launch_resident_for(const ko::LayerNormBackwardArgs<T> &a, const ko::DeviceInfo &info, int *partial_rows, cudaStream_t s) {
#define KO_TRY(columns, lanes) \
    if (a.cols <= (columns) * (lanes)) return launch_resident<T, E, (columns) / E, lanes>(a, info, partial_rows, s)
    if constexpr (E > 1) {
        KO_TRY(8, 8); KO_TRY(16, 8); KO_TRY(16, 16); KO_TRY(16, 32);
        if constexpr (E == 4) { KO_TRY(12, 64); }
        KO_TRY(16, 64);
        if constexpr (E == 4) { KO_TRY(12, 96); }
        KO_TRY(16, 96); KO_TRY(16, 128); KO_TRY(16, 160); KO_TRY(16, 192); KO_TRY(16, 224); KO_TRY(16, 256); KO_TRY(16, 320); KO_TRY(16, 384);
        KO_TRY(16, 448); KO_TRY(16, 512);
    } else {
        KO_TRY(8, 32); KO_TRY(16, 32); KO_TRY(16, 64); KO_TRY(16, 96); KO_TRY(16, 128); KO_TRY(16, 192); KO_TRY(16, 256); KO_TRY(16, 384); KO_TRY(16, 512);
    }
#undef KO_TRY
    return ko::fail(KO_ERR_SHAPE, "layernorm backward: %d columns are too many for the resident kernels", a.cols);
}

template <typename T, int E>
int launch(const ko::LayerNormBackwardArgs<T> &a, int dtype, const Plan &plan, const ko::DeviceInfo &info, ko::LayerNormRowTerms *terms,
           float *dgamma, float *dbeta, cudaStream_t s) {
    int partial_rows = plan.row_chunks;
    const int st = a.cols <= kResidentColumns ? launch_resident_for<T, E>(a, info, &partial_rows, s) : launch_two_pass<T, E>(a, plan, info, terms, s);
    return st ? st : launch_fold(a, partial_rows, dgamma, dbeta, s);
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
    for (const T *p : {dy, x, (const T *)dx, gamma, residual})
        KO_REQUIRE(ko::aligned_to(p, sizeof(T)), KO_ERR_ALIGN, "layernorm backward: an operand is not aligned to its element");
    KO_REQUIRE(ko::aligned_to(dgamma, 4) && ko::aligned_to(dbeta, 4), KO_ERR_ALIGN, "layernorm backward: dgamma and dbeta must be aligned to 4 bytes");
    KO_REQUIRE(dgamma == nullptr || dgamma != dbeta, KO_ERR_INVALID_ARG, "layernorm backward: dgamma and dbeta must not be the same buffer");
    ko::DeviceInfo info;
    if (int st = ko::current_device_info(&info)) return st;
    const bool aligned = ko::aligned16(dy) && ko::aligned16(x) && ko::aligned16(dx) && (!gamma || ko::aligned16(gamma)) &&
                         (!residual || ko::aligned16(residual));
    const bool vec = aligned && can_use_vectors(dtype, cols);
    const size_t need = workspace_for(dtype, rows, cols, info);
    KO_REQUIRE(workspace != nullptr && workspace_bytes >= need, KO_ERR_INVALID_ARG,
               "layernorm backward: the workspace needs %zu bytes, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    KO_REQUIRE(ko::aligned16(workspace), KO_ERR_ALIGN, "layernorm backward: the workspace must be 16-byte aligned");
    const Plan plan = plan_for(dtype, rows, cols, vec, info);
    auto *terms = static_cast<ko::LayerNormRowTerms *>(workspace);
    float *partials = dgamma || dbeta ? reinterpret_cast<float *>(static_cast<char *>(workspace) + plan.terms_bytes) : nullptr;
    const ko::LayerNormBackwardArgs<T> a{dy, x, dx, rows, cols, eps, gamma, residual, partials, ddof};
    return vec ? launch<T, ko::RowIo<T>::kPerVec>(a, dtype, plan, info, terms, dgamma, dbeta, s)
               : launch<T, 1>(a, dtype, plan, info, terms, dgamma, dbeta, s);
}

}  // namespace ln_backward
}  // namespace ko
