// TMA descriptors of the tensor-core GEMM kernels' operands.
#pragma once

#include "ko_internal.h"

#include <mutex>

#include <cudaTypedefs.h>

#include "../nn_operators/gemm/tensor_core_gemm.h"

namespace ko {

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline int get_encode_fn(EncodeTiledFn *out) {
    static std::mutex mu;
    static EncodeTiledFn cached = nullptr;
    std::lock_guard<std::mutex> lock(mu);
    if (!cached) {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult qres;
        KO_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres));
        KO_REQUIRE(qres == cudaDriverEntryPointSuccess && fn != nullptr, KO_ERR_CUDA,
                   "cuTensorMapEncodeTiled is not available from this driver");
        cached = reinterpret_cast<EncodeTiledFn>(fn);
    }
    *out = cached;
    return KO_OK;
}

// 2-D map over a K-contiguous 16-bit matrix [rows, K]; box = 64 (K) x box_rows, 128-byte swizzle,
// out-of-range elements read as zero
inline int make_map(EncodeTiledFn encode, CUtensorMap *map, int fmt, const void *base, int64_t rows, int64_t K, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)K * 2};
    const cuuint32_t box[2] = {(cuuint32_t)ko::tc::kBK, (cuuint32_t)box_rows};
    const cuuint32_t elem_strides[2] = {1, 1};
    const CUtensorMapDataType dt = fmt == 0 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const CUresult r = encode(map, dt, 2, const_cast<void *>(base), dims, strides, box, elem_strides,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    KO_REQUIRE(r == CUDA_SUCCESS, KO_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return KO_OK;
}

// 2-D map over a row-major 16-bit B[K, N] (N contiguous); box = 64 columns x 64 K-rows, 128-byte swizzle
inline int make_map_b_row_major(EncodeTiledFn encode, CUtensorMap *map, int fmt, const void *base, int64_t K, int64_t N) {
    const cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)K};
    const cuuint64_t strides[1] = {(cuuint64_t)N * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)ko::tc::kBK};
    const cuuint32_t elem_strides[2] = {1, 1};
    const CUtensorMapDataType dt = fmt == 0 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const CUresult r = encode(map, dt, 2, const_cast<void *>(base), dims, strides, box, elem_strides,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    KO_REQUIRE(r == CUDA_SUCCESS, KO_ERR_CUDA, "cuTensorMapEncodeTiled (row-major B) failed with CUresult %d", (int)r);
    return KO_OK;
}

// [M, N] row-major output (or an operand read in the same shape), boxes of 32 rows x 32 columns: FP32 rows of 128 bytes with
// the 128-byte swizzle, 16-bit rows of 64 bytes with the 64-byte swizzle; 64 columns of 16 bits: 128 bytes again
inline int make_store_map(EncodeTiledFn encode, CUtensorMap *map, int out_fmt, void *D, int64_t M, int64_t N, int columns = 32) {
    const cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)M};
    const cuuint64_t strides[1] = {(cuuint64_t)N * (out_fmt == 0 ? 4 : 2)};
    const cuuint32_t box[2] = {(cuuint32_t)columns, 32};
    const cuuint32_t elem_strides[2] = {1, 1};
    const CUtensorMapDataType dt = out_fmt == 0   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : out_fmt == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const CUresult r = encode(map, dt, 2, D, dims, strides, box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              columns * (out_fmt == 0 ? 4 : 2) == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                              CU_TENSOR_MAP_L2_PROMOTION_NONE,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    KO_REQUIRE(r == CUDA_SUCCESS, KO_ERR_CUDA, "cuTensorMapEncodeTiled (D) failed with CUresult %d", (int)r);
    return KO_OK;
}

}  // namespace ko
