// Fused epilogues of the tensor-core GEMM kernels for the linear layer and its gradients:
//   forward        Y = act(X W^T + bias) + residual, and Z = X W^T + bias (16 bits) when the backward pass wants it
//   input grad     dX = (dY W) * act'(Z)
//   weight grad    dW = dY^T X + C   (A = dY stored [tokens, features]: MN-major operand)
// An accumulator chunk of 32 rows x 32 columns stays in registers from tensor memory to the store; what it is combined
// with (residual, Z or C: one row segment of 64 or 128 bytes per lane; the bias: the same 64 bytes for all lanes) is
// loaded one chunk ahead, the first chunk's while the tile is still being multiplied.  Everything is FP32 until one
// rounding to the stored type.  Eight epilogue warps, two per quadrant of TMEM lanes: an activation is 10 to 20
// instructions an element, and four warps alone could not hide them behind the MMAs of the next tile.
#pragma once

#include <type_traits>

#include "../gemm/tensor_core_gemm.h"
#include "activation.h"

namespace ko {

enum class LinearMode { kForward, kInputGrad, kWeightGrad };

struct LinearParams : tc::GemmParams {
    const void *bias;   // forward: [N], element type of the inputs; may be null
    const void *extra;  // forward: residual, weight grad: C (both of D's type); input grad: Z (the inputs' type); may be null
    void *pre;          // forward: Z out (the inputs' type); may be null
    int activation;
    int bias_vec, extra_vec;  // 16-byte accesses allowed: base aligned, row pitch a multiple of 16 bytes
    alignas(64) CUtensorMap map_pre;
};

// two 16-bit values of type kBf16 ? BF16 : FP16 as FP32
template <bool kBf16>
__device__ __forceinline__ void widen16(uint32_t w, float &lo, float &hi) {
    if constexpr (kBf16) {
        lo = bf16_lo(w);
        hi = bf16_hi(w);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        lo = f.x;
        hi = f.y;
    }
}
template <bool kBf16>
__device__ __forceinline__ float widen16_at(const void *base, size_t i) {
    const uint32_t w = static_cast<const uint16_t *>(base)[i];
    float lo, hi;
    widen16<kBf16>(w, lo, hi);
    return lo;
}

// The same epilogue for one element, where speed does not depend on it: acc -> the value to be stored (before rounding);
// Z is written here.
template <LinearMode kMode, bool kBf16, bool kOut16>
__device__ __forceinline__ float linear_finish_one(const LinearParams &p, float acc, int row, int col) {
    const size_t at = (size_t)row * p.N + col;
    float v = acc;
    if constexpr (kMode == LinearMode::kForward) {
        if (p.bias) v += widen16_at<kBf16>(p.bias, (size_t)col);
        if (p.pre) static_cast<uint16_t *>(p.pre)[at] = (uint16_t)tc::pack16(v, 0.f, kBf16 ? 2 : 1);
        with_activation(p.activation, [&](auto act) { v = activate<act.value, !kOut16>(v); });
    }
    if (p.extra) {
        if constexpr (kMode == LinearMode::kInputGrad) {
            const float z = widen16_at<kBf16>(p.extra, at);
            with_activation(p.activation, [&](auto act) { v *= activation_slope<act.value, !kOut16>(z); });
        } else if constexpr (kOut16) {
            v += widen16_at<kBf16>(p.extra, at);
        } else {
            v += static_cast<const float *>(p.extra)[at];
        }
    }
    return v;
}
template <bool kBf16, bool kOut16>
__device__ __forceinline__ void linear_store_one(const LinearParams &p, float v, int row, int col) {
    const size_t at = (size_t)row * p.N + col;
    if constexpr (kOut16) static_cast<uint16_t *>(p.D)[at] = (uint16_t)tc::pack16(v, 0.f, kBf16 ? 2 : 1);
    else static_cast<float *>(p.D)[at] = v;
}

template <LinearMode kMode, bool kOut16>
struct LinearEpilogue {
    using Params = LinearParams;
    static constexpr int kWarps = 8;
    static constexpr bool kTransA = kMode == LinearMode::kWeightGrad;
    static constexpr bool kFused = true;
    static constexpr bool kExtra16 = kMode == LinearMode::kInputGrad || kOut16;
    static constexpr int kExtraVecs = kExtra16 ? 4 : 8;  // 16-byte vectors per lane and chunk
    // 4 KB of staging per warp: two boxes of 32 x 32 16-bit values, or one of FP32 (then Z, if any, takes its turn in it)
    static constexpr int kBoxes = kOut16 ? 2 : 1;
    static constexpr uint32_t kBoxBytes = kOut16 ? 2048 : 4096;

    struct Operands {
        uint4 extra[kExtraVecs];
        uint4 bias[4];
    };

    // 32 columns of row `row` from column `col` on; what lies outside the matrix is left at zero
    __device__ __forceinline__ static void load(Operands &o, const Params &p, int row, int col) {
#pragma unroll
        for (int j = 0; j < kExtraVecs; ++j) o.extra[j] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int j = 0; j < 4; ++j) o.bias[j] = make_uint4(0u, 0u, 0u, 0u);
        if (p.extra != nullptr && row < p.M) {
            constexpr int kPer = kExtra16 ? 8 : 4;
            const char *at = static_cast<const char *>(p.extra) + ((size_t)row * p.N + col) * (kExtra16 ? 2 : 4);
            if (p.extra_vec) {
#pragma unroll
                for (int j = 0; j < kExtraVecs; ++j)
                    if (col + j * kPer < p.N) o.extra[j] = *reinterpret_cast<const uint4 *>(at + j * 16);
            } else {
                load_singly<kExtraVecs, kExtra16>(o.extra, at, p.N - col);
            }
        }
        if constexpr (kMode == LinearMode::kForward) {
            if (p.bias != nullptr) {
                const char *at = static_cast<const char *>(p.bias) + (size_t)col * 2;
                if (p.bias_vec) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (col + j * 8 < p.N) o.bias[j] = *reinterpret_cast<const uint4 *>(at + j * 16);
                } else {
                    load_singly<4, true>(o.bias, at, p.N - col);
                }
            }
        }
    }

    // the chunks c_begin, c_begin + 8 * kWarps, ... of this warp's 32 rows (accumulator at TMEM address t_row) to D and Z
    template <bool kTmaStore>
    __device__ __forceinline__ static void block(const CUtensorMap *map_d, const Params &p, Operands &next, uint32_t t_row, int row_base,
                                                 int col0, int bn, int c_begin, int lane, uint32_t boxes, uint32_t &store_seq) {
#pragma unroll 1
        for (int c0 = c_begin; c0 < bn; c0 += 8 * kWarps) {
            uint32_t r[32];
            tc::tmem_ld_32x32_issue(t_row + c0, r);
            const Operands o = next;
            if (c0 + 8 * kWarps < bn) load(next, p, row_base + lane, col0 + c0 + 8 * kWarps);
            tc::tmem_ld_wait();
            if (p.fmt) chunk<kTmaStore, true>(map_d, p, o, r, row_base, col0 + c0, lane, boxes, store_seq);
            else chunk<kTmaStore, false>(map_d, p, o, r, row_base, col0 + c0, lane, boxes, store_seq);
        }
    }

private:
    template <int kVecs, bool k16>
    __device__ __forceinline__ static void load_singly(uint4 (&v)[kVecs], const char *at, int left) {
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
            uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = j * 4 + e;  // 32-bit word of the segment
                if constexpr (k16) {
                    const uint16_t *h = reinterpret_cast<const uint16_t *>(at);
                    if (2 * i < left) w[e] = h[2 * i];
                    if (2 * i + 1 < left) w[e] |= (uint32_t)h[2 * i + 1] << 16;
                } else {
                    if (i < left) w[e] = reinterpret_cast<const uint32_t *>(at)[i];
                }
            }
            v[j] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    template <bool kBf16, int kVecs>
    __device__ __forceinline__ static void unpack16(const uint4 (&v)[kVecs], float (&f)[32]) {
        static_assert(kVecs == 4, "32 values of 16 bits");
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            widen16<kBf16>(v[j].x, f[8 * j], f[8 * j + 1]);
            widen16<kBf16>(v[j].y, f[8 * j + 2], f[8 * j + 3]);
            widen16<kBf16>(v[j].z, f[8 * j + 4], f[8 * j + 5]);
            widen16<kBf16>(v[j].w, f[8 * j + 6], f[8 * j + 7]);
        }
    }

    template <bool kTmaStore, bool kBf16>
    __device__ __forceinline__ static void put(const CUtensorMap *map, void *base, int out_fmt, const Params &p, const float (&v)[32],
                                               int row_base, int col, int lane, uint32_t boxes, uint32_t &store_seq) {
        if constexpr (kTmaStore) {
            uint32_t bits[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) bits[i] = __float_as_uint(v[i]);
            tc::stage_chunk<kBoxes>(map, p.M, p.N, out_fmt, bits, row_base, col, lane, boxes, kBoxBytes, store_seq);
        } else {
            const int row = row_base + lane;
            if (row >= p.M || col >= p.N) return;
            tc::GemmParams q = p;
            q.C = nullptr;
            q.D = base;
            if (out_fmt == 0) tc::store_row_segment<float>(v, q, row, col);
            else if (kBf16) tc::store_row_segment<__nv_bfloat16>(v, q, row, col);
            else tc::store_row_segment<__half>(v, q, row, col);
        }
    }

    template <bool kTmaStore, bool kBf16>
    __device__ __forceinline__ static void chunk(const CUtensorMap *map_d, const Params &p, const Operands &o, const uint32_t (&r)[32],
                                                 int row_base, int col, int lane, uint32_t boxes, uint32_t &store_seq) {
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        if constexpr (kMode == LinearMode::kForward) {
            if (p.bias) {
                float b[32];
                unpack16<kBf16>(o.bias, b);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] += b[i];
            }
            if (p.pre) put<kTmaStore, kBf16>(&p.map_pre, p.pre, kBf16 ? 2 : 1, p, v, row_base, col, lane, boxes, store_seq);
            with_activation(p.activation, [&](auto act) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = activate<act.value, !kOut16>(v[i]);
            });
        }
        if (p.extra) {
            float x[32];
            if constexpr (kExtra16) {
                unpack16<kBf16>(o.extra, x);
            } else {
#pragma unroll
                for (int j = 0; j < kExtraVecs; ++j) {
                    x[4 * j] = __uint_as_float(o.extra[j].x);
                    x[4 * j + 1] = __uint_as_float(o.extra[j].y);
                    x[4 * j + 2] = __uint_as_float(o.extra[j].z);
                    x[4 * j + 3] = __uint_as_float(o.extra[j].w);
                }
            }
            if constexpr (kMode == LinearMode::kInputGrad) {
                with_activation(p.activation, [&](auto act) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] *= activation_slope<act.value, !kOut16>(x[i]);
                });
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] += x[i];
            }
        }
        put<kTmaStore, kBf16>(map_d, p.D, kOut16 ? (kBf16 ? 2 : 1) : 0, p, v, row_base, col, lane, boxes, store_seq);
    }
};

// Second step of a product cut into K slices (see tc::gemm_slice_sum_kernel): the slices of a 32 x 32 chunk are added in
// K order, then the epilogue.  One block per chunk, thread i takes columns 4 * (i % 8) .. + 3 of row i / 8.
template <LinearMode kMode, bool kOut16>
__global__ void __launch_bounds__(256) linear_slice_sum_kernel(const LinearParams p, int bn) {
    const int chunks_n = bn / 32, chunks_per_tile = (tc::kBM / 32) * chunks_n;
    const long long t = blockIdx.x / chunks_per_tile;
    const int chunk = (int)(blockIdx.x - t * chunks_per_tile);
    const int tiles_m = (p.M + tc::kBM - 1) / tc::kBM, tiles_n = (p.N + bn - 1) / bn;
    int tm, tn;
    tc::tile_coords(t, tiles_m, tiles_n, tm, tn);
    const int row = tm * tc::kBM + (chunk / chunks_n) * 32 + (int)threadIdx.x / 8;
    const int col = tn * bn + (chunk % chunks_n) * 32 + ((int)threadIdx.x & 7) * 4;
    grid_launch_dependents();
    grid_dependency_wait();  // the slices are complete and visible
    if (row >= p.M || col >= p.N) return;
    const size_t slot_vecs = (size_t)tc::kBM * bn / 4;
    const float4 *src = reinterpret_cast<const float4 *>(p.partials) + (size_t)t * p.split_k * slot_vecs + ((size_t)chunk << 8) + threadIdx.x;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < p.split_k; s0 += 4) {
        float4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (s0 + i < p.split_k) v[i] = __ldcg(src + (size_t)(s0 + i) * slot_vecs);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (s0 + i < p.split_k) {
                if (s0 + i == 0) sum = v[0];
                else { sum.x += v[i].x; sum.y += v[i].y; sum.z += v[i].z; sum.w += v[i].w; }
            }
    }
    const float acc[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (col + e >= p.N) break;
        if (p.fmt) linear_store_one<true, kOut16>(p, linear_finish_one<kMode, true, kOut16>(p, acc[e], row, col + e), row, col + e);
        else linear_store_one<false, kOut16>(p, linear_finish_one<kMode, false, kOut16>(p, acc[e], row, col + e), row, col + e);
    }
}

// Column sums of a 16-bit [rows, cols] matrix (the bias gradient), cols a multiple of 8: a warp takes 256 columns of every
// (8 * gridDim.y)-th row, the block's warps add through shared memory, one partial row per block; with a single block
// along the rows the partial row is the result.
template <bool kBf16>
__global__ void __launch_bounds__(256) column_sum_kernel(const uint16_t *in, long long rows, int cols, float *partials) {
    constexpr int E = 8;
    __shared__ float fold[8][32 * E + 1];
    grid_launch_dependents();
    grid_dependency_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = (int)(blockIdx.x * 32 + lane) * E;
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0.f;
    if (c < cols) {
#pragma unroll 4
        for (long long r = (long long)blockIdx.y * 8 + warp; r < rows; r += (long long)gridDim.y * 8) {
            const uint16_t *at = in + (size_t)r * cols + c;
            const uint4 v = *reinterpret_cast<const uint4 *>(at);
            float f[8];
            widen16<kBf16>(v.x, f[0], f[1]);
            widen16<kBf16>(v.y, f[2], f[3]);
            widen16<kBf16>(v.z, f[4], f[5]);
            widen16<kBf16>(v.w, f[6], f[7]);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += f[e];
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) fold[warp][lane * E + e] = sum[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * E; i += 256) {
        const int col = (int)blockIdx.x * 32 * E + i;
        float total = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) total += fold[w][i];
        if (col < cols) partials[(size_t)blockIdx.y * cols + col] = total;
    }
}
// out = the partial rows added in order: a block takes 32 columns, warp w the partial rows w, w + 8, ...
template <int kWarps = 8>
__global__ void __launch_bounds__(32 * kWarps) column_fold_kernel(const float *partials, int partial_rows, int cols, float *out) {
    __shared__ float fold[kWarps][32];
    grid_launch_dependents();
    grid_dependency_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int col = (int)blockIdx.x * 32 + lane;
    float sum = 0.f;
    if (col < cols)
#pragma unroll 4
        for (int p = warp; p < partial_rows; p += kWarps) sum += __ldcg(partials + (size_t)p * cols + col);
    fold[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && col < cols) {
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += fold[w][lane];
        out[col] = sum;
    }
}

}  // namespace ko
