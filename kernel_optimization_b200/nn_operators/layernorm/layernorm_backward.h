// LayerNorm backward: dx, dgamma, dbeta of y = (x - mean) * rstd * gamma + beta, row-major [rows, cols].
//
// With n columns, d = n - ddof, rstd = (M2 / d + eps)^(-1/2), xhat = (x - mean) * rstd and w = dy * gamma,
//     dx_j     = rstd * (w_j - sum(w) / n - xhat_j * sum(w * xhat) / d)  [+ residual_j]
//     dgamma_j = sum over rows of dy_j * xhat_j          dbeta_j = sum over rows of dy_j
// (d M2 / d x_j = 2 (x_j - mean): the mean's own derivative drops out because deviations sum to zero.)
// mean and rstd are formed again from x, in the exact two-pass form, instead of being kept by the forward pass: x has
// to be read here anyway, so this costs one more reduction over values already in registers and no memory traffic.
// All sums and statistics are FP32; dx is rounded once to the element type; dgamma and dbeta stay FP32.
// Column sums are formed per block in a fixed row order, written as partial rows to the workspace and added in block
// order by a second kernel: no atomics, the same call gives the same bits.
//
// Everything a thread writes of dx it has read before (dy, x, residual at the same place), so dx may be the same
// buffer as any of them.
#pragma once

#include "layernorm.h"

namespace ko {

// a thread's unit of access: E consecutive elements, 16 bytes of them or a single one
template <typename T, int E>
struct RowChunk {
    using Raw = typename RowIo<T>::Raw;
    static_assert(E == RowIo<T>::kPerVec, "16-byte vectors or single elements");
    __device__ __forceinline__ static Raw load(const T *p) { return *reinterpret_cast<const Raw *>(p); }
    __device__ __forceinline__ static void store(T *p, const Raw &r) { *reinterpret_cast<Raw *>(p) = r; }
    __device__ __forceinline__ static void unpack(const Raw &r, float (&f)[E]) { RowIo<T>::unpack(r, f); }
    __device__ __forceinline__ static Raw pack(const float (&f)[E]) { return RowIo<T>::pack(f); }
    __device__ __forceinline__ static Raw zero() { return Raw{}; }
};
template <typename T>
struct RowChunk<T, 1> {
    using Raw = T;
    __device__ __forceinline__ static Raw load(const T *p) { return *p; }
    __device__ __forceinline__ static void store(T *p, const Raw &r) { *p = r; }
    __device__ __forceinline__ static void unpack(const Raw &r, float (&f)[1]) { f[0] = RowIo<T>::to_float(r); }
    __device__ __forceinline__ static Raw pack(const float (&f)[1]) { return RowIo<T>::from_float(f[0]); }
    __device__ __forceinline__ static Raw zero() { return RowIo<T>::from_float(0.f); }
};

template <typename T>
struct LayerNormBackwardArgs {
    const T *dy, *x;
    T *dx;
    long long rows;
    int cols;
    float eps;
    const T *gamma;     // may be null
    const T *residual;  // may be null; added to dx
    float *partials;    // [partial rows][2][cols]: dgamma, dbeta; null when neither is wanted
    int ddof;
};

// what a row's elements need of the row: dx_j = rstd * (w_j - c1 - (x_j - mean) * c2), with c2 holding rstd
struct LayerNormRowTerms {
    float mean, rstd, c1, c2;
};

// block-wide sum of N values, the result in every thread; `scratch` holds 32 * N floats and is free again on return
template <int N>
__device__ __forceinline__ void block_allreduce_sums(float (&v)[N], float *scratch) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_allreduce_sum(v[i]);
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) scratch[warp * N + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
    for (int w = 0; w < warps; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += scratch[w * N + i];
    __syncthreads();
}

// Rows of any length: one block per row forms the row's terms in two passes over x (the second one and dy come from
// the L1 / L2).
template <typename T, int E>
__global__ void __launch_bounds__(256) layernorm_backward_terms_kernel(const LayerNormBackwardArgs<T> a, LayerNormRowTerms *terms) {
    using Chunk = RowChunk<T, E>;
    __shared__ float scratch[3 * 32];
    grid_launch_dependents();
    grid_dependency_wait();
    const float inv_n = 1.0f / (float)a.cols, inv_d = a.cols > a.ddof ? 1.0f / (float)(a.cols - a.ddof) : 0.f;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = a.x + (size_t)r * a.cols, *dy = a.dy + (size_t)r * a.cols;
        float total[1] = {0.f};
        for (int c = threadIdx.x * E; c < a.cols; c += 256 * E) {
            float f[E];
            Chunk::unpack(Chunk::load(x + c), f);
#pragma unroll
            for (int e = 0; e < E; ++e) total[0] += f[e];
        }
        block_allreduce_sums<1>(total, scratch);
        const float mean = total[0] * inv_n;
        float sums[3] = {0.f, 0.f, 0.f};  // squared deviations, w, w * deviation
        for (int c = threadIdx.x * E; c < a.cols; c += 256 * E) {
            float f[E], g[E], w[E];
            Chunk::unpack(Chunk::load(x + c), f);
            Chunk::unpack(Chunk::load(dy + c), g);
            if (a.gamma) {
                Chunk::unpack(Chunk::load(a.gamma + c), w);
#pragma unroll
                for (int e = 0; e < E; ++e) w[e] *= g[e];
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) w[e] = g[e];
            }
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float dev = f[e] - mean;
                sums[0] = fmaf(dev, dev, sums[0]);
                sums[1] += w[e];
                sums[2] = fmaf(w[e], dev, sums[2]);
            }
        }
        block_allreduce_sums<3>(sums, scratch);
        if (threadIdx.x == 0) {
            const float rstd = rsqrtf(fmaf(sums[0], inv_d, a.eps));
            terms[r] = {mean, rstd, sums[1] * inv_n, sums[2] * rstd * inv_d * rstd};
        }
    }
}

// dx and the column sums once the rows' terms are known.  A warp takes 32 * E columns of every 8 * gridDim.y-th row;
// the block's eight warps add their column sums through shared memory and write one partial row.
template <typename T, int E>
__global__ void __launch_bounds__(256) layernorm_backward_apply_kernel(const LayerNormBackwardArgs<T> a, const LayerNormRowTerms *terms) {
    using Chunk = RowChunk<T, E>;
    __shared__ float fold[8][32 * E + 1];
    grid_launch_dependents();
    grid_dependency_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = (int)(blockIdx.x * 32 + lane) * E;
    const bool active = c < a.cols;
    float gamma[E], dgamma[E], dbeta[E];
#pragma unroll
    for (int e = 0; e < E; ++e) gamma[e] = 1.f, dgamma[e] = 0.f, dbeta[e] = 0.f;
    if (active) {
        if (a.gamma) Chunk::unpack(Chunk::load(a.gamma + c), gamma);
#pragma unroll 2
        for (long long r = (long long)blockIdx.y * 8 + warp; r < a.rows; r += (long long)gridDim.y * 8) {
            const size_t at = (size_t)r * a.cols + c;
            const float4 t4 = __ldcg(reinterpret_cast<const float4 *>(terms + r));  // written by the kernel before: past the L1
            const LayerNormRowTerms t = {t4.x, t4.y, t4.z, t4.w};
            float f[E], g[E], res[E], o[E];
            Chunk::unpack(Chunk::load(a.x + at), f);
            Chunk::unpack(Chunk::load(a.dy + at), g);
            Chunk::unpack(a.residual ? Chunk::load(a.residual + at) : Chunk::zero(), res);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float dev = f[e] - t.mean;
                dgamma[e] = fmaf(g[e], dev * t.rstd, dgamma[e]);
                dbeta[e] += g[e];
                o[e] = fmaf(t.rstd, fmaf(-dev, t.c2, fmaf(g[e], gamma[e], -t.c1)), res[e]);
            }
            Chunk::store(a.dx + at, Chunk::pack(o));
        }
    }
    if (a.partials == nullptr) return;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
#pragma unroll
        for (int e = 0; e < E; ++e) fold[warp][lane * E + e] = which ? dbeta[e] : dgamma[e];
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * E; i += 256) {
            const int col = (int)blockIdx.x * 32 * E + i;
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) sum += fold[w][i];
            if (col < a.cols) a.partials[((size_t)blockIdx.y * 2 + which) * a.cols + col] = sum;
        }
        __syncthreads();
    }
}

// dgamma / dbeta = the partial rows added in order: a block takes 32 columns, warp w the partial rows w, w + 8, ...
// (a template only so that the header may be included by several translation units)
template <int kWarps = 8>
__global__ void __launch_bounds__(32 * kWarps) layernorm_backward_fold_kernel(const float *partials, int partial_rows, int cols,
                                                                              float *dgamma, float *dbeta) {
    __shared__ float fold[2][kWarps][32];
    grid_launch_dependents();
    grid_dependency_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int col = (int)blockIdx.x * 32 + lane;
    float g = 0.f, b = 0.f;
    if (col < cols)
#pragma unroll 4
        for (int p = warp; p < partial_rows; p += kWarps) {
            g += __ldcg(partials + (size_t)p * 2 * cols + col);
            b += __ldcg(partials + ((size_t)p * 2 + 1) * cols + col);
        }
    fold[0][warp][lane] = g;
    fold[1][warp][lane] = b;
    __syncthreads();
    if (warp < 2 && col < cols) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += fold[warp][w][lane];
        if (warp == 0 && dgamma) dgamma[col] = sum;
        if (warp == 1 && dbeta) dbeta[col] = sum;
    }
}

}  // namespace ko
