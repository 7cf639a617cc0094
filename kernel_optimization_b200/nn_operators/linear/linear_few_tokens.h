// The linear layer for a handful of tokens (decoding): Y[m, n] = act(sum_k X[m, k] W[n, k] + bias[n]) + residual, m < 32.
//
// With few tokens the weights are read once and used a handful of times, so the kernel is bound by how fast W streams
// in: a 128-row tensor-core tile would be nearly empty, and its pipeline's fill and drain cost more than the whole read.
// Here W is the 16-row operand of mma.sync m16n8k16 and the tokens are the 8-wide one.  Both operands come straight from
// global memory into fragments: the inner dimension may be permuted as long as both agree, so a thread takes 8
// consecutive k (16 bytes) of W row g, of W row g + 8 and of token g, and feeds them to two MMAs as if they were the
// columns the instruction names (2t, 2t + 1, 2t + 8, 2t + 9).  No shared memory, no barrier in the loop.
//
// A block takes kSlabs * 16 rows of W; its warps, and the blocks of its cluster, take 32 * kChunks-wide pieces of K in
// turn, so that the whole device reads even when N is small.  FP32 partial sums are added in a fixed order, first over
// the block's warps, then over the cluster's blocks through distributed shared memory.
#pragma once

#include <cooperative_groups.h>

#include "linear_epilogue.h"

namespace ko {

constexpr int kFewTokens = 32;  // the most this kernel takes

template <bool kBf16>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (kBf16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of W: read once by one thread, so they pass the L1 by (they stay in the L2: the next token reads them again)
__device__ __forceinline__ uint4 ld_weights(const uint16_t *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

struct FewTokensParams {
    LinearParams p;
    const void *X, *W;
};

// kTiles: token tiles of 8; kChunks: 32-wide pieces of K a warp loads together; kPromote: for FP32 results, and 16-bit ones of long sums
template <bool kBf16, bool kOut16, bool kPromote, int kTiles, int kSlabs, int kChunks, int kWarps>
__global__ void __launch_bounds__(32 * kWarps) linear_few_tokens_kernel(const __grid_constant__ FewTokensParams q) {
    const LinearParams &p = q.p;
    constexpr int kRows = 16 * kSlabs, kCols = 8 * kTiles;
    __shared__ float part[kWarps][kRows][kCols + 1];
    __shared__ float sums[kRows * kCols];
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = (int)(blockIdx.x / ranks) * kRows;
    float acc[kSlabs][kTiles][4];
#pragma unroll
    for (int s = 0; s < kSlabs; ++s)
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[s][i][e] = 0.f;
    // rows of W past N and tokens past M are read from the last one there is and never stored
    const uint16_t *w_row[kSlabs][2], *x_row[kTiles];
#pragma unroll
    for (int s = 0; s < kSlabs; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            w_row[s][h] = static_cast<const uint16_t *>(q.W) + (size_t)min(n0 + s * 16 + h * 8 + g, p.N - 1) * p.K + t * 8;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) x_row[i] = static_cast<const uint16_t *>(q.X) + (size_t)min(i * 8 + g, p.M - 1) * p.K + t * 8;
    grid_launch_dependents();
    // The previous kernel may still be running, and W may be what it writes: nothing is read yet, but a warp's first piece of W can
    // be on its way into the L2 (1 x 4096 x 4096 9.3 -> 8.7 us, 1 x 14336 x 4096 25.3 -> 24.4).  Not where a cluster of four or
    // eight shares few rows: the pieces are then most of K (4 x 1024 x 8192 6.1 -> 6.7), nor
    // for 32 rows a block (32 x 8192 x 2048 13.2 either way).
    const int first = (rank * kWarps + warp) * 32 * kChunks;
    if (kSlabs == 1 && ranks <= 2 && t == 0)
#pragma unroll
        for (int c = 0; c < kChunks; c += 2)
#pragma unroll
            for (int s = 0; s < kSlabs; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (first + c * 32 < p.K) asm volatile("prefetch.global.L2 [%0];" ::"l"(w_row[s][h] + first + c * 32));
    grid_dependency_wait();
    const int stride = ranks * kWarps * 32 * kChunks;
    // A result is not to show how the matrix instructions cut their accumulators off (see LinearEpilogue): every 1024 values of
    // K a warp adds them to sums of its own.
    float sum[kPromote ? kSlabs : 1][kPromote ? kTiles : 1][4] = {};
    int pieces = 0;
    for (int k0 = first; k0 < p.K; k0 += stride) {
        uint4 w[kChunks][kSlabs][2], x[kChunks][kTiles];
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int k = k0 + c * 32;
            const bool in = k + t * 8 < p.K;  // K is a multiple of 8: a vector lies inside or outside as a whole
#pragma unroll
            for (int s = 0; s < kSlabs; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) w[c][s][h] = in ? ld_weights(w_row[s][h] + k) : zero;
#pragma unroll
            for (int i = 0; i < kTiles; ++i) x[c][i] = in ? *reinterpret_cast<const uint4 *>(x_row[i] + k) : zero;
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int s = 0; s < kSlabs; ++s)
#pragma unroll
                for (int i = 0; i < kTiles; ++i) {
                    mma_16x8x16<kBf16>(acc[s][i], w[c][s][0].x, w[c][s][1].x, w[c][s][0].y, w[c][s][1].y, x[c][i].x, x[c][i].y);
                    mma_16x8x16<kBf16>(acc[s][i], w[c][s][0].z, w[c][s][1].z, w[c][s][0].w, w[c][s][1].w, x[c][i].z, x[c][i].w);
                }
        if constexpr (kPromote) {
            if (++pieces == 1024 / (32 * kChunks)) {
                pieces = 0;
#pragma unroll
                for (int s = 0; s < kSlabs; ++s)
#pragma unroll
                    for (int i = 0; i < kTiles; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            sum[s][i][e] += acc[s][i][e];
                            acc[s][i][e] = 0.f;
                        }
            }
        }
    }
#pragma unroll
    for (int s = 0; s < kSlabs; ++s)
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                part[warp][s * 16 + (e >> 1) * 8 + g][i * 8 + 2 * t + (e & 1)] = kPromote ? sum[s * kPromote][i * kPromote][e] + acc[s][i][e] : acc[s][i][e];
    __syncthreads();
    // element i of the block: token i / kRows, W row i % kRows (stores of a token's outputs are then contiguous)
    for (int i = threadIdx.x; i < kRows * kCols; i += 32 * kWarps) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += part[w][i % kRows][i / kRows];
        sums[i] = v;
    }
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    // the cluster's blocks share the outputs: each adds its part of them over the blocks, in rank order
    for (int i = rank * 32 * kWarps + threadIdx.x; i < kRows * kCols; i += ranks * 32 * kWarps) {
        float v = 0.f;
        for (int r = 0; r < ranks; ++r) v += ranks > 1 ? *cluster.map_shared_rank(sums + i, r) : sums[i];
        const int token = i / kRows, n = n0 + i % kRows;
        if (token < p.M && n < p.N) {
            v = linear_finish_one<LinearMode::kForward, kBf16, kOut16>(p, v, token, n);
            linear_store_one<kBf16, kOut16>(p, v, token, n);
        }
    }
    if (ranks > 1) cluster.sync();  // nobody leaves while its sums may still be read
}

}  // namespace ko
