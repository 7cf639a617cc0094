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

// Rows that fit the registers of up to 16 warps: one pass over memory.  kLanes threads (part of a warp, or whole warps) hold a
// row, each of them kVecs chunks of E columns of x and dy; a block takes kRows consecutive rows at a time and persists over
// the rows, so a thread meets the same columns in every row: gamma stays in registers and so do its dgamma and dbeta, which
// leave once per block.  Per row two reductions of two values each: sum x and sum w, then, with the mean, sum dev^2 and
// sum w dev.
//
// Rows are consecutive bytes: the first warp brings a step's rows of x, dy and the residual into a shared-memory ring by bulk
// copies (cp.async.bulk, counted in bytes on an mbarrier), several steps ahead, so the bytes in flight depend neither on
// registers nor on how many warps the row's reductions keep waiting.  Bulk copies want 16-byte boundaries: rows of single
// elements (E == 1: odd widths, unaligned operands) come by plain loads instead.
//
// 16-bit rows leave about 34 instruction slots per element at full bandwidth (6 bytes an element, 22 bytes per clock and
// SM), so arithmetic runs on packed FP32 pairs, elements are unpacked once, and a thread holds 16 columns to spread the
// reductions' shuffles over many elements.
//
// Measured (B200, with the kernel that adds the partial rows; copy bandwidth 6447 GB/s): BF16 [32768, 4096] with residual
// 190 us = 5.64 TB/s (177 us = 4.55 TB/s without: there the instruction slots bind, 70 % of them taken), FP32 [16384, 768]
// 30 us = 5.0 TB/s of which the second kernel is 3, FP32 [8192, 5120] with residual 103 us = 6.5 TB/s, FP16 [30000, 1001]
// 54 us = 3.3 TB/s (two-byte loads).
constexpr int kBackwardWarpsPerSm = 16;  // at 128 registers a thread
constexpr int kBackwardMaxStages = 8;

// warps of a block for rows of `lanes` threads: whole rows, about eight warps
__host__ __device__ constexpr int backward_warps(int lanes) {
    const int group = lanes <= 32 ? 1 : lanes / 32;
    if (group == 3 || group == 5) return 15;
    return group >= 8 ? group : group * (8 / group);
}
__host__ __device__ constexpr int backward_blocks_per_sm(int lanes) { return kBackwardWarpsPerSm / backward_warps(lanes); }

// sums of two values over the kLanes threads of a row, in every thread of it
template <int kLanes>
struct RowReduce {
    float *scratch;  // [2][warps of a row][2], 16-byte aligned; only for rows of several warps
    int barrier;     // named barrier of the row's warps
    int turn = 0;
    __device__ __forceinline__ void operator()(float &a, float &b) {
        constexpr int kWidth = kLanes < 32 ? kLanes : 32;
        // the lower half of the lanes goes on with a, the upper half with b: five exchanges for both sums
        const int lane = threadIdx.x & 31;
        const bool upper = lane & (kWidth / 2);
        float v = upper ? b : a;
        v += __shfl_xor_sync(kFullMask, upper ? a : b, kWidth / 2);
#pragma unroll
        for (int m = kWidth / 4; m > 0; m >>= 1) v += __shfl_xor_sync(kFullMask, v, m);
        if constexpr (kLanes <= 32) {
            a = __shfl_sync(kFullMask, v, 0, kWidth);
            b = __shfl_sync(kFullMask, v, kWidth / 2, kWidth);
        } else {
            // Two scratch halves in turn: whoever writes a half again has passed the barrier of the reduction in between, so
            // everyone has read it.
            constexpr int kGroup = kLanes / 32;
            float *half = scratch + turn * 2 * kGroup;
            turn ^= 1;
            if ((lane & 15) == 0) half[2 * ((threadIdx.x >> 5) % kGroup) + (lane >> 4)] = v;
            asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(kLanes) : "memory");
            f32x2 sum = *reinterpret_cast<const f32x2 *>(half);
#pragma unroll
            for (int w = 1; w < kGroup; ++w) sum = pair_add(sum, *reinterpret_cast<const f32x2 *>(half + 2 * w));
            pair_split(sum, a, b);
        }
    }
};

// Rows of more than a warp have a place of their own in the ring, as wide as the columns their threads cover: every address is
// then a constant away from the stage's, and the columns past the row's end read zeros that are written once.  Each row is a
// copy of its own then, which shorter rows do not bear (131072 x 256 BF16 60 us against 47 with one copy for a step's rows).
template <int kLanes>
constexpr bool kBackwardPadded = kLanes >= 64;
template <typename T, int E, int kVecs, int kLanes>
__host__ __device__ constexpr uint32_t backward_pitch(int cols) {
    return (uint32_t)((kBackwardPadded<kLanes> ? kLanes * kVecs * E : cols) * (int)sizeof(T));
}

// stages: steps of kRows rows in the ring (dynamic shared memory: [stages][x, dy(, residual)][kRows][pitch], at least
// 2 * kCapacity floats for the column sums at the end); status: the staged row operators' device status word
template <typename T, int E, int kVecs, int kLanes>
__global__ void __launch_bounds__(32 * backward_warps(kLanes), backward_blocks_per_sm(kLanes))
layernorm_backward_resident_kernel(const LayerNormBackwardArgs<T> a, int stages, unsigned *status) {
    using Chunk = RowChunk<T, E>;
    using Raw = typename Chunk::Raw;
    constexpr int kWarps = backward_warps(kLanes), kRows = 32 * kWarps / kLanes;
    constexpr int kCapacity = kLanes * kVecs * E, kPairs = kVecs * E / 2;
    constexpr bool kSingles = E == 1;  // a pair then spans two chunks, and rows come by plain loads
    constexpr bool kPadded = kBackwardPadded<kLanes>;
    const uint32_t pitch = backward_pitch<T, E, kVecs, kLanes>(a.cols);
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ __align__(16) float scratch[kLanes > 32 ? kRows : 1][kLanes > 32 ? 4 * (kLanes / 32) : 1];
    __shared__ uint64_t full[kBackwardMaxStages], empty[kBackwardMaxStages];
    __shared__ int abort_flag;
    const int slot = threadIdx.x / kLanes, t = threadIdx.x % kLanes;
    RowReduce<kLanes> reduce{kLanes > 32 ? scratch[slot] : nullptr, 1 + slot};
    const float inv_n = 1.0f / (float)a.cols, inv_d = a.cols > a.ddof ? 1.0f / (float)(a.cols - a.ddof) : 0.f;
    f32x2 gamma[kPairs], dgamma[kPairs], dbeta[kPairs];
    bool active[kVecs];
#pragma unroll
    for (int v = 0; v < kVecs; ++v) active[v] = (t + v * kLanes) * E < a.cols;

    auto unpack = [](const Raw (&raw)[kVecs], f32x2 (&p)[kPairs]) {
        if constexpr (kSingles) {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) p[i] = pair_of(RowIo<T>::to_float(raw[2 * i]), RowIo<T>::to_float(raw[2 * i + 1]));
        } else {
#pragma unroll
            for (int v = 0; v < kVecs; ++v) RowIo<T>::unpack_pairs(raw[v], p + v * (E / 2));
        }
    };
    // the thread's chunks of a row in global memory; zeros past the row's end, or everywhere in a row that is not there
    auto load = [&](const T *row, bool there, f32x2 (&p)[kPairs]) {
        Raw raw[kVecs];
#pragma unroll
        for (int v = 0; v < kVecs; ++v) raw[v] = active[v] && there ? Chunk::load(row + (t + v * kLanes) * E) : Chunk::zero();
        unpack(raw, p);
    };
    // the same of a row in the ring, at the address of the thread's first chunk
    auto staged = [&](uint32_t at, bool there, f32x2 (&p)[kPairs]) {
        if constexpr (!kSingles) {
            Raw raw[kVecs];
#pragma unroll
            for (int v = 0; v < kVecs; ++v) {
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (kPadded || (active[v] && there))
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                                 : "r"(at + (uint32_t)(v * kLanes * 16)));
                raw[v] = *reinterpret_cast<const Raw *>(&w);
            }
            unpack(raw, p);
        }
    };

    // ring: step s of this block, rows first_row + s * stride .. + kRows - 1, lives in stage s % stages
    const uint32_t tensor_bytes = kRows * pitch, stage_bytes = tensor_bytes * (a.residual ? 3u : 2u);
    const long long first_row = (long long)blockIdx.x * kRows, stride = (long long)gridDim.x * kRows;
    const int steps = (int)((a.rows - 1 - first_row) / stride) + 1;  // the grid has no idle block
    auto bring = [&](long long row, uint32_t stage) {  // whole warp 0: one copy per tensor, or padded a lane per row
        const int lane = threadIdx.x, rows = (int)(a.rows - row < kRows ? a.rows - row : kRows);
        const uint32_t row_bytes = (uint32_t)a.cols * (uint32_t)sizeof(T), bar = smem_u32(full + stage);
        if (lane == 0) mbar_expect_tx(bar, (a.residual ? 3u : 2u) * (uint32_t)rows * row_bytes);
        __syncwarp();
        if (lane < (kPadded ? rows : 1)) {
            const uint32_t bytes = kPadded ? row_bytes : (uint32_t)rows * row_bytes;
            const size_t at = (size_t)(row + lane) * a.cols;
            const uint32_t dst = smem_u32(ring) + stage * stage_bytes + (uint32_t)lane * pitch;
            bulk_load_1d(dst, a.x + at, bytes, bar);
            bulk_load_1d(dst + tensor_bytes, a.dy + at, bytes, bar);
            if (a.residual) bulk_load_1d(dst + 2 * tensor_bytes, a.residual + at, bytes, bar);
        }
    };
    auto give_up = [&](unsigned code) {  // a wait ran out: the rest runs through without waiting, the host is told
        atomicCAS(status, 0u, code);
        *(volatile int *)&abort_flag = 1;
    };

    if constexpr (!kSingles) {
        if constexpr (kPadded) {  // zeros behind every row of the ring, where the copies do not reach
            const int pad = kCapacity / E - a.cols / E, pads = stages * (a.residual ? 3 : 2) * kRows * pad;
            for (int i = threadIdx.x; i < pads; i += 32 * kWarps)
                *reinterpret_cast<uint4 *>(ring + (size_t)(i / pad) * pitch + (size_t)(a.cols / E + i % pad) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        if (threadIdx.x == 0) {
            for (int s = 0; s < stages; ++s) {
                mbar_init(smem_u32(full + s), 1);
                mbar_init(smem_u32(empty + s), kWarps);
            }
            abort_flag = 0;
            fence_barrier_init();
            fence_proxy_async();
        }
        __syncthreads();
    }
    grid_launch_dependents();
    grid_dependency_wait();
    if (!kSingles && threadIdx.x < 32)
        for (int i = 0; i < stages && i < steps; ++i) bring(first_row + i * stride, (uint32_t)i);
    // a row's columns past the last one: x = dy = gamma = 0
    if (a.gamma) {
        load(a.gamma, true, gamma);
    } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            const float lo = active[2 * i / E] ? 1.f : 0.f, hi = active[(2 * i + 1) / E] ? 1.f : 0.f;
            gamma[i] = pair_of(lo, hi);
        }
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i) dgamma[i] = dbeta[i] = pair_of(0.f, 0.f);

    uint32_t stage = 0, phase = 0;
    long long r = first_row + slot;
    T *dx = a.dx + (size_t)r * a.cols + t * E;
    const uint32_t my_chunks = smem_u32(ring) + (uint32_t)slot * pitch + (uint32_t)t * 16u;
    for (int step = 0; step < steps; ++step, r += stride, dx += (size_t)stride * a.cols) {
        const bool there = r < a.rows;
        // Rows past the end are met in the last step only.  Whole warps leave; parts of a warp stay for its shuffles, with
        // zeros, and store nothing.  Single elements stay as well, and find their row's address anew at the store: with the early way
        // out, and the address carried through the loop, the 128 registers do not do (8 bytes spilled; FP16 [30000, 1001] 62.7 us
        // against 54.5, [30000, 501] 36.2 against 29.5).
        if (!kSingles && kLanes >= 32 && !there) break;
        f32x2 x[kPairs], dy[kPairs];
        const uint32_t here = my_chunks + stage * stage_bytes;
        if constexpr (kSingles) {
            load(a.x + (size_t)r * a.cols, there, x);
            load(a.dy + (size_t)r * a.cols, there, dy);
        } else {
            if (!warp_all(mbar_wait(smem_u32(full + stage), phase, &abort_flag))) give_up(2u);
            staged(here, there, x);
            staged(here + tensor_bytes, there, dy);
        }
        f32x2 sum_x2 = x[0], sum_w2 = pair_mul(dy[0], gamma[0]);
#pragma unroll
        for (int i = 1; i < kPairs; ++i) {
            sum_x2 = pair_add(sum_x2, x[i]);
            sum_w2 = pair_fma(dy[i], gamma[i], sum_w2);
        }
        float lo, hi, sum_x, sum_w;
        pair_split(sum_x2, lo, hi);
        sum_x = lo + hi;
        pair_split(sum_w2, lo, hi);
        sum_w = lo + hi;
        reduce(sum_x, sum_w);
        // the stage of the step before: by now every warp of this row is done with it
        if (!kSingles && threadIdx.x < 32 && step > 0 && step - 1 + stages < steps) {
            const uint32_t before = stage ? stage - 1 : (uint32_t)stages - 1;
            if (!warp_all(mbar_wait(smem_u32(empty + before), stage ? phase : phase ^ 1u, &abort_flag))) give_up(3u);
            else bring(r - slot + (stages - 1) * stride, before);
        }
        const float mean = sum_x * inv_n;
        f32x2 minus_mean[kSingles ? kPairs : kVecs];  // 0 past the row's end: the deviation is 0 there
#pragma unroll
        for (int i = 0; i < (kSingles ? kPairs : kVecs); ++i)
            minus_mean[i] = kSingles ? pair_of(active[(2 * i) % kVecs] ? -mean : 0.f, active[(2 * i + 1) % kVecs] ? -mean : 0.f)
                                     : (active[i] ? pair_of(-mean, -mean) : pair_of(0.f, 0.f));
        f32x2 m2_2 = pair_of(0.f, 0.f), sum_wd2 = m2_2;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            x[i] = pair_add(x[i], minus_mean[kSingles ? i : 2 * i / E]);  // x holds the deviations from here on
            m2_2 = pair_fma(x[i], x[i], m2_2);
            sum_wd2 = pair_fma(pair_mul(dy[i], gamma[i]), x[i], sum_wd2);
        }
        float m2, sum_wd;
        pair_split(m2_2, lo, hi);
        m2 = lo + hi;
        pair_split(sum_wd2, lo, hi);
        sum_wd = lo + hi;
        reduce(m2, sum_wd);
        const float rstd = there ? rsqrtf(fmaf(m2, inv_d, a.eps)) : 0.f;  // (eps may be 0, and then 0 * rstd no longer is)
        // dx = rstd w - rstd c1 - xhat rstd c2, c1 = sum(w) / n, c2 = sum(w xhat) / d
        const float offset = -rstd * sum_w * inv_n, slope = -rstd * (sum_wd * rstd * inv_d);
        const f32x2 rstd2 = pair_of(rstd, rstd), offset2 = pair_of(offset, offset), slope2 = pair_of(slope, slope);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            const f32x2 xhat = pair_mul(x[i], rstd2);
            dgamma[i] = pair_fma(dy[i], xhat, dgamma[i]);
            dbeta[i] = pair_add(dbeta[i], dy[i]);
            x[i] = pair_fma(xhat, slope2, pair_fma(pair_mul(dy[i], gamma[i]), rstd2, offset2));
        }
        if (a.residual) {
            f32x2 add[kPairs];
            if constexpr (kSingles) load(a.residual + (size_t)r * a.cols, there, add);
            else staged(here + 2 * tensor_bytes, there, add);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) x[j] = pair_add(x[j], add[j]);
        }
        if constexpr (!kSingles) {
            __syncwarp();
            if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(empty + stage));
            if (++stage == (uint32_t)stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if ((!kSingles && kLanes >= 32) || there) {
            T *out = kSingles ? a.dx + (size_t)r * a.cols + t : dx;
#pragma unroll
            for (int v = 0; v < kVecs; ++v)
                if (active[v]) {
                    if constexpr (kSingles) {
                        float lo, hi;
                        pair_split(x[v / 2], lo, hi);
                        out[v * kLanes] = RowIo<T>::from_float(v & 1 ? hi : lo);
                    } else {
                        Chunk::store(out + v * kLanes * E, RowIo<T>::pack_pairs(x + v * (E / 2)));
                    }
                }
        }
    }
    if (!kSingles && threadIdx.x == 0 && *(volatile int *)&abort_flag) {
        // copies on their way still land in this block's shared memory: wait (bounded) for each stage's last one
        for (int s = 0; s < stages; ++s)
            for (uint32_t parity = 0; parity < 2; ++parity)
                for (uint32_t spin = 0; spin < kSpinLimit / 64 && !mbar_try_wait(smem_u32(full + s), parity); ++spin) {}
    }
    if (a.partials == nullptr) return;
    auto column = [&](int i) { return kSingles ? t + i * kLanes : (t + (i / E) * kLanes) * E + i % E; };  // of the thread's i-th value
    float *out = a.partials + (size_t)blockIdx.x * 2 * a.cols;
    if constexpr (kRows > 1) {
        float *fold = reinterpret_cast<float *>(ring);  // every stage has been read: the ring is free
        __syncthreads();
        // the block's rows add their column sums one after the other, then the block writes one partial row
        for (int turn = 0; turn < kRows; ++turn) {
            if (slot == turn) {
#pragma unroll
                for (int i = 0; i < kPairs; ++i)
#pragma unroll
                    for (int which = 0; which < 2; ++which) {
                        float v[2];
                        pair_split(which ? dbeta[i] : dgamma[i], v[0], v[1]);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float *at = fold + which * kCapacity + column(2 * i + h);
                            *at = turn ? *at + v[h] : v[h];
                        }
                    }
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < a.cols; i += 32 * kWarps) {
            out[i] = fold[i];
            out[a.cols + i] = fold[kCapacity + i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                float v[2];
                pair_split(which ? dbeta[i] : dgamma[i], v[0], v[1]);
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (column(2 * i + h) < a.cols) out[which * a.cols + column(2 * i + h)] = v[h];
            }
    }
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

// dgamma / dbeta = the partial rows added in a fixed order: a block takes 32 columns, warp w of 32 the partial rows w, w + 32,
// ... (few loads per thread, all in flight: the kernel is latency)
// (a template only so that the header may be included by several translation units)
template <int kWarps = 32>
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
