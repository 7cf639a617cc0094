// Fused epilogues of the tensor-core GEMM kernels for the linear layer and its gradients:
//   forward        Y = act(X W^T + bias) + residual, and Z = X W^T + bias (16 bits) when the backward pass wants it
//   input grad     dX = (dY W) * act'(Z)
//   weight grad    dW = dY^T X + C   (A = dY stored [tokens, features]: MN-major operand)
// An accumulator chunk of 32 rows x 128 bytes of output (64 columns of 16 bits, 32 of FP32) goes from tensor memory through
// registers to a swizzled box in shared memory and out by one TMA store of full 128-byte lines.  What it is combined with
// (residual, Z or C) comes the other way: one TMA load per chunk into a box of the warp's own, issued a chunk ahead -- the
// first chunk's while the tile is still being multiplied -- so neither direction takes issue slots or L1 from the warps.
// Everything is FP32 until one rounding to the stored type.  Eight epilogue warps, two per quadrant of TMEM lanes: an
// activation costs about ten issue slots an element, which four warps alone could not hide behind the next tile's MMAs.
// (Four for the weight gradient, which only stores.)
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
    // weight grad, the column sums of dY (see ColumnSums): tiles of a row of tiles that share them (0: none are wanted), where
    // their parts go, [split_k * sum_shares, M] (a single part: dbias itself), and where the parts' sum goes
    int sum_shares;
    float *sum_parts, *dbias;
    alignas(64) CUtensorMap map_pre, map_extra;
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
// Z is written here.  (__fadd_rn: no contraction with an activation's last product, so that every form of the epilogue
// gives the same bits.)
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
            v = __fadd_rn(v, widen16_at<kBf16>(p.extra, at));
        } else {
            v = __fadd_rn(v, static_cast<const float *>(p.extra)[at]);
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

// Column sums of dY, the bias gradient, by two warps beside the product: dY's tiles lie in shared memory for the matrix
// instructions anyway, so the sums cost neither the L2 nor DRAM another reading of it.  (A kernel of their own beside or ahead
// of the product cost 20 us in 147 at 16384 tokens of 4096 features, x 1024.)  All tiles of the same rows of dW see the same dY; the
// first sum_shares of them (of a pair: of those whose leaders hold the rows) take its K-blocks in turn, so that no CTA's shared memory
// serves much more than the others'.
// A warp takes 64 columns, a lane eight of them in every fourth of a K-block's 64 rows; the rows of a K-block are added first,
// then the K-blocks: chains of 16 and K / 64 FP32 additions.
struct ColumnSums {
    f32x2 sum[4] = {pair_of(0.f, 0.f), pair_of(0.f, 0.f), pair_of(0.f, 0.f), pair_of(0.f, 0.f)};

    // box: shared-memory address of 64 rows x 64 columns, 128-byte rows with their 16-byte pieces swizzled by the row
    template <bool kBf16>
    __device__ __forceinline__ void add_box(uint32_t box, int lane) {
        f32x2 part[4];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int row = 4 * i + (lane >> 3);
            uint32_t w[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "r"(box + row * 128 + (((lane & 7) ^ (row & 7)) << 4))
                         : "memory");
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float lo, hi;
                widen16<kBf16>(w[j], lo, hi);
                part[j] = i ? pair_add(part[j], pair_of(lo, hi)) : pair_of(lo, hi);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] = pair_add(sum[j], part[j]);
    }
    __device__ __forceinline__ void add(const LinearParams &p, uint32_t box, int lane) {
        if (p.fmt) add_box<true>(box, lane);
        else add_box<false>(box, lane);
    }
    // part: number of this part; row: first of the warp's 64 rows of the product
    __device__ __forceinline__ void store(const LinearParams &p, int part, int row, int lane) const {
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) pair_split(sum[j], v[2 * j], v[2 * j + 1]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] += __shfl_xor_sync(kFullMask, v[i], 16);
            v[i] += __shfl_xor_sync(kFullMask, v[i], 8);
        }
        const int at = row + lane * 8;
        if (lane >= 8 || at >= p.M) return;  // M is a multiple of 8
        float *to = p.sum_parts + (size_t)part * p.M + at;
#pragma unroll
        for (int i = 0; i < 8; ++i) to[i] = v[i];
    }
};

// the parts of row `row`, added in their order
__device__ __forceinline__ float fold_sum_parts(const LinearParams &p, int row) {
    const int parts = p.sum_shares * p.split_k;
    float total = 0.f;
    for (int i0 = 0; i0 < parts; i0 += 8) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i0 + i < parts ? __ldcg(p.sum_parts + (size_t)(i0 + i) * p.M + row) : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) total += v[i];
    }
    return total;
}
// where no kernel adds slices of the product
template <int kBlock = 256>
__global__ void __launch_bounds__(kBlock) linear_fold_sums_kernel(const LinearParams p) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int row = blockIdx.x * kBlock + threadIdx.x;
    if (row < p.M) p.dbias[row] = fold_sum_parts(p, row);
}

// kPromote (FP32 results of more than 1024 values of K, 16-bit ones of more than 16384): the tensor cores cut their accumulator off
// at every addition instead of rounding it, so an error grows with K on the side of smaller magnitudes -- 4.5e-6 of the result
// (2-norm) at K = 4096, 1.9e-5 at 16384, where a blocked FP32 sum is off by 6e-7 and 1.5e-6.  A tile is then taken in periods of 896
// values of K, each into the other of the two accumulators, and the epilogue warps add the periods' sums, rounded to nearest, in
// registers (128 a thread for a tile 256 columns wide) while the next period is being multiplied: 9e-7 at any K.  Hidden where a CTA
// has one tile (16384 x 4096 x 1024 dW: 101 us either way).  With several the total holds one of the accumulators while it is being
// stored, and the next tile gets no further than a period meanwhile: 4096^3 to FP32 101 -> 135 .. 145 us.  (Storing from the registers
// instead spilled them: 206 with periods of 1024; periods of 512, too short for the additions: 204.)
// K-blocks of 64 that one accumulator may take.  16-bit results: what is cut off stays below a sixteenth of half a step of FP16,
// 2^-15, up to 16384 values of K (terms of one sign: 2^-25 of the result for each of K / 16 instructions).  In one accumulator over
// 400000 positive terms FP16 results were off by more than a step.  Their periods are of 8192 (dW of 65536 tokens, 2048 x 2048, to
// BF16 366 -> 383 us; with periods of 896 422).
constexpr int blocks_in_one_accumulator(bool out16) { return out16 ? 256 : 16; }

template <LinearMode kMode, bool kOut16, bool kPromoteSums = false>
struct LinearEpilogue {
    using Params = LinearParams;
    static constexpr bool kTransA = kMode == LinearMode::kWeightGrad;
    static constexpr bool kPromote = kPromoteSums;
    static constexpr int kPeriod = kOut16 ? 128 : 14;  // K-blocks of an accumulator: 896 values of K, or 8192
    static constexpr int kWarps = kTransA && !kPromote ? 4 : 8;
    static constexpr bool kFused = true;
    static constexpr int kSumWarps = kTransA ? 2 : 0;  // 64 columns of dY each, see ColumnSums
    using Sums = ColumnSums;
    static constexpr bool kExtra16 = kMode == LinearMode::kInputGrad || kOut16;
    static constexpr int kChunk = kOut16 ? 64 : 32;           // columns
    static constexpr int kStep = kChunk * (kWarps / 4);        // from one chunk of a warp to its next
    static constexpr uint32_t kBoxBytes = 4096;
    static constexpr int kBoxesPerWarp = 2;

    // a warp's boxes and mbarrier, and where it stands with them
    struct State {
        uint32_t boxes, bar;
        uint32_t stores = 0;  // TMA stores issued
        uint32_t phase = 0;   // of the extra operand's box
        bool coming = false;  // an extra load has been issued and not waited for
    };

    // The promoted sums of a tile's `periods` accumulators, the first of them number `first` of the CTA's sequence: all but the
    // last are added up in registers -- this warp's 32 rows of the chunks share * 32, share * 32 + 64, ... -- and given
    // back; the last receives the total, for the rest of the epilogue to find there.  wide: the chunks are those of a 16-bit result, 64
    // columns from share * 64, from there + 128 and so on.  t_rows: TMEM address of the warp's
    // rows in accumulator 0; ready, free: the accumulators' mbarriers (free as a shared::cluster address where the MMAs are
    // issued by another CTA).  False when a wait ran out.  A function of its own, so that its registers and those of the
    // code around it do not add up.
    template <int BN, bool kRemote>
    __device__ __noinline__ static bool promote(uint32_t t_rows, int share, bool wide, int periods, uint32_t first, uint32_t ready, uint32_t free,
                                                volatile int *abort_flag) {
        constexpr int kChunks = BN / 64;
        f32x2 sums[kChunks][16];
        for (uint32_t n = first; n < first + (uint32_t)periods; ++n) {
            const uint32_t acc = n & 1u, t_row = t_rows + acc * BN + share * (wide ? 64 : 32);
            if (!warp_all(mbar_wait(ready + 8u * acc, (n >> 1) & 1u, abort_flag))) return false;
            tc::tc_fence_after();
            const bool last = n + 1 == first + (uint32_t)periods;
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                float f[32];
                const uint32_t at = t_row + (wide ? (j >> 1) * 128 + (j & 1) * 32 : j * 64);
                tc::tmem_ld_32x32(at, f);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const f32x2 part = pair_of(f[2 * i], f[2 * i + 1]);
                    sums[j][i] = n == first ? part : pair_add(sums[j][i], part);
                }
                if (last) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) pair_split(sums[j][i], f[2 * i], f[2 * i + 1]);
                    tc::tmem_st_32x32(at, f);
                }
            }
            if (last) {
                tc::tmem_st_wait();
            } else {
                tc::tc_fence_before();
                __syncwarp();
                if ((threadIdx.x & 31) == 0) {
                    if constexpr (kRemote) mbar_arrive_cluster(free + 8u * acc);
                    else mbar_arrive(free + 8u * acc);
                }
            }
        }
        return true;
    }

    // the extra operand's chunk at (row_base, col) on its way into box 1
    __device__ __forceinline__ static void bring(State &st, const Params &p, int row_base, int col) {
        if (p.extra == nullptr || row_base >= p.M || col >= p.N) return;
        if (tc::elect_one()) {
            // a box is filled whole: what lies outside the matrix arrives as zeros and counts
            mbar_expect_tx(st.bar, kExtra16 && !kOut16 ? kBoxBytes / 2 : kBoxBytes);
            tc::tma_load_2d(st.boxes + kBoxBytes, &p.map_extra, col, row_base, st.bar);
        }
        st.coming = true;
    }

    // rows row_base .. + 31 of a tile, this warp's chunks c_begin, c_begin + kStep, ... of the accumulator at TMEM address t_row, to
    // D and Z; false when a wait ran out
    template <bool kTmaStore>
    __device__ __forceinline__ static bool block(const CUtensorMap *map_d, const Params &p, State &st, uint32_t t_row, int row_base,
                                                 int col0, int bn, int c_begin, int lane, volatile int *abort_flag) {
#pragma unroll 1
        for (int c0 = c_begin; c0 < bn; c0 += kStep) {
            if (row_base >= p.M || col0 + c0 >= p.N) break;
            if constexpr (kTmaStore) {
                if (st.coming) {
                    if (!warp_all(mbar_wait(st.bar, st.phase, abort_flag))) return false;
                    st.phase ^= 1u;
                    st.coming = false;
                }
                if (p.fmt) chunk<true>(map_d, p, st, t_row + c0, row_base, col0 + c0, c0 + kStep < bn, lane);
                else chunk<false>(map_d, p, st, t_row + c0, row_base, col0 + c0, c0 + kStep < bn, lane);
            } else {
#pragma unroll 1
                for (int h = 0; h < kChunk; h += 32) {
                    const int c = c0 + h, next = h + 32 < kChunk ? c + 32 : c0 + kStep;
                    const bool more = p.extra && next < bn && col0 + next < p.N;
                    float coming[32];  // the extra operand of the next chunk, on its way meanwhile
                    if (more) fetch_rows(p, coming, row_base, col0 + next + lane);
                    f32x2 r[16];
                    sums_at(t_row + c, r);
                    if (p.fmt) chunk_by_rows<true>(p, r, row_base, col0 + c, lane, st.boxes);
                    else chunk_by_rows<false>(p, r, row_base, col0 + c, lane, st.boxes);
                    if (more) keep_rows(st, coming, lane);
                }
            }
        }
        return true;
    }

    // the first chunk's extra operand for the row-wise form
    __device__ __forceinline__ static void bring_rows(State &st, const Params &p, int row_base, int col, int lane) {
        if (p.extra == nullptr || row_base >= p.M || col >= p.N) return;
        float x[32];
        fetch_rows(p, x, row_base, col + lane);
        keep_rows(st, x, lane);
    }

    // before the block leaves: nothing may still arrive in its shared memory or be read from it
    __device__ __forceinline__ static void finish(State &st) {
        if (st.coming)
            for (uint32_t spin = 0; spin < kSpinLimit && !mbar_try_wait(st.bar, st.phase); ++spin) {}
        if (tc::elect_one()) tc::bulk_wait_group_read<0>();
    }

private:
    // Rows that start anywhere (odd N, unaligned operands): the chunk is turned in shared memory (4 KB, column c of row r at
    // c ^ r: no bank conflict either way) so that a lane has one column, and every access is 32 neighbouring elements of
    // a row.  Written straight from a lane's own row, each store touched 32 sectors: 1021 x 2053 x 1096 FP32 22 us.
    // Instructions count: with 46 of them for a row's 32 elements the same call took 17.2 us, now 14.0 (30 -> 15.2 with a residual).
    template <bool kBf16>
    __device__ __forceinline__ static void chunk_by_rows(const Params &p, const f32x2 (&r)[16], int row_base, int col, int lane, uint32_t box) {
        using Stored = std::conditional_t<kOut16, uint16_t, float>;
        __syncwarp();
        const uint32_t own = box + (uint32_t)lane * 132u;  // boxes are aligned to their size
#pragma unroll
        for (int c = 0; c < 32; ++c) {
            float lo, hi;
            pair_split(r[c / 2], lo, hi);
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(own ^ (uint32_t)(c * 4)), "f"(c & 1 ? hi : lo) : "memory");
        }
        __syncwarp();
        const int c = col + lane, rows = min(32, p.M - row_base);
        if (c >= p.N) return;
        float bias = 0.f;
        if (kMode == LinearMode::kForward && p.bias) bias = widen16_at<kBf16>(p.bias, (size_t)c);
        const size_t at = (size_t)row_base * p.N + c;
        Stored *out = static_cast<Stored *>(p.D) + at;
        uint16_t *pre = kMode == LinearMode::kForward && p.pre ? static_cast<uint16_t *>(p.pre) + at : nullptr;
        const uint32_t column = box + (uint32_t)lane * 4u;
        constexpr int kRows = 8;
#pragma unroll 1
        for (int i0 = 0; i0 < rows; i0 += kRows) {
            const uint32_t from = (column + (uint32_t)i0 * 128u) ^ (uint32_t)(i0 * 4), extra = column + kBoxBytes + (uint32_t)i0 * 128u;
            const int left = rows - i0;
            float v[kRows];
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[i]) : "r"((from ^ (uint32_t)(i * 4)) + (uint32_t)i * 128u) : "memory");
                if constexpr (kMode == LinearMode::kForward)
                    if (p.bias) v[i] += bias;
            }
            if constexpr (kMode == LinearMode::kForward)
                if (pre) {
                    uint16_t z[kRows];
#pragma unroll
                    for (int i = 0; i < kRows; ++i) z[i] = (uint16_t)tc::pack16(v[i], 0.f, kBf16 ? 2 : 1);
                    put_rows(pre, z, p.N, left);
                }
            float x[kRows];
            if (p.extra)
#pragma unroll
                for (int i = 0; i < kRows; ++i) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x[i]) : "r"(extra + (uint32_t)i * 128u) : "memory");
            if (p.activation != kActNone)
                with_activation(p.activation, [&](auto act) {
#pragma unroll
                    for (int i = 0; i < kRows; i += 2) {
                        if constexpr (kMode == LinearMode::kInputGrad) {
                            float s0 = 0.f, s1 = 0.f;
                            if constexpr (kOut16) pair_split(slope_pair<act.value>(pair_of(x[i], x[i + 1])), s0, s1);
                            else s0 = slope_exact<act.value>(x[i]), s1 = slope_exact<act.value>(x[i + 1]);
                            v[i] *= s0;
                            v[i + 1] *= s1;
                        } else if constexpr (kOut16) {
                            pair_split(activate_pair<act.value>(pair_of(v[i], v[i + 1])), v[i], v[i + 1]);
                        } else {
                            v[i] = activate_exact<act.value>(v[i]);
                            v[i + 1] = activate_exact<act.value>(v[i + 1]);
                        }
                    }
                });
            if (kMode != LinearMode::kInputGrad && p.extra)
#pragma unroll
                for (int i = 0; i < kRows; ++i) v[i] = __fadd_rn(v[i], x[i]);
            Stored y[kRows];
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                if constexpr (kOut16) y[i] = (uint16_t)tc::pack16(v[i], 0.f, kBf16 ? 2 : 1);
                else y[i] = v[i];
            }
            put_rows(out, y, p.N, left);
        }
    }
    // v[i] to row i of the rows that are left, `to` moved past them
    template <class T, int kRows>
    __device__ __forceinline__ static void put_rows(T *&to, const T (&v)[kRows], int pitch, int left) {
        if (left >= kRows) {
#pragma unroll
            for (int i = 0; i < kRows; ++i, to += pitch) *to = v[i];
        } else {
#pragma unroll
            for (int i = 0; i < kRows; ++i, to += pitch)
                if (i < left) *to = v[i];
        }
    }
    // The extra operand of 32 rows in column c, by plain loads that are all on their way together (in batches of eight, each
    // batch's between two batches of stores, 1021 x 2053 x 1096 with a residual took 30 us), kept as FP32 in the warp's
    // second box, where each lane finds its own column again.
    __device__ __forceinline__ static void fetch_rows(const Params &p, float (&x)[32], int row_base, int c) {
        const int rows = min(32, p.M - row_base);
        const size_t at = (size_t)row_base * p.N + c;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            x[i] = 0.f;
            if (c < p.N && i < rows) {
                if constexpr (kExtra16) x[i] = __uint_as_float(static_cast<const uint16_t *>(p.extra)[at + (size_t)i * p.N]);
                else x[i] = static_cast<const float *>(p.extra)[at + (size_t)i * p.N];
            }
        }
        if constexpr (kExtra16) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                float lo, hi;
                if (p.fmt) widen16<true>(__float_as_uint(x[i]), lo, hi);
                else widen16<false>(__float_as_uint(x[i]), lo, hi);
                x[i] = lo;
            }
        }
    }
    __device__ __forceinline__ static void keep_rows(State &st, const float (&x)[32], int lane) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(st.boxes + kBoxBytes + (uint32_t)(i * 128 + lane * 4)), "f"(x[i]) : "memory");
    }

    // address of 16-byte piece j of row `lane` of a box: rows of 128 bytes with the 128-byte swizzle, or of 64 bytes with the
    // 64-byte one
    template <int kRowBytes>
    __device__ __forceinline__ static uint32_t piece(uint32_t box, int lane, int j) {
        return kRowBytes == 128 ? box + (uint32_t)lane * 128u + (uint32_t)((j ^ (lane & 7)) << 4)
                                : box + (uint32_t)lane * 64u + (uint32_t)((j ^ ((lane >> 1) & 3)) << 4);
    }
    __device__ __forceinline__ static void put_piece(uint32_t at, const uint4 &v) {
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
    }
    __device__ __forceinline__ static uint4 get_piece(uint32_t at) {
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
        return v;
    }
    template <bool kBf16>
    __device__ __forceinline__ static f32x2 widen(uint32_t w) {
        float lo, hi;
        widen16<kBf16>(w, lo, hi);
        return pair_of(lo, hi);
    }
    template <bool kBf16>
    __device__ __forceinline__ static uint32_t narrow(f32x2 v) {
        float lo, hi;
        pair_split(v, lo, hi);
        if constexpr (kBf16) return pack_bf16(lo, hi);
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    // 32 values as 16-bit pieces j0 .. j0 + 3 of the lane's row
    template <bool kBf16, int kRowBytes>
    __device__ __forceinline__ static void put16(const f32x2 (&v)[16], uint32_t box, int lane, int j0) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            put_piece(piece<kRowBytes>(box, lane, j0 + j),
                      make_uint4(narrow<kBf16>(v[4 * j]), narrow<kBf16>(v[4 * j + 1]), narrow<kBf16>(v[4 * j + 2]), narrow<kBf16>(v[4 * j + 3])));
    }
    // the box D leaves from, free to be written: box 0 where box 1 belongs to the extra operand or to Z, else both in turn
    __device__ __forceinline__ static uint32_t free_box(State &st, const Params &p) {
        const bool turns = p.extra == nullptr && p.pre == nullptr;
        if (tc::elect_one()) {
            if (turns) tc::bulk_wait_group_read<1>();
            else tc::bulk_wait_group_read<0>();
        }
        __syncwarp();
        return st.boxes + (turns ? (st.stores & 1u) * kBoxBytes : 0u);
    }
    __device__ __forceinline__ static void send(State &st, const CUtensorMap *map, uint32_t box, int row_base, int col) {
        fence_proxy_async();
        __syncwarp();
        if (tc::elect_one()) {
            tc::tma_store_2d(map, col, row_base, box);  // rows and columns beyond the matrix are clipped by the map
            tc::bulk_commit_group();
        }
        ++st.stores;
    }
    __device__ __forceinline__ static void sums_at(uint32_t taddr, f32x2 (&v)[16]) {
        uint32_t r[32];
        tc::tmem_ld_32x32_issue(taddr, r);
        tc::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = pair_of(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
    }
    // 32 sums (columns col .. of the matrix) plus the bias
    template <bool kBf16>
    __device__ __forceinline__ static void biased(const Params &p, uint32_t taddr, int col, f32x2 (&v)[16]) {
        uint4 bias[4];
        if constexpr (kMode == LinearMode::kForward) {
            if (p.bias) {
                const uint4 *at = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.bias) + col);
#pragma unroll
                for (int j = 0; j < 4; ++j) bias[j] = col + j * 8 < p.N ? at[j] : make_uint4(0u, 0u, 0u, 0u);
            }
        }
        sums_at(taddr, v);
        if constexpr (kMode == LinearMode::kForward) {
            if (p.bias) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[4 * j] = pair_add(v[4 * j], widen<kBf16>(bias[j].x));
                    v[4 * j + 1] = pair_add(v[4 * j + 1], widen<kBf16>(bias[j].y));
                    v[4 * j + 2] = pair_add(v[4 * j + 2], widen<kBf16>(bias[j].z));
                    v[4 * j + 3] = pair_add(v[4 * j + 3], widen<kBf16>(bias[j].w));
                }
            }
        }
    }

    template <bool kBf16>
    __device__ __forceinline__ static void chunk(const CUtensorMap *map_d, const Params &p, State &st, uint32_t taddr, int row_base, int col,
                                                 bool more, int lane) {
        constexpr int kHalves = kChunk / 32;
        constexpr int kRow16 = kOut16 ? 128 : 64;  // bytes of a 16-bit tensor's box row
        const bool keep_z = kMode == LinearMode::kForward && p.pre != nullptr;
        if (keep_z && p.extra) {  // box 1 is taken: Z goes ahead through box 0, from a reading of the sums of its own
            const uint32_t box = free_box(st, p);
#pragma unroll 1
            for (int h = 0; h < kHalves; ++h) {
                f32x2 v[16];
                biased<kBf16>(p, taddr + h * 32, col + h * 32, v);
                put16<kBf16, kRow16>(v, box, lane, h * 4);
            }
            send(st, &p.map_pre, box, row_base, col);
        }
        const uint32_t d_box = free_box(st, p), z_box = st.boxes + kBoxBytes;
        if constexpr (kOut16) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint4 extra[4];
                if (p.extra)
#pragma unroll
                    for (int j = 0; j < 4; ++j) extra[j] = get_piece(piece<128>(z_box, lane, h * 4 + j));
                if (h == 1) next_extra(st, p, row_base, col, more);
                f32x2 v[16];
                biased<kBf16>(p, taddr + h * 32, col + h * 32, v);
                if constexpr (kMode == LinearMode::kForward) {
                    if (keep_z && !p.extra) put16<kBf16, 128>(v, z_box, lane, h * 4);
                    with_activation(p.activation, [&](auto act) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = activate_pair<act.value>(v[i]);
                    });
                }
                if (p.extra) {
                    f32x2 x[16];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[4 * j] = widen<kBf16>(extra[j].x);
                        x[4 * j + 1] = widen<kBf16>(extra[j].y);
                        x[4 * j + 2] = widen<kBf16>(extra[j].z);
                        x[4 * j + 3] = widen<kBf16>(extra[j].w);
                    }
                    if constexpr (kMode == LinearMode::kInputGrad) {
                        with_activation(p.activation, [&](auto act) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = pair_mul(v[i], slope_pair<act.value>(x[i]));
                        });
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = pair_add(v[i], x[i]);
                    }
                }
                put16<kBf16, 128>(v, d_box, lane, h * 4);
            }
        } else {
            // FP32 results: the accumulators go to the box as they are; activation, slope or addition (library functions of
            // some 40 instructions) then work on the lane's row of it, four values at a time
            f32x2 v[16];
            biased<kBf16>(p, taddr, col, v);
            if (keep_z && !p.extra) put16<kBf16, 64>(v, z_box, lane, 0);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float4 f;
                pair_split(v[2 * j], f.x, f.y);
                pair_split(v[2 * j + 1], f.z, f.w);
                put_piece(piece<128>(d_box, lane, j), make_uint4(__float_as_uint(f.x), __float_as_uint(f.y), __float_as_uint(f.z), __float_as_uint(f.w)));
            }
            if (p.extra || (kMode == LinearMode::kForward && p.activation != kActNone)) {
                with_activation(kMode == LinearMode::kWeightGrad ? (int)kActNone : p.activation, [&](auto act) {
#pragma unroll 1
                    for (int j = 0; j < 8; ++j) {
                        const uint4 w = get_piece(piece<128>(d_box, lane, j));
                        float f[4] = {__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w)}, x[4] = {-0.f, -0.f, -0.f, -0.f};  // what adds nothing
                        if (p.extra) {
                            if constexpr (kExtra16) {
                                const uint4 e = get_piece(piece<64>(z_box, lane, j >> 1));
                                widen16<kBf16>(j & 1 ? e.z : e.x, x[0], x[1]);
                                widen16<kBf16>(j & 1 ? e.w : e.y, x[2], x[3]);
                            } else {
                                const uint4 e = get_piece(piece<128>(z_box, lane, j));
                                x[0] = __uint_as_float(e.x), x[1] = __uint_as_float(e.y), x[2] = __uint_as_float(e.z), x[3] = __uint_as_float(e.w);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if constexpr (kMode == LinearMode::kInputGrad) f[i] *= slope_exact<act.value>(x[i]);
                            else f[i] = __fadd_rn(activate_exact<act.value>(f[i]), x[i]);
                        }
                        put_piece(piece<128>(d_box, lane, j), make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])));
                    }
                });
            }
            next_extra(st, p, row_base, col, more);
        }
        if (keep_z && !p.extra) {  // both boxes in one group of stores
            fence_proxy_async();
            __syncwarp();
            if (tc::elect_one()) tc::tma_store_2d(&p.map_pre, col, row_base, z_box);
        }
        send(st, map_d, d_box, row_base, col);
    }
    // the extra operand's box has been read: the next chunk's may come
    __device__ __forceinline__ static void next_extra(State &st, const Params &p, int row_base, int col, bool more) {
        if (p.extra == nullptr) return;
        __syncwarp();
        if (more) bring(st, p, row_base, col + kStep);
    }
};

// Second step of a product cut into K slices (see tc::gemm_slice_sum_kernel): the slices of a 32 x 32 chunk are added in
// K order, then the epilogue.  tile_m, bn: the product's tile.  One block per chunk, thread i takes columns 4 * (i % 8) .. + 3 of row i / 8.
template <LinearMode kMode, bool kOut16>
__global__ void __launch_bounds__(256) linear_slice_sum_kernel(const LinearParams p, int tile_m, int bn) {
    const int chunks_n = bn / 32, chunks_per_tile = (tile_m / 32) * chunks_n;
    const long long t = blockIdx.x / chunks_per_tile;
    const int chunk = (int)(blockIdx.x - t * chunks_per_tile);
    const int tiles_m = (p.M + tile_m - 1) / tile_m, tiles_n = (p.N + bn - 1) / bn;
    int tm, tn;
    tc::tile_coords(t, tiles_m, tiles_n, tm, tn);
    const int row = tm * tile_m + (chunk / chunks_n) * 32 + (int)threadIdx.x / 8;
    const int col = tn * bn + (chunk % chunks_n) * 32 + ((int)threadIdx.x & 7) * 4;
    grid_launch_dependents();
    grid_dependency_wait();  // the slices are complete and visible
    if constexpr (kMode == LinearMode::kWeightGrad) {  // the blocks of dW's first 32 columns fold the column sums of their rows
        const int sum_row = tm * tile_m + (chunk / chunks_n) * 32 + (int)threadIdx.x;
        if (p.sum_shares && tn == 0 && chunk % chunks_n == 0 && threadIdx.x < 32 && sum_row < p.M) p.dbias[sum_row] = fold_sum_parts(p, sum_row);
    }
    if (row >= p.M || col >= p.N) return;
    const size_t slot_vecs = (size_t)tile_m * bn / 4;
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

// Column sums of a 16-bit [rows, cols] matrix, cols a multiple of 8: the bias gradient of a layer without input features, whose
// product has no tiles.  A block takes 64 columns, a lane eight of them; speed does not matter here.
template <bool kBf16>
__global__ void __launch_bounds__(256) column_sum_kernel(const uint16_t *in, long long rows, int cols, float *out) {
    __shared__ float sums[8][64];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c0 = (int)blockIdx.x * 64, c = c0 + (lane & 7) * 8;
    float sum[8] = {};
    if (c < cols)
        for (long long r = warp * 4 + (lane >> 3); r < rows; r += 32) {
            const uint4 v = __ldcg(reinterpret_cast<const uint4 *>(in + (size_t)r * cols + c));
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float lo, hi;
                widen16<kBf16>(w[j], lo, hi);
                sum[2 * j] += lo;
                sum[2 * j + 1] += hi;
            }
        }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        sum[i] += __shfl_xor_sync(kFullMask, sum[i], 16);
        sum[i] += __shfl_xor_sync(kFullMask, sum[i], 8);
        if (lane < 8) sums[warp][lane * 8 + i] = sum[i];
    }
    __syncthreads();
    if (threadIdx.x >= 64 || c0 + (int)threadIdx.x >= cols) return;
    float total = 0.f;
    for (int w = 0; w < 8; ++w) total += sums[w][threadIdx.x];
    out[c0 + threadIdx.x] = total;
}

}  // namespace ko
