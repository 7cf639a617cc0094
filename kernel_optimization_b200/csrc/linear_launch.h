// Host side shared by the linear layer's entry points: how a product is cut up, and its launch on the tensor-core kernels.
#pragma once

#include "ko_internal.h"
#include "row_launch.h"
#include "tensor_maps.h"

#include <algorithm>
#include <atomic>

#include "../nn_operators/gemm/tensor_core_gemm_pair.h"
#include "../nn_operators/linear/linear_epilogue.h"

namespace ko {

// D[M, N] = A B over K, in 128 x bn tiles of one CTA or 256 x 256 tiles of a pair of CTAs, K cut into `split` slices
struct ProductPlan {
    bool pair;
    int bn, split;
    int rows() const { return pair ? 256 : 128; }
    size_t bytes() const { return split > 1 ? (size_t)tiles * split * rows() * bn * sizeof(float) : 0; }
    long long tiles;
};

// tma: D can be stored by TMA; without it only the 128 x 128 tile is built.  element_bytes: what the epilogue moves per element
// of D (D itself, Z, the extra operand).  Modelled microseconds per candidate: start, then rounds of work units x (K-blocks
// of 64 x time per K-block + epilogue time that the next tile does not hide); slices add a second kernel (2 us of the
// device, 4 of the host with the workspace; 5 is what they have to gain) and the partial tiles' way through the L2 (written once,
// read once) at 5 TB/s.  Fitted to forced plans, BF16, measured (modelled), pair / 128 x 128 / 128 x 256:
// 16384 x 4096 x 1024 101 (100), 135 (135), 114 (107); 4096^3 96 (93), 118 (110), 117 (101); 8192 x 768 x 768 18.8 (15.6), 18.1
// (14.5), 20.2 (16.1); 1024 x 1024 x 4096 26 (27), 19.8 (18.3), 33 (28), 128 x 128 in two slices 20.2 (20.7).  Slices, where a few
// tiles leave most SMs idle: 512 x 2048 x 32768 (a weight gradient) pair in four 65 (61), 128 x 256 in four 77 (65), uncut 156 (171);
// 768 x 768 x 16384 128 x 128 in four 24.5, uncut 53.
// sums: column sums are wanted, which a pair can take where a row of tiles has two (see sum_shares).
inline ProductPlan plan_product(int64_t M, int64_t N, int64_t K, bool tma, int element_bytes, int sms, bool sums) {
    const long long k_blocks = (K + tc::kBK - 1) / tc::kBK;
    ProductPlan best{false, 128, 1, 0};
    double best_cost = 1e300;
    struct Tile {
        bool pair;
        int bn;
        double start, per_block, once, per_byte;  // us: a launch, a K-block, an epilogue and each byte of its elements
    };
    for (const Tile &tile : {Tile{true, 256, 4.5, 0.32, 0.3, 0.7}, Tile{false, 128, 3.0, 0.22, 0.5, 0.35}, Tile{false, 256, 4.3, 0.35, 0.5, 0.6}}) {
        if (tile.bn == 256 && (!tma || N <= 128 || (tile.pair && (M <= 128 || (sums && N <= 256))))) continue;
        const int rows = tile.pair ? 256 : 128, bn = tile.bn, at_once = tile.pair ? sms / 2 : sms;
        const double per_block = tile.per_block, start = tile.start;
        const auto per_tile = [&](int bytes) { return tile.once + tile.per_byte * bytes; };
        const long long tiles = ((M + rows - 1) / rows) * ((N + bn - 1) / bn);
        const long long most = std::min<long long>(std::max<long long>(at_once / tiles, 1), std::max<long long>(k_blocks / 4, 1));
        for (int split = 1; split <= most && split <= 64; ++split) {
            const long long rounds = (tiles * split + at_once - 1) / at_once;
            double cost = start + (double)rounds * ((double)((k_blocks + split - 1) / split) * per_block + per_tile(split > 1 ? 4 : element_bytes));
            if (split > 1) {
                const double written = (double)((M + 31) / 32 * 32) * (double)N * split, read = (double)M * (double)N * split;
                cost += 5.0 + ((written + read) * 4.0 + (double)M * (double)N * element_bytes) / 5e6;
            }
            if (cost < best_cost) {
                best_cost = cost;
                best = {tile.pair, bn, split, tiles};
            }
        }
    }
    return best;
}

// a plan pinned by a tuning call: tile 0 = choose, 128 / 256 = columns of a CTA's tile, 2048 = the pair of CTAs; slices 0 =
// choose (1 with a pinned tile)
struct PinnedPlan {
    int tile = 0, slices = 0;
};
inline int pin_product(const PinnedPlan &pin, int64_t M, int64_t N, int64_t K, bool tma, bool sums, const char *name, ProductPlan *plan) {
    if (pin.tile == 0 && pin.slices == 0) return KO_OK;
    KO_REQUIRE(pin.tile == 128 || pin.tile == 256 || pin.tile == 2048, KO_ERR_INVALID_ARG, "%s: tile code %d not in {128,256,2048}", name, pin.tile);
    KO_REQUIRE(tma || pin.tile == 128, KO_ERR_SHAPE, "%s: without TMA stores there is only the 128-column tile", name);
    KO_REQUIRE(pin.tile != 2048 || !sums || N > 256, KO_ERR_SHAPE, "%s: a pair of CTAs sums the columns of dY only where dW has more than 256", name);
    const long long k_blocks = (K + tc::kBK - 1) / tc::kBK;
    KO_REQUIRE(pin.slices >= 0 && pin.slices <= 64 && pin.slices <= k_blocks, KO_ERR_INVALID_ARG,
               "%s: %d K slices out of range", name, pin.slices);
    plan->pair = pin.tile == 2048;
    plan->bn = plan->pair ? 256 : pin.tile;
    plan->split = pin.slices > 1 ? pin.slices : 1;
    plan->tiles = ((M + plan->rows() - 1) / plan->rows()) * ((N + plan->bn - 1) / plan->bn);
    return KO_OK;
}

// Tiles of a row of tiles that share the column sums of dY (see ColumnSums): one, whose sums are dbias, or four, whose parts
// have to be added.  One that takes all K-blocks falls behind the others (a K-block's sums take longer than its MMAs in the 128 x 128
// tile), adding parts is a launch, 1.2 us of the device, where K is not cut anyway.  One / four, without the sums (us): 777 tokens of
// 1000 x 520 9.6 / 10.9, 9.5; 1024 tokens of 1024 x 1024 10.4 / 10.2, 8.7; 2048 tokens 16.7 / 14.2, 12.4; in
// pairs, 16384 of 4096 x 1024, 104 with the two shares that four columns of tiles give, 103.
// Of a pair of CTAs only the leader adds, the upper rows of its tile in even columns of tiles and the lower ones in odd columns: two
// columns of tiles for every share.
inline int sum_shares(const ProductPlan &plan, int64_t N, int64_t K) {
    const long long tiles_n = (N + plan.bn - 1) / plan.bn, unit_blocks = ((K + tc::kBK - 1) / tc::kBK + plan.split - 1) / plan.split;
    return unit_blocks < 32 ? 1 : (int)std::min<long long>(plan.pair ? tiles_n / 2 : tiles_n, 4);
}
inline size_t sum_bytes(const ProductPlan &plan, int64_t M, int64_t N, int64_t K) {  // room for their parts; a single one is dbias
    const size_t parts = (size_t)sum_shares(plan, N, K) * plan.split;
    return parts > 1 ? parts * (size_t)M * sizeof(float) : 0;
}

// room for whatever plan a call of this shape may take: with or without TMA, any operands, column sums
inline size_t product_workspace(int64_t M, int64_t N, int64_t K, int sms, bool sums = false) {
    if (M == 0 || N == 0 || K == 0) return 0;
    size_t most = 0;
    for (int element_bytes = 2; element_bytes <= 10; element_bytes += 2)
        for (bool tma : {true, false})
            for (int with = 0; with <= (sums ? 1 : 0); ++with) {
                const ProductPlan plan = plan_product(M, N, K, tma, element_bytes, sms, with);
                most = std::max(most, plan.bytes() + (with ? sum_bytes(plan, M, N, K) : 0));
            }
    return most;
}

// clusters of two CTAs of a pair kernel that the current device holds at once; `cached`: per device, 0 = not asked yet (whoever asks at the
// same time gets the same answer)
inline int resident_pairs_of(const void *kernel, unsigned threads, size_t smem, int device, std::atomic<int> *cached, int *out) {
    int n = cached[device].load(std::memory_order_relaxed);
    if (n == 0) {
        if (int st = max_resident_clusters(kernel, threads, 2, smem, &n)) return st;
        cached[device].store(n, std::memory_order_relaxed);
    }
    *out = n;
    return KO_OK;
}

template <class Epi, int BN, bool kTmaStore>
int launch_product_tile(const CUtensorMap &ma, const CUtensorMap &mb, const CUtensorMap &md, const LinearParams &p, int sms, cudaStream_t s) {
    using Cfg = typename tc::TileConfigFor<BN, 1, 2, Epi>::type;
    auto kernel = tc::gemm_tcgen05_kernel<BN, kTmaStore, 1, 2, Epi>;
    if (int st = ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), Cfg::kSmemBytes)) return st;
    const long long units = (long long)((p.M + 127) / 128) * ((p.N + BN - 1) / BN) * p.split_k;
    return launch_overlapped(kernel, (unsigned)std::min<long long>(units, sms), 64u + 32u * (Epi::kWarps + Epi::kSumWarps), (size_t)Cfg::kSmemBytes, s, ma,
                             mb, mb, md, p);
}

template <class Epi>
int launch_product_pair(const CUtensorMap &ma, const CUtensorMap &mb, const CUtensorMap &md, const LinearParams &p, const DeviceInfo &info, cudaStream_t s) {
    using Cfg = typename tc::PairConfigFor<Epi>::type;
    auto kernel = tc::gemm_tcgen05_pair_kernel<true, Epi>;
    const void *id = reinterpret_cast<const void *>(kernel);
    constexpr unsigned threads = 64u + 32u * (Epi::kWarps + Epi::kSumWarps);
    if (int st = ensure_dynamic_smem(id, Cfg::kSmemBytes)) return st;
    static std::atomic<int> cached[64];  // device ordinals, see current_device_info
    int resident = 0;
    if (int st = resident_pairs_of(id, threads, Cfg::kSmemBytes, info.device, cached, &resident)) return st;
    const long long units = (long long)((p.M + 255) / 256) * ((p.N + 255) / 256) * p.split_k;
    return launch_clustered_overlapped(kernel, 2u * (unsigned)std::min<long long>(units, resident), threads, 2u, (size_t)Cfg::kSmemBytes, s, ma,
                                       mb, mb, md, p);
}

// Runs the product that `p` describes (M, N, K, D, fmt, out_fmt, b_row_major, bias, extra, pre, activation set by the
// caller; the rest filled in here).  A: [M, K], or [K, M] for the weight gradient; B: [N, K], or [K, N] with b_row_major.
// Everything has been checked but the workspace.
template <class Epi>
int launch_product(const ProductPlan &plan, bool tma, const CUtensorMap &ma, const CUtensorMap &mb, const CUtensorMap &md, const LinearParams &p,
                   const DeviceInfo &info, cudaStream_t s) {
    const int sms = info.sm_count;
    if (plan.pair) return launch_product_pair<Epi>(ma, mb, md, p, info, s);
    if (!tma) return launch_product_tile<Epi, 128, false>(ma, mb, md, p, sms, s);
    if (plan.bn == 128) return launch_product_tile<Epi, 128, true>(ma, mb, md, p, sms, s);
    return launch_product_tile<Epi, 256, true>(ma, mb, md, p, sms, s);
}

template <LinearMode kMode, bool kOut16>
int run_product(LinearParams p, const void *A, const void *B, void *workspace, size_t workspace_bytes, cudaStream_t s, const DeviceInfo &info,
                const char *name, const PinnedPlan &pin = {}) {
    using Epi = LinearEpilogue<kMode, kOut16>;
    EncodeTiledFn encode = nullptr;
    if (int st = get_encode_fn(&encode)) return st;
    // 16-byte row pitches and bases of everything the epilogue touches: TMA and vector loads; else its row-wise form
    const bool sixteen = kOut16 || p.pre || p.bias || (p.extra && Epi::kExtra16);
    const bool tma = p.N % (sixteen ? 8 : 4) == 0 && aligned16(p.D) && aligned16(p.pre) && aligned16(p.bias) && aligned16(p.extra);
    const int element_bytes = (kOut16 ? 2 : 4) + (p.pre ? 2 : 0) + (p.extra ? (Epi::kExtra16 ? 2 : 4) : 0);
    ProductPlan plan = plan_product(p.M, p.N, p.K, tma, element_bytes, info.sm_count, p.dbias != nullptr);
    if (int st = pin_product(pin, p.M, p.N, p.K, tma, p.dbias != nullptr, name, &plan)) return st;
    p.sum_shares = p.dbias ? sum_shares(plan, p.N, p.K) : 0;
    const size_t parts_bytes = p.dbias ? sum_bytes(plan, p.M, p.N, p.K) : 0;
    const bool fold = parts_bytes != 0;
    const size_t bytes = plan.bytes() + parts_bytes;
    KO_REQUIRE(bytes == 0 || (workspace != nullptr && workspace_bytes >= bytes), KO_ERR_INVALID_ARG,
               "%s: the workspace needs %zu bytes, got %zu", name, bytes, workspace ? workspace_bytes : (size_t)0);
    KO_REQUIRE(aligned16(workspace), KO_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", name);
    p.C = nullptr;
    p.tiles_n = p.wide_tiles_n = p.bn_wide = p.bn_narrow = 0;
    p.split_k = plan.split;
    p.partials = static_cast<float *>(workspace);
    p.sum_parts = fold ? static_cast<float *>(workspace) + plan.bytes() / sizeof(float) : p.dbias;
    if (int st = device_status_word(0, &p.status)) return st;

    alignas(64) CUtensorMap map_a, map_b, map_d;
    if (Epi::kTransA) {
        if (int st = make_map_b_row_major(encode, &map_a, p.fmt, A, p.K, p.M)) return st;
    } else {
        if (int st = make_map(encode, &map_a, p.fmt, A, p.M, p.K, tc::kBM)) return st;
    }
    if (p.b_row_major) {
        if (int st = make_map_b_row_major(encode, &map_b, p.fmt, B, p.K, p.N)) return st;
    } else {
        if (int st = make_map(encode, &map_b, p.fmt, B, p.N, p.K, plan.pair ? 128 : plan.bn)) return st;
    }
    map_d = map_a;  // unused by the direct-store epilogue
    p.map_pre = p.map_extra = map_a;
    if (tma) {
        if (int st = make_store_map(encode, &map_d, p.out_fmt, p.D, p.M, p.N, Epi::kChunk)) return st;
        if (p.pre)
            if (int st = make_store_map(encode, &p.map_pre, p.fmt + 1, p.pre, p.M, p.N, Epi::kChunk)) return st;
        if (p.extra)
            if (int st = make_store_map(encode, &p.map_extra, Epi::kExtra16 ? p.fmt + 1 : 0, const_cast<void *>(p.extra), p.M, p.N, Epi::kChunk)) return st;
    }
    // long sums: those of parts are promoted (see LinearEpilogue)
    const long long unit_blocks = ((p.K + tc::kBK - 1) / tc::kBK + plan.split - 1) / plan.split;
    const int st = unit_blocks > blocks_in_one_accumulator(kOut16)
                       ? launch_product<LinearEpilogue<kMode, kOut16, true>>(plan, tma, map_a, map_b, map_d, p, info, s)
                       : launch_product<Epi>(plan, tma, map_a, map_b, map_d, p, info, s);
    if (st != KO_OK) return st;
    if constexpr (kMode == LinearMode::kWeightGrad)
        if (fold && plan.split == 1) return launch_overlapped(linear_fold_sums_kernel<256>, (unsigned)((p.M + 255) / 256), 256u, (size_t)0, s, p);
    if (plan.split <= 1) return KO_OK;
    const long long chunks = plan.tiles * (plan.rows() / 32) * (plan.bn / 32);
    return launch_overlapped(linear_slice_sum_kernel<kMode, kOut16>, (unsigned)chunks, 256u, (size_t)0, s, p, plan.rows(), plan.bn);
}

// the checks that the three entry points share; M tokens, N output features, K input features
int check_linear(const char *name, int in_fmt, int out_fmt, int activation, int64_t M, int64_t N, int64_t K);

}  // namespace ko
