// How matmul_quantized.cu's kernel takes a product: its tiles' sizes, and the choice among
// them. Host code alone, without CUDA's headers.
#pragma once

#include <cstddef>
#include <cstdint>

namespace tlb {

// How the tensor-core kernel takes a product (plan_product).
struct ProductPlan {
    int tile_tokens;           // tokens of a tile, a multiple of 16, 224 at most
    int split;                 // CTAs (a cluster) that share a tile's width
    bool pair;                 // two CTAs take 256 features as one
    int chunks;                // of 128 values of the width a stage
    bool pieces;               // 16-bit results by way of a warp's 32 features
    int stages;
    int ctas;
    size_t smem;
};

namespace product {

constexpr int kFeatures = 128;             // of a CTA's tile (M)
constexpr int kChunk = 128;                // bytes of K of a shared-memory row
constexpr int kMaxTokens = 224;            // of a tile (N): two accumulators and the scales
constexpr int kWeightBytes = kFeatures * kChunk;  // of a chunk
constexpr int kResultWarps = 8;
constexpr int kMaxStages = 12;
constexpr int kTail = 512;                 // bytes of barriers and flags, after the stages
// CTAs that share a tile. Eight were slower everywhere (64 x 8192 -> 2048: 17.7 us where four
// took 10.4, 9.4 by now): fewer than 16 clusters of that many large CTAs run at once.
constexpr int kMaxSplit = 4;
// scales on their way to tensor memory: words (of four groups) of a row at a time, two
// buffers of the tokens' rows and the weights' behind them
constexpr int kWordsAtOnce = 4;
constexpr int kScalePitch = kWordsAtOnce + 1;  // words: rows in different banks
constexpr int kScaleRows = kMaxTokens + 1;
constexpr int kScaleBytes = 2 * kScaleRows * kScalePitch * 4;
constexpr size_t kMaxSmem = 232448;        // of a CTA

// Results in shared memory: two buffers of 2 KB a warp, or sums of the whole tile or of
// 64 tokens.
inline int parts_bytes_of(int tokens, int split, bool pieces) {
    return pieces ? kResultWarps * 4096 : (split > 1 ? tokens : 64) * kFeatures * 4;
}
inline size_t smem_of(int tokens, int split, bool pair, int chunks, bool pieces, int stages) {
    const int rows = pair ? tokens / 2 : tokens;
    return 1024 + (size_t)stages * chunks * (kWeightBytes + rows * kChunk) + kTail +
           parts_bytes_of(tokens, split, pieces) + kScaleBytes;
}

}  // namespace product

// Which tile, and how many CTAs share it: the plan whose time, in microseconds by the
// measurements below (short runs, at 1.9 GHz), is the shortest.
//   * A chunk of a tile of n tokens takes 0.13 + n / 1000 (the issuing thread, then the
//     tensor cores; 16 tokens 0.17, 160 0.29), of a pair's 0.13 + n / 1250 (160 tokens
//     0.26, 224 0.31); at least its bytes at 115 GB/s an SM (from the L2), and where every
//     weight is read once, all CTAs' weights at 6.3 TB/s. Weights too many for the L2 cost
//     0.7 of that where several tiles read them (33 x 4096 -> 28672: 23.6 us in a tile of
//     48 tokens, 33.5 in two of 32).
//   * A tile's end takes 0.5, and a tile no less than its results' way to memory, 0.3 and
//     0.0118 a token (13863 x 208 -> 9928: 106 us with single CTAs, 91 with pairs, 275 MB).
//   * Pairs start 1.2 later (1024 x 2048 -> 2560: 9.0 us with single CTAs, 9.7 with pairs;
//     4096 x 4096 -> 4096: 59.4 and 53.1; 16384 x 4096 -> 8192: 426 and 399).
//   * Sharing a tile costs 0.9 + n / 40 (64 x 8192 -> 2048: 15.2 us alone, 10.7 by two,
//     9.4 by four CTAs; 64 x 2048 -> 2560: 6.2, 6.2 and 6.4).
// half: results in 16 bits.
inline ProductPlan plan_product(int64_t num_tokens, int64_t features, int64_t width, bool half,
                                int sms) {
    using namespace product;
    const int64_t chunks = (width + kChunk - 1) / kChunk;
    ProductPlan best{};
    double best_time = 0;
    auto consider = [&](int split, bool pair, int tokens) {
        const int per_cta = pair ? 2 * kFeatures : kFeatures, cluster = pair ? 2 : split;
        const int units = sms / cluster;
        if (units == 0) return;
        const int64_t tiles_t = (num_tokens + tokens - 1) / tokens;
        const int64_t tiles = (features + per_cta - 1) / per_cta * tiles_t;
        const int64_t rounds = (tiles + units - 1) / units;
        const int ctas = (int)(tiles < units ? tiles : units) * cluster;
        double chunk = 0.13 + tokens * (pair ? 0.8e-3 : 1e-3);
        const double copy = (kWeightBytes + (pair ? tokens / 2 : tokens) * kChunk) / 115e3;
        if (copy > chunk) chunk = copy;
        double stream = ctas * (double)kWeightBytes / 6.3e6;
        if (tiles_t > 1) stream *= features * width > (64 << 20) ? 0.7 : 0;
        if (stream > chunk) chunk = stream;
        double tile = (double)((chunks + split - 1) / split) * chunk + 0.5;
        if (tile < 0.3 + 0.0118 * tokens) tile = 0.3 + 0.0118 * tokens;
        double time = rounds * tile + (pair ? 1.2 : 0);
        if (split > 1) time += rounds * (0.9 + tokens / 40.0);
        if (best_time == 0 || time < best_time) {
            best_time = time;
            best.tile_tokens = tokens;
            best.split = split;
            best.pair = pair;
            best.ctas = ctas;
        }
    };
    for (int tokens = 16; tokens <= kMaxTokens; tokens += 16) {
        if (tokens != 16 && tokens - 16 >= num_tokens) break;
        for (int split = 1; split <= (tokens <= 128 ? kMaxSplit : 1) && 2 * split <= chunks + 1;
             split *= 2)
            consider(split, false, tokens);
        if (tokens % 32 == 0 && tokens >= 64) consider(1, true, tokens);
    }
    best.chunks = best.pair || best.tile_tokens < 128 || best.split > 1 ? 2 : 1;
    best.pieces = best.split == 1 && half;
    int stages = kMaxStages;
    auto smem = [&] {
        return smem_of(best.tile_tokens, best.split, best.pair, best.chunks, best.pieces, stages);
    };
    while (smem() > kMaxSmem) --stages;
    best.stages = stages;
    // One CTA an SM, also where two would fit: each takes all tensor memory, and two
    // clusters could otherwise wait for one another's.
    best.smem = smem() < 120 * 1024 ? 120 * 1024 : smem();
    return best;
}

}  // namespace tlb
