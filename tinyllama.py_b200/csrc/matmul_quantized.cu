// Product of 8-bit rows with 8-bit weights on the tensor cores:
//   out[t, n] = sum over groups g of 2^(xs[t,g] + ws[n/128,g]) sum_{k in g} x[t,k] w[n,k]
//
// The scales are powers of two, so the tensor cores apply them: kind::mxf8f6f4
// takes an E8M0 scale for each row and 32 values of K, and gets the scale of the
// row's 128 four times. The sums stay in tensor memory in fp32 from the first
// value of K to the last.
//
// The weights are the M side (128 features, so a weight block of 128 x 128 has one
// scale for all lanes of a tile), the tokens the N side, of any multiple of 16:
// the number of tokens is what varies from call to call, and a tile of few tokens
// costs few bytes and few cycles. For few tokens a cluster of 2, 4 or 8 CTAs shares a
// tile's width, and the CTAs send one another their part of the sums over
// distributed shared memory.
//
// Warps of a CTA: 0-3 load the scales and write them to tensor memory (each the
// 32 lanes it can reach), 4-7 read the sums and write the results, 8 issues the TMA
// copies (128 bytes of K a stage), 9 the tensor instructions. The accumulator is
// double buffered: a tile is written out while the next one is summed.
#include <atomic>

#include "kernels.h"
#include "quant.cuh"
#include "tcgen05.cuh"

namespace tlb {

namespace {

constexpr int kFeatures = 128;             // of a tile (M)
constexpr int kDepth = 128;                // bytes of K of a stage
constexpr int kMaxTokens = 224;            // of a tile (N): two accumulators and the scales
constexpr int kWeightBytes = kFeatures * kDepth;
constexpr int kThreads = 320;
constexpr int kMaxStages = 12;
constexpr int kScaleSets = 4;              // sets of scales in tensor memory, 4 stages each
constexpr int kSetColumns = 12;            // 4 of the weights, 8 of the tokens
constexpr int kScaleColumn = 512 - kScaleSets * kSetColumns;
constexpr int kColumns = 512;
static_assert(2 * kMaxTokens <= kScaleColumn, "tensor memory");
// mbarriers
constexpr int kBarFull = 0, kBarEmpty = kMaxStages, kBarScales = 2 * kMaxStages,
              kBarScalesFree = kBarScales + kScaleSets, kBarSums = kBarScalesFree + kScaleSets,
              kBarSumsFree = kBarSums + 2, kBarParts = kBarSumsFree + 2,
              kBarPartsFree = kBarParts + 1, kBarDrain = kBarPartsFree + 1,
              kNumBars = kBarDrain + 1;
constexpr int kTail = 512;                 // bytes after the stages: barriers, tmem address, flag
static_assert(kNumBars * 8 + 16 <= kTail, "barriers");
constexpr int kMaxSplit = 8;

struct Work {
    ProductParams p;
    int tile_tokens;
    int blocks;              // of 128 bytes of K
    int stages;
    int split;
    int tiles_n, tiles_t;
    int band;                // token tiles whose weights' tiles follow one another
    unsigned wait_limit;
    bool overlap;
    bool x_words, w_words;   // rows of scales allow 4-byte loads
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                     : "memory");
}
// Address in the cluster's CTA `rank` of what is at `addr` here.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void store_cluster(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, uint32_t limit) {
    for (uint32_t i = 0; i < limit; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
        if (ok) return true;
    }
    return false;
}

// The scale bytes of groups 4 w .. 4 w + 3 of a row, those past the last group 127.
__device__ __forceinline__ uint32_t scale_word(const uint8_t* row, int w, int groups, bool words) {
    if (words && 4 * w + 4 <= groups) return *reinterpret_cast<const uint32_t*>(row + 4 * w);
    uint32_t v = 0x7f7f7f7fu;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (4 * w + i < groups) {
            const uint32_t b = row[4 * w + i];
            v = (v & ~(0xffu << (8 * i))) | (b << (8 * i));
        }
    return v;
}

// Tile `i` of the order in which a band of token tiles goes through all features.
__device__ __forceinline__ void tile_at(const Work& w, int i, int& tn, int& tt) {
    const int per_band = w.band * w.tiles_n, b = i / per_band, rest = i % per_band;
    const int height = min(w.band, w.tiles_t - b * w.band);
    tn = rest / height;
    tt = b * w.band + rest % height;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_w,
                   const __grid_constant__ CUtensorMap map_x, const Work w) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    const uint32_t base = smem_u32(smem);
    const ProductParams& p = w.p;
    const uint32_t stage_bytes = kWeightBytes + w.tile_tokens * kDepth;
    const uint32_t tail = base + w.stages * stage_bytes, parts = tail + kTail;
    uint8_t* tail_ptr = smem + w.stages * stage_bytes;
    auto bar = [tail](int i) { return tail + 8u * i; };
    const uint32_t slot = tail + kNumBars * 8;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = w.split;
    const uint32_t rank = split > 1 ? cluster_rank() : 0;

    if (tid == 0) {
        for (int i = 0; i < w.stages; ++i) {
            mbar_init(bar(kBarFull + i), 1);
            mbar_init(bar(kBarEmpty + i), 1);
        }
        for (int i = 0; i < kScaleSets; ++i) {
            mbar_init(bar(kBarScales + i), 4);
            mbar_init(bar(kBarScalesFree + i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(kBarSums + i), 1);
            mbar_init(bar(kBarSumsFree + i), 4);
        }
        mbar_init(bar(kBarParts), 4 * split);
        mbar_init(bar(kBarPartsFree), 4 * split);
        mbar_init(bar(kBarDrain), 1);
        fence_mbar_init();
    }
    if (warp == 9) tc5::alloc(slot, kColumns);
    if (tid == 256) {
        prefetch_tensormap(&map_w);
        prefetch_tensormap(&map_x);
    }
    tc5::fence_before_sync();
    __syncthreads();
    if (split > 1) cluster_sync();  // all barriers of the cluster are set up
    tc5::fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tail_ptr + kNumBars * 8);

    // this CTA's tiles, and its part of their width
    const int tiles = w.tiles_n * w.tiles_t, units = gridDim.x / split, unit = blockIdx.x / split;
    const int k_first = (int)((long long)w.blocks * rank / split);
    const int k_last = (int)((long long)w.blocks * (rank + 1) / split);
    const uint32_t limit = w.wait_limit;
    bool ok = true;

    if (warp == 8) {
        // ------------------------------------------------------------ copies
        if (elect_one()) {
            const uint64_t keep = l2_policy_evict_last();
            const uint64_t once = l2_policy_evict_first();
            // weights that only this tile's tokens want pass through the L2
            const uint64_t w_policy = w.tiles_t > 1 ? keep : once;
            int n = 0;  // stages issued
            bool waited = false;
            int ahead = 0;  // stages whose weights were issued before the wait
            if (w.overlap) {
                int i = unit, kb = k_first;
                for (; ahead < w.stages && i < tiles; ++ahead) {
                    if (kb == k_last) {
                        kb = k_first;
                        i += units;
                        if (i >= tiles) break;
                    }
                    int tn, tt;
                    tile_at(w, i, tn, tt);
                    mbar_arrive_expect_tx(bar(kBarFull + ahead), stage_bytes);
                    tma_load_2d(base + ahead * stage_bytes, &map_w, kb * kDepth, tn * kFeatures,
                                bar(kBarFull + ahead), w_policy);
                    ++kb;
                }
            }
            for (int i = unit; i < tiles && ok; i += units) {
                int tn, tt;
                tile_at(w, i, tn, tt);
                for (int kb = k_first; kb < k_last; ++kb, ++n) {
                    const int s = n % w.stages, round = n / w.stages;
                    if (round > 0 &&
                        !mbar_wait_bounded(bar(kBarEmpty + s), (round - 1) & 1, limit)) {
                        ok = false;
                        break;
                    }
                    if (!waited) {
                        grid_dependency_wait();
                        waited = true;
                    }
                    const uint32_t at = base + s * stage_bytes;
                    if (n >= ahead) {
                        mbar_arrive_expect_tx(bar(kBarFull + s), stage_bytes);
                        tma_load_2d(at, &map_w, kb * kDepth, tn * kFeatures, bar(kBarFull + s),
                                    w_policy);
                    }
                    tma_load_2d(at + kWeightBytes, &map_x, kb * kDepth, tt * w.tile_tokens,
                                bar(kBarFull + s), keep);
                }
            }
            if (!waited) grid_dependency_wait();
            // After a wait that gave up, the copies in flight land before the CTA ends.
            if (!ok)
                for (int k = n > w.stages ? n - w.stages : 0; k < n; ++k)
                    mbar_wait_bounded(bar(kBarFull + k % w.stages), (k / w.stages) & 1);
        }
    } else if (warp == 9) {
        // ------------------------------------------------ tensor instructions
        if (elect_one()) {
            int n = 0, group = 0, it = 0;
            bool issued = false;
            for (int i = unit; i < tiles && ok; i += units, ++it) {
                const int b = it & 1;
                if (it >= 2 && !mbar_wait_bounded(bar(kBarSumsFree + b), ((it >> 1) - 1) & 1, limit)) {
                    ok = false;
                    break;
                }
                tc5::fence_after_sync();
                const uint32_t sums = tmem + b * kMaxTokens;
                for (int kb = k_first; kb < k_last; ++kb, ++n) {
                    const int set = group % kScaleSets;
                    if ((kb == k_first || (kb & 3) == 0) &&
                        !mbar_wait_bounded(bar(kBarScales + set), (group / kScaleSets) & 1, limit)) {
                        ok = false;
                        break;
                    }
                    const int s = n % w.stages;
                    if (!mbar_wait_bounded(bar(kBarFull + s), (n / w.stages) & 1, limit)) {
                        ok = false;
                        break;
                    }
                    tc5::fence_after_sync();
                    const uint32_t at = base + s * stage_bytes;
                    const uint32_t scales = tmem + kScaleColumn + set * kSetColumns;
                    const uint32_t idesc = tc5::idesc_mxf8(kFeatures, w.tile_tokens, kb & 3);
                    const int steps = min(4, (p.width - kb * kDepth + 31) / 32);
                    for (int k = 0; k < steps; ++k)
                        tc5::mma_mxf8(sums, tc5::desc_sw128(at + 32 * k, 16, 1024),
                                      tc5::desc_sw128(at + kWeightBytes + 32 * k, 16, 1024), idesc,
                                      scales, scales + 4, kb > k_first || k > 0);
                    issued = true;
                    tc5::commit(bar(kBarEmpty + s));
                    if ((kb & 3) == 3 || kb + 1 == k_last) {
                        tc5::commit(bar(kBarScalesFree + set));
                        ++group;
                    }
                }
                if (ok) tc5::commit(bar(kBarSums + b));
            }
            if (!ok && issued) {  // nothing runs on when the CTA ends
                tc5::commit(bar(kBarDrain));
                mbar_wait_bounded(bar(kBarDrain), 0);
            }
        }
    } else if (warp < 4) {
        // ------------------------------------------------------------ scales
        grid_dependency_wait();
        grid_launch_dependents();
        int group = 0;
        const uint32_t lanes = (uint32_t)warp << 21;  // 32 warp, in the address's upper half
        const int groups = w.blocks;
        for (int i = unit; i < tiles && ok; i += units) {
            int tn, tt;
            tile_at(w, i, tn, tt);
            const uint8_t* w_row = p.weight_scales + tn * p.weight_scales_stride;
            const long long t0 = (long long)tt * w.tile_tokens + lane;
            for (int word = k_first >> 2; word <= (k_last - 1) >> 2; ++word, ++group) {
                uint32_t x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const long long t = t0 + 32 * j;
                    x[j] = 0x7f7f7f7fu;
                    if (32 * j < w.tile_tokens && t < p.num_tokens)
                        x[j] = scale_word(p.x_scales + t * p.x_scales_stride, word, groups, w.x_words);
                }
                const uint32_t wt = scale_word(w_row, word, groups, w.w_words);
                const int set = group % kScaleSets;
                if (group >= kScaleSets &&
                    !__all_sync(0xffffffffu, mbar_wait_bounded(bar(kBarScalesFree + set),
                                                               (group / kScaleSets - 1) & 1, limit))) {
                    ok = false;
                    break;
                }
                tc5::fence_after_sync();
                const uint32_t to = tmem + lanes + kScaleColumn + set * kSetColumns;
                tc5::st4(to, wt);
                tc5::st8(to + 4, x);
                tc5::st_wait();
                tc5::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(kBarScales + set));
            }
        }
    } else {
        // ----------------------------------------------------------- results
        grid_dependency_wait();
        const int quarter = warp & 3, feature = quarter * 32 + lane;
        int it = 0;
        for (int i = unit; i < tiles && ok; i += units, ++it) {
            int tn, tt;
            tile_at(w, i, tn, tt);
            const long long n = (long long)tn * kFeatures + feature;
            const long long t0 = (long long)tt * w.tile_tokens;
            const int here = (int)min((long long)w.tile_tokens, p.num_tokens - t0);
            const bool on = n < p.features;
            float bias = 0.f;
            if (p.bias && on) bias = Elem<T>::to_f(reinterpret_cast<const T*>(p.bias)[n]);
            T* out = reinterpret_cast<T*>(p.out) + t0 * p.out_stride + n;
            const int b = it & 1;
            if (!__all_sync(0xffffffffu,
                            mbar_wait_bounded(bar(kBarSums + b), (it >> 1) & 1, limit))) {
                ok = false;
                break;
            }
            tc5::fence_after_sync();
            const uint32_t sums = tmem + ((uint32_t)quarter << 21) + b * kMaxTokens;
            const int share = (here + split - 1) / split;  // tokens that a CTA of the cluster joins
            if (split > 1 && it > 0 &&
                !__all_sync(0xffffffffu, wait_cluster(bar(kBarPartsFree), (it - 1) & 1, limit))) {
                ok = false;
                break;
            }
            for (int j0 = 0; j0 < here; j0 += 32) {
                float v[32];
                tc5::ld32(sums + j0, v);
                if (split == 1) {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (on && j0 + j < here)
                            out[(j0 + j) * p.out_stride] = Elem<T>::from_f(v[j] + bias);
                } else {
                    // token j of the tile goes to CTA j / share, at [from][j % share][feature]
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        if (j0 + j >= here) break;
                        const int to = (j0 + j) / share, row = (j0 + j) - to * share;
                        store_cluster(map_rank(parts, to) +
                                          4u * (((int)rank * share + row) * kFeatures + feature),
                                      v[j]);
                    }
                }
            }
            tc5::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kBarSumsFree + b));
            if (split > 1) {
                if (lane < split) arrive_cluster(map_rank(bar(kBarParts), lane));
                if (!__all_sync(0xffffffffu, wait_cluster(bar(kBarParts), it & 1, limit))) {
                    ok = false;
                    break;
                }
                const int first = (int)rank * share, mine = max(0, min(share, here - first));
                const float* in = reinterpret_cast<const float*>(tail_ptr + kTail) + feature;
                for (int row = 0; row < mine; ++row) {
                    float v = 0.f;
                    for (int from = 0; from < split; ++from)
                        v += in[(from * share + row) * kFeatures];
                    if (on) out[(first + row) * p.out_stride] = Elem<T>::from_f(v + bias);
                }
                __syncwarp();
                if (lane < split) arrive_cluster(map_rank(bar(kBarPartsFree), lane));
            }
        }
    }
    if (!ok) flag_status(TLB_STATUS_WAIT_TIMEOUT);
    __syncwarp();
    tc5::fence_before_sync();
    __syncthreads();
    if (split > 1) cluster_sync();  // no CTA ends while another one may write to it
    if (warp == 9) {
        tc5::fence_after_sync();
        tc5::dealloc(tmem, kColumns);
    }
}

size_t smem_of(int tokens, int split, int stages) {
    const size_t parts = split > 1 ? (size_t)(tokens + split) * kFeatures * 4 : 0;
    return 1024 + (size_t)stages * (kWeightBytes + tokens * kDepth) + kTail + parts;
}

template <typename T>
cudaError_t launch(const Work& w, const ProductPlan& plan, const CUtensorMap& map_w,
                   const CUtensorMap& map_x, cudaStream_t st) {
    auto kernel = product_kernel<T>;
    // the attribute is the kernel's on one device: set once for each
    static std::atomic<unsigned long long> set{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (!(set.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
        if (e != cudaSuccess) return e;
        set.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = plan.split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(plan.ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = plan.smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = plan.split > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, map_w, map_x, w);
}

}  // namespace

ProductPlan plan_product(int64_t num_tokens, int64_t features, int64_t width, int sms) {
    const int64_t blocks = (width + kDepth - 1) / kDepth;
    const int64_t tiles_n = (features + kFeatures - 1) / kFeatures;
    ProductPlan best{};
    double best_cost = 0;
    for (int split = 1; split <= kMaxSplit && split <= blocks; split *= 2) {
        const int units = sms / split;
        if (units == 0) break;
        for (int tokens = 16; tokens <= (split > 1 ? 128 : kMaxTokens); tokens += 16) {
            if (tokens != 16 && tokens - 16 >= num_tokens) break;
            const int64_t tiles = tiles_n * ((num_tokens + tokens - 1) / tokens);
            const int64_t rounds = (tiles + units - 1) / units;
            // cycles of a stage: the tensor cores' or the copies', whichever is longer
            const double mma = 2.0 * tokens, copy = (kWeightBytes + tokens * kDepth) / 32.0;
            const double per = (double)((blocks + split - 1) / split) * (mma > copy ? mma : copy);
            const double cost = rounds * (per + 300) + (split > 1 ? 1500 + 4.0 * tokens : 0);
            if (best_cost == 0 || cost < best_cost) {
                best_cost = cost;
                best.tile_tokens = tokens;
                best.split = split;
                best.ctas = (int)(tiles < units ? tiles : units) * split;
            }
        }
    }
    int stages = kMaxStages;
    while (smem_of(best.tile_tokens, best.split, stages) > 232448) --stages;
    best.stages = stages;
    // One CTA an SM, also where two would fit: each takes all tensor memory, and two
    // clusters could otherwise wait for one another's.
    best.smem = smem_of(best.tile_tokens, best.split, stages);
    if (best.smem < 120 * 1024) best.smem = 120 * 1024;
    return best;
}

cudaError_t launch_product(int out_dtype, const ProductParams& p, const ProductPlan& plan,
                           const CUtensorMap& map_w, const CUtensorMap& map_x, bool overlap,
                           unsigned wait_limit, cudaStream_t st) {
    Work w{};
    w.p = p;
    w.tile_tokens = plan.tile_tokens;
    w.blocks = (p.width + kDepth - 1) / kDepth;
    w.stages = plan.stages;
    w.split = plan.split;
    w.tiles_n = (int)((p.features + kFeatures - 1) / kFeatures);
    w.tiles_t = (int)((p.num_tokens + plan.tile_tokens - 1) / plan.tile_tokens);
    w.band = w.tiles_t < 8 ? w.tiles_t : 8;
    w.wait_limit = wait_limit;
    w.overlap = overlap;
    auto words = [](const uint8_t* s, long long stride) {
        return reinterpret_cast<uintptr_t>(s) % 4 == 0 && stride % 4 == 0;
    };
    w.x_words = words(p.x_scales, p.x_scales_stride);
    w.w_words = words(p.weight_scales, p.weight_scales_stride);
    switch (out_dtype) {
        case TLB_FLOAT16: return launch<__half>(w, plan, map_w, map_x, st);
        case TLB_BFLOAT16: return launch<__nv_bfloat16>(w, plan, map_w, map_x, st);
        default: return launch<float>(w, plan, map_w, map_x, st);
    }
}

}  // namespace tlb
