// Product of 8-bit rows with 8-bit weights on the tensor cores:
//   out[t, n] = sum over groups g of 2^(xs[t,g] + ws[n/128,g]) sum_{k in g} x[t,k] w[n,k]
//
// The scales are powers of two, so the tensor cores apply them: kind::mxf8f6f4
// takes an E8M0 scale for each row and 32 values of K, and gets the scale of the
// row's 128 four times. The sums stay in tensor memory in fp32 from the first
// value of K to the last.
//
// The weights are the M side (128 features a CTA, so a weight block of 128 x 128 has
// one scale for all lanes of a tile), the tokens the N side, of any multiple of 16:
// the number of tokens is what varies from call to call, and a tile of few tokens
// costs few bytes and few cycles. For few tokens a cluster of 2 or 4 CTAs shares a
// tile's width, and each joins the sums of some of its tokens, reading the others'
// over distributed shared memory. For many tokens two CTAs of a pair take 256
// features as one, each fetching half of the tokens' rows.
//
// Warps of a CTA: 0-3 bring the scales to tensor memory (each the 32 lanes it can
// reach), 4-11 read the sums and write the results, 12 issues the TMA copies (one or
// two chunks of 128 of K a stage), 13 the tensor instructions. The accumulator is
// double buffered: a tile is written out while the next one is summed.
#include <atomic>
#include <type_traits>

#include "kernels.h"
#include "quant.cuh"
#include "tcgen05.cuh"

namespace tlb {

using namespace product;

namespace {

constexpr int kThreads = 448;
constexpr int kResultThreads = 32 * kResultWarps;
constexpr int kCopyWarp = 12, kTensorWarp = 13;
constexpr int kScaleSets = 4;              // sets of scales in tensor memory, a word each
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
// behind the barriers, in kTail bytes with them: the tensor-memory address, the number of
// stages issued, and whether a wait gave up
constexpr int kSlot = kNumBars * 8, kIssued = kSlot + 4, kGaveUp = kSlot + 8;
static_assert(kGaveUp + 4 <= kTail, "barriers");
struct Work {
    ProductParams p;
    int tile_tokens;
    int depths;              // stages of a tile's whole width
    int groups;              // scales of a row
    int stages;
    int split;
    int tiles_n, tiles_t;
    int band;                // token tiles whose weights' tiles follow one another
    unsigned wait_limit;
    bool words;              // rows of scales allow 4-byte loads, and are whole words
    int parts_bytes;         // of shared memory for the results
    bool aligned;            // results allow stores of four features
    bool pieces;             // 16-bit results of one CTA a tile
    bool tma_out;            // whose rows allow TMA stores
    bool pairs_out;          // whose rows allow stores of two features
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
// The same where nothing written before has to be seen.
__device__ __forceinline__ void cluster_sync_relaxed() {
    asm volatile(
        "barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// Address in the cluster's CTA `rank` of what is at `addr` here.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 load_cluster(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ int load_cluster_int(uint32_t addr) {
    int v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
                 : "memory");
}
// The same where nothing written before has to be seen: a release waits for it.
__device__ __forceinline__ void arrive_cluster_relaxed(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
                 : "memory");
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

// A tile load into this CTA that completes at a barrier of either CTA of its pair.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int32_t x,
                                              int32_t y, uint32_t bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        ".cta_group::2.L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar), "l"(policy)
        : "memory");
}

// Tile `i` of the order in which a band of token tiles goes through all features.
__device__ __forceinline__ void tile_at(const Work& w, int i, int& tn, int& tt) {
    if (w.tiles_t == 1) {  // few tokens: the divisions would be in front of the first load
        tn = i;
        tt = 0;
        return;
    }
    const int per_band = w.band * w.tiles_n, b = i / per_band, rest = i % per_band;
    const int height = min(w.band, w.tiles_t - b * w.band);
    tn = rest / height;
    tt = b * w.band + rest % height;
}

// Whether `ok` holds in every thread of the kCount that meet at a barrier: they go on or
// give up together.
template <int kBarrier, int kCount>
__device__ __forceinline__ bool all_agree(bool ok) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.and.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(all)
        : "r"(ok ? 1u : 0u), "n"(kBarrier), "n"(kCount)
        : "memory");
    return all != 0;
}

// The scale bytes of groups 4 word .. 4 word + 3 of a row (past the last group: its
// byte again, which no instruction reads).
template <bool kWords>
__device__ __forceinline__ uint32_t scale_word(const uint8_t* row, int word, int groups) {
    if constexpr (kWords) return reinterpret_cast<const uint32_t*>(row)[word];
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) v |= (uint32_t)row[min(4 * word + i, groups - 1)] << (8 * i);
    return v;
}

// The scales' way to tensor memory (four warps). A tile's scales are read kWordsAtOnce
// words (of four groups) of every row at a time, each word once, and kept in shared
// memory, while the words before them go to tensor memory: four columns of the tile's
// weight scale, the same in all lanes, and a column for each 32 tokens. Each warp
// writes the 32 lanes it can reach. False: a wait gave up.
constexpr int kRowsAtOnce = 128 / kWordsAtOnce;

template <bool kPair, bool kWords>
__device__ __forceinline__ bool feed_scales(const Work& w, uint8_t* buffers, uint32_t tmem,
                                            uint32_t tail, int tid, int unit, int units, int tiles,
                                            int word_first, int word_end, int rank) {
    const ProductParams& p = w.p;
    const int warp = tid >> 5, lane = tid & 31;
    const long long last_block = (p.features - 1) / kFeatures;
    constexpr int kItems = kMaxTokens * kWordsAtOnce / 128;
    uint32_t x[kItems], ws = 0;
    int tile = unit, word = word_first, tn = 0, tt = 0;  // of the next read
    tile_at(w, tile, tn, tt);  // its divisions before the wait
    grid_dependency_wait();
    grid_launch_dependents();
    auto read = [&]() {
        if (tile >= tiles) return;
        const int at = min(word + (tid & (kWordsAtOnce - 1)), word_end - 1);
        const long long last = p.num_tokens - 1;
        long long t = (long long)tt * w.tile_tokens + tid / kWordsAtOnce;
#pragma unroll
        for (int m = 0; m < kItems; ++m, t += kRowsAtOnce)
            if (kRowsAtOnce * m < w.tile_tokens)
                x[m] = scale_word<kWords>(p.x_scales + min(t, last) * p.x_scales_stride, at, w.groups);
        if (tid < kWordsAtOnce) {
            const long long block = kPair ? min(2ll * tn + rank, last_block) : tn;
            ws = scale_word<kWords>(p.weight_scales + block * p.weight_scales_stride, at, w.groups);
        }
        word += kWordsAtOnce;
        if (word >= word_end) {
            word = word_first;
            tile += units;
            if (tile < tiles) tile_at(w, tile, tn, tt);
        }
    };
    read();
    int set = 0, half = 0;
    uint32_t parity = 1;  // of the wait for a free set: the first round's holds
    const uint32_t lanes = (uint32_t)warp << 21;  // 32 warp, in the address's upper half
    for (int i = unit; i < tiles; i += units)
        for (int first = word_first; first < word_end; first += kWordsAtOnce, half ^= 1) {
            uint32_t* buf = reinterpret_cast<uint32_t*>(buffers) + half * (kScaleRows * kScalePitch);
#pragma unroll
            for (int m = 0; m < kItems; ++m)
                if (kRowsAtOnce * m < w.tile_tokens)
                    buf[(tid / kWordsAtOnce + kRowsAtOnce * m) * kScalePitch +
                        (tid & (kWordsAtOnce - 1))] = x[m];
            if (tid < kWordsAtOnce) buf[kMaxTokens * kScalePitch + tid] = ws;
            named_bar_sync(2, 128);  // the other half's readers are past it too
            const int count = min(kWordsAtOnce, word_end - first);
            for (int k = 0; k < count; ++k) {
                // a CTA's warps give up together: they meet at the barrier above
                if (!all_agree<2, 128>(mbar_wait_bounded(tail + 8u * (kBarScalesFree + set), parity,
                                                    w.wait_limit)))
                    return false;
                tc5::fence_after_sync();
                uint32_t v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    v[j] = buf[min(32 * j + lane, kMaxTokens - 1) * kScalePitch + k];
                const uint32_t to = tmem + lanes + kScaleColumn + set * kSetColumns;
                tc5::st4(to, buf[kMaxTokens * kScalePitch + k]);
                tc5::st8(to + 4, v);
                tc5::st_wait();
                tc5::fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    const uint32_t full = tail + 8u * (kBarScales + set);
                    // wait::st has completed the stores to tensor memory; a release would
                    // wait for all others as well (a quarter of a pair's time)
                    if constexpr (kPair) arrive_cluster_relaxed(map_rank(full, 0));
                    else mbar_arrive(full);
                }
                if (++set == kScaleSets) {
                    set = 0;
                    parity ^= 1;
                }
                // early; bytes are waited for at once, so after the last word
                if (k == (kWords ? 0 : count - 1)) read();
            }
        }
    return true;
}

__device__ __forceinline__ void store_box(const CUtensorMap* map, int x, int y, uint32_t from) {
    asm volatile(
        "cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
            reinterpret_cast<uint64_t>(map)),
        "r"(x), "r"(y), "r"(from)
        : "memory");
}

// A warp's 32 features of up to 32 tokens where the rows of results are off 16 bytes
// (features no multiple of 8): two features a lane and two tokens at a time, or, off 4
// bytes, one and one.
template <typename T>
__device__ __forceinline__ void store_rows(const Work& w, uint32_t from, long long n0, long long t0,
                                           int rows, int lane) {
    const ProductParams& p = w.p;
    const int left = (int)min(32ll, p.features - n0);
    // feature f of token t: byte 2 (f % 8) of unit f / 8 ^ t / 2 % 4 of the token's 64
    auto at = [from](int t, int f) {
        return from + t * 64 + (((f >> 3) ^ ((t >> 1) & 3)) << 4) + (f & 7) * 2;
    };
    if (w.pairs_out) {
        const int f = (lane & 15) * 2;
        T* out = reinterpret_cast<T*>(p.out) + (t0 + (lane >> 4)) * p.out_stride + n0 + f;
#pragma unroll 4
        for (int t = lane >> 4; t < rows; t += 2, out += 2 * p.out_stride) {
            uint32_t v;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at(t, f)) : "memory");
            const uint16_t low = (uint16_t)v;
            if (f + 1 < left)
                *reinterpret_cast<uint32_t*>(out) = v;
            else if (f < left)
                memcpy(out, &low, 2);
        }
    } else {
        T* out = reinterpret_cast<T*>(p.out) + t0 * p.out_stride + n0 + lane;
#pragma unroll 4
        for (int t = 0; t < rows; ++t, out += p.out_stride) {
            uint16_t v;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at(t, lane)) : "memory");
            if (lane < left) memcpy(out, &v, 2);
        }
    }
}

// A tile's results in 16 bits, a warp's 32 features and 32 tokens at a time: the sums
// leave tensor memory in the layout of matrix fragments, are rounded in pairs of
// tokens and turned round by stmatrix, so that a token's 32 features lie side by side
// in shared memory (the 64-byte swizzle: unit u of 16 bytes at u ^ token / 2 % 4, free
// of bank conflicts); a TMA store takes them from there, past the tensor's ends as
// well (or the lanes do, store_rows). The warps of a feature quarter take every other 32 tokens; each has two buffers
// of its own (`turn` is the next), so the warps do not wait for one another; the next
// sums are read under the stores. 32 tokens take about 500 cycles of a warp (640 written
// by the lanes): with four warps, more than the instructions of a tile 1024 wide.
template <typename T>
__device__ __forceinline__ void store_pieces(const Work& w, const CUtensorMap* map, uint32_t sums,
                                             uint32_t stage, long long n0, long long t0, int here,
                                             int warp, int lane, uint32_t& turn) {
    if constexpr (sizeof(T) == 2) {
        const ProductParams& p = w.p;
        const int first = (warp >> 2) * 32;  // of this warp's tokens
        n0 += (warp & 3) * 32;
        if (n0 >= p.features || first >= here) return;
        const int box = w.tile_tokens % 32 == 0 ? 32 : 16;  // of the map
        float bias[4] = {};
        if (p.bias)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const long long n = n0 + 8 * i + (lane >> 2);
                if (n < p.features) bias[i] = Elem<T>::to_f(reinterpret_cast<const T*>(p.bias)[n]);
            }
        const uint32_t buf = stage + warp * 4096;  // two of 2 KB
        // token 8 g + lane % 8, unit lane / 8
        const uint32_t put = buf + (lane & 7) * 64 + (((lane >> 3) ^ ((lane >> 1) & 3)) << 4);
        uint32_t a[16], c[16];
        tc5::ld_rows16(sums + first, a);
        tc5::ld_rows16(sums + first + (16u << 16), c);
#pragma unroll 1
        for (int j = first; j < here; j += 64, turn ^= 2048) {
            tc5::ld_wait();
            uint32_t m[16];
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t* v = (i < 2 ? a : c) + 4 * g + 2 * (i & 1);
                    m[4 * g + i] = pack2<T>(__uint_as_float(v[0]) + bias[i],
                                            __uint_as_float(v[1]) + bias[i]);
                }
            if (j + 64 < here) {
                tc5::ld_rows16(sums + j + 64, a);
                tc5::ld_rows16(sums + j + 64 + (16u << 16), c);
            }
            // the store before the last one has read this buffer
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            __syncwarp();
#pragma unroll
            for (int g = 0; g < 4; ++g)
                asm volatile(
                    "stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                        put + turn + 512 * g),
                    "r"(m[4 * g]), "r"(m[4 * g + 1]), "r"(m[4 * g + 2]), "r"(m[4 * g + 3])
                    : "memory");
            if (!w.tma_out) {
                __syncwarp();
                store_rows<T>(w, buf + turn, n0, t0 + j, min(32, here - j), lane);
                continue;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                store_box(map, (int)n0, (int)t0 + j, buf + turn);
                // of 16 tokens where a tile may end after them
                if (box == 16 && j + 16 < w.tile_tokens)
                    store_box(map, (int)n0, (int)t0 + j + 16, buf + turn + 1024);
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
        }
    }
}

// A tile's results by way of fp32 sums in shared memory: of a cluster's CTAs, each
// joins its share of the tile's tokens, reading its part of the sums from every CTA
// (in the order of their ranks, so results do not depend on which is first). Also
// for one CTA's fp32 results. False: a wait gave up.
template <typename T>
__device__ __forceinline__ bool store_joined(const Work& w, uint32_t sums, uint8_t* stage,
                                             uint32_t parts, uint32_t bar, uint32_t parity,
                                             long long n0, long long t0, int here, int warp,
                                             int lane, int rank) {
    const ProductParams& p = w.p;
    const int split = w.split, f0 = lane * 4;
    const int wide = (int)min(4ll, p.features - n0 - f0);  // features of this lane
    float bias[4] = {};
    if (p.bias)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < wide) bias[k] = Elem<T>::to_f(reinterpret_cast<const T*>(p.bias)[n0 + f0 + k]);
    T* out = reinterpret_cast<T*>(p.out) + t0 * p.out_stride + n0 + f0;
    // tokens at a time: all of a cluster's tile, else 64
    const int rows = split > 1 ? w.tile_tokens : 64;
    float* column = reinterpret_cast<float*>(stage) + (warp & 3) * 32 + lane;
    for (int j0 = 0; j0 < here; j0 += rows) {
        const int count = min(rows, here - j0);
        for (int j = (warp >> 2) * 32; j < count; j += 64) {
            float v[32];
            tc5::ld32(sums + j0 + j, v);
#pragma unroll
            for (int k = 0; k < 32; ++k)
                if (j + k < rows) column[(j + k) * kFeatures] = v[k];
        }
        int first = 0, mine = count;
        if (split > 1) {
            const int share = (count + split - 1) / split;
            first = rank * share;
            mine = max(0, min(share, count - first));
            __syncwarp();
            if (lane < split) arrive_cluster(map_rank(bar, lane));
            if (!all_agree<1, kResultThreads>(wait_cluster(bar, parity, w.wait_limit))) return false;
        } else {
            named_bar_sync(1, kResultThreads);
        }
        const uint32_t from = parts + f0 * 4;
        for (int r0 = warp; r0 < mine; r0 += 2 * kResultWarps) {  // two rows of all CTAs in flight
            float4 v[2], x[kMaxSplit][2];
#pragma unroll
            for (int c = 0; c < kMaxSplit; ++c) {
                if (c >= split) break;
                const uint32_t at = split > 1 ? map_rank(from, c) : from;
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    x[c][k] = load_cluster(at + (first + min(r0 + kResultWarps * k, mine - 1)) *
                                                    (kFeatures * 4));
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                v[k] = x[0][k];
#pragma unroll
                for (int c = 1; c < kMaxSplit; ++c) {
                    if (c >= split) break;
                    v[k].x += x[c][k].x;
                    v[k].y += x[c][k].y;
                    v[k].z += x[c][k].z;
                    v[k].w += x[c][k].w;
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int row = r0 + kResultWarps * k;
                if (row >= mine) break;
                T* to = out + (j0 + first + row) * p.out_stride;
                const float y[4] = {v[k].x + bias[0], v[k].y + bias[1], v[k].z + bias[2],
                                    v[k].w + bias[3]};
                if (wide == 4 && w.aligned) {
                    if constexpr (sizeof(T) == 2)
                        *reinterpret_cast<uint2*>(to) =
                            make_uint2(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]));
                    else
                        *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e < wide) to[e] = Elem<T>::from_f(y[e]);
                }
            }
        }
        if (j0 + rows < here) named_bar_sync(1, kResultThreads);  // read before it is written again
    }
    return true;
}

// kChunks: of 128 values of K a stage. Two halve the waits and commits of the one thread
// that issues the tensor instructions, which a tile of few tokens is bounded by; one
// gives a wide tile's stages finer steps (64 x 2048 -> 2560 in tiles of 16 tokens: 7.4 us
// with one, 6.6 with two; 1024 x 2048 -> 2560 in tiles of 160: 9.0 and 9.9).
template <typename T, bool kPair, int kChunks>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_w,
                   const __grid_constant__ CUtensorMap map_x,
                   const __grid_constant__ CUtensorMap map_out, const Work w) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    const uint32_t base = smem_u32(smem);
    constexpr int kDepth = kChunks * kChunk;  // of a stage
    constexpr int kPerWord = 512 / kDepth;    // stages of a word of scales
    const ProductParams& p = w.p;
    const int x_rows = kPair ? w.tile_tokens / 2 : w.tile_tokens;  // of this CTA's stages
    const uint32_t x_bytes = x_rows * kChunk;                      // of a chunk
    const uint32_t stage_bytes = kChunks * (kWeightBytes + x_bytes);
    const uint32_t tail = base + w.stages * stage_bytes, parts = tail + kTail;
    uint8_t* tail_ptr = smem + w.stages * stage_bytes;
    auto bar = [tail](int i) { return tail + 8u * i; };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // CTAs of a cluster: of a pair, or sharing a tile's width
    const int split = kPair ? 1 : w.split, cluster = kPair ? 2 : split;
    const int rank = cluster > 1 ? (int)cluster_rank() : 0;

    if (tid < kNumBars) {  // a barrier a thread
        int arrivals = 1;
        if (tid >= kBarScales && tid < kBarScalesFree) arrivals = kPair ? 8 : 4;
        if (tid >= kBarSumsFree && tid < kBarParts) arrivals = (kPair ? 2 : 1) * kResultWarps;
        if (tid >= kBarParts && tid < kBarDrain) arrivals = kResultWarps * split;
        mbar_init(bar(tid), arrivals);
        fence_mbar_init();
        if (tid == 0) *reinterpret_cast<volatile int*>(tail_ptr + kGaveUp) = 0;
    }
    if (warp == kTensorWarp) {
        if constexpr (kPair) tc5::alloc_pair(tail + kSlot, kColumns);
        else tc5::alloc(tail + kSlot, kColumns);
    }
    if (tid == 32 * kCopyWarp) {
        prefetch_tensormap(&map_w);
        prefetch_tensormap(&map_x);
    }
    tc5::fence_before_sync();
    __syncthreads();
    if (cluster > 1) cluster_sync();  // all barriers of the cluster are set up
    tc5::fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tail_ptr + kSlot);

    auto commit = [](uint32_t b) {
        if constexpr (kPair) tc5::commit_pair(b);
        else tc5::commit(b);
    };
    // this CTA's tiles, and its part of their width
    const int tiles = w.tiles_n * w.tiles_t;
    const int units = gridDim.x / cluster, unit = blockIdx.x / cluster;
    const int d_first = (int)((long long)w.depths * (split > 1 ? rank : 0) / split);
    const int d_last = (int)((long long)w.depths * (split > 1 ? rank + 1 : 1) / split);
    const int word_first = d_first / kPerWord, word_end = (d_last - 1) / kPerWord + 1;
    const uint32_t limit = w.wait_limit;
    bool ok = true, issues = false;  // issues: this thread, the tensor instructions

    if (warp == kCopyWarp) {
        // ------------------------------------------------------------ copies
        if (elect_one()) {
            // tiles read both operands again: 2 to 4 % faster than without a policy
            const uint64_t keep = l2_policy_evict_last();
            const uint64_t once = l2_policy_evict_first();
            // weights that only this tile's tokens want pass through the L2
            const uint64_t w_policy = w.tiles_t > 1 ? keep : once;
            const uint32_t full0 = kPair && rank == 1 ? map_rank(bar(kBarFull), 0) : bar(kBarFull);
            auto load = [](uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t b,
                           uint64_t policy) {
                if constexpr (kPair) tma_load_pair(dst, map, x, y, b, policy);
                else tma_load_2d(dst, map, x, y, b, policy);
            };
            // The weights too: fetched under the kernel before (which mostly does not write
            // them), a norm and a product of 64 x 2048 -> 2560 took 9.1 us, so 8.5.
            int tn, tt;
            tile_at(w, unit, tn, tt);
            grid_dependency_wait();
            // One thread issues everything, so its instructions are what a stage costs:
            // counters instead of divisions.
            int s = 0, issued = 0;
            uint32_t parity = 1;  // of the wait for a free stage: the first round's holds
            uint32_t at = base;
            for (int i = unit; i < tiles && ok; i += units) {
                if (i != unit) tile_at(w, i, tn, tt);
                const int wy = (kPair ? 2 * tn + rank : tn) * kFeatures;
                const int xy = tt * w.tile_tokens + (kPair ? rank * x_rows : 0);
                for (int d = d_first; d < d_last; ++d) {
                    const uint32_t full = full0 + 8 * s;
                    if (!mbar_wait_bounded(bar(kBarEmpty + s), parity, limit)) {
                        ok = false;
                        break;
                    }
                    const int k = d * kDepth;
                    const bool both = kChunks == 2 && k + kChunk < p.width;
                    // a pair's bytes are expected by its even CTA; copies may complete first
                    if (!kPair || rank == 0)
                        mbar_arrive_expect_tx(
                            full, (kPair ? 2 : 1) * (both ? stage_bytes : stage_bytes / kChunks));
                    load(at, &map_w, k, wy, full, w_policy);
                    load(at + kChunks * kWeightBytes, &map_x, k, xy, full, keep);
                    if (both) {
                        load(at + kWeightBytes, &map_w, k + kChunk, wy, full, w_policy);
                        load(at + kChunks * kWeightBytes + x_bytes, &map_x, k + kChunk, xy, full, keep);
                    }
                    ++issued;
                    at += stage_bytes;
                    if (++s == w.stages) {
                        s = 0;
                        parity ^= 1;
                        at = base;
                    }
                }
            }
            *reinterpret_cast<volatile int*>(tail_ptr + kIssued) = issued;
        }
    } else if (warp == kTensorWarp) {
        // ------------------------------------------------ tensor instructions
        if ((!kPair || rank == 0) && elect_one()) {
            issues = true;
            const uint64_t whole = tc5::desc_sw128(base, 16, 1024);
            const uint32_t first = (uint32_t)whole, high = (uint32_t)(whole >> 32);
            const uint32_t idesc = tc5::idesc_mxf8(kPair ? 256 : 128, w.tile_tokens, 0);
            uint32_t desc = first;
            int s = 0, set = 0, it = 0;
            uint32_t parity = 0, set_parity = 0;
            // Nothing is read here, but the scales and stages come no earlier: a bounded wait
            // begun before this would count the rest of the kernel before as well, which
            // may be longer than the bound.
            grid_dependency_wait();
            for (int i = unit; i < tiles && ok; i += units, ++it) {
                const int b = it & 1;
                if (it >= 2 && !mbar_wait_bounded(bar(kBarSumsFree + b), ((it >> 1) - 1) & 1, limit)) {
                    ok = false;
                    break;
                }
                tc5::fence_after_sync();
                const uint32_t sums = tmem + b * kMaxTokens;
                bool accumulate = false;
                for (int word = word_first; word < word_end && ok; ++word) {
                    if (!mbar_wait_bounded(bar(kBarScales + set), set_parity, limit)) {
                        ok = false;
                        break;
                    }
                    const uint32_t scales = tmem + kScaleColumn + set * kSetColumns;
#pragma unroll
                    for (int h = 0; h < kPerWord; ++h) {
                        const int d = kPerWord * word + h;
                        if (d < d_first || d >= d_last) continue;
                        if (!mbar_wait_bounded(bar(kBarFull + s), parity, limit)) {
                            ok = false;
                            break;
                        }
                        tc5::fence_after_sync();
                        const int left = p.width - d * kDepth;
#pragma unroll
                        for (int k = 0; k < 4 * kChunks; ++k) {
                            if (32 * k >= left) break;
                            const uint32_t sf = kChunks * h + k / 4;
                            tc5::mma_mxf8<kPair>(
                                sums, desc + (k / 4) * (kWeightBytes >> 4) + 2 * (k % 4),
                                desc + (kChunks * kWeightBytes >> 4) + (k / 4) * (x_bytes >> 4) +
                                    2 * (k % 4),
                                high, idesc | sf << 4 | sf << 29, scales, scales + 4, accumulate);
                            accumulate = true;
                        }
                        commit(bar(kBarEmpty + s));
                        desc += stage_bytes >> 4;
                        if (++s == w.stages) {
                            s = 0;
                            parity ^= 1;
                            desc = first;
                        }
                    }
                    commit(bar(kBarScalesFree + set));
                    if (++set == kScaleSets) {
                        set = 0;
                        set_parity ^= 1;
                    }
                }
                if (ok) commit(bar(kBarSums + b));
            }
        }
    } else if (warp < 4) {
        // ------------------------------------------------------------ scales
        uint8_t* buffers = tail_ptr + kTail + w.parts_bytes;
        ok = w.words ? feed_scales<kPair, true>(w, buffers, tmem, tail, tid, unit, units, tiles,
                                                word_first, word_end, rank)
                     : feed_scales<kPair, false>(w, buffers, tmem, tail, tid, unit, units, tiles,
                                                 word_first, word_end, rank);
    } else {
        // ----------------------------------------------------------- results
        grid_dependency_wait();
        const int mine = warp - 4;
        uint8_t* stage = tail_ptr + kTail;
        uint32_t turn = 0;
        int it = 0;
        for (int i = unit; i < tiles; i += units, ++it) {
            int tn, tt;
            tile_at(w, i, tn, tt);
            const long long n0 = (kPair ? 2ll * tn + rank : tn) * kFeatures;
            const long long t0 = (long long)tt * w.tile_tokens;
            const int here = (int)min((long long)w.tile_tokens, p.num_tokens - t0);
            const int b = it & 1;
            const uint32_t sums = tmem + ((uint32_t)(warp & 3) << 21) + b * kMaxTokens;
            ok = mbar_wait_bounded(bar(kBarSums + b), (it >> 1) & 1, limit);
            if (split > 1 && it > 0)
                ok = wait_cluster(bar(kBarPartsFree), (it - 1) & 1, limit) && ok;
            if (w.pieces) {
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc5::fence_after_sync();
                store_pieces<T>(w, &map_out, sums, parts, n0, t0, here, mine, lane, turn);
            } else {
                ok = all_agree<1, kResultThreads>(ok);
                if (!ok) break;
                tc5::fence_after_sync();
                ok = store_joined<T>(w, sums, stage, parts, bar(kBarParts), it & 1, n0, t0, here,
                                     mine, lane, rank);
            }
            tc5::fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                // the sums have been read (wait::ld); nothing was written for the other CTA
                if constexpr (kPair) arrive_cluster_relaxed(map_rank(bar(kBarSumsFree + b), 0));
                else mbar_arrive(bar(kBarSumsFree + b));
            }
            if (!ok) break;
            // a release waits for the results' stores: only where another tile follows
            if (split > 1 && i + units < tiles && lane < split)
                arrive_cluster(map_rank(bar(kBarPartsFree), lane));
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    if (!ok) {
        flag_status(TLB_STATUS_WAIT_TIMEOUT);
        *reinterpret_cast<volatile int*>(tail_ptr + kGaveUp) = 1;
    }
    __syncwarp();
    tc5::fence_before_sync();
    __syncthreads();
    // No CTA ends while another one may read its sums or arrive at its barriers (a pair's
    // also tell one another whether a wait gave up).
    if constexpr (kPair) cluster_sync();
    else if (split > 1) cluster_sync_relaxed();
    bool gave_up = *reinterpret_cast<volatile int*>(tail_ptr + kGaveUp) != 0;
    if constexpr (kPair)
        gave_up = gave_up || load_cluster_int(map_rank(tail + kGaveUp, rank ^ 1)) != 0;
    // After a wait that gave up, the tensor instructions that were issued complete before the
    // tensor memory is freed, whichever thread gave up (results that were read were complete,
    // but a thread that waits for them may have given up where the one that issues them went
    // on to its end), of a pair in both CTAs, whose operands they read.
    if (gave_up && issues) commit(bar(kBarDrain));
    if (gave_up && tid == 32 * kTensorWarp) mbar_wait_bounded(bar(kBarDrain), 0);
    // And the copies that were issued land before the CTA ends (they have otherwise: their
    // stages were used).
    if (gave_up && tid == 0 && (!kPair || rank == 0)) {
        const int mine = *reinterpret_cast<volatile int*>(tail_ptr + kIssued);
        int most = mine;
        if constexpr (kPair) {
            // both CTAs' copies complete here: expect those of the other CTA alone, and
            // make up for those that it did not issue
            const int other = load_cluster_int(map_rank(tail + kIssued, 1));
            most = max(mine, other);
            for (int k = min(mine, other); k < most; ++k) {
                const int s = k % w.stages, x = k % w.depths * kDepth;
                const uint32_t at = base + s * stage_bytes;
                const bool both = kChunks == 2 && x + kChunk < p.width;
                if (k >= mine) {
                    mbar_arrive_expect_tx(bar(kBarFull + s),
                                          both ? stage_bytes : stage_bytes / kChunks);
                    continue;
                }
                for (int c = 0; c < (both ? 2 : 1); ++c) {
                    tma_load_2d(at + c * kWeightBytes, &map_w, x, 0, bar(kBarFull + s),
                                l2_policy_evict_first());
                    tma_load_2d(at + kChunks * kWeightBytes + c * x_bytes, &map_x, x, 0,
                                bar(kBarFull + s), l2_policy_evict_first());
                }
            }
        }
        for (int k = max(0, most - w.stages); k < most; ++k)
            mbar_wait_bounded(bar(kBarFull + k % w.stages), (k / w.stages) & 1);
    }
    if (gave_up) __syncthreads();
    if constexpr (kPair) cluster_sync();
    if (warp == kTensorWarp) {
        tc5::fence_after_sync();
        if constexpr (kPair) tc5::dealloc_pair(tmem, kColumns);
        else tc5::dealloc(tmem, kColumns);
    }
}

template <typename T, bool kPair, int kChunks>
cudaError_t launch(const Work& w, const ProductPlan& plan, const CUtensorMap& map_w,
                   const CUtensorMap& map_x, const CUtensorMap& map_out, cudaStream_t st) {
    auto kernel = product_kernel<T, kPair, kChunks>;
    // the attribute is the kernel's on one device: set once for each
    static std::atomic<unsigned long long> set{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (!(set.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)kMaxSmem);
        if (e != cudaSuccess) return e;
        set.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kPair ? 2 : plan.split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(plan.ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = plan.smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = kPair || plan.split > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, map_w, map_x, map_out, w);
}

}  // namespace

cudaError_t launch_product(int out_dtype, const ProductParams& p, const ProductPlan& plan,
                           const CUtensorMap& map_w, const CUtensorMap& map_x,
                           const CUtensorMap& map_out, bool tma_out, unsigned wait_limit,
                           cudaStream_t st) {
    Work w{};
    w.p = p;
    w.tile_tokens = plan.tile_tokens;
    const int depth = plan.chunks * kChunk;
    w.depths = (p.width + depth - 1) / depth;
    w.groups = (p.width + kChunk - 1) / kChunk;
    w.stages = plan.stages;
    w.split = plan.split;
    const int per_cta = plan.pair ? 2 * kFeatures : kFeatures;
    w.tiles_n = (int)((p.features + per_cta - 1) / per_cta);
    w.tiles_t = (int)((p.num_tokens + plan.tile_tokens - 1) / plan.tile_tokens);
    // 2048 x 4096 -> 14336 sustained: 112.6 us in bands of 8, 109.4 in bands of 16 or 32
    w.band = w.tiles_t < 16 ? w.tiles_t : 16;
    w.wait_limit = wait_limit;
    auto words = [](const uint8_t* s, long long stride) {
        return reinterpret_cast<uintptr_t>(s) % 4 == 0 && stride % 4 == 0;
    };
    w.words = w.groups % 4 == 0 && words(p.x_scales, p.x_scales_stride) &&
              words(p.weight_scales, p.weight_scales_stride);
    w.parts_bytes = parts_bytes_of(plan.tile_tokens, plan.split, plan.pieces);
    const int e = out_dtype == TLB_FLOAT32 ? 4 : 2;
    w.aligned = reinterpret_cast<uintptr_t>(p.out) % (4 * e) == 0 && p.out_stride % 4 == 0;
    w.pieces = plan.pieces;
    w.tma_out = tma_out;
    w.pairs_out = reinterpret_cast<uintptr_t>(p.out) % 4 == 0 && p.out_stride % 2 == 0;
    auto start = [&](auto pair, auto chunks) {
        constexpr bool kPair = decltype(pair)::value;
        constexpr int kChunks = decltype(chunks)::value;
        switch (out_dtype) {
            case TLB_FLOAT16: return launch<__half, kPair, kChunks>(w, plan, map_w, map_x, map_out, st);
            case TLB_BFLOAT16:
                return launch<__nv_bfloat16, kPair, kChunks>(w, plan, map_w, map_x, map_out, st);
            default: return launch<float, kPair, kChunks>(w, plan, map_w, map_x, map_out, st);
        }
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    if (plan.pair) return start(std::true_type{}, Two{});
    return plan.chunks == 1 ? start(std::false_type{}, One{}) : start(std::false_type{}, Two{});
}

}  // namespace tlb
