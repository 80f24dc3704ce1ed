// Decode attention whose keys and values may be held in 8 bits and whose
// scores may be capped, biased by distance or limited to a window.
//
// For query head h of sequence s with L tokens, token j of its context scores
//   x_j = scale * 2^Ek_j * (q . k_j)            (no scale byte: Ek = 0)
//   x_j = cap * tanh(x_j / cap)                 (softcap > 0)
//   x_j += slope_h * (j - (L - 1))              (alibi_slopes)
// over the tokens first <= j < L, first = max(0, L - window) (window > 0) or 0,
// whose block is not a hole, and out = sum_j softmax(x)_j * 2^Ev_j * v_j.
//
// What bounds it: the stream of cache rows (two flops a byte and query head),
// so the work is laid out for bytes in flight and even ranges:
//  * A tile is kTT tokens of one (sequence, kv head), 8 KB of keys and values:
//    16 to 64 rows by their width. The tiles of all units, with a charge of
//    kUnitCost tiles for starting a unit, form one line, cut evenly over all
//    warps of the grid (one CTA per SM; 12 warps for units of up to 8 heads, 8
//    for 16). Each warp streams its contiguous part through a ring of its own
//    (TMA boxes of a block's rows, scale bytes by cp.async) and never waits for
//    another warp, so units of any mix of lengths keep every SM busy and a short
//    sequence costs one warp one tile.
//  * S^T = K Q^T and O^T += V^T P^T with mma.m16n8k16: the tokens (then the
//    dims) fill m = 16 and the query heads of the kv head n = 8, so a group of
//    8 wastes nothing; 8-bit values become fp16 in registers, exactly. bf16
//    queries meet 8-bit keys as fp16 scaled by a power of two per head (their
//    8 significant bits fit in fp16's 11; elements 2^-29 below the head's largest
//    start to lose bits).
//  * The softmax is online, in fp32, with a lazy reference: the running
//    maximum m moves only when a score passes it by 2^8, so most tiles pay one
//    vote instead of shuffles and a rescale. Values' scales fold into the
//    weights: w_j = 2^(x_j + Ev_j - mv) with a running maximum mv of its own,
//    so w_j fits fp16 whatever the scales of the rows are. fp16 weights are
//    held 2^7 higher (up to 2^15 with the lazy reference), so that what
//    fp16 rounds by 2^-25 below its normal range is 2^-32 of the reference.
//  * Where there are no more units than SMs and none has more than
//    kAlignedTiles tiles a warp, a CTA takes a whole unit instead: even ranges
//    would gain little, and neither a scan nor a joining of CTAs is needed.
//  * A unit cut by range ends leaves fp32 partials: warps of one CTA join
//    theirs in shared memory, CTAs through the workspace: the last CTA to
//    publish its partial sums them all. The order of every sum is fixed, so
//    results are the same bits on every run.
// Measured: 256 sequences of 7000-8192 tokens, 14 + 2 heads of 64, bf16 over e4m3
// (508 MB), 90 to 97 us on three B200s (5.6 to 5.2 TB/s; 86 us back to back on three
// inputs). 64 sequences of 128-4096 tokens, 16 + 2 heads of 128, bf16 over e4m3
// (71.6 MB), 22.2 us: the rows stream until 15 us, the joins take the rest. An L2
// policy of evict_normal for the rows cost 4 % of the latter. Without the scale
// bytes' copies the former, at 133 us then, took 128 us; without its arithmetic
// 92 us.
#pragma once

#include <atomic>
#include <type_traits>

#include "kernels.h"
#include "quant.cuh"

namespace tlb {
namespace scored {

constexpr int kUnitCost = 1;       // tiles charged for starting a unit
constexpr float kLazy = 8.f;       // log2 of how far a score may pass the reference
constexpr float kLog2e = 1.4426950408889634f;

// Flags of a tile and, or-ed over a piece, of a partial. Above them the unit's
// number of query heads (bits 4-8) and, in a tile's header, its first one.
constexpr int kFirst = 1;      // first tile of a piece in this warp's range
constexpr int kLast = 2;       // last tile of a piece in this warp's range
constexpr int kUnitBegin = 4;  // first tile of its unit
constexpr int kUnitEnd = 8;    // last tile of its unit
constexpr int kHeadsShift = 4, kHeadsMask = 31 << kHeadsShift, kHead0Shift = 9;

template <typename QT, typename CT, int D, int NT>
struct Cfg {
    static constexpr int kBytes = sizeof(CT);
    static constexpr bool kQ8 = kBytes == 1;
    static constexpr int kRow = D * kBytes;         // bytes per row
    static constexpr int kTT = tile_tokens(kRow);   // tokens per tile
    static constexpr int kChunks = kRow / 16;
    static constexpr int kHalfStage = kTT * kRow;   // K (or V) bytes of a stage
    static constexpr int kStage = 2 * kHalfStage;
    static constexpr int kWarps = warps_for(8 * NT);
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kStages = kWarps > 8 ? 2 : 3;
    static constexpr int kRingBytes = kStages * kStage;  // per warp
    static constexpr int kColumns = kRow > 128 ? 2 : 1;  // 128-byte columns of a row
    static constexpr int kGroup = 8 * NT;           // heads per unit
    static constexpr int kTiles = D / 16;           // dim tiles
    // float4 fragments of a partial: [nt][dim tile][lane]
    static constexpr int kFrags = NT * kTiles * 32;
    // P is carried as a hi + lo pair where one 16-bit rounding would show in
    // the output: bf16 weights (8 bits) always, fp16 weights with fp16 outputs
    static constexpr bool kSplit = !(kQ8 && std::is_same<QT, __nv_bfloat16>::value);
    // weights are held 2^kLift above the reference where they are fp16
    static constexpr int kLift = kQ8 || std::is_same<QT, __half>::value ? 7 : 0;
    // Partials of pieces that end inside a warp's range: the first kParts of a
    // CTA in shared memory, others in the workspace.
    static constexpr int kPartBytes = kFrags * 16;
    static constexpr int kParts = 24576 / kPartBytes;
    // shared memory
    static constexpr int kPartOff = kWarps * kRingBytes;
    static constexpr int kBarOff = kPartOff + kParts * kPartBytes;
    static constexpr int kHdrOff = kBarOff + (kWarps * kStages * 8 + 15) / 16 * 16;
    static constexpr int kScaleOff = kHdrOff + kWarps * kStages * 16;
    static constexpr int kMlOff = kScaleOff + (kQ8 ? kWarps * kStages * 2 * kTT : 0);
    static constexpr int kWeightOff = kMlOff + 2 * kWarps * kGroup * 8;
    static constexpr int kUnitOff = kWeightOff + 2 * kWarps * kGroup * 8;
    static constexpr int kPointOff = kUnitOff + 2 * kWarps * 16;
    static constexpr int kPrefixOff = kPointOff + (2 * kWarps * 8 + kWarps * kStages * 4 + 15) / 16 * 16;
    static constexpr int kSmem = kPrefixOff + (kThreads + kWarps) * 4 + 1024;  // + alignment slack
    static_assert(kSmem <= 232448, "one CTA per SM");
};

// Byte offset of 16-byte chunk c of row r in a tile, as the TMA boxes leave it:
// rows of 128 bytes with 128-byte swizzle, 256-byte rows as two such columns,
// 64-byte rows two to a line with 64-byte swizzle. ldmatrix's eight rows of one
// chunk then hit all banks.
template <int CH, int TT>
__device__ __forceinline__ uint32_t tile_offset(int r, int c) {
    if constexpr (CH == 4) {
        const int line = r >> 1;
        return (uint32_t)(line * 128 + (((((r & 1) << 2) | c) ^ (line & 3)) << 4));
    } else {
        return (uint32_t)((c >> 3) * TT * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
    }
}

__device__ __forceinline__ void cp_async_4_zfill(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(src)), "r"(on ? 4 : 0)
                 : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Four bytes of one row (dims 4t .. 4t + 3) -> fp16 pairs (0, 1) and (2, 3).
template <typename C> __device__ __forceinline__ void widen_row(uint32_t x, uint32_t& a, uint32_t& b);
// Bytes {token 2t: dims 2g, 2g+1; token 2t+1: the same dims}, as a transposed
// 16-bit ldmatrix leaves them -> the token pairs of dim 2g and of dim 2g + 1.
template <typename C> __device__ __forceinline__ void widen_col(uint32_t x, uint32_t& a, uint32_t& b);
template <> __device__ __forceinline__ void widen_row<E4M3>(uint32_t x, uint32_t& a, uint32_t& b) {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(a), "=r"(b)
        : "r"(x));
}
template <> __device__ __forceinline__ void widen_col<E4M3>(uint32_t x, uint32_t& a, uint32_t& b) {
    widen_row<E4M3>(__byte_perm(x, 0, 0x3120), a, b);
}
// int8: the byte with its sign bit flipped is x + 128; under 0x64 it is the
// fp16 number 1024 + x + 128, and the subtraction is exact.
__device__ __forceinline__ uint32_t minus_1152(uint32_t h) {
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&h), __float2half2_rn(1152.f));
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ void widen_row<int8_t>(uint32_t x, uint32_t& a, uint32_t& b) {
    x ^= 0x80808080u;
    a = minus_1152(__byte_perm(x, 0x64646464u, 0x4140));
    b = minus_1152(__byte_perm(x, 0x64646464u, 0x4342));
}
template <> __device__ __forceinline__ void widen_col<int8_t>(uint32_t x, uint32_t& a, uint32_t& b) {
    x ^= 0x80808080u;
    a = minus_1152(__byte_perm(x, 0x64646464u, 0x4240));
    b = minus_1152(__byte_perm(x, 0x64646464u, 0x4341));
}

// A score in log2 units from the scaled product (scale, scales and the query's
// power of two already applied): the cap, then the distance bias.
struct ScoreMod {
    float cap_log2;  // softcap * log2(e), 0: none
    float inv_cap;   // 1 / softcap
    bool alibi;
    __device__ __forceinline__ float cap(float x) const {
        // tanh(u) = 1 - 2 / (e^2u + 1) loses its leading digits near 0, where
        // u - u^3/3 + 2 u^5/15 is good to 1e-9
        const float u = x * inv_cap;
        const float e = ex2(2.f * kLog2e * u);
        const float big = 1.f - __fdividef(2.f, e + 1.f);
        const float u2 = u * u;
        const float small = u * (1.f + u2 * (-1.f / 3.f + u2 * (2.f / 15.f)));
        return cap_log2 * (fabsf(u) < 0.05f ? small : big);
    }
};

// Weight of a partial whose reference is m against the joint reference M
// (-inf: an empty partial).
__device__ __forceinline__ float piece_weight(float m, float M) {
    return m == -INFINITY ? 0.f : ex2(m - M);
}

// 1 / the sum of weights; 0 for an empty softmax (NaN stays NaN).
__device__ __forceinline__ float inverse(float sum) {
    return sum > 0.f || sum != sum ? __fdividef(1.f, sum) : 0.f;
}

// Largest x of the lanes in `mask`, each of which calls this with its own set.
__device__ __forceinline__ float max_of(uint32_t mask, float x) {
    // as integers of the same order (NaN above or below all numbers)
    const int b = __float_as_int(x);
    const int m = __reduce_max_sync(mask, b ^ ((b >> 31) & 0x7fffffff));
    return __int_as_float(m ^ ((m >> 31) & 0x7fffffff));
}

// One fragment (dim tile i, lane) of a unit's output, whose first head is row
// `row` of the [sequences * heads] output: (v.x, v.y) are heads 2t, 2t + 1 of
// one dim, (v.z, v.w) of another: with 8-bit values the next dim (dims 2g,
// 2g + 1 of the tile), otherwise dims g and g + 8.
template <typename QT, bool Q8, int D>
__device__ __forceinline__ void write_frag(void* out, int row, int heads, int nt, int i, int lane,
                                           float4 v, float inv0, float inv1) {
    const int g = lane >> 2, h = nt * 8 + 2 * (lane & 3);
    const int d0 = 16 * i + (Q8 ? 2 * g : g);
    QT* o = reinterpret_cast<QT*>(out) + (long long)(row + h) * D + d0;
    if constexpr (Q8) {
        if (h < heads) *reinterpret_cast<uint32_t*>(o) = pack2<QT>(v.x * inv0, v.z * inv0);
        if (h + 1 < heads) *reinterpret_cast<uint32_t*>(o + D) = pack2<QT>(v.y * inv1, v.w * inv1);
    } else {
        if (h < heads) {
            o[0] = Elem<QT>::from_f(v.x * inv0);
            o[8] = Elem<QT>::from_f(v.z * inv0);
        }
        if (h + 1 < heads) {
            o[D] = Elem<QT>::from_f(v.y * inv1);
            o[D + 8] = Elem<QT>::from_f(v.w * inv1);
        }
    }
}

// Tokens of sequence s that are read: [first, len).
struct Span {
    int len, first;
};
__device__ __forceinline__ Span span_of(int s, const Params& p) {
    Span r;
    r.len = min(max(p.seq_lens[s], 0), p.max_tokens);
    r.first = p.window > 0 ? max(0, r.len - p.window) : 0;
    return r;
}

template <typename QT, typename CT, int D, int NT>
__global__ void __launch_bounds__(Cfg<QT, CT, D, NT>::kThreads, 1)
    scored_attention_kernel(const __grid_constant__ CUtensorMap map_k,
                            const __grid_constant__ CUtensorMap map_v, const Params p) {
    using F = Cfg<QT, CT, D, NT>;
    // element type of the matrix products: 8-bit values become fp16
    using MT = typename std::conditional<F::kQ8, __half, QT>::type;
    constexpr int TT = F::kTT, CH = F::kChunks, ST = F::kStages, G = F::kGroup;
    constexpr int W = F::kWarps, THREADS = F::kThreads;
    constexpr int MT_TILES = TT / 16;  // 16-token tiles of a stage
    // the swizzled boxes need a 1024-byte aligned base, which nothing promises
    // of the dynamic array itself
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_base = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw_base + 1023u) & ~1023u) - raw_base);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t4 = lane & 3;
    int4* hdr = reinterpret_cast<int4*>(smem + F::kHdrOff) + warp * ST;
    uint8_t* sc = smem + F::kScaleOff + warp * ST * 2 * TT;
    float2* ml = reinterpret_cast<float2*>(smem + F::kMlOff);      // [2 W][G] (m, l)
    float2* wl = reinterpret_cast<float2*>(smem + F::kWeightOff);  // [2 W][G] joint weight, times l
    int4* ids = reinterpret_cast<int4*>(smem + F::kUnitOff);       // [2 W] (row, flags, part)
    int2* points = reinterpret_cast<int2*>(smem + F::kPointOff);   // [2 W] a unit's (first cost point, tiles)
    int* hdr_point = reinterpret_cast<int*>(points + 2 * W) + warp * ST;  // first cost point
    int* pre = reinterpret_cast<int*>(smem + F::kPrefixOff);       // [THREADS] cost before, in warp
    int* wsum = pre + THREADS;                                     // [W] cost of a warp's threads
    __shared__ int parts_used;
    __shared__ bool last_cta[2];
    __shared__ int4 shared_unit[2];
    const uint32_t bars = smem_u32(smem + F::kBarOff) + warp * ST * 8;
    const uint32_t ring = smem_u32(smem) + warp * F::kRingBytes;

    if (!p.overlap) grid_dependency_wait();
    // ---- cost line: thread i holds the sequences [i * per, (i + 1) * per)
    auto cost_of = [&](int s) {
        const Span sp = span_of(s, p);
        return sp.len > 0
                   ? ((sp.len + TT - 1) / TT - sp.first / TT + kUnitCost) * p.units_per_seq : 0;
    };
    if (lane < 2) ids[2 * warp + lane] = make_int4(-1, 0, 0, 0);
    if (tid == 0) parts_used = 0;
    if (lane == 0) {
        prefetch_tensormap(&map_k);
        prefetch_tensormap(&map_v);
        for (int i = 0; i < ST; ++i) mbar_init(bars + 8 * i, 1);
        fence_mbar_init();
    }
    // ---- cursor of the tile loads
    int seq = 0, kvh = 0, chunk = 0, tile = 0, tile_begin = 0, tile_end = 0;
    int rel = 0, lim = 0;  // cost points from this warp's range start
    unsigned total = 0, range0 = 0;  // cost points of the line, and where this range starts
    // cost point at which warp w of the grid starts: total * w / nw, nw = W * gridDim.x,
    // by multiplication with ceil(2^64 / nw): exact below 2^64 / nw. Lines shorter
    // than nw go to the first warps, a point each: every CTA up to a unit's last
    // one then holds a part of it.
    auto start_of = [&](unsigned w) {
        return total < W * gridDim.x ? min(w, total)
                                     : (unsigned)__umul64hi((unsigned long long)total * w, p.inv_warps);
    };
    Span span{0, 0};
    auto enter_seq = [&](int s) {
        seq = s;
        span = span_of(s, p);
        tile_begin = span.first / TT;
        tile_end = (span.len + TT - 1) / TT;
    };
    bool fresh = true;  // next tile starts a piece
    if (p.aligned) {
        // one unit for each CTA, its tiles cut evenly over the warps
        const int s = blockIdx.x / p.units_per_seq, sub = blockIdx.x - s * p.units_per_seq;
        enter_seq(s);
        kvh = sub / p.head_chunks;
        chunk = sub - kvh * p.head_chunks;
        const int n = tile_end - tile_begin;
        tile = tile_begin + n * warp / W;
        lim = tile_begin + n * (warp + 1) / W - tile;
        __syncthreads();
    } else {
        const int per = (p.num_seqs + THREADS - 1) / THREADS;
        int mine = 0;
        for (int s = tid * per; s < min((tid + 1) * per, p.num_seqs); ++s) mine += cost_of(s);
        int inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        pre[tid] = inc - mine;
        if (lane == 31) wsum[warp] = inc;
        __syncthreads();
        // lane i: cost before warp i's threads
        const int own = lane < W ? wsum[lane] : 0;
        int before = own;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += v;
        }
        total = __shfl_sync(0xffffffffu, before, W - 1);
        before -= own;
        const unsigned wi = blockIdx.x * W + warp;
        {
            const unsigned a = range0 = start_of(wi);
            lim = (int)(start_of(wi + 1) - a);
            if (lim > 0) {
                // the sequence whose costs hold point a: the last thread whose
                // cost before it is at most a (an empty one shares its number
                // with the next)
                const int w =
                    31 - __clz(__ballot_sync(0xffffffffu, lane < W && (unsigned)before <= a));
                const unsigned at_lane = __shfl_sync(0xffffffffu, before, w) + pre[w * 32 + lane];
                const int i = 31 - __clz(__ballot_sync(0xffffffffu, at_lane <= a));
                unsigned at = a - __shfl_sync(0xffffffffu, at_lane, i);  // a's place from there
                int s = (w * 32 + i) * per;
                while (true) {
                    const unsigned cost = cost_of(s);
                    if (at < cost) break;
                    at -= cost;
                    ++s;
                }
                enter_seq(s);
                const unsigned unit_cost = tile_end - tile_begin + kUnitCost;
                // at / unit_cost: the quotient is below 2^16, so the estimate is
                // off by one at most
                int sub = (int)__fdividef((float)at, (float)unit_cost);
                int off = (int)(at - sub * unit_cost);
                if (off < 0) {
                    --sub;
                    off += unit_cost;
                } else if (off >= (int)unit_cost) {
                    ++sub;
                    off -= unit_cost;
                }
                kvh = p.head_chunks == 1 ? sub : sub / p.head_chunks;
                chunk = sub - kvh * p.head_chunks;
                // a unit's tiles sit at the end of its cost points
                const int skip = max(off - kUnitCost, 0);
                tile = tile_begin + skip;
                rel = skip + kUnitCost - off;
            }
        }
    }
    // Boxes of a tile: box_rows rows (a block or a part of one) each. Lane i
    // holds the block id of box i of the next tile, and its offset in the block.
    const int shift = p.box_shift, boxes = TT >> shift;
    const int32_t* table = p.block_tables + (long long)seq * p.max_blocks;
    int bid_next = -1, off_next = 0;
    auto fetch_bid = [&]() {
        bid_next = -1;
        const int pos = tile * TT + (lane << shift);
        // a box past the context's end reads no table
        if (rel < lim && lane < boxes && pos < span.len) {
            const int b = p.block_of(pos);
            bid_next = table[b];
            off_next = pos - b * p.block_size;
        }
    };
    const uint64_t policy = l2_policy_evict_first();

    auto load_tile = [&](int slot) {
        if (rel < lim) {
            const int pos0 = tile * TT;
            const int bid = bid_next;
            const int lo = max(span.first - pos0, 0), hi = min(span.len - pos0, TT);
            // boxes with a token in the span and a block of the pool
            const int row0 = lane << shift;
            const bool overlaps = lane < boxes && row0 < hi && row0 + (1 << shift) > lo;
            const bool on = overlaps && bid >= 0 && bid < p.num_blocks;
            if (overlaps && bid >= p.num_blocks) flag_status(TLB_STATUS_BAD_BLOCK_ID);
            const uint32_t box_mask = __ballot_sync(0xffffffffu, on);
            // first cache row of this lane's box
            const int row = on ? (bid * p.num_kv_heads + kvh) * p.block_size + off_next : 0;
            const uint32_t bar = bars + 8 * slot;
            if (lane == 0)
                mbar_arrive_expect_tx(bar, (uint32_t)__popc(box_mask) * 2u * F::kRow << shift);
            __syncwarp();
            uint32_t dst = ring + slot * F::kStage;
            for (int i = 0; i < boxes; ++i) {
                const int y = __shfl_sync(0xffffffffu, row, i);
                if (((box_mask >> i) & 1) && elect_one()) {
#pragma unroll
                    for (int c = 0; c < F::kColumns; ++c) {
                        const int x = c * (128 / F::kBytes);
                        tma_load_2d(dst + c * TT * 128, &map_k, x, y, bar, policy);
                        tma_load_2d(dst + c * TT * 128 + F::kHalfStage, &map_v, x, y, bar, policy);
                    }
                }
                dst += (F::kRow < 128 ? F::kRow : 128) << shift;
            }
            if constexpr (F::kQ8) {
                // four key scales each for the first TT / 4 lanes, value scales next
                const int tok = 4 * (lane & (TT / 4 - 1)), box = tok >> shift;
                const int srow = __shfl_sync(0xffffffffu, row, box) + tok - (box << shift);
                if (lane < TT / 2)
                    cp_async_4_zfill(smem_u32(sc) + slot * 2 * TT + lane * 4,
                                     (lane < TT / 4 ? p.key_scales : p.value_scales) + srow,
                                     (box_mask >> box) & 1);
                cp_async_commit();
            }
            const int in_group = chunk * p.unit_heads;
            int flags = (fresh ? kFirst : 0) | (tile == tile_begin ? kUnitBegin : 0) |
                        (tile + 1 == tile_end ? kUnitEnd : 0) |
                        min(p.unit_heads, p.group - in_group) << kHeadsShift |
                        (kvh * p.group + in_group) << kHead0Shift;
            const int u = seq;
            const int point = (int)range0 + rel - (tile - tile_begin);
            // every token seen: box_mask 0 stands for it
            const uint32_t seen = box_mask == (1u << boxes) - 1u && lo == 0 && hi == TT
                                      ? 0u : 1u << 31 | box_mask << 16 | hi << 8 | lo;
            // advance
            fresh = false;
            ++tile;
            ++rel;
            if (tile == tile_end) {
                fresh = true;
                rel += kUnitCost;
                if (++chunk == p.head_chunks) {
                    chunk = 0;
                    if (++kvh == p.num_kv_heads) {
                        kvh = 0;
                        if (rel < lim) {
                            int s = seq + 1;
                            while (s < p.num_seqs && cost_of(s) == 0) ++s;
                            if (s < p.num_seqs) {
                                enter_seq(s);
                                table = p.block_tables + (long long)seq * p.max_blocks;
                            } else {
                                lim = rel;
                            }
                        }
                    }
                }
                tile = tile_begin;
            }
            if (fresh || rel >= lim) flags |= kLast;
            if (lane == 0) {
                hdr[slot] = make_int4((int)seen, pos0, u, flags);
                hdr_point[slot] = point;
            }
            fetch_bid();
        } else {
            if (lane == 0) hdr[slot] = make_int4(0, 0, -1, 0);
            if constexpr (F::kQ8) cp_async_commit();
        }
    };
    // whether token t of a tile that is not all seen is
    auto is_seen = [&](uint32_t seen, int t) {
        return t >= (int)(seen & 255) && t < (int)((seen >> 8) & 255) &&
               ((seen >> 16) >> (t >> shift)) & 1;
    };

    fetch_bid();
    grid_dependency_wait();
    grid_launch_dependents();

    // the CTAs (from this one down, from this one up) whose ranges hold cost
    // points x0 <= x1 of a unit that this CTA has a part of; 32 CTAs a step
    auto first_cta = [&](unsigned x0) {
        for (int c = blockIdx.x;; c -= 32) {
            const int mine = c - lane;
            const uint32_t at = __ballot_sync(0xffffffffu, mine <= 0 || start_of(mine * W) <= x0);
            if (at) return c - (__ffs(at) - 1);
        }
    };
    auto final_cta = [&](unsigned x1) {
        for (int c = blockIdx.x;; c += 32) {
            const int mine = c + lane;
            const uint32_t at = __ballot_sync(0xffffffffu, mine >= (int)gridDim.x - 1 ||
                                                               start_of((mine + 1) * W) > x1);
            if (at) return c + __ffs(at) - 1;
        }
    };

    // ---- state of the piece in flight
    uint32_t qf[NT][F::kTiles][2];
    float o[NT][F::kTiles][4];
    float m[NT][2], mv[NT][2], l[NT][2], qs[NT][2], slope[NT][2];
    int piece_flags = 0, last_pos = 0;
    int row = 0, heads = 0;  // output row of the unit's first head, its heads
    const ScoreMod mod{p.cap_log2, p.inv_cap, p.alibi_slopes != nullptr};
    QT* out = reinterpret_cast<QT*>(p.out);
    float4* part_a = p.warp_partials + ((long long)blockIdx.x * W + warp) * F::kFrags;

    int slot = 0;
    uint32_t parity = 0;
    bool failed = false;
    int ahead = 0;  // tiles loaded before the first is used
    while (true) {
        load_tile(ahead < ST - 1 ? ahead : slot == 0 ? ST - 1 : slot - 1);
        if (ahead < ST - 1) {
            ++ahead;
            continue;
        }
        __syncwarp();
        const int4 h = hdr[slot];
        if (h.z < 0) break;
        if (h.w & kFirst) {
            piece_flags = h.w & (kUnitBegin | kHeadsMask);
            heads = (h.w & kHeadsMask) >> kHeadsShift;
            const int head0 = h.w >> kHead0Shift;
            row = h.z * p.num_heads + head0;
            last_pos = min(max(p.seq_lens[h.z], 0), p.max_tokens) - 1;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int head = nt * 8 + g;
                const bool there = head < heads;
                const QT* q = reinterpret_cast<const QT*>(p.query) +
                              h.z * p.query_stride + (long long)(head0 + head) * D;
                float scale_q = p.cap_log2 > 0.f ? p.scale : p.scale * kLog2e;
                if constexpr (F::kQ8) {
                    uint2 raw[F::kTiles];
                    uint32_t top = 0;
#pragma unroll
                    for (int i = 0; i < F::kTiles; ++i) {
                        raw[i] = there ? *reinterpret_cast<const uint2*>(q + 16 * i + 4 * t4)
                                       : make_uint2(0, 0);
                        float a, b;
                        unpack2<QT>(raw[i].x, a, b);
                        top = max(top, max(finite_abs_bits(a), finite_abs_bits(b)));
                        unpack2<QT>(raw[i].y, a, b);
                        top = max(top, max(finite_abs_bits(a), finite_abs_bits(b)));
                    }
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    // 2^n that brings the head's largest element into [2^14, 2^15):
                    // n >= 14 - 127; at most 110, so that 2^-n leaves room for the scale
                    const int n = min(14 - ((int)(top >> 23) - 127), 110);
                    const float up = __uint_as_float((uint32_t)(n + 127) << 23);
                    scale_q *= __uint_as_float((uint32_t)(127 - n) << 23);
#pragma unroll
                    for (int i = 0; i < F::kTiles; ++i) {
                        float a, b;
                        unpack2<QT>(raw[i].x, a, b);
                        qf[nt][i][0] = pack2<__half>(mul_keep(a, up), mul_keep(b, up));
                        unpack2<QT>(raw[i].y, a, b);
                        qf[nt][i][1] = pack2<__half>(mul_keep(a, up), mul_keep(b, up));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < F::kTiles; ++i) {
                        qf[nt][i][0] =
                            there ? *reinterpret_cast<const uint32_t*>(q + 16 * i + 2 * t4) : 0u;
                        qf[nt][i][1] =
                            there ? *reinterpret_cast<const uint32_t*>(q + 16 * i + 8 + 2 * t4) : 0u;
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    // this lane's score columns are heads 2 t4 + e
                    qs[nt][e] = __shfl_sync(0xffffffffu, scale_q, (2 * t4 + e) * 4);
                    const int hh = nt * 8 + 2 * t4 + e;
                    slope[nt][e] = mod.alibi && hh < heads
                                       ? p.alibi_slopes[head0 + hh] * kLog2e : 0.f;
                    m[nt][e] = mv[nt][e] = -INFINITY;
                    l[nt][e] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < F::kTiles; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
            }
        }
        const uint32_t kbase = ring + slot * F::kStage, vbase = kbase + F::kHalfStage;
        // the tile's rows (bounded: see TLB_STATUS_WAIT_TIMEOUT) and scales
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(bars + 8 * slot, parity, p.wait_limit))) {
            failed = true;
            break;
        }
        if constexpr (F::kQ8) {
            cp_async_wait<ST - 1>();
            __syncwarp();
        }
        const uint32_t seen = (uint32_t)h.x;
        const bool full = seen == 0;
        if (!full) {
            // value rows that are not seen may hold anything (0 * NaN): zeros
            for (int i = lane; i < TT * CH; i += 32)
                if (!is_seen(seen, i / CH))
                    *reinterpret_cast<uint4*>(smem + (vbase - smem_u32(smem)) +
                                              tile_offset<CH, TT>(i / CH, i % CH)) =
                        make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();  // before a later copy into this slot
            __syncwarp();
        }

        // ---- S^T = K Q^T
        float s[NT][MT_TILES][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int mt = 0; mt < MT_TILES; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[nt][mt][e] = 0.f;
        {
            const int lr = (lane & 7) + ((lane >> 3) & 1) * 8, lc = lane >> 4;
            if constexpr (F::kQ8) {
#pragma unroll
                for (int c = 0; c < F::kTiles; c += 2)
#pragma unroll
                    for (int mt = 0; mt < MT_TILES; ++mt) {
                        uint32_t r0, r1, r2, r3;
                        ldsm_x4(kbase + tile_offset<CH, TT>(mt * 16 + lr, c + lc), r0, r1, r2, r3);
                        uint32_t a[4], b[4];
                        widen_row<CT>(r0, a[0], a[2]);
                        widen_row<CT>(r1, a[1], a[3]);
                        widen_row<CT>(r2, b[0], b[2]);
                        widen_row<CT>(r3, b[1], b[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816<MT>(s[nt][mt], a, qf[nt][c][0], qf[nt][c][1]);
                            mma16816<MT>(s[nt][mt], b, qf[nt][c + 1][0], qf[nt][c + 1][1]);
                        }
                    }
            } else {
#pragma unroll
                for (int c = 0; c < F::kTiles; ++c)
#pragma unroll
                    for (int mt = 0; mt < MT_TILES; ++mt) {
                        uint32_t a[4];
                        ldsm_x4(kbase + tile_offset<CH, TT>(mt * 16 + lr, 2 * c + lc), a[0], a[1], a[2],
                                a[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma16816<MT>(s[nt][mt], a, qf[nt][c][0], qf[nt][c][1]);
                    }
            }
        }

        // ---- scores in log2 units
        float ev[MT_TILES][2];
#pragma unroll
        for (int mt = 0; mt < MT_TILES; ++mt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int tok = mt * 16 + r * 8 + g;
                float ks = 1.f;
                ev[mt][r] = 0.f;
                if constexpr (F::kQ8) {
                    ks = scale_value(sc[slot * 2 * TT + tok]);
                    // byte - 127, through the mantissa of 2^23
                    ev[mt][r] = __uint_as_float(0x4b000000u | sc[slot * 2 * TT + TT + tok]) - 8388735.f;
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        // the two scales first: the product of the stored
                        // values is of moderate size, so nothing overflows
                        // that the score itself does not
                        s[nt][mt][2 * r + e] *= F::kQ8 ? ks * qs[nt][e] : qs[nt][e];
            }
        if (p.cap_log2 > 0.f) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int mt = 0; mt < MT_TILES; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nt][mt][e] = mod.cap(s[nt][mt][e]);
        }
        if (mod.alibi) {
            const float back = (float)(h.y + g - last_pos);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int mt = 0; mt < MT_TILES; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[nt][mt][e] = fmaf(slope[nt][e & 1], back + (float)(mt * 16 + (e >> 1) * 8),
                                            s[nt][mt][e]);
        }
        if (!full) {
#pragma unroll
            for (int mt = 0; mt < MT_TILES; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool on = is_seen(seen, mt * 16 + (e >> 1) * 8 + g);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        s[nt][mt][e] = on ? s[nt][mt][e] : -INFINITY;
                }
        }
        // ---- weights
        bool over = false;
        float cm[NT][2], cv[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float a = -INFINITY, b = -INFINITY;
#pragma unroll
                for (int mt = 0; mt < MT_TILES; ++mt)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        a = fmaxf(a, s[nt][mt][2 * r + e]);
                        if constexpr (F::kQ8) b = fmaxf(b, s[nt][mt][2 * r + e] + ev[mt][r]);
                    }
                cm[nt][e] = a;
                cv[nt][e] = b;
                over |= a > m[nt][e] + kLazy;
                if constexpr (F::kQ8) over |= b > mv[nt][e] + kLazy;
            }
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float a = cm[nt][e], b = cv[nt][e];
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) {
                        a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, d));
                        if constexpr (F::kQ8) b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, d));
                    }
                    const float M = fmaxf(m[nt][e], a);
                    const float al = piece_weight(m[nt][e], M);
                    l[nt][e] *= al;
                    m[nt][e] = M;
                    float av = al;
                    if constexpr (F::kQ8) {
                        const float MV = fmaxf(mv[nt][e], b);
                        av = piece_weight(mv[nt][e], MV);
                        mv[nt][e] = MV;
                    }
#pragma unroll
                    for (int i = 0; i < F::kTiles; ++i) {
                        o[nt][i][e] *= av;
                        o[nt][i][e + 2] *= av;
                    }
                }
        }
        uint32_t ph[NT][MT_TILES][2], pl[NT][MT_TILES][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float ref[2], refv[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                ref[e] = m[nt][e] == -INFINITY ? 0.f : m[nt][e];
                refv[e] = mv[nt][e] == -INFINITY ? 0.f : mv[nt][e] - F::kLift;
            }
#pragma unroll
            for (int mt = 0; mt < MT_TILES; ++mt)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float w[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float x = s[nt][mt][2 * r + e];
                        const float pr = ex2(x - ref[e]);
                        l[nt][e] += pr;
                        w[e] = F::kQ8 ? ex2(x + ev[mt][r] - refv[e]) : pr * (float)(1 << F::kLift);
                    }
                    const uint32_t hi = pack2<MT>(w[0], w[1]);
                    ph[nt][mt][r] = movmatrix_trans(hi);
                    if constexpr (F::kSplit) {
                        float h0, h1;
                        unpack2<MT>(hi, h0, h1);
                        pl[nt][mt][r] = movmatrix_trans(pack2<MT>(w[0] - h0, w[1] - h1));
                    }
                }
        }

        // ---- O^T += V^T P^T
        {
            const int lr = (lane & 7) + ((lane >> 3) & 1) * 8, lc = lane >> 4;
#pragma unroll
            for (int mt = 0; mt < MT_TILES; ++mt)
                if constexpr (F::kQ8) {
#pragma unroll
                    for (int c = 0; c < F::kTiles; c += 2) {
                        uint32_t r0, r1, r2, r3;
                        ldsm_x4_trans(vbase + tile_offset<CH, TT>(mt * 16 + lr, c + lc), r0, r1, r2, r3);
                        uint32_t a[4], b[4];
                        widen_col<CT>(r0, a[0], a[1]);
                        widen_col<CT>(r1, a[2], a[3]);
                        widen_col<CT>(r2, b[0], b[1]);
                        widen_col<CT>(r3, b[2], b[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816<MT>(o[nt][c], a, ph[nt][mt][0], ph[nt][mt][1]);
                            mma16816<MT>(o[nt][c + 1], b, ph[nt][mt][0], ph[nt][mt][1]);
                            if constexpr (F::kSplit) {
                                mma16816<MT>(o[nt][c], a, pl[nt][mt][0], pl[nt][mt][1]);
                                mma16816<MT>(o[nt][c + 1], b, pl[nt][mt][0], pl[nt][mt][1]);
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < F::kTiles; ++c) {
                        // (tokens 0-7, dims 0-7), (tokens 8-15, dims 0-7), then dims 8-15
                        uint32_t a[4];
                        ldsm_x4_trans(vbase + tile_offset<CH, TT>(mt * 16 + lr, 2 * c + lc), a[0], a[2],
                                      a[1], a[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816<MT>(o[nt][c], a, ph[nt][mt][0], ph[nt][mt][1]);
                            if constexpr (F::kSplit)
                                mma16816<MT>(o[nt][c], a, pl[nt][mt][0], pl[nt][mt][1]);
                        }
                    }
                }
        }

        if (h.w & kLast) {
            piece_flags |= h.w & kUnitEnd;
            const bool whole = (piece_flags & ~kHeadsMask) == (kUnitBegin | kUnitEnd);
            // the last piece of the range stays in shared memory (the ring is
            // free: no tile follows), an earlier one goes to the workspace
            const bool end = hdr[slot + 1 == ST ? 0 : slot + 1].z < 0;
            const int entry = 2 * warp + (end ? 1 : 0);
            int part = 0;
            float4* dst = reinterpret_cast<float4*>(smem + warp * F::kRingBytes);
            if (!end && !whole) {
                if (lane == 0) part = atomicAdd(&parts_used, 1);
                part = __shfl_sync(0xffffffffu, part, 0);
                dst = part < F::kParts
                          ? reinterpret_cast<float4*>(smem + F::kPartOff + part * F::kPartBytes)
                          : part_a;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float inv[2], fac[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float sum = l[nt][e];
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                    // weights relative to mv, lifted -> relative to m
                    fac[e] = !F::kQ8                  ? 1.f / (1 << F::kLift)
                             : mv[nt][e] == -INFINITY ? 0.f
                                                      : ex2(mv[nt][e] - m[nt][e] - F::kLift);
                    inv[e] = inverse(sum);
                    if (!whole && g == 0)
                        ml[entry * G + nt * 8 + 2 * t4 + e] = make_float2(m[nt][e], sum);
                }
#pragma unroll
                for (int i = 0; i < F::kTiles; ++i) {
                    const float4 v = make_float4(o[nt][i][0] * fac[0], o[nt][i][1] * fac[1],
                                                 o[nt][i][2] * fac[0], o[nt][i][3] * fac[1]);
                    if (whole)
                        write_frag<QT, F::kQ8, D>(p.out, row, heads, nt, i, lane, v, inv[0], inv[1]);
                    else
                        dst[(nt * F::kTiles + i) * 32 + lane] = v;
                }
            }
            if (!whole && lane == 0) {
                ids[entry] = make_int4(row, piece_flags, part, 0);
                const Span sp = span_of(h.z, p);
                points[entry] = make_int2(hdr_point[slot], (sp.len + TT - 1) / TT - sp.first / TT);
            }
        }
        __syncwarp();
        if (++slot == ST) {
            slot = 0;
            parity ^= 1;
        }
    }
    if (failed) {
        // a copy did not arrive in time: report it, give the copies in flight
        // (this slot's and the following ones') the same time to land, and stop
        if (lane == 0) {
            flag_status(TLB_STATUS_WAIT_TIMEOUT);
            ids[2 * warp] = ids[2 * warp + 1] = make_int4(-1, 0, 0, 0);
        }
        for (int i = 0; i < ST; ++i) {
            if (hdr[slot].z >= 0) mbar_wait_bounded(bars + 8 * slot, parity, kWaitLimit);
            if (++slot == ST) {
                slot = 0;
                parity ^= 1;
            }
        }
    }
    if constexpr (F::kQ8) cp_async_wait<0>();
    __syncthreads();

    // ---- join the CTA's partials, in range order. Lane e of every warp holds
    // entry e: the piece that ended inside warp e / 2's range (even e) or was
    // the last of its range (odd e).
    const int4 mine = lane < 2 * W ? ids[lane] : make_int4(-1, 0, 0, 0);
    const uint32_t run = __match_any_sync(0xffffffffu, mine.x);  // entries of the same unit
    const uint32_t there = __ballot_sync(0xffffffffu, mine.x >= 0);
    if (there) {
        // weights of the entries, a warp for each head
        if (mine.x >= 0)
            for (int h = warp; h < G; h += W) {
                const float2 v = ml[lane * G + h];
                const float M = max_of(run, v.x);
                const float w = piece_weight(v.x, M);
                wl[lane * G + h] = make_float2(w, w * v.y);
                ml[lane * G + h].x = M;
            }
        if (warp >= W - 2) {
            // units that other CTAs share, one for each of these warps: [0] begins
            // before this CTA, [1] ends after it. (output row or -1, heads, CTA of
            // the unit's first tile, CTAs that hold a part)
            const int side = warp - (W - 2);
            const int e1 = side ? 31 - __clz(there) : __ffs(there) - 1;
            const uint32_t k = __shfl_sync(0xffffffffu, run, e1);
            const int e0 = __ffs(k) - 1;
            const int begin = __shfl_sync(0xffffffffu, mine.y, e0);
            const int end = __shfl_sync(0xffffffffu, mine.y, 31 - __clz(k));
            int4 unit = make_int4(-1, (begin & kHeadsMask) >> kHeadsShift, 0, 0);
            if (side ? (begin & kUnitBegin) && !(end & kUnitEnd) : !(begin & kUnitBegin)) {
                const int2 pt = points[e0];
                unit.x = __shfl_sync(0xffffffffu, mine.x, e0);
                unit.z = first_cta(pt.x);
                unit.w = final_cta(pt.x + pt.y - 1) - unit.z + 1;
            }
            if (lane == 0) shared_unit[side] = unit;
        }
        __syncthreads();
        // byte offset of the entry's partial in shared memory, -1: workspace
        const int from = (lane & 1) ? (lane >> 1) * F::kRingBytes
                         : mine.z < F::kParts ? F::kPartOff + mine.z * F::kPartBytes : -1;
        // a warp for each 32 fragments of each unit
        constexpr int FG = F::kFrags / 32;
#pragma unroll 1
        for (int task = warp;; task += W) {
            int e0 = 0;
            uint32_t rest = there, entries = 0;
            for (int i = task / FG;; --i) {
                if (!rest) break;
                e0 = __ffs(rest) - 1;
                entries = __shfl_sync(0xffffffffu, run, e0);
                if (i == 0) break;
                rest &= ~entries;
            }
            if (!rest) break;
            // the first entry says whether the unit begins here, the last
            // whether it ends
            const int flags = __shfl_sync(0xffffffffu, mine.y, e0) |
                              __shfl_sync(0xffffffffu, mine.y, 31 - __clz(entries));
            const int u = __shfl_sync(0xffffffffu, mine.x, e0);
            const int f = task % FG * 32 + lane, nt = f / (F::kTiles * 32);
            const int i = (f >> 5) % F::kTiles, h0 = nt * 8 + 2 * (lane & 3);
            float L0 = 0.f, L1 = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f), v, w;
            auto fetch = [&](int e) {
                const int off = __shfl_sync(0xffffffffu, from, e);
                v = off >= 0 ? *reinterpret_cast<const float4*>(smem + off + 16 * f)
                             : p.warp_partials[((long long)blockIdx.x * W + (e >> 1)) * F::kFrags + f];
                w = *reinterpret_cast<const float4*>(wl + e * G + h0);
            };
            fetch(e0);
#pragma unroll 1
            for (uint32_t k = entries & (entries - 1);; k &= k - 1) {
                const float4 v0 = v, w0 = w;
                if (k) fetch(__ffs(k) - 1);
                acc.x = fmaf(w0.x, v0.x, acc.x);
                acc.y = fmaf(w0.z, v0.y, acc.y);
                acc.z = fmaf(w0.x, v0.z, acc.z);
                acc.w = fmaf(w0.z, v0.w, acc.w);
                L0 += w0.y;
                L1 += w0.w;
                if (!k) break;
            }
            if ((flags & ~kHeadsMask) == (kUnitBegin | kUnitEnd)) {
                write_frag<QT, F::kQ8, D>(p.out, u, (flags & kHeadsMask) >> kHeadsShift, nt, i, lane,
                                          acc, inverse(L0), inverse(L1));
            } else {
                const int at = 2 * blockIdx.x + ((flags & kUnitBegin) ? 1 : 0);
                p.cta_partials[(long long)at * F::kFrags + f] = acc;
                if (i == 0 && lane < 4)
                    *reinterpret_cast<float4*>(p.cta_ml + at * G + h0) =
                        make_float4(ml[e0 * G + h0].x, L0, ml[e0 * G + h0 + 1].x, L1);
            }
        }
    }
    // ---- join units across CTAs: the last CTA to publish its partial of a unit
    // sums all of them, in range order whichever CTA it is. The counters are
    // zero between calls.
    if (there && (shared_unit[0].x >= 0 || shared_unit[1].x >= 0)) {
        __syncthreads();
        if (lane == 0 && warp < 2) {
            const int4 unit = shared_unit[warp];
            // releases what the barrier has made this thread see: all the CTA's
            // stores of its partial
            last_cta[warp] = unit.x >= 0 && atomic_inc_acq_rel(p.counters + unit.z, unit.w - 1) ==
                                                (unsigned)unit.w - 1;
        }
        __syncthreads();
#pragma unroll 1
        for (int sd = 0; sd < 2; ++sd) {
            if (!last_cta[sd]) continue;
            const int4 unit = shared_unit[sd];
            const int c0 = unit.z, n = unit.w;
#pragma unroll 1
            for (int f = tid; f < F::kFrags; f += THREADS) {
                const int nt = f / (F::kTiles * 32), i = (f >> 5) % F::kTiles;
                const int h0 = nt * 8 + 2 * (lane & 3);
                float M0 = -INFINITY, M1 = -INFINITY, L0 = 0.f, L1 = 0.f;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                float4 v, w;
                auto fetch = [&](int k) {
                    const int at = k == 0 ? 2 * c0 + 1 : 2 * (c0 + k);
                    v = __ldcg(p.cta_partials + (long long)at * F::kFrags + f);
                    w = __ldcg(reinterpret_cast<const float4*>(p.cta_ml + at * G + h0));
                };
                auto add = [&](const float4& x, const float4& y) {
                    const float N0 = fmaxf(M0, y.x), N1 = fmaxf(M1, y.z);
                    const float a0 = piece_weight(M0, N0), a1 = piece_weight(M1, N1);
                    const float b0 = piece_weight(y.x, N0), b1 = piece_weight(y.z, N1);
                    L0 = L0 * a0 + y.y * b0;
                    L1 = L1 * a1 + y.w * b1;
                    acc.x = acc.x * a0 + x.x * b0;
                    acc.y = acc.y * a1 + x.y * b1;
                    acc.z = acc.z * a0 + x.z * b0;
                    acc.w = acc.w * a1 + x.w * b1;
                    M0 = N0;
                    M1 = N1;
                };
                // four partials' loads in flight
                int k = 0;
                while (k < n) {
                    fetch(k);
                    const float4 v0 = v, w0 = w;
                    fetch(min(k + 1, n - 1));
                    const float4 v1 = v, w1 = w;
                    fetch(min(k + 2, n - 1));
                    const float4 v2 = v, w2 = w;
                    fetch(min(k + 3, n - 1));
                    float4 x = v0, y = w0;
#pragma unroll 1
                    for (int j = 0;; ++j) {
                        add(x, y);
                        if (++k == n || j == 3) break;
                        x = j == 0 ? v1 : j == 1 ? v2 : v;
                        y = j == 0 ? w1 : j == 1 ? w2 : w;
                    }
                }
                write_frag<QT, F::kQ8, D>(p.out, unit.x, unit.y, nt, i, lane, acc, inverse(L0),
                                          inverse(L1));
            }
        }
    }
    // ---- sequences with no token: zeros
    for (int s = blockIdx.x; s < p.num_seqs; s += gridDim.x) {
        if (p.seq_lens[s] > p.max_tokens && tid == 0) flag_status(TLB_STATUS_SEQ_TOO_LONG);
        if (p.seq_lens[s] <= 0)
            for (int i = tid; i < p.num_heads * D; i += THREADS)
                out[(long long)s * p.num_heads * D + i] = Elem<QT>::from_f(0.f);
    }
}

template <typename QT, typename CT, int D, int NT>
cudaError_t launch_fast(const Params& p, const CUtensorMap& map_k, const CUtensorMap& map_v,
                        int ctas, cudaStream_t st) {
    using F = Cfg<QT, CT, D, NT>;
    auto kern = scored_attention_kernel<QT, CT, D, NT>;
    // the attribute is the kernel's on one device: set once for each
    static std::atomic<unsigned long long> set{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (!(set.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem);
        if (e != cudaSuccess) return e;
        set.fetch_or(bit, std::memory_order_relaxed);
    }
    return launch_early(kern, ctas, F::kThreads, F::kSmem, st, map_k, map_v, p);
}

template <typename QT, typename CT>
cudaError_t launch_fast_shape(const Params& p, const CUtensorMap& map_k, const CUtensorMap& map_v,
                              int ctas, cudaStream_t st) {
    if (p.head_dim == 128)
        return p.unit_heads <= 8 ? launch_fast<QT, CT, 128, 1>(p, map_k, map_v, ctas, st)
                                 : launch_fast<QT, CT, 128, 2>(p, map_k, map_v, ctas, st);
    return p.unit_heads <= 8 ? launch_fast<QT, CT, 64, 1>(p, map_k, map_v, ctas, st)
                             : launch_fast<QT, CT, 64, 2>(p, map_k, map_v, ctas, st);
}

}  // namespace scored
}  // namespace tlb
