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
//  * A tile is kTT tokens of one (sequence, kv head): 32 rows of 8-bit values
//    or 16 of 16-bit ones, 8 KB of keys and values at head_dim 128. The tiles
//    of all units, with a charge of kUnitCost tiles for starting a unit, form
//    one line, cut evenly over all warps of the grid (one CTA of 8 warps per
//    SM). Each warp streams its contiguous part through a ring of its own
//    (24 KB, cp.async) and never waits for another warp, so units of any mix
//    of lengths keep every SM busy and a short sequence costs one warp one tile.
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
//  * A unit cut by range ends leaves fp32 partials: warps of one CTA join
//    theirs in shared memory, CTAs through the workspace in a second small
//    kernel (programmatic launch). The order of every sum is fixed: results
//    are the same bits on every run. Nothing in the workspace outlives a call.
#pragma once

#include <type_traits>

#include "kernels.h"
#include "quant.cuh"

namespace tlb {
namespace scored {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kRingBytes = 24576;  // per warp
constexpr int kUnitCost = 1;       // tiles charged for starting a unit
constexpr float kLazy = 8.f;       // log2 of how far a score may pass the reference
constexpr float kLog2e = 1.4426950408889634f;

// Flags of a tile and, or-ed over a piece, of a partial.
constexpr int kFirst = 1;      // first tile of a piece in this warp's range
constexpr int kLast = 2;       // last tile of a piece in this warp's range
constexpr int kUnitBegin = 4;  // first tile of its unit
constexpr int kUnitEnd = 8;    // last tile of its unit

template <typename QT, typename CT, int D, int NT>
struct Cfg {
    static constexpr int kBytes = sizeof(CT);
    static constexpr bool kQ8 = kBytes == 1;
    static constexpr int kTT = kQ8 ? 32 : 16;       // tokens per tile
    static constexpr int kRow = D * kBytes;         // bytes per row
    static constexpr int kChunks = kRow / 16;
    static constexpr int kHalfStage = kTT * kRow;   // K (or V) bytes of a stage
    static constexpr int kStage = 2 * kHalfStage;
    static constexpr int kStages = kRingBytes / kStage;
    static constexpr int kGroup = 8 * NT;           // heads per unit
    static constexpr int kTiles = D / 16;           // dim tiles
    // float4 fragments of a partial: [nt][dim tile][lane]
    static constexpr int kFrags = NT * kTiles * 32;
    // P is carried as a hi + lo pair where one 16-bit rounding would show in
    // the output: bf16 weights (8 bits) always, fp16 weights with fp16 outputs
    static constexpr bool kSplit = !(kQ8 && std::is_same<QT, __nv_bfloat16>::value);
    // weights are held 2^kLift above the reference where they are fp16
    static constexpr int kLift = kQ8 || std::is_same<QT, __half>::value ? 7 : 0;
    // shared memory: rings, tile headers, scale bytes, partial (m, l), ids, prefix
    static constexpr int kHdrOff = kWarps * kRingBytes;
    static constexpr int kScaleOff = kHdrOff + kWarps * kStages * 16;
    static constexpr int kMlOff = kScaleOff + (kQ8 ? kWarps * kStages * 64 : 0);
    static constexpr int kUnitOff = kMlOff + 2 * kWarps * kGroup * 8;
    static constexpr int kPrefixOff = kUnitOff + 2 * kWarps * 8;
    static constexpr int kSmem = kPrefixOff + (kThreads + 1) * 8 + 64;
};

// Byte offset of 16-byte chunk c of row r in a tile: rows of a 128-byte line
// are xor-swizzled so that ldmatrix's eight rows of one chunk hit all banks.
template <int CH>
__device__ __forceinline__ uint32_t tile_offset(int r, int c) {
    if constexpr (CH == 4) {  // two 64-byte rows per line
        const int line = r >> 1;
        return (uint32_t)(line * 128 + (((((r & 1) << 2) | c) ^ (line & 3)) << 4));
    } else {
        return (uint32_t)(r * CH * 16 + ((c ^ (r & 7)) << 4));
    }
}

__device__ __forceinline__ void cp_async_16_zfill(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(src)), "r"(on ? 16 : 0)
                 : "memory");
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
    a = e4m3x2_to_half2(x);
    b = e4m3x2_to_half2(x >> 16);
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

// Unit u: sequence, kv head and chunk of its query heads.
struct Unit {
    int s, kvh, head0, heads;
};
__device__ __forceinline__ Unit unit_of(int u, const Params& p) {
    Unit r;
    r.s = u / p.units_per_seq;
    const int sub = u - r.s * p.units_per_seq;
    r.kvh = sub / p.head_chunks;
    const int hc = sub - r.kvh * p.head_chunks;
    const int first = hc * p.unit_heads;
    r.heads = min(p.unit_heads, p.group - first);
    r.head0 = r.kvh * p.group + first;
    return r;
}

// One fragment (dim tile i, lane) of a unit's output: (v.x, v.y) are heads
// 2t, 2t + 1 of one dim, (v.z, v.w) of another: with 8-bit values the next
// dim (dims 2g, 2g + 1 of the tile), otherwise dims g and g + 8.
template <typename QT, bool Q8>
__device__ __forceinline__ void write_frag(QT* out, const Params& p, const Unit& u, int D, int nt,
                                           int i, int lane, float4 v, float inv0, float inv1) {
    const int g = lane >> 2, h = nt * 8 + 2 * (lane & 3);
    const int d0 = 16 * i + (Q8 ? 2 * g : g), d1 = Q8 ? d0 + 1 : d0 + 8;
    QT* o = out + ((long long)u.s * p.num_heads + u.head0 + h) * D;
    if (h < u.heads) {
        o[d0] = Elem<QT>::from_f(v.x * inv0);
        o[d1] = Elem<QT>::from_f(v.z * inv0);
    }
    if (h + 1 < u.heads) {
        o[D + d0] = Elem<QT>::from_f(v.y * inv1);
        o[D + d1] = Elem<QT>::from_f(v.w * inv1);
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
__global__ void __launch_bounds__(kThreads, 1) scored_attention_kernel(const Params p) {
    using F = Cfg<QT, CT, D, NT>;
    // element type of the matrix products: 8-bit values become fp16
    using MT = typename std::conditional<F::kQ8, __half, QT>::type;
    constexpr int TT = F::kTT, CH = F::kChunks, ST = F::kStages, G = F::kGroup;
    constexpr int MT_TILES = TT / 16;  // 16-token tiles of a stage
    extern __shared__ __align__(1024) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t4 = lane & 3;
    int4* hdr = reinterpret_cast<int4*>(smem + F::kHdrOff) + warp * ST;
    uint8_t* sc = smem + F::kScaleOff + warp * ST * 64;
    float2* ml = reinterpret_cast<float2*>(smem + F::kMlOff);       // [2 W][G] (m, l)
    int2* ids = reinterpret_cast<int2*>(smem + F::kUnitOff);        // [2 W] (unit, flags)
    long long* pre = reinterpret_cast<long long*>(smem + F::kPrefixOff);
    __shared__ long long wsum[kWarps];

    grid_launch_dependents();
    // ---- cost line: thread i holds the sequences [i * per, (i + 1) * per)
    auto tiles_of = [&](int s) {
        const Span sp = span_of(s, p);
        return sp.len > 0 ? (sp.len + TT - 1) / TT - sp.first / TT : 0;
    };
    const int per = (p.num_seqs + kThreads - 1) / kThreads;
    {
        long long mine = 0;
        for (int s = tid * per; s < min((tid + 1) * per, p.num_seqs); ++s) {
            const int n = tiles_of(s);
            if (n > 0) mine += (long long)(n + kUnitCost) * p.units_per_seq;
        }
        long long inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) wsum[warp] = inc;
        __syncthreads();
        long long before = 0;
        for (int w = 0; w < warp; ++w) before += wsum[w];
        pre[tid] = before + inc - mine;
        if (tid == kThreads - 1) pre[kThreads] = before + inc;
        if (tid < 2 * kWarps) ids[tid] = make_int2(-1, 0);
        __syncthreads();
    }
    const long long total = pre[kThreads];
    // CTAs that take part: at least kMinTiles tiles' cost per warp
    const long long want = (total + kWarps * p.min_cost - 1) / (kWarps * p.min_cost);
    const long long nw = (long long)kWarps * max(1ll, min((long long)gridDim.x, want));
    const long long wi = (long long)blockIdx.x * kWarps + warp;

    // ---- cursor of the tile loads
    int seq = 0, sub = 0, tile = 0, tile_begin = 0, tile_end = 0;
    int rel = 0, lim = 0;  // cost points from this warp's range start
    Span span{0, 0};
    auto enter_seq = [&](int s) {
        seq = s;
        span = span_of(s, p);
        tile_begin = span.first / TT;
        tile_end = (span.len + TT - 1) / TT;
    };
    bool fresh = true;  // next tile starts a piece
    if (wi < nw) {
        const long long a = total * wi / nw, b = total * (wi + 1) / nw;
        lim = (int)(b - a);
        if (lim > 0) {
            // the sequence whose costs hold point a
            int lo = 0, hi = kThreads;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (pre[mid] <= a) lo = mid; else hi = mid;
            }
            long long at = pre[lo];
            int s = lo * per;
            long long cost;
            while (true) {
                const int n = tiles_of(s);
                cost = n > 0 ? (long long)(n + kUnitCost) * p.units_per_seq : 0;
                if (a < at + cost) break;
                at += cost;
                ++s;
            }
            enter_seq(s);
            const int unit_cost = tile_end - tile_begin + kUnitCost;
            sub = (int)((a - at) / unit_cost);
            const int off = (int)((a - at) - (long long)sub * unit_cost);
            // a unit's tiles sit at the end of its cost points
            const int skip = max(off - kUnitCost, 0);
            tile = tile_begin + skip;
            rel = skip + kUnitCost - off;
        }
    }
    int bid_next = -1;
    auto fetch_bid = [&]() {
        // this lane's token of the next tile (tokens of its group of four that
        // are all outside the context read no table)
        bid_next = -1;
        if (rel < lim) {
            const int pos = tile * TT + (lane & (TT - 1));
            if ((pos & ~3) < span.len)
                bid_next = p.block_tables[(long long)seq * p.max_blocks + p.block_of(pos)];
        }
    };
    const unsigned char* kc = reinterpret_cast<const unsigned char*>(p.key_cache);
    const unsigned char* vc = reinterpret_cast<const unsigned char*>(p.value_cache);
    const uint32_t ring = smem_u32(smem) + warp * kRingBytes;

    auto load_tile = [&](int slot) {
        if (rel < lim) {
            const int r0 = lane & (TT - 1);
            const int pos = tile * TT + r0;
            const int bid = bid_next;
            const bool in_pool = bid >= 0 && bid < p.num_blocks;
            const bool in_span = pos >= span.first && pos < span.len;
            if (in_span && bid >= p.num_blocks) flag_status(TLB_STATUS_BAD_BLOCK_ID);
            const int kvh = sub / p.head_chunks;
            const uint32_t row = in_pool ? ((uint32_t)bid * p.num_kv_heads + kvh) * p.block_size +
                                               (pos - p.block_of(pos) * p.block_size)
                                         : 0u;
            uint32_t mask = __ballot_sync(0xffffffffu, in_pool && in_span);
            if constexpr (TT == 16) mask &= 0xffffu;
            const uint32_t base = ring + slot * F::kStage;
            constexpr int RPI = 32 / CH;  // rows per instruction
            const int cc = lane & (CH - 1);
#pragma unroll
            for (int i = 0; i < TT / RPI; ++i) {
                const int r = i * RPI + lane / CH;
                const uint64_t off = (uint64_t)__shfl_sync(0xffffffffu, row, r) * F::kRow + cc * 16;
                const bool on = (mask >> r) & 1;
                const uint32_t dst = base + tile_offset<CH>(r, cc);
                cp_async_16_zfill(dst, kc + off, on);
                cp_async_16_zfill(dst + F::kHalfStage, vc + off, on);
            }
            if constexpr (F::kQ8) {
                // lanes 0-7: four key scales each, lanes 8-15: value scales
                const uint32_t srow = __shfl_sync(0xffffffffu, row, 4 * (lane & 7));
                const bool on = (mask >> (4 * (lane & 7))) & 15;
                if (lane < 16)
                    cp_async_4_zfill(smem_u32(sc) + slot * 64 + lane * 4,
                                     (lane < 8 ? p.key_scales : p.value_scales) + srow, on);
            }
            int flags = (fresh ? kFirst : 0) | (tile == tile_begin ? kUnitBegin : 0) |
                        (tile + 1 == tile_end ? kUnitEnd : 0);
            const int u = seq * p.units_per_seq + sub;
            const int pos0 = tile * TT;
            // advance
            fresh = false;
            ++tile;
            ++rel;
            if (tile == tile_end) {
                fresh = true;
                rel += kUnitCost;
                if (++sub == p.units_per_seq) {
                    sub = 0;
                    if (rel < lim) {
                        int s = seq + 1;
                        while (s < p.num_seqs && tiles_of(s) == 0) ++s;
                        if (s < p.num_seqs) enter_seq(s); else lim = rel;
                    }
                }
                tile = tile_begin;
            }
            if (fresh || rel >= lim) flags |= kLast;
            if (lane == 0) hdr[slot] = make_int4((int)mask, pos0, u, flags);
            fetch_bid();
        } else if (lane == 0) {
            hdr[slot] = make_int4(0, 0, -1, 0);
        }
        cp_async_commit();
    };

    fetch_bid();
    grid_dependency_wait();
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) load_tile(i);

    // ---- state of the piece in flight
    uint32_t qf[NT][F::kTiles][2];
    float o[NT][F::kTiles][4];
    float m[NT][2], mv[NT][2], l[NT][2], qs[NT][2], slope[NT][2];
    int piece_flags = 0, last_pos = 0;
    Unit un{0, 0, 0, 0};
    const ScoreMod mod{p.cap_log2, p.inv_cap, p.alibi_slopes != nullptr};
    QT* out = reinterpret_cast<QT*>(p.out);
    float4* part_a = p.warp_partials + ((long long)blockIdx.x * kWarps + warp) * F::kFrags;

    int slot = 0;
    while (true) {
        {
            int next = slot + ST - 1;
            if (next >= ST) next -= ST;
            load_tile(next);
        }
        cp_async_wait<ST - 1>();
        __syncwarp();
        const int4 h = hdr[slot];
        if (h.z < 0) break;
        const uint32_t mask = (uint32_t)h.x;
        if (h.w & kFirst) {
            piece_flags = h.w & kUnitBegin;
            un = unit_of(h.z, p);
            last_pos = min(max(p.seq_lens[un.s], 0), p.max_tokens) - 1;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int head = nt * 8 + g;
                const bool there = head < un.heads;
                const QT* q = reinterpret_cast<const QT*>(p.query) +
                              (long long)un.s * p.query_stride + (long long)(un.head0 + head) * D;
                float scale_q = p.scale;
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
                    // 2^n that brings the head's largest element into [2^14, 2^15)
                    const int n = min(max(14 - ((int)(top >> 23) - 127), -110), 110);
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
                    slope[nt][e] = mod.alibi && hh < un.heads
                                       ? p.alibi_slopes[un.head0 + hh] * kLog2e : 0.f;
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
                        ldsm_x4(kbase + tile_offset<CH>(mt * 16 + lr, c + lc), r0, r1, r2, r3);
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
                        ldsm_x4(kbase + tile_offset<CH>(mt * 16 + lr, 2 * c + lc), a[0], a[1], a[2],
                                a[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma16816<MT>(s[nt][mt], a, qf[nt][c][0], qf[nt][c][1]);
                    }
            }
        }

        // ---- scores in log2 units, weights
        float ev[MT_TILES][2];
#pragma unroll
        for (int mt = 0; mt < MT_TILES; ++mt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int tok = mt * 16 + r * 8 + g;
                float ks = 1.f;
                if constexpr (F::kQ8) {
                    ks = scale_value(sc[slot * 64 + tok]);
                    ev[mt][r] = (float)((int)sc[slot * 64 + 32 + tok] - 127);
                } else {
                    ev[mt][r] = 0.f;
                }
                const bool seen = (mask >> tok) & 1;
                const float back = (float)(h.y + tok - last_pos);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        // the two scales first: the product of the stored
                        // values is of moderate size, so nothing overflows
                        // that the score itself does not
                        float x = s[nt][mt][2 * r + e] * (ks * qs[nt][e]);
                        x = p.cap_log2 > 0.f ? mod.cap(x) : x * kLog2e;
                        x = fmaf(slope[nt][e], back, x);
                        s[nt][mt][2 * r + e] = seen ? x : -INFINITY;
                    }
            }
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
                        ldsm_x4_trans(vbase + tile_offset<CH>(mt * 16 + lr, c + lc), r0, r1, r2, r3);
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
                        ldsm_x4_trans(vbase + tile_offset<CH>(mt * 16 + lr, 2 * c + lc), a[0], a[2],
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
            const bool whole = piece_flags == (kUnitBegin | kUnitEnd);
            // the last piece of the range stays in shared memory (the ring is
            // free: every load has landed), an earlier one goes to the workspace
            const bool end = rel >= lim && hdr[slot + 1 == ST ? 0 : slot + 1].z < 0;
            const int entry = 2 * warp + (end ? 1 : 0);
            if (end && !whole) {
                cp_async_wait<0>();
                __syncwarp();
            }
            float4* dst = end ? reinterpret_cast<float4*>(smem + warp * kRingBytes) : part_a;
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
                    inv[e] = sum > 0.f || sum != sum ? __fdividef(1.f, sum) : 0.f;
                    if (!whole && g == 0)
                        ml[entry * G + nt * 8 + 2 * t4 + e] = make_float2(m[nt][e], sum);
                }
#pragma unroll
                for (int i = 0; i < F::kTiles; ++i) {
                    const float4 v = make_float4(o[nt][i][0] * fac[0], o[nt][i][1] * fac[1],
                                                 o[nt][i][2] * fac[0], o[nt][i][3] * fac[1]);
                    if (whole)
                        write_frag<QT, F::kQ8>(out, p, un, D, nt, i, lane, v, inv[0], inv[1]);
                    else
                        dst[(nt * F::kTiles + i) * 32 + lane] = v;
                }
            }
            if (!whole && lane == 0) ids[entry] = make_int2(h.z, piece_flags);
        }
        __syncwarp();
        if (++slot == ST) slot = 0;
    }
    cp_async_wait<0>();
    __syncthreads();

    // ---- join the CTA's partials, in range order
    {
        const int slot0 = 2 * blockIdx.x;
        int2 left = make_int2(-1, 0), right = make_int2(-1, 0);
        int e0 = 0;
        while (e0 < 2 * kWarps) {
            if (ids[e0].x < 0) {
                ++e0;
                continue;
            }
            const int u = ids[e0].x;
            int flags = ids[e0].y, e1 = e0 + 1;
            for (; e1 < 2 * kWarps; ++e1) {
                if (ids[e1].x < 0) continue;
                if (ids[e1].x != u) break;
                flags |= ids[e1].y;
            }
            const bool whole = flags == (kUnitBegin | kUnitEnd);
            const int side = (flags & kUnitBegin) ? 1 : 0;
            if (!whole) {
                if (side) right = make_int2(u, flags); else left = make_int2(u, flags);
            }
            const Unit w = unit_of(u, p);
            for (int f = tid; f < F::kFrags; f += kThreads) {
                const int nt = f / (F::kTiles * 32), fl = f & 31;
                const int h0 = nt * 8 + 2 * (fl & 3);
                float M0 = -INFINITY, M1 = -INFINITY;
                for (int e = e0; e < e1; ++e) {
                    if (ids[e].x < 0) continue;
                    M0 = fmaxf(M0, ml[e * G + h0].x);
                    M1 = fmaxf(M1, ml[e * G + h0 + 1].x);
                }
                float L0 = 0.f, L1 = 0.f;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int e = e0; e < e1; ++e) {
                    if (ids[e].x < 0) continue;
                    const float2 a = ml[e * G + h0], b = ml[e * G + h0 + 1];
                    const float w0 = piece_weight(a.x, M0), w1 = piece_weight(b.x, M1);
                    const float4* src = (e & 1) ? reinterpret_cast<const float4*>(
                                                      smem + (e >> 1) * kRingBytes)
                                                : p.warp_partials + ((long long)blockIdx.x * kWarps +
                                                                     (e >> 1)) * F::kFrags;
                    const float4 v = src[f];
                    L0 += w0 * a.y;
                    L1 += w1 * b.y;
                    acc.x += w0 * v.x;
                    acc.y += w1 * v.y;
                    acc.z += w0 * v.z;
                    acc.w += w1 * v.w;
                }
                if (whole) {
                    write_frag<QT, F::kQ8>(out, p, w, D, nt, (f >> 5) % F::kTiles, fl, acc,
                                           L0 > 0.f || L0 != L0 ? __fdividef(1.f, L0) : 0.f,
                                           L1 > 0.f || L1 != L1 ? __fdividef(1.f, L1) : 0.f);
                } else {
                    p.cta_partials[(long long)(slot0 + side) * F::kFrags + f] = acc;
                    if ((f >> 5) % F::kTiles == 0 && fl < 4) {
                        p.cta_ml[(slot0 + side) * G + h0] = make_float2(M0, L0);
                        p.cta_ml[(slot0 + side) * G + h0 + 1] = make_float2(M1, L1);
                    }
                }
            }
            e0 = e1;
        }
        if (tid == 0) {
            p.cta_ids[slot0] = left;
            p.cta_ids[slot0 + 1] = right;
        }
    }
    // ---- sequences with no token: zeros
    for (int s = blockIdx.x; s < p.num_seqs; s += gridDim.x) {
        if (p.seq_lens[s] > p.max_tokens && tid == 0) flag_status(TLB_STATUS_SEQ_TOO_LONG);
        if (tiles_of(s) == 0)
            for (int i = tid; i < p.num_heads * D; i += kThreads)
                out[(long long)s * p.num_heads * D + i] = Elem<QT>::from_f(0.f);
    }
}

// Units that several CTAs share: CTA c takes the unit whose first partial is
// c's right one; its others are the left partials of the CTAs after c, up to
// the one that holds the unit's end. blockIdx.y takes a quarter of the
// fragments; the threads split the partials of a fragment between them.
constexpr int kJoinParts = 4;

template <typename QT, bool Q8, int D, int NT>
__global__ void __launch_bounds__(256) scored_join_kernel(const Params p, int ctas) {
    constexpr int kTiles = D / 16, kFrags = NT * kTiles * 32, G = 8 * NT;
    constexpr int P = kFrags / kJoinParts;  // fragments of this block
    constexpr int LANES = 256 / P;          // threads per fragment
    static_assert(P <= 256 && 256 % P == 0, "fragments split over the block");
    __shared__ int last_s;
    __shared__ float sM[G], sL[G];
    __shared__ float4 red[256];
    const int c = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    grid_dependency_wait();
    const int2 id = p.cta_ids[2 * c + 1];
    if (id.x < 0) return;
    if (tid == 0) last_s = ctas;
    __syncthreads();
    for (int i = c + 1 + tid; i < ctas; i += 256)
        if (p.cta_ids[2 * i].x == id.x && (p.cta_ids[2 * i].y & kUnitEnd)) atomicMin(&last_s, i);
    __syncthreads();
    const int n = min(last_s, ctas - 1) - c + 1;  // partials
    auto slot = [&](int i) { return i == 0 ? 2 * c + 1 : 2 * (c + i); };
    for (int h = warp; h < G; h += 8) {
        float M = -INFINITY;
        for (int i = lane; i < n; i += 32) M = fmaxf(M, p.cta_ml[slot(i) * G + h].x);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
        float L = 0.f;
        for (int i = lane; i < n; i += 32) {
            const float2 v = p.cta_ml[slot(i) * G + h];
            L += piece_weight(v.x, M) * v.y;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) L += __shfl_xor_sync(0xffffffffu, L, d);
        if (lane == 0) {
            sM[h] = M;
            sL[h] = L;
        }
    }
    __syncthreads();
    const int f = blockIdx.y * P + tid % P, part = tid / P;
    const int nt = f / (kTiles * 32), fl = f & 31, h0 = nt * 8 + 2 * (fl & 3);
    const float M0 = sM[h0], M1 = sM[h0 + 1];
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = part; i < n; i += LANES) {
        const float4 v = p.cta_partials[(long long)slot(i) * kFrags + f];
        const float w0 = piece_weight(p.cta_ml[slot(i) * G + h0].x, M0);
        const float w1 = piece_weight(p.cta_ml[slot(i) * G + h0 + 1].x, M1);
        acc.x += w0 * v.x;
        acc.y += w1 * v.y;
        acc.z += w0 * v.z;
        acc.w += w1 * v.w;
    }
    red[tid] = acc;
    __syncthreads();
    if (part == 0) {
        for (int i = 1; i < LANES; ++i) {
            const float4 v = red[i * P + tid];
            acc.x += v.x;
            acc.y += v.y;
            acc.z += v.z;
            acc.w += v.w;
        }
        const float L0 = sL[h0], L1 = sL[h0 + 1];
        write_frag<QT, Q8>(reinterpret_cast<QT*>(p.out), p, unit_of(id.x, p), D, nt,
                           (f >> 5) % kTiles, fl, acc,
                           L0 > 0.f || L0 != L0 ? __fdividef(1.f, L0) : 0.f,
                           L1 > 0.f || L1 != L1 ? __fdividef(1.f, L1) : 0.f);
    }
}

template <typename QT, typename CT, int D, int NT>
cudaError_t launch_fast(const Params& p, int ctas, bool overlap, cudaStream_t st) {
    using F = Cfg<QT, CT, D, NT>;
    auto kern = scored_attention_kernel<QT, CT, D, NT>;
    cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = F::kSmem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = overlap ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess || ctas == 1) return e;
    cfg.gridDim = dim3(ctas, kJoinParts);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, scored_join_kernel<QT, F::kQ8, D, NT>, p, ctas);
}

template <typename QT, typename CT>
cudaError_t launch_fast_shape(const Params& p, int head_dim, int ctas, bool overlap,
                              cudaStream_t st) {
    if (head_dim == 128)
        return p.unit_heads <= 8 ? launch_fast<QT, CT, 128, 1>(p, ctas, overlap, st)
                                 : launch_fast<QT, CT, 128, 2>(p, ctas, overlap, st);
    return p.unit_heads <= 8 ? launch_fast<QT, CT, 64, 1>(p, ctas, overlap, st)
                             : launch_fast<QT, CT, 64, 2>(p, ctas, overlap, st);
}

}  // namespace scored
}  // namespace tlb
