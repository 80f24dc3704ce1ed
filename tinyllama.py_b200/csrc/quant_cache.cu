// Quantised KV-cache rows: the cache write, reading blocks back, and the
// per-head norm of queries and keys with their rotation (and cache write).
//
// All three are streaming kernels bounded by HBM; each row is held in the
// registers of a few lanes between its one read and its one write.
#include "kernels.h"
#include "quant_rows.cuh"

namespace tlb {

namespace {

__device__ __forceinline__ long long load_int(const void* p, bool wide, long long i) {
    return wide ? (long long)reinterpret_cast<const int64_t*>(p)[i]
                : (long long)reinterpret_cast<const int32_t*>(p)[i];
}

// Row index of (slot's block, head 0, slot's offset) in a
// [blocks, kv_heads, block_size] cache, or -1 to skip the token.
__device__ __forceinline__ long long slot_row(long long slot, const QuantCacheParams& p) {
    if (slot < 0) return -1;
    int off;
    long long blk;
    if (p.block_shift >= 0) {
        blk = slot >> p.block_shift;
        off = (int)(slot & (p.block_size - 1));
    } else {
        blk = divide(slot, p.block_size, off);
    }
    if (blk >= p.num_blocks) {
        flag_status(TLB_STATUS_BAD_SLOT);
        return -1;
    }
    return blk * p.num_kv_heads * p.block_size + off;
}

// The row of token t at position pos through its block-table row.
__device__ __forceinline__ long long table_row(long long t, long long pos,
                                               const QuantCacheParams& p) {
    int off = 0;
    const long long logical = pos < 0 ? -1 : divide(pos, p.block_size, off);
    if (logical < 0 || logical >= p.max_blocks) {
        flag_status(TLB_STATUS_BAD_SLOT);
        return -1;
    }
    const long long blk = p.block_tables[t * p.max_blocks + logical];
    if (blk < 0) return -1;
    if (blk >= p.num_blocks) {
        flag_status(TLB_STATUS_BAD_SLOT);
        return -1;
    }
    return blk * p.num_kv_heads * p.block_size + off;
}

// A warp's place in its share of the work: rows [first, first + step) of token
// t's `rows` rows, taken `step` at a time by each of the `parts` warps that share
// a token; then the same of a later token.
// The token's position and slot are loaded when the place is taken, a step
// before they are used.
struct Place {
    long long item, t, pos, slot;
    int first;
    bool valid;
};
__device__ __forceinline__ Place place_of(long long item, long long items, int parts, int step,
                                          const QuantCacheParams& p) {
    Place c{item, 0, 0, -1, 0, item < items};
    if (c.valid) {
        c.t = item;
        if (parts != 1) {
            int part;
            c.t = divide(item, parts, part);
            c.first = part * step;
        }
        if (p.positions) c.pos = load_int(p.positions, p.positions64, c.t);
        if (p.slots) c.slot = load_int(p.slots, p.slots64, c.t);
    }
    return c;
}
__device__ __forceinline__ Place next_place(const Place& c, long long items, int parts, int step,
                                            int rows, const QuantCacheParams& p) {
    Place n = c;
    n.first += parts * step;
    if (n.first < rows) return n;
    return place_of(c.item + (long long)gridDim.x * 8, items, parts, step, p);
}

// ------------------------------------------------------------- cache write
// HBM bound: e D bytes in, D + 1 out for each row of e-byte values. A warp takes
// rows of one token: all keys, then all values. A row is held by LANES lanes, 16
// values each (two 16-byte loads, 8-byte stores) between its one read and its one
// write; kWriteRows rows of a group are read while kWriteRows are quantised and
// stored. 16381 fp16 tokens of 8 heads of 128 to int8 (101 MB): 19.7 us with 4
// rows and 16 warps an SM, 21.3 us with 2, 23.5 us with 1 row and 24 warps. Of
// 24 us, 3 went into the scales' single bytes and 5.5 into the rows' stores.
// Rows of other widths and alignments take a warp each, element by element, and
// are read twice.
constexpr int kWriteRows = 4;

template <typename T, typename C, int LANES>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) quantize_write_kernel(const QuantCacheParams p, int parts) {
    grid_dependency_wait();
    grid_launch_dependents();
    constexpr int GROUPS = 32 / LANES, STEP = GROUPS * kWriteRows;
    const int lane = threadIdx.x & 31, grp = lane / LANES, sub = lane % LANES;
    const uint32_t mask = group_mask<LANES>();
    const int D = p.head_size, kvh = p.num_kv_heads, rows = 2 * kvh;
    const bool on = sub * 16 < D;
    const int i0 = sub * 8, i1 = i0 + D / 2;
    const long long items = p.num_tokens * parts;
    const int head_stride = p.block_size * D;  // of a cache, in values

    Raw8<T> a0[kWriteRows], a1[kWriteRows], b0[kWriteRows], b1[kWriteRows];
    auto load = [&](const Place& c, Raw8<T> (&x0)[kWriteRows], Raw8<T> (&x1)[kWriteRows]) {
        const T* key = reinterpret_cast<const T*>(p.key) + c.t * p.key_stride;
        const T* value = reinterpret_cast<const T*>(p.value) + c.t * p.value_stride;
#pragma unroll
        for (int i = 0; i < kWriteRows; ++i) {
            const int r = c.first + i * GROUPS + grp;
            x0[i].zero();
            x1[i].zero();
            if (c.valid && r < rows && on) {
                const T* src = r < kvh ? key + r * D : value + (r - kvh) * D;
                x0[i].load_stream(src + i0);
                x1[i].load_stream(src + i1);
            }
        }
    };
    long long known = -1;  // the token looked up last, and its rows of head 0
    uint8_t *key_row = nullptr, *value_row = nullptr, *key_scale = nullptr, *value_scale = nullptr;
    auto store = [&](const Place& c, Raw8<T> (&x0)[kWriteRows], Raw8<T> (&x1)[kWriteRows]) {
        if (known != c.t) {
            known = c.t;
            const long long base = slot_row(c.slot, p);
            key_row = nullptr;
            if (base >= 0) {
                key_row = reinterpret_cast<uint8_t*>(p.key_cache) + base * D;
                value_row = reinterpret_cast<uint8_t*>(p.value_cache) + base * D;
                key_scale = p.key_scales + base;
                value_scale = p.value_scales + base;
            }
        }
        if (key_row == nullptr) return;
#pragma unroll
        for (int i = 0; i < kWriteRows; ++i) {
            const int r = c.first + i * GROUPS + grp;
            if (r >= rows) break;
            const bool is_value = r >= kvh;
            const int h = is_value ? r - kvh : r;
            uint2 q0, q1;
            const uint32_t byte = quantize_pieces<T, C, LANES>(
                x0[i], x1[i], group_top<LANES, T>(max_top<T>(x0[i].top(), x1[i].top()), mask), mask,
                q0, q1);
            uint8_t* dst = (is_value ? value_row : key_row) + h * head_stride;
            if (on) {
                *reinterpret_cast<uint2*>(dst + i0) = q0;
                *reinterpret_cast<uint2*>(dst + i1) = q1;
            }
            if (sub == 0) (is_value ? value_scale : key_scale)[h * p.block_size] = (uint8_t)byte;
        }
    };
    Place c = place_of(blockIdx.x * 8 + threadIdx.x / 32, items, parts, STEP, p);
    load(c, a0, a1);
    while (c.valid) {
        Place n = next_place(c, items, parts, STEP, rows, p);
        load(n, b0, b1);
        store(c, a0, a1);
        if (!n.valid) break;
        c = next_place(n, items, parts, STEP, rows, p);
        load(c, a0, a1);
        store(n, b0, b1);
    }
}

template <typename T, typename C>
__global__ void __launch_bounds__(256) quantize_write_any_kernel(const QuantCacheParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const int lane = threadIdx.x & 31, D = p.head_size;
    const long long rows = p.num_tokens * 2 * p.num_kv_heads;
    for (long long r = blockIdx.x * 8 + threadIdx.x / 32; r < rows; r += gridDim.x * 8) {
        int h;
        const long long th = divide(r, p.num_kv_heads, h), t = th >> 1;
        const bool is_value = th & 1;
        const long long base = slot_row(load_int(p.slots, p.slots64, t), p);
        if (base < 0) continue;
        const long long row = base + (long long)h * p.block_size;
        const T* src = reinterpret_cast<const T*>(is_value ? p.value : p.key) +
                       t * (is_value ? p.value_stride : p.key_stride) + (long long)h * D;
        C* dst = reinterpret_cast<C*>(is_value ? p.value_cache : p.key_cache) + row * D;
        uint32_t m = 0;
        for (int i = lane; i < D; i += 32) m = max(m, finite_abs_bits(Elem<T>::to_f(src[i])));
        const uint32_t byte = scale_byte<C>(group_max<32>(m, 0xffffffffu));
        const float inv = inverse_scale(byte);
        for (int i = lane; i < D; i += 32) store_quantized1(dst + i, Elem<T>::to_f(src[i]), inv);
        if (lane == 0) (is_value ? p.value_scales : p.key_scales)[row] = (uint8_t)byte;
    }
}

// -------------------------------------------------------------- read back
// HBM bound: D + 1 bytes in, e D out for each row. Flat over 16-value pieces of
// the listed blocks (pieces never straddle a row), a piece of each cache for a
// thread and step. The values go past the caches (streaming stores): 9000 blocks
// of 2 x 16 rows of 128 (222 MB) take 38.7 us, with plain stores and two pieces
// in flight 42.5. IX: index type of the piece arithmetic (32-bit unsigned where
// it fits).
template <typename T, typename C>
__device__ __forceinline__ void widen16(T* out, uint4 u, float scale) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            f[j] = mul_keep(dequantize1<C>((w[2 * half + (j >> 2)] >> (8 * (j & 3))) & 0xff), scale);
        Raw8<T> r;
        r.set(f);
        r.store_stream(out + 8 * half);
    }
}

template <typename T, typename C, typename IX>
__global__ void __launch_bounds__(256) dequantize_blocks_kernel(const DequantParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const unsigned row_pieces = p.head_size / 16;
    const IX pieces = (IX)p.rows_per_block * row_pieces;  // of a block
    const IX total = pieces * (IX)p.num_ids;
    const uint8_t* kc = reinterpret_cast<const uint8_t*>(p.key_cache);
    const uint8_t* vc = reinterpret_cast<const uint8_t*>(p.value_cache);
    for (IX i = (IX)blockIdx.x * 256 + threadIdx.x; i < total; i += (IX)gridDim.x * 256) {
        const IX n = i / pieces;
        const unsigned piece = (unsigned)(i - n * pieces);
        const long long blk = load_int(p.ids, p.ids64, n);
        uint4 k = make_uint4(0, 0, 0, 0), v = k;
        uint32_t ks = 0, vs = 0;
        if (blk >= p.num_blocks) flag_status(TLB_STATUS_BAD_BLOCK_ID);
        if (blk >= 0 && blk < p.num_blocks) {
            const long long from = (blk * (long long)pieces + piece) * 16;
            const long long row = blk * p.rows_per_block + piece / row_pieces;
            k = __ldcs(reinterpret_cast<const uint4*>(kc + from));
            v = __ldcs(reinterpret_cast<const uint4*>(vc + from));
            ks = p.key_scales[row];
            vs = p.value_scales[row];
        }
        widen16<T, C>(reinterpret_cast<T*>(p.key_out) + (long long)i * 16, k, scale_value(ks));
        widen16<T, C>(reinterpret_cast<T*>(p.value_out) + (long long)i * 16, v, scale_value(vs));
    }
}

// Any row width and alignment, value by value.
template <typename T, typename C>
__global__ void __launch_bounds__(256) dequantize_any_kernel(const DequantParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const long long block_values = (long long)p.rows_per_block * p.head_size;
    const long long total = block_values * p.num_ids;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total;
         i += (long long)gridDim.x * 256) {
        const long long n = i / block_values, at = i - n * block_values;
        const long long blk = load_int(p.ids, p.ids64, n);
        float k = 0.f, v = 0.f;
        if (blk >= p.num_blocks) flag_status(TLB_STATUS_BAD_BLOCK_ID);
        if (blk >= 0 && blk < p.num_blocks) {
            const long long from = blk * block_values + at;
            const long long row = blk * p.rows_per_block + at / p.head_size;
            k = mul_keep(dequantize1<C>(reinterpret_cast<const uint8_t*>(p.key_cache)[from]),
                         scale_value(p.key_scales[row]));
            v = mul_keep(dequantize1<C>(reinterpret_cast<const uint8_t*>(p.value_cache)[from]),
                         scale_value(p.value_scales[row]));
        }
        reinterpret_cast<T*>(p.key_out)[i] = Elem<T>::from_f(k);
        reinterpret_cast<T*>(p.value_out)[i] = Elem<T>::from_f(v);
    }
}

// ------------------------------------------------- query / key norm + RoPE
// For each head row x of a token's query and key
//   y_i = x_i * rsqrt(mean(x^2) + eps) * w_i
// then the rotation of pairs (i, i + rot/2), in fp32 with one rounding to the
// storage type. Keys go to key_out, or with a cache to their slot there; the
// value row goes to its slot beside them. A quantised cache takes the row as
// rounded to the storage type, so the bytes are those of a separate
// quantising write of this kernel's key.
//
// HBM bound (every row read and written once). A warp takes rows of one token,
// so that position, cos/sin row and slot are looked up once: query heads, key
// heads, value heads. A row is held by LANES lanes, 16 values each: lane
// l < rot/16 the eight values at 8 l and their partners at 8 l + rot/2 (so the
// rotation needs no exchange), the others 16 values beyond rot. A group keeps
// its weights while it stays with queries or with keys; kRows of its rows are
// read while kRows are worked on, with the next token's position and slot: 16383
// fp16 tokens of 32 + 8 heads of 128, half of each rotated (338 MB), take 61.8 us
// (62.7 and 64.6 on two other B200s; on the first, 66.6 without the next position
// and slot, 79 one buffer of rows). Four neighbouring tokens for the four groups
// of a warp, which would make the kind of row uniform, took 71.4 us. Other widths
// and alignments: a warp for each row, by element.
constexpr int kRows = 2;

enum RowKind { kQuery = 0, kKey = 1, kValue = 2 };

struct NormRow {
    RowKind kind;
    int h;
};
__device__ __forceinline__ NormRow norm_row(int r, const QuantCacheParams& p) {
    if (r < p.num_heads) return {kQuery, r};
    r -= p.num_heads;
    return r < p.num_kv_heads ? NormRow{kKey, r} : NormRow{kValue, r - p.num_kv_heads};
}

// x' = x cos - y sin, y' = y cos + x sin, a rounding less than rope_pair has: what
// comes in is an unrounded fp32 value, so there are no bits to agree with.
__device__ __forceinline__ void turn_pair(float x, float y, float c, float s, float& xo, float& yo) {
    xo = fmaf(x, c, -(y * s));
    yo = fmaf(y, c, x * s);
}

template <typename T, typename C, int LANES>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) qk_norm_rope_kernel(const QuantCacheParams p, int parts) {
    constexpr int GROUPS = 32 / LANES, STEP = GROUPS * kRows;
    const int lane = threadIdx.x & 31, grp = lane / LANES, sub = lane % LANES;
    const uint32_t mask = group_mask<LANES>();
    const int D = p.head_size, rot = p.rot_dim, half = rot / 2;
    const int H = p.num_heads, kvh = p.num_kv_heads;
    const bool with_cache = p.key_cache != nullptr;
    const int rows = H + kvh * (with_cache ? 2 : 1);
    const int pairs = rot / 16;  // lanes that rotate
    const bool on = sub * 16 < D, turn = on && sub < pairs;
    const int i0 = sub < pairs ? 8 * sub : rot + 16 * (sub - pairs);
    const int i1 = sub < pairs ? i0 + half : i0 + 8;
    const float inv_d = 1.f / (float)D;
    const long long items = p.num_tokens * parts;
    const int head_stride = p.block_size * D;  // of a cache, in values

    Raw8<T> a0[kRows], a1[kRows], b0[kRows], b1[kRows];
    auto load = [&](const Place& c, Raw8<T> (&x0)[kRows], Raw8<T> (&x1)[kRows]) {
        const T* query = reinterpret_cast<const T*>(p.query) + c.t * p.query_stride;
        const T* key = reinterpret_cast<const T*>(p.key) + c.t * p.key_stride;
        const T* value = reinterpret_cast<const T*>(p.value) + c.t * p.value_stride;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int r = c.first + i * GROUPS + grp;
            x0[i].zero();
            x1[i].zero();
            if (c.valid && r < rows && on) {
                const T* src = r < H         ? query + r * D
                               : r < H + kvh ? key + (r - H) * D
                                             : value + (r - H - kvh) * D;
                x0[i].load_stream(src + i0);
                x1[i].load_stream(src + i1);
            }
        }
    };
    long long known = -1;  // the token looked up last
    long long base = -1;   // its first cache row
    bool rotate = false;
    float cs[8], sn[8];  // cos and sin of the lane's pairs
    float w0[8], w1[8];  // weights of the kind of row the group had last
    int have = -1;
    auto process = [&](const Place& c, Raw8<T> (&x0)[kRows], Raw8<T> (&x1)[kRows]) {
        if (known != c.t) {
            known = c.t;
            const long long pos = c.pos;
            rotate = false;
            if (pos >= 0 && pos < p.cache_rows) {
                rotate = turn;
                if (turn) {
                    const T* table = reinterpret_cast<const T*>(p.cos_sin) + pos * rot;
                    Raw8<T> u, v;
                    u.load(table + i0);
                    v.load(table + half + i0);
                    u.get(cs);
                    v.get(sn);
                }
            } else {
                flag_status(TLB_STATUS_BAD_POSITION);
            }
            if (with_cache)
                base = p.slots ? slot_row(c.slot, p) : table_row(c.t, pos, p);
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int r = c.first + i * GROUPS + grp;
            if (r >= rows) break;
            const int kind = r < H ? kQuery : r < H + kvh ? kKey : kValue;
            if (kind != kValue) {
                if (have != kind) {
                    have = kind;
                    const T* w = reinterpret_cast<const T*>(kind == kQuery ? p.query_weight
                                                                           : p.key_weight);
                    Raw8<T> u, v;
                    u.zero();
                    v.zero();
                    if (on) {
                        u.load(w + i0);
                        v.load(w + i1);
                    }
                    u.get(w0);
                    v.get(w1);
                }
                float a[8], b[8];
                x0[i].get(a);
                x1[i].get(b);
                float sa = 0.f, sb = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    sa = fmaf(a[j], a[j], sa);
                    sb = fmaf(b[j], b[j], sb);
                }
                const float inv = rsqrtf(group_sum<LANES>(sa + sb, mask) * inv_d + p.eps);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    a[j] = a[j] * inv * w0[j];
                    b[j] = b[j] * inv * w1[j];
                }
                if (rotate) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float x, y;
                        turn_pair(a[j], b[j], cs[j], sn[j], x, y);
                        a[j] = x;
                        b[j] = y;
                    }
                }
                x0[i].set(a);
                x1[i].set(b);
            }
            if (kind == kQuery || !with_cache) {
                T* dst = kind == kQuery
                             ? reinterpret_cast<T*>(p.out) + c.t * (H * D) + r * D
                             : reinterpret_cast<T*>(p.key_out) + c.t * (kvh * D) + (r - H) * D;
                if (on) {
                    x0[i].store(dst + i0);
                    x1[i].store(dst + i1);
                }
                continue;
            }
            if (base < 0) continue;
            const int h = kind == kKey ? r - H : r - H - kvh;
            const long long at = base * D + (long long)h * head_stride;
            if constexpr (sizeof(C) == 1) {
                uint2 q0, q1;
                const uint32_t byte = quantize_pieces<T, C, LANES>(
                    x0[i], x1[i], group_top<LANES, T>(max_top<T>(x0[i].top(), x1[i].top()), mask),
                    mask, q0, q1);
                uint8_t* dst =
                    reinterpret_cast<uint8_t*>(kind == kValue ? p.value_cache : p.key_cache) + at;
                if (on) {
                    *reinterpret_cast<uint2*>(dst + i0) = q0;
                    *reinterpret_cast<uint2*>(dst + i1) = q1;
                }
                if (sub == 0)
                    (kind == kValue ? p.value_scales : p.key_scales)[base + (long long)h *
                                                                                p.block_size] =
                        (uint8_t)byte;
            } else if (on) {
                T* dst = reinterpret_cast<T*>(kind == kValue ? p.value_cache : p.key_cache) + at;
                x0[i].store(dst + i0);
                x1[i].store(dst + i1);
            }
        }
    };
    grid_dependency_wait();
    grid_launch_dependents();
    Place c = place_of(blockIdx.x * 8 + threadIdx.x / 32, items, parts, STEP, p);
    load(c, a0, a1);
    while (c.valid) {
        Place n = next_place(c, items, parts, STEP, rows, p);
        load(n, b0, b1);
        process(c, a0, a1);
        if (!n.valid) break;
        c = next_place(n, items, parts, STEP, rows, p);
        load(c, a0, a1);
        process(n, b0, b1);
    }
}

template <typename T>
__device__ __forceinline__ float rounded(float x) {
    return Elem<T>::to_f(Elem<T>::from_f(x));
}

template <typename T, typename C>
__global__ void __launch_bounds__(256) qk_norm_rope_any_kernel(const QuantCacheParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const int lane = threadIdx.x & 31, D = p.head_size, rot = p.rot_dim, half = rot / 2;
    const bool with_cache = p.key_cache != nullptr;
    const int rows = p.num_heads + p.num_kv_heads * (with_cache ? 2 : 1);
    const long long items = p.num_tokens * rows;
    for (long long it = blockIdx.x * 8 + threadIdx.x / 32; it < items; it += gridDim.x * 8) {
        int r;
        const long long t = divide(it, rows, r);
        const NormRow nr = norm_row(r, p);
        const long long pos = load_int(p.positions, p.positions64, t);
        const T* cs = nullptr;
        if (pos >= 0 && pos < p.cache_rows)
            cs = reinterpret_cast<const T*>(p.cos_sin) + pos * rot;
        else
            flag_status(TLB_STATUS_BAD_POSITION);
        long long row = -1;  // cache row of this item
        if (with_cache && nr.kind != kQuery) {
            row = p.slots ? slot_row(load_int(p.slots, p.slots64, t), p) : table_row(t, pos, p);
            if (row < 0) continue;
            row += (long long)nr.h * p.block_size;
        }
        const T* src = nr.kind == kQuery ? reinterpret_cast<const T*>(p.query) + t * p.query_stride
                       : nr.kind == kKey ? reinterpret_cast<const T*>(p.key) + t * p.key_stride
                                         : reinterpret_cast<const T*>(p.value) + t * p.value_stride;
        src += (long long)nr.h * D;
        const T* w = reinterpret_cast<const T*>(nr.kind == kQuery ? p.query_weight : p.key_weight);
        float inv = 0.f;
        if (nr.kind != kValue) {
            float ss = 0.f;
            for (int i = lane; i < D; i += 32) {
                const float x = Elem<T>::to_f(src[i]);
                ss = fmaf(x, x, ss);
            }
            inv = rsqrtf(group_sum<32>(ss, 0xffffffffu) * (1.f / (float)D) + p.eps);
        }
        auto out = [&](int i) -> float {
            float x = Elem<T>::to_f(src[i]);
            if (nr.kind == kValue) return x;
            x = x * inv * Elem<T>::to_f(w[i]);
            if (i >= rot || !cs) return x;
            const bool first = i < half;
            const int j = first ? i + half : i - half, k = first ? i : j;
            const float y = Elem<T>::to_f(src[j]) * inv * Elem<T>::to_f(w[j]);
            float xo, yo;
            turn_pair(first ? x : y, first ? y : x, Elem<T>::to_f(cs[k]),
                      Elem<T>::to_f(cs[half + k]), xo, yo);
            return first ? xo : yo;
        };
        if (nr.kind == kQuery || !with_cache) {
            T* dst = nr.kind == kQuery
                         ? reinterpret_cast<T*>(p.out) + (t * p.num_heads + nr.h) * D
                         : reinterpret_cast<T*>(p.key_out) + (t * p.num_kv_heads + nr.h) * D;
            for (int i = lane; i < D; i += 32) dst[i] = Elem<T>::from_f(out(i));
            continue;
        }
        C* dst = reinterpret_cast<C*>(nr.kind == kValue ? p.value_cache : p.key_cache) + row * D;
        if constexpr (sizeof(C) == 1) {
            uint32_t m = 0;
            for (int i = lane; i < D; i += 32) m = max(m, finite_abs_bits(rounded<T>(out(i))));
            const uint32_t byte = scale_byte<C>(group_max<32>(m, 0xffffffffu));
            const float qs = inverse_scale(byte);
            for (int i = lane; i < D; i += 32) store_quantized1(dst + i, rounded<T>(out(i)), qs);
            if (lane == 0) (nr.kind == kValue ? p.value_scales : p.key_scales)[row] = (uint8_t)byte;
        } else {
            for (int i = lane; i < D; i += 32) dst[i] = Elem<T>::from_f(out(i));
        }
    }
}

// ------------------------------------------------------------------- host
int sm_count() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
        return 148;
    return n;
}
// CTAs of 256 threads that stride over `items` items of `per_cta` a CTA.
int grid_of(long long items, int per_cta, int ctas_per_sm = 8) {
    const long long need = (items + per_cta - 1) / per_cta, cap = (long long)sm_count() * ctas_per_sm;
    return (int)(need < cap ? (need > 0 ? need : 1) : cap);
}
// Warps that share a token's `rows` rows, `step` rows each time: as many as keep
// 16 warps an SM busy, one where there are tokens enough.
int parts_of(long long tokens, int rows, int step) {
    const int most = (rows + step - 1) / step;
    const long long want = (16ll * sm_count() + tokens - 1) / tokens;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

template <typename T, typename C, int LANES>
cudaError_t write_lanes(const QuantCacheParams& p, cudaStream_t st) {
    const int parts = parts_of(p.num_tokens, 2 * p.num_kv_heads, 32 / LANES * kWriteRows);
    return launch_early(quantize_write_kernel<T, C, LANES>, grid_of(p.num_tokens * parts, 8, 2), 256,
                        0, st, p, parts);
}
template <typename T, typename C>
cudaError_t write_tc(const QuantCacheParams& p, bool vec, cudaStream_t st) {
    const int units = vec ? p.head_size / 16 : 33;
    if (units <= 4) return write_lanes<T, C, 4>(p, st);
    if (units <= 8) return write_lanes<T, C, 8>(p, st);
    if (units <= 16) return write_lanes<T, C, 16>(p, st);
    if (units <= 32) return write_lanes<T, C, 32>(p, st);
    return launch_early(quantize_write_any_kernel<T, C>,
                        grid_of(p.num_tokens * 2 * p.num_kv_heads, 8), 256, 0, st, p);
}
template <typename T>
cudaError_t write_t(int cache_dtype, const QuantCacheParams& p, bool vec, cudaStream_t st) {
    return cache_dtype == TLB_INT8 ? write_tc<T, int8_t>(p, vec, st) : write_tc<T, E4M3>(p, vec, st);
}

template <typename T, typename C>
cudaError_t dequant_tc(const DequantParams& p, bool vec, cudaStream_t st) {
    const long long values = p.num_ids * p.rows_per_block * p.head_size;
    // 32-bit piece numbers, with room for a step past the end
    if (vec && values / 16 < (1ll << 31))
        return launch_early(dequantize_blocks_kernel<T, C, unsigned>, grid_of(values / 16, 256), 256,
                            0, st, p);
    if (vec)
        return launch_early(dequantize_blocks_kernel<T, C, unsigned long long>,
                            grid_of(values / 16, 256), 256, 0, st, p);
    return launch_early(dequantize_any_kernel<T, C>, grid_of(values, 256), 256, 0, st, p);
}
template <typename T>
cudaError_t dequant_t(int cache_dtype, const DequantParams& p, bool vec, cudaStream_t st) {
    return cache_dtype == TLB_INT8 ? dequant_tc<T, int8_t>(p, vec, st)
                                   : dequant_tc<T, E4M3>(p, vec, st);
}

template <typename T, typename C, int LANES>
cudaError_t norm_lanes(const QuantCacheParams& p, int rows, cudaStream_t st) {
    const int parts = parts_of(p.num_tokens, rows, 32 / LANES * kRows);
    return launch_early(qk_norm_rope_kernel<T, C, LANES>, grid_of(p.num_tokens * parts, 8, 2), 256, 0,
                        st, p, parts);
}
template <typename T, typename C>
cudaError_t norm_tc(const QuantCacheParams& p, bool vec, cudaStream_t st) {
    const int rows = p.num_heads + p.num_kv_heads * (p.key_cache != nullptr ? 2 : 1);
    const int units = vec ? p.head_size / 16 : 33;
    if (units <= 4) return norm_lanes<T, C, 4>(p, rows, st);
    if (units <= 8) return norm_lanes<T, C, 8>(p, rows, st);
    if (units <= 16) return norm_lanes<T, C, 16>(p, rows, st);
    if (units <= 32) return norm_lanes<T, C, 32>(p, rows, st);
    return launch_early(qk_norm_rope_any_kernel<T, C>, grid_of(p.num_tokens * rows, 8), 256, 0, st, p);
}
template <typename T>
cudaError_t norm_t(int cache_dtype, const QuantCacheParams& p, bool vec, cudaStream_t st) {
    if (cache_dtype == TLB_INT8) return norm_tc<T, int8_t>(p, vec, st);
    if (cache_dtype == TLB_FLOAT8_E4M3) return norm_tc<T, E4M3>(p, vec, st);
    return norm_tc<T, T>(p, vec, st);
}

}  // namespace

cudaError_t launch_quantize_write(int dtype, int cache_dtype, const QuantCacheParams& p, bool vec,
                                  cudaStream_t stream) {
    switch (dtype) {
        case TLB_FLOAT32: return write_t<float>(cache_dtype, p, vec, stream);
        case TLB_FLOAT16: return write_t<__half>(cache_dtype, p, vec, stream);
        default: return write_t<__nv_bfloat16>(cache_dtype, p, vec, stream);
    }
}
cudaError_t launch_dequantize_blocks(int out_dtype, int cache_dtype, const DequantParams& p,
                                     bool vec, cudaStream_t stream) {
    switch (out_dtype) {
        case TLB_FLOAT32: return dequant_t<float>(cache_dtype, p, vec, stream);
        case TLB_FLOAT16: return dequant_t<__half>(cache_dtype, p, vec, stream);
        default: return dequant_t<__nv_bfloat16>(cache_dtype, p, vec, stream);
    }
}
cudaError_t launch_qk_norm_rope(int dtype, int cache_dtype, const QuantCacheParams& p, bool vec,
                                cudaStream_t stream) {
    switch (dtype) {
        case TLB_FLOAT32: return norm_t<float>(cache_dtype, p, vec, stream);
        case TLB_FLOAT16: return norm_t<__half>(cache_dtype, p, vec, stream);
        default: return norm_t<__nv_bfloat16>(cache_dtype, p, vec, stream);
    }
}

}  // namespace tlb
