// Quantised KV-cache rows: the cache write, reading blocks back, and the
// per-head norm of queries and keys with their rotation (and cache write).
//
// All three are streaming kernels bounded by HBM; each row is held in the
// registers of a few lanes between its one read and its one write.
#include "kernels.h"
#include "quant.cuh"

namespace tlb {

namespace {

// Eight elements <-> registers, 16-byte accesses for half types, two for fp32.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
    constexpr int N = 8 * sizeof(T) / 16;
    uint4 u[N];
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
    const T* e = reinterpret_cast<const T*>(u);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = Elem<T>::to_f(e[i]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
    constexpr int N = 8 * sizeof(T) / 16;
    uint4 u[N];
    T* e = reinterpret_cast<T*>(u);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = Elem<T>::from_f(f[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<uint4*>(p)[i] = u[i];
}

__device__ __forceinline__ uint32_t max_abs8(const float (&f)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, finite_abs_bits(f[i]));
    return m;
}

template <typename C>
__device__ __forceinline__ void store_quantized8(C* dst, const float (&f)[8], float inv) {
    uint2 u;
    u.x = quantize4<C>(mul_keep(f[0], inv), mul_keep(f[1], inv), mul_keep(f[2], inv),
                       mul_keep(f[3], inv));
    u.y = quantize4<C>(mul_keep(f[4], inv), mul_keep(f[5], inv), mul_keep(f[6], inv),
                       mul_keep(f[7], inv));
    *reinterpret_cast<uint2*>(dst) = u;
}
template <typename C>
__device__ __forceinline__ void store_quantized1(C* dst, float x, float inv) {
    *reinterpret_cast<uint8_t*>(dst) = (uint8_t)quantize4<C>(mul_keep(x, inv), 0.f, 0.f, 0.f);
}

// Maximum over the `lanes` (a power of two) lanes of a group, which `mask`
// names.
__device__ __forceinline__ uint32_t group_max(uint32_t v, int lanes, uint32_t mask) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(mask, v, o));
    return v;
}
__device__ __forceinline__ float group_sum(float v, int lanes, uint32_t mask) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
    return v;
}
__device__ __forceinline__ uint32_t group_mask(int lanes) {
    const uint32_t ones = lanes == 32 ? 0xffffffffu : (1u << lanes) - 1u;
    return ones << ((threadIdx.x & 31) / lanes * lanes);
}

__device__ __forceinline__ long long load_int(const void* p, bool wide, long long i) {
    return wide ? (long long)reinterpret_cast<const int64_t*>(p)[i]
                : (long long)reinterpret_cast<const int32_t*>(p)[i];
}

// Row index of (slot's block, head 0, slot's offset) in a
// [blocks, kv_heads, block_size] cache, or -1 to skip the token.
__device__ __forceinline__ long long slot_row(long long slot, const QuantCacheParams& p) {
    if (slot < 0) return -1;
    const long long blk = slot / p.block_size;
    if (blk >= p.num_blocks) {
        flag_status(TLB_STATUS_BAD_SLOT);
        return -1;
    }
    return blk * p.num_kv_heads * p.block_size + (slot - blk * p.block_size);
}

// The row of token t at position pos through its block-table row.
__device__ __forceinline__ long long table_row(long long t, long long pos,
                                               const QuantCacheParams& p) {
    const long long logical = pos < 0 ? -1 : pos / p.block_size;
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
    return blk * p.num_kv_heads * p.block_size + (pos - logical * p.block_size);
}

// ------------------------------------------------------------- cache write
// A row is read by `lanes` lanes, eight elements each (VEC), which keep it in
// registers between the maximum and the store; rows of other widths or
// alignments take a warp each, element by element, and read the row twice.
template <typename T, typename C, bool VEC>
__global__ void __launch_bounds__(256) quantize_write_kernel(const QuantCacheParams p, int lanes) {
    const int per_block = 256 / lanes;
    const int sub = threadIdx.x % lanes;
    const uint32_t mask = group_mask(lanes);
    const long long rows = p.num_tokens * 2 * p.num_kv_heads;
    const int D = p.head_size;
    for (long long r = (long long)blockIdx.x * per_block + threadIdx.x / lanes; r < rows;
         r += (long long)gridDim.x * per_block) {
        const long long th = r / p.num_kv_heads;
        const int h = (int)(r - th * p.num_kv_heads);
        const long long t = th >> 1;
        const bool is_value = th & 1;
        const long long base = slot_row(load_int(p.slots, p.slots64, t), p);
        if (base < 0) continue;
        const long long row = base + (long long)h * p.block_size;
        const T* src = reinterpret_cast<const T*>(is_value ? p.value : p.key) +
                       t * (is_value ? p.value_stride : p.key_stride) + (long long)h * D;
        C* dst = reinterpret_cast<C*>(is_value ? p.value_cache : p.key_cache) + row * D;
        uint8_t* scale = (is_value ? p.value_scales : p.key_scales) + row;
        if constexpr (VEC) {
            const bool on = sub * 8 < D;
            float f[8] = {};
            if (on) load8(src + sub * 8, f);
            const uint32_t byte = scale_byte<C>(group_max(max_abs8(f), lanes, mask));
            if (on) store_quantized8(dst + sub * 8, f, inverse_scale(byte));
            if (sub == 0) *scale = (uint8_t)byte;
        } else {
            uint32_t m = 0;
            for (int i = sub; i < D; i += lanes) m = max(m, finite_abs_bits(Elem<T>::to_f(src[i])));
            const uint32_t byte = scale_byte<C>(group_max(m, lanes, mask));
            const float inv = inverse_scale(byte);
            for (int i = sub; i < D; i += lanes)
                store_quantized1(dst + i, Elem<T>::to_f(src[i]), inv);
            if (sub == 0) *scale = (uint8_t)byte;
        }
    }
}

// -------------------------------------------------------------- read back
// Flat over 16-value pieces of the listed blocks; the two caches' pieces of a
// thread are in flight together. Pieces never straddle a row.
template <typename T, typename C, int VEC>
__global__ void __launch_bounds__(256) dequantize_blocks_kernel(const DequantParams p) {
    const long long block_values = (long long)p.rows_per_block * p.head_size;
    const long long pieces = block_values / VEC;
    const long long total = pieces * p.num_ids;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total;
         i += (long long)gridDim.x * 256) {
        const long long n = i / pieces;
        const long long at = (i - n * pieces) * VEC;  // value within the block
        const long long blk = load_int(p.ids, p.ids64, n);
        T* ok = reinterpret_cast<T*>(p.key_out) + n * block_values + at;
        T* ov = reinterpret_cast<T*>(p.value_out) + n * block_values + at;
        const bool there = blk >= 0 && blk < p.num_blocks;
        if (blk >= p.num_blocks) flag_status(TLB_STATUS_BAD_BLOCK_ID);
        const long long from = there ? blk * block_values + at : 0;
        const long long row = there ? blk * p.rows_per_block + at / p.head_size : 0;
        if constexpr (VEC == 16) {
            uint4 uk = make_uint4(0, 0, 0, 0), uv = uk;
            uint32_t bk = 0, bv = 0;
            if (there) {
                uk = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(p.key_cache) +
                                                     from);
                uv = *reinterpret_cast<const uint4*>(
                    reinterpret_cast<const uint8_t*>(p.value_cache) + from);
                bk = p.key_scales[row];
                bv = p.value_scales[row];
            }
            const float sk = scale_value(bk), sv = scale_value(bv);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float f[8];
                const uint32_t k0 = half ? uk.z : uk.x, k1 = half ? uk.w : uk.y;
                const uint32_t v0 = half ? uv.z : uv.x, v1 = half ? uv.w : uv.y;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    f[j] = mul_keep(dequantize1<C>(((j < 4 ? k0 : k1) >> (8 * (j & 3))) & 0xff), sk);
                store8(ok + 8 * half, f);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    f[j] = mul_keep(dequantize1<C>(((j < 4 ? v0 : v1) >> (8 * (j & 3))) & 0xff), sv);
                store8(ov + 8 * half, f);
            }
        } else {
            float fk = 0.f, fv = 0.f;
            if (there) {
                fk = mul_keep(dequantize1<C>(reinterpret_cast<const uint8_t*>(p.key_cache)[from]),
                              scale_value(p.key_scales[row]));
                fv = mul_keep(dequantize1<C>(reinterpret_cast<const uint8_t*>(p.value_cache)[from]),
                              scale_value(p.value_scales[row]));
            }
            *ok = Elem<T>::from_f(fk);
            *ov = Elem<T>::from_f(fv);
        }
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
// An item is one row kind (query, key, value) of one token. VEC: `lanes`
// lanes hold a row, 16 values each: lane l < rot/16 the eight values at 8 l and
// their partners at 8 l + rot/2 (so the rotation needs no exchange), the
// others 16 values beyond rot. Otherwise a warp walks the row by element.
template <typename T, typename C>
__device__ __forceinline__ void store_row16(C* cache, uint8_t* scales, long long row, int D, int i0,
                                            int i1, bool on, int sub, const float (&a)[8],
                                            const float (&b)[8], int lanes, uint32_t mask) {
    if constexpr (sizeof(C) == 1) {
        const uint32_t m = on ? max(max_abs8(a), max_abs8(b)) : 0u;
        const uint32_t byte = scale_byte<C>(group_max(m, lanes, mask));
        const float inv = inverse_scale(byte);
        if (on) {
            store_quantized8(cache + row * D + i0, a, inv);
            store_quantized8(cache + row * D + i1, b, inv);
        }
        if (sub == 0) scales[row] = (uint8_t)byte;
    } else if (on) {
        store8(cache + row * D + i0, a);
        store8(cache + row * D + i1, b);
    }
}

template <typename T>
__device__ __forceinline__ float rounded(float x) {
    return Elem<T>::to_f(Elem<T>::from_f(x));
}

enum RowKind { kQuery = 0, kKey = 1, kValue = 2 };

template <typename T, typename C, bool VEC>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const QuantCacheParams p, int lanes) {
    grid_launch_dependents();
    const int per_block = 256 / lanes;
    const int sub = threadIdx.x % lanes;
    const uint32_t mask = group_mask(lanes);
    const int D = p.head_size, rot = p.rot_dim, half = rot / 2;
    const bool with_cache = p.key_cache != nullptr;
    const int per_token = p.num_heads + p.num_kv_heads * (with_cache ? 2 : 1);
    const long long items = p.num_tokens * per_token;
    for (long long it = (long long)blockIdx.x * per_block + threadIdx.x / lanes; it < items;
         it += (long long)gridDim.x * per_block) {
        const long long t = it / per_token;
        int h = (int)(it - t * per_token);
        RowKind kind = kQuery;
        if (h >= p.num_heads) {
            h -= p.num_heads;
            kind = kKey;
            if (h >= p.num_kv_heads) {
                h -= p.num_kv_heads;
                kind = kValue;
            }
        }
        const long long pos = load_int(p.positions, p.positions64, t);
        const T* cs = nullptr;
        if (pos >= 0 && pos < p.cache_rows)
            cs = reinterpret_cast<const T*>(p.cos_sin) + pos * rot;
        else if (kind != kValue)
            flag_status(TLB_STATUS_BAD_POSITION);
        long long row = -1;  // cache row of this item
        if (with_cache && kind != kQuery) {
            row = p.slots ? slot_row(load_int(p.slots, p.slots64, t), p) : table_row(t, pos, p);
            if (row < 0) continue;
            row += (long long)h * p.block_size;
        }
        const T* src;
        T* dst = nullptr;
        if (kind == kQuery) {
            src = reinterpret_cast<const T*>(p.query) + t * p.query_stride + (long long)h * D;
            dst = reinterpret_cast<T*>(p.out) + (t * p.num_heads + h) * D;
        } else if (kind == kKey) {
            src = reinterpret_cast<const T*>(p.key) + t * p.key_stride + (long long)h * D;
            if (!with_cache) dst = reinterpret_cast<T*>(p.key_out) + (t * p.num_kv_heads + h) * D;
        } else {
            src = reinterpret_cast<const T*>(p.value) + t * p.value_stride + (long long)h * D;
        }
        C* cache = reinterpret_cast<C*>(kind == kValue ? p.value_cache : p.key_cache);
        uint8_t* scales = kind == kValue ? p.value_scales : p.key_scales;
        const T* w = reinterpret_cast<const T*>(kind == kQuery ? p.query_weight : p.key_weight);
        if constexpr (VEC) {
            const int pairs = rot / 16;  // lanes that rotate
            const bool on = sub * 16 < D, turn = sub < pairs;
            const int i0 = turn ? 8 * sub : rot + 16 * (sub - pairs);
            const int i1 = turn ? i0 + half : i0 + 8;
            float a[8] = {}, b[8] = {}, wa[8], wb[8], c[8], s[8];
            if (on && kind != kValue) {
                load8(w + i0, wa);
                load8(w + i1, wb);
                if (turn && cs) {
                    load8(cs + i0, c);
                    load8(cs + half + i0, s);
                }
            }
            grid_dependency_wait();
            if (on) {
                load8(src + i0, a);
                load8(src + i1, b);
            }
            if (kind != kValue) {
                float ss = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) ss += a[j] * a[j] + b[j] * b[j];
                ss = group_sum(ss, lanes, mask);
                const float inv = rsqrtf(ss / (float)D + p.eps);
                if (on) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        a[j] = a[j] * inv * wa[j];
                        b[j] = b[j] * inv * wb[j];
                    }
                    if (turn && cs) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            float x, y;
                            rope_pair(a[j], b[j], c[j], s[j], x, y);
                            a[j] = x;
                            b[j] = y;
                        }
                    }
                }
            }
            if (dst) {
                if (on) {
                    store8(dst + i0, a);
                    store8(dst + i1, b);
                }
            } else {
                if constexpr (sizeof(C) == 1) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        a[j] = rounded<T>(a[j]);
                        b[j] = rounded<T>(b[j]);
                    }
                }
                store_row16<T, C>(cache, scales, row, D, i0, i1, on, sub, a, b, lanes, mask);
            }
        } else {
            grid_dependency_wait();
            float inv = 0.f;
            if (kind != kValue) {
                float ss = 0.f;
                for (int i = sub; i < D; i += lanes) {
                    const float x = Elem<T>::to_f(src[i]);
                    ss += x * x;
                }
                inv = rsqrtf(group_sum(ss, lanes, mask) / (float)D + p.eps);
            }
            auto value = [&](int i) -> float {
                float x = Elem<T>::to_f(src[i]);
                if (kind == kValue) return x;
                x = x * inv * Elem<T>::to_f(w[i]);
                if (i >= rot || !cs) return x;
                const bool first = i < half;
                const int j = first ? i + half : i - half, k = first ? i : j;
                const float y = Elem<T>::to_f(src[j]) * inv * Elem<T>::to_f(w[j]);
                float xo, yo;
                rope_pair(first ? x : y, first ? y : x, Elem<T>::to_f(cs[k]),
                          Elem<T>::to_f(cs[half + k]), xo, yo);
                return first ? xo : yo;
            };
            if (dst) {
                for (int i = sub; i < D; i += lanes) dst[i] = Elem<T>::from_f(value(i));
            } else if constexpr (sizeof(C) == 1) {
                uint32_t m = 0;
                for (int i = sub; i < D; i += lanes)
                    m = max(m, finite_abs_bits(rounded<T>(value(i))));
                const uint32_t byte = scale_byte<C>(group_max(m, lanes, mask));
                const float qs = inverse_scale(byte);
                for (int i = sub; i < D; i += lanes)
                    store_quantized1(cache + row * D + i, rounded<T>(value(i)), qs);
                if (sub == 0) scales[row] = (uint8_t)byte;
            } else {
                for (int i = sub; i < D; i += lanes) cache[row * D + i] = Elem<T>::from_f(value(i));
            }
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
// CTAs of 256 threads for `items` items of `lanes` lanes: all of them up to
// eight CTAs per SM, which then stride.
int grid_of(long long items, int lanes) {
    const long long need = (items * lanes + 255) / 256, cap = (long long)sm_count() * 8;
    return (int)(need < cap ? (need > 0 ? need : 1) : cap);
}
// Lanes of a row of `units` units: the power of two that holds them.
int lanes_for(int units) {
    int n = 1;
    while (n < units) n <<= 1;
    return n;
}

template <typename T, typename C>
cudaError_t write_tc(const QuantCacheParams& p, bool vec, cudaStream_t st) {
    const long long rows = p.num_tokens * 2 * p.num_kv_heads;
    if (vec && p.head_size <= 256) {
        const int lanes = lanes_for(p.head_size / 8);
        quantize_write_kernel<T, C, true><<<grid_of(rows, lanes), 256, 0, st>>>(p, lanes);
    } else {
        quantize_write_kernel<T, C, false><<<grid_of(rows, 32), 256, 0, st>>>(p, 32);
    }
    return cudaGetLastError();
}
template <typename T>
cudaError_t write_t(int cache_dtype, const QuantCacheParams& p, bool vec, cudaStream_t st) {
    return cache_dtype == TLB_INT8 ? write_tc<T, int8_t>(p, vec, st) : write_tc<T, E4M3>(p, vec, st);
}

template <typename T, typename C>
cudaError_t dequant_tc(const DequantParams& p, bool vec, cudaStream_t st) {
    const long long values = p.num_ids * p.rows_per_block * p.head_size;
    if (vec)
        dequantize_blocks_kernel<T, C, 16><<<grid_of(values / 16, 1), 256, 0, st>>>(p);
    else
        dequantize_blocks_kernel<T, C, 1><<<grid_of(values, 1), 256, 0, st>>>(p);
    return cudaGetLastError();
}
template <typename T>
cudaError_t dequant_t(int cache_dtype, const DequantParams& p, bool vec, cudaStream_t st) {
    return cache_dtype == TLB_INT8 ? dequant_tc<T, int8_t>(p, vec, st)
                                   : dequant_tc<T, E4M3>(p, vec, st);
}

template <typename T, typename C>
cudaError_t norm_tc(const QuantCacheParams& p, bool vec, cudaStream_t st) {
    const long long rows =
        p.num_tokens * (p.num_heads + p.num_kv_heads * (p.key_cache != nullptr ? 2 : 1));
    vec = vec && p.head_size <= 512;
    const int lanes = vec ? lanes_for(p.head_size / 16) : 32;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid_of(rows, lanes));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.overlap ? 1 : 0;
    if (vec) return cudaLaunchKernelEx(&cfg, qk_norm_rope_kernel<T, C, true>, p, lanes);
    return cudaLaunchKernelEx(&cfg, qk_norm_rope_kernel<T, C, false>, p, lanes);
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
