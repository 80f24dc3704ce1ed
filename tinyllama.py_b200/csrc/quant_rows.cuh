// Rows of fp16, bf16 or fp32 values on their way to 8 bits: eight elements of a
// lane as read, their largest magnitude, and the reductions of a group of lanes.
// Shared by the kernels that quantise cache rows and those that quantise
// activations.
#pragma once

#include <type_traits>

#include "quant.cuh"

namespace tlb {

// Of two words of elements the larger magnitudes, NaN kept.
template <typename T> __device__ __forceinline__ uint32_t max_top(uint32_t a, uint32_t b) {
    uint32_t m;
    if constexpr (std::is_same<T, __half>::value)
        asm("{\n\t.reg .b32 x, y;\n\tabs.f16x2 x, %1;\n\tabs.f16x2 y, %2;\n\t"
            "max.NaN.f16x2 %0, x, y;\n\t}" : "=r"(m) : "r"(a), "r"(b));
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm("{\n\t.reg .b32 x, y;\n\tabs.bf16x2 x, %1;\n\tabs.bf16x2 y, %2;\n\t"
            "max.NaN.bf16x2 %0, x, y;\n\t}" : "=r"(m) : "r"(a), "r"(b));
    else
        m = max(a & 0x7fffffffu, b & 0x7fffffffu);
    return m;
}
// fp32 bits of the largest magnitude of such a word: infinities and NaN come
// above all numbers.
template <typename T> __device__ __forceinline__ uint32_t top_bits(uint32_t m) {
    if constexpr (sizeof(T) == 2) {
        const uint16_t h = (uint16_t)max(m & 0xffffu, m >> 16);
        T e;
        memcpy(&e, &h, 2);
        return __float_as_uint(Elem<T>::to_f(e)) & 0x7fffffffu;
    } else {
        return m;
    }
}

// Eight elements, as read: 16 bytes of half types, 32 of fp32.
template <typename T> struct Raw8 {
    static constexpr int N = 8 * sizeof(T) / 16;
    uint4 u[N];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    // read once, by one SM
    __device__ __forceinline__ void load_stream(const T* p) {
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        const T* e = reinterpret_cast<const T*>(u);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = Elem<T>::to_f(e[i]);
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
        if constexpr (sizeof(T) == 2) {
            u[0] = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]),
                              pack2<T>(f[6], f[7]));
        } else {
            T* e = reinterpret_cast<T*>(u);
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = f[i];
        }
    }
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int i = 0; i < N; ++i) reinterpret_cast<uint4*>(p)[i] = u[i];
    }
    __device__ __forceinline__ void store_stream(T* p) const {
#pragma unroll
        for (int i = 0; i < N; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, u[i]);
    }
    // The largest magnitude, for half types one of the even and one of the odd
    // elements packed; NaN where there is one.
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) m = max_top<T>(m, w[k]);
        }
        return m;
    }
};

__device__ __forceinline__ uint32_t max_finite8(const float (&f)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, finite_abs_bits(f[i]));
    return m;
}

template <typename C, bool kBounded>
__device__ __forceinline__ uint2 quantized8(const float (&f)[8], float inv) {
    uint2 u;
    u.x = quantize4<C, kBounded>(f[0], f[1], f[2], f[3], inv);
    u.y = quantize4<C, kBounded>(f[4], f[5], f[6], f[7], inv);
    return u;
}

// fp16 values scaled and converted in pairs. The product with 2^-E is exact where
// it is a normal fp16 number; below 2^-14 it may be rounded, but then the
// stored value is 0 either way (e4m3 rounds to 0 up to 2^-10, int8 up to 1/2).
// int8: x * 2^-E + 1.5 * 2^10 is the nearest integer, to even, in the low bits.
template <typename C>
__device__ __forceinline__ uint2 quantized8_half(const uint4& u, __half2 inv) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 x = *reinterpret_cast<const __half2*>(&w[i]);
        if constexpr (Quant8<C>::kTopExponent == 8) {  // e4m3
            const __half2 y = __hmul2(x, inv);
            q[i] = __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(y), __NV_SATFINITE, __NV_E4M3);
        } else {
            const __half2 y = __hfma2(x, inv, __float2half2_rn(1536.f));
            q[i] = *reinterpret_cast<const uint32_t*>(&y);
        }
    }
    if constexpr (Quant8<C>::kTopExponent == 8)
        return make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
    else
        return make_uint2(__byte_perm(q[0], q[1], 0x6420), __byte_perm(q[2], q[3], 0x6420));
}

template <typename C>
__device__ __forceinline__ void store_quantized1(C* dst, float x, float inv) {
    *reinterpret_cast<uint8_t*>(dst) = (uint8_t)quantize4<C, false>(x, 0.f, 0.f, 0.f, inv);
}

// Over the LANES (a power of two) lanes of a group, which `mask` names.
template <int LANES>
__device__ __forceinline__ uint32_t group_max(uint32_t v, uint32_t mask) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(mask, v, o));
    return v;
}
template <int LANES, typename T>
__device__ __forceinline__ uint32_t group_top(uint32_t v, uint32_t mask) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = max_top<T>(v, __shfl_xor_sync(mask, v, o));
    return top_bits<T>(v);
}
template <int LANES>
__device__ __forceinline__ float group_sum(float v, uint32_t mask) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
    return v;
}
// A row's lane's two pieces quantised, and the row's scale byte, from the group's
// maximum (group_top).
template <typename T, typename C, int LANES>
__device__ __forceinline__ uint32_t quantize_pieces(const Raw8<T>& x0, const Raw8<T>& x1,
                                                    uint32_t top, uint32_t mask, uint2& q0,
                                                    uint2& q1) {
    const uint32_t byte = scale_byte<C>(top);
    if constexpr (std::is_same<T, __half>::value) {
        // finite rows whose 2^-E is an fp16 number (E >= -15)
        if (top < 0x7f800000u && byte >= 112) {
            const __half2 inv = __half2half2(__float2half_rn(inverse_scale(byte)));
            q0 = quantized8_half<C>(x0.u[0], inv);
            q1 = quantized8_half<C>(x1.u[0], inv);
            return byte;
        }
    }
    float a[8], b[8];
    x0.get(a);
    x1.get(b);
    if (top < 0x7f800000u) {
        q0 = quantized8<C, true>(a, inverse_scale(byte));
        q1 = quantized8<C, true>(b, inverse_scale(byte));
        return byte;
    }
    const uint32_t finite = scale_byte<C>(group_max<LANES>(max(max_finite8(a), max_finite8(b)), mask));
    q0 = quantized8<C, false>(a, inverse_scale(finite));
    q1 = quantized8<C, false>(b, inverse_scale(finite));
    return finite;
}
template <int LANES> __device__ __forceinline__ uint32_t group_mask() {
    constexpr uint32_t ones = LANES == 32 ? 0xffffffffu : (1u << (LANES & 31)) - 1u;
    return ones << ((threadIdx.x & 31) / LANES * LANES);
}

// (quotient, remainder) by a positive 32-bit divisor; 32-bit division when the
// dividend fits, a quarter of the instructions.
__device__ __forceinline__ long long divide(long long x, int by, int& rest) {
    if (x < (1ll << 32)) {
        const unsigned q = (unsigned)x / (unsigned)by;
        rest = (int)((unsigned)x - q * (unsigned)by);
        return q;
    }
    const long long q = x / by;
    rest = (int)(x - q * by);
    return q;
}

}  // namespace tlb
