// 8-bit cache rows: one row (a token of one kv head) is head_dim values of
// e4m3 or int8 and one scale 2^E held as a biased exponent byte (E8M0).
//
// E is the smallest integer with max|x| <= qmax * 2^E (qmax 448 for e4m3, 127
// for int8), so x * 2^-E is exact in fp32 and the stored value is x * 2^-E
// rounded once, to nearest even: the bits depend on no division or rounding
// of a scale. A power of two costs e4m3 nothing (its own exponent takes the
// rest up) and int8 at most one of its seven bits; in exchange the scale is a
// byte instead of four (a 128-wide row reads 129 bytes) and scores fold it in
// as an exponent.
//
// Rows with infinities or NaN: the scale comes from the finite values,
// infinities saturate, NaN stays NaN in e4m3 and becomes 0 in int8.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace tlb {

template <typename T> struct Same {
    using type = T;
};
// Launches that may begin while the kernel before them on the stream ends
// (programmatic stream serialization). Their kernels wait for it
// (grid_dependency_wait) before they touch memory, the decode kernel with its
// `overlap` flag before it touches anything but lengths and tables; what is saved
// is the launch itself. They let the next launch begin (grid_launch_dependents)
// only after that wait: what the next kernel reads early may have been written
// by the kernel before this one, which is then complete.
template <typename... Args>
cudaError_t launch_early(void (*kernel)(Args...), dim3 grid, int threads, size_t smem,
                         cudaStream_t stream, typename Same<Args>::type... args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Storage tag of an e4m3 cache (one byte per value, as int8_t is for int8).
struct E4M3 {
    uint8_t bits;
};
static_assert(sizeof(E4M3) == 1, "one byte per value");

template <typename C> struct Quant8;
template <> struct Quant8<E4M3> {
    static constexpr uint32_t kTopMantissa = 0x600000u;  // 448 = 1.75 * 2^8
    static constexpr int kTopExponent = 8;
};
template <> struct Quant8<int8_t> {
    static constexpr uint32_t kTopMantissa = 0x7E0000u;  // 127 = 1.984375 * 2^6
    static constexpr int kTopExponent = 6;
};

// Multiplication that keeps subnormal operands and results (the build flushes
// them elsewhere): a row may hold values below 2^-126 in bf16 or fp32.
__device__ __forceinline__ float mul_keep(float a, float b) {
    float d;
    asm("mul.rn.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// |x| as ordered bits, 0 for infinities and NaN.
__device__ __forceinline__ uint32_t finite_abs_bits(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}

// Biased exponent byte of the row's scale from the bits of its largest
// finite magnitude: 1 .. 254 (E in [-126, 127]).
template <typename C>
__device__ __forceinline__ uint32_t scale_byte(uint32_t max_bits) {
    // max = (1 + mant / 2^23) * 2^(e - 127); the smallest E with
    // max <= qmax * 2^E is e - 127 - kTopExponent, one more above qmax's mantissa
    const int e = (int)(max_bits >> 23);
    const int byte = e - Quant8<C>::kTopExponent +
                     ((max_bits & 0x7fffffu) > Quant8<C>::kTopMantissa ? 1 : 0);
    return (uint32_t)min(max(byte, 1), 254);
}

// 2^-E as a float (exact; E <= 122 for any finite maximum).
__device__ __forceinline__ float inverse_scale(uint32_t byte) {
    return __uint_as_float((254u - byte) << 23);
}
// 2^E (E >= -126; byte 0, which the writes never store, gives 0 here, and 2^-127 where
// the decode kernel adds exponents: telling it apart there costs 0.7 % of a long case).
__device__ __forceinline__ float scale_value(uint32_t byte) { return __uint_as_float(byte << 23); }

// Four values times 2^-E -> four stored bytes (first in the low byte). kBounded:
// all are finite (and so at most qmax), which spares int8 the conversion unit:
// x * 2^-E + 1.5 * 2^23, rounded once, is the nearest integer, to even, in the low
// bits.
template <typename C, bool kBounded>
__device__ __forceinline__ uint32_t quantize4(float a, float b, float c, float d, float inv) {
    if constexpr (Quant8<C>::kTopExponent == 8) {  // e4m3
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(mul_keep(a, inv), mul_keep(b, inv)),
                                                     __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(mul_keep(c, inv), mul_keep(d, inv)),
                                                     __NV_SATFINITE, __NV_E4M3);
        return lo | (hi << 16);
    } else if constexpr (kBounded) {
        auto one = [inv](float x) {
            float y;  // subnormal x kept, as in mul_keep
            asm("fma.rn.f32 %0, %1, %2, 0f4B400000;" : "=f"(y) : "f"(x), "f"(inv));
            return __float_as_uint(y);
        };
        const uint32_t lo = __byte_perm(one(a), one(b), 0x0040);
        const uint32_t hi = __byte_perm(one(c), one(d), 0x0040);
        return __byte_perm(lo, hi, 0x5410);
    } else {
        auto one = [inv](float x) {
            // NaN converts to 0, infinities to the integer bounds
            return (uint32_t)min(max(__float2int_rn(mul_keep(x, inv)), -127), 127) & 0xffu;
        };
        return one(a) | (one(b) << 8) | (one(c) << 16) | (one(d) << 24);
    }
}

// One stored byte -> its unscaled value.
template <typename C> __device__ __forceinline__ float dequantize1(uint32_t byte);
template <> __device__ __forceinline__ float dequantize1<E4M3>(uint32_t byte) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3);
    return __half2float(__half(h));
}
template <> __device__ __forceinline__ float dequantize1<int8_t>(uint32_t byte) {
    return (float)(int)(int8_t)byte;
}

}  // namespace tlb
