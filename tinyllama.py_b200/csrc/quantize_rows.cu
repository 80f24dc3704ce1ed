// Rows in 8 bits for the block-scaled product: plain rows, the gated activation
// silu(gate) * up, and the RMS norm with the residual's addition.
//
// A row of K values is held as K e4m3 values and a power-of-two scale for each
// 128 of them (the last group of a row may be shorter): the format of the 8-bit
// cache rows, with groups in the place of heads. All three stream their input
// once and are bounded by HBM; what they compute stays in the registers of the
// lanes that read it until it is quantised.
//
// A lane holds eight neighbouring values, so a group is 16 lanes and its largest
// magnitude takes four shuffles; a warp reads 512 bytes of a 16-bit row and
// stores 256 in one access each.
#include <cfloat>

#include "kernels.h"
#include "quant_rows.cuh"

namespace tlb {

namespace {

constexpr int kGroup = 128;
constexpr int kLanes = kGroup / 8;

// Sum that keeps subnormal operands and results (the build flushes them
// elsewhere): the residual of bf16 or fp32 may hold values below 2^-126.
__device__ __forceinline__ float add_keep(float a, float b) {
    float d;
    asm("add.rn.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// Two floats in one register pair: an instruction for both, subnormal values kept.
struct Pair {
    uint64_t v;
    Pair() = default;
    __device__ __forceinline__ Pair(float a, float b) {
        asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    }
    __device__ __forceinline__ void get(float& a, float& b) const {
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
    }
};
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}

// g[i] = silu(g[i]) * u[i] as g / (1 + exp(-g)) * u. The reciprocal of a denominator above
// 2^126 would be 0, and the formula's own reach is 2^128, so it is taken of a quarter of it.
// Gates below -88.7, where exp(-g) passes fp32, give 0. Products keep subnormal values: a far
// one of the other operand makes up for them. Off by at most 4 + 0.7 |g| units of 2^-23, of
// which the exponent's rounding is (1 + |g|) / 2: far below the 8-bit rounding behind it,
// which it moves for about one value in 10^5. In pairs as fast as one by one with neither of
// the two (4853 x 5632 fp16 23.5 us, 23.4); one by one it took 24.9.
template <int N>
__device__ __forceinline__ void silu_mul(float (&g)[N], const float (&u)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const Pair gate(g[i], g[i + 1]);
        float a, b;
        fma2(gate, Pair(-1.44269504f, -1.44269504f), Pair(-2.f, -2.f)).get(a, b);  // 1 / ln 2
        (Pair(exp2f(a), exp2f(b)) + Pair(0.25f, 0.25f)).get(a, b);
        const Pair quarter(__fdividef(1.f, a), __fdividef(1.f, b));
        (gate * (quarter * Pair(0.25f, 0.25f)) * Pair(u[i], u[i + 1])).get(g[i], g[i + 1]);
    }
}

// sum / width, rounded once: the inverse comes as a sum of two floats. The build's default
// division is off by up to 2 ulp where the width is no power of two, which broke ties of
// values that the norm leaves on a border of 8 bits; a rounded one took 0.2 us longer
// (4853 x 896 fp16). The rest may be 0, so an infinite sum stays out of its product.
__device__ __forceinline__ float mean_of(float sum, const RowQuantParams& p) {
    return fmaf(sum, p.inverse_width, fminf(sum, FLT_MAX) * p.inverse_width_rest);
}

// 1 / sqrt(m) as a sum of two floats: rsqrtf and what Newton's step adds to it, from the
// residual 1 - m r^2 with the product's own rounding error taken in. (Sums of the lanes
// in fp64 as well: no fewer values on the other side of a border, 3 to 8 % slower.)
struct InverseRoot {
    float high, low;
    __device__ __forceinline__ explicit InverseRoot(float m) : high(rsqrtf(m)) {
        const float t = m * high, error = fmaf(m, high, -t);
        const float rest = fmaf(-t, high, 1.f) - error * high;
        low = isfinite(high) && high > 0.f ? 0.5f * high * rest : 0.f;
    }
    // x * w / sqrt(m), for values of 16 bits (whose product is exact) rounded once: a row's
    // values are rounded to 8 bits next, and each rounding before that moves some of
    // them over a border (16383 x 4096: 31 to 44 of 67 M, 50 to 190 with one rounding for
    // each step).
    template <int N>
    __device__ __forceinline__ void scale(float (&x)[N], const float (&w)[N]) const {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const Pair v = Pair(x[i], x[i + 1]) * Pair(w[i], w[i + 1]);
            fma2(v, Pair(high, high), v * Pair(low, low)).get(x[i], x[i + 1]);
        }
    }
};

// A row's values are taken this much larger (smaller) where their squares would leave fp32's
// range: a mean below 2^-100 has lost squares below 2^-126, and an infinite one may come from
// finite values. Rows are at most 2^30 wide, so the former's squares then sum to less than
// 2^122, the latter's to less than 2^126. Results do not depend on it. fp16 has no such rows.
template <typename T> __device__ __forceinline__ float range_shift(float mean) {
    if (std::is_same<T, __half>::value || (mean >= 0x1p-100f && mean < INFINITY)) return 1.f;
    return mean < 0x1p-100f ? 0x1p96f : 0x1p-80f;
}
template <int N>
__device__ __forceinline__ void shift(float (&x)[N], float by) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = mul_keep(x[i], by);
}
template <int N>
__device__ __forceinline__ float squares(const float (&x)[N], float sum) {
#pragma unroll
    for (int i = 0; i < N; ++i) sum = fmaf(x[i], x[i], sum);
    return sum;
}

// Eight fp32 values of a lane -> their 8 stored bytes, and the scale byte of the
// 16 lanes' group.
__device__ __forceinline__ uint2 quantize_group(const float (&f)[8], uint32_t mask,
                                                uint32_t& byte) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
    top = group_max<kLanes>(top, mask);
    if (top < 0x7f800000u) {
        byte = scale_byte<E4M3>(top);
    } else {  // infinities or NaN in the group: the scale comes from the others
        byte = scale_byte<E4M3>(group_max<kLanes>(max_finite8(f), mask));
    }
    return quantized8<E4M3, false>(f, inverse_scale(byte));
}

// A plain group's lane: eight elements as read. The magnitudes are compared, and fp16
// values converted, in pairs (as in the cache write).
template <typename T>
__device__ __forceinline__ uint2 quantize_raw(const Raw8<T>& x, uint32_t mask, uint32_t& byte) {
    const uint32_t top = group_top<kLanes, T>(x.top(), mask);
    if (top < 0x7f800000u) {
        byte = scale_byte<E4M3>(top);
        if constexpr (std::is_same<T, __half>::value) {
            if (byte >= 112)  // 2^-E is an fp16 number (E >= -15)
                return quantized8_half<E4M3>(x.u[0],
                                             __half2half2(__float2half_rn(inverse_scale(byte))));
        }
        float f[8];
        x.get(f);
        return quantized8<E4M3, true>(f, inverse_scale(byte));
    }
    float f[8];
    x.get(f);
    byte = scale_byte<E4M3>(group_max<kLanes>(max_finite8(f), mask));
    return quantized8<E4M3, false>(f, inverse_scale(byte));
}

// x / d for x < 2^31 and d < 2^31 by a product with the inverse, rounded up (Granlund and
// Montgomery, Division by invariant integers using multiplication, 1994): 32-bit division
// took a fifth of these kernels' instructions.
struct FastDivisor {
    uint32_t by, inverse;
    int shift;
    FastDivisor() = default;
    explicit FastDivisor(uint32_t d) : by(d), shift(0) {
        while ((1ull << shift) < d) ++shift;
        inverse = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t divide(uint32_t x) const {
        return (__umulhi(x, inverse) + x) >> shift;
    }
};

// ------------------------------------------------- plain rows, gated activation
// Flat over the eight-value pieces of all rows, each row's filled up to whole groups
// (so that a group is half a warp wherever it lies), kSteps pieces of a lane in flight.
// Bounded by HBM and, the gated form, nearly as much by its instructions.
template <typename T, bool kSilu, int kSteps>
__global__ void __launch_bounds__(256) quantize_pieces_kernel(const RowQuantParams p,
                                                              const FastDivisor padded,
                                                              const uint32_t pieces) {
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t mask = group_mask<kLanes>();
    const uint32_t step = gridDim.x * 256 * kSteps, row_pieces = p.width / 8;
    for (uint32_t base = blockIdx.x * 256 * kSteps; base < pieces; base += step) {
        Raw8<T> x[kSteps], u[kSilu ? kSteps : 1];
        long long to[kSteps];  // the piece's place in the result, -1: none
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const uint32_t i = base + s * 256 + threadIdx.x;
            x[s].zero();
            if constexpr (kSilu) u[s].zero();
            const uint32_t r = padded.divide(i), piece = i - r * padded.by;
            to[s] = -1;
            if (i < pieces && piece < row_pieces) {
                to[s] = (long long)r * row_pieces + piece;
                const T* src = reinterpret_cast<const T*>(p.x) + r * p.x_stride + piece * 8;
                x[s].load_stream(src);
                if constexpr (kSilu) u[s].load_stream(src + p.width);
            }
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const uint32_t i = base + s * 256 + threadIdx.x;
            uint32_t byte;
            uint2 q;
            if constexpr (kSilu) {
                float f[8], v[8];
                x[s].get(f);
                u[s].get(v);
                silu_mul(f, v);
                q = quantize_group(f, mask, byte);
            } else {
                q = quantize_raw<T>(x[s], mask, byte);
            }
            if (to[s] >= 0) {
                reinterpret_cast<uint2*>(p.out)[to[s]] = q;
                if ((threadIdx.x & (kLanes - 1)) == 0) p.scales[i / kLanes] = (uint8_t)byte;
            }
        }
    }
}

// ------------------------------------------------------------------- RMS norm
// A row is held by the warps of a CTA, kPieces pieces a lane, between its one read and
// its writes; the warps' sums of squares meet in shared memory. (A warp for each short
// row, eight a CTA, gained nothing: 4853 rows of 896 fp16 5.7 us instead of 6.0, fp32 7.3
// instead of 6.7.)
template <typename T, bool kResidual, int kPieces>
__global__ void rms_norm_kernel(const RowQuantParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    __shared__ float sums[32];
    const int threads = blockDim.x, tid = threadIdx.x;
    const int row_pieces = p.width / 8;
    const uint32_t mask = group_mask<kLanes>();
    const long long r = blockIdx.x;
    Raw8<T> x[kPieces];
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < kPieces; ++s) {
        const int i = tid + s * threads;
        x[s].zero();
        if (i < row_pieces) x[s].load_stream(reinterpret_cast<const T*>(p.x) + r * p.x_stride + i * 8);
    }
    if constexpr (kResidual) {
        Raw8<T> y[kPieces];
#pragma unroll
        for (int s = 0; s < kPieces; ++s) {
            const int i = tid + s * threads;
            y[s].zero();
            if (i < row_pieces)
                y[s].load_stream(reinterpret_cast<const T*>(p.residual) + r * p.residual_stride + i * 8);
        }
#pragma unroll
        for (int s = 0; s < kPieces; ++s) {
            const int i = tid + s * threads;
            float a[8], b[8];
            x[s].get(a);
            y[s].get(b);
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j] = add_keep(a[j], b[j]);
            x[s].set(a);  // the norm is that of the residual as stored
            if (i < row_pieces)
                x[s].store(reinterpret_cast<T*>(p.residual_out) + r * p.residual_out_stride + i * 8);
        }
    }
    // of the CTA's threads, the same bits in all of them
    auto total = [&](float v) {
        v = group_sum<32>(v, 0xffffffffu);
        if (threads > 32) {
            if ((tid & 31) == 0) sums[tid >> 5] = v;
            __syncthreads();
            v = group_sum<32>((tid & 31) < threads / 32 ? sums[tid & 31] : 0.f, 0xffffffffu);
        }
        return v;
    };
#pragma unroll
    for (int s = 0; s < kPieces; ++s) {
        float a[8];
        x[s].get(a);
        sum = squares(a, sum);
    }
    float mean = mean_of(total(sum), p) + p.eps;
    const float by = range_shift<T>(mean);
    if (by != 1.f) {
        sum = 0.f;
#pragma unroll
        for (int s = 0; s < kPieces; ++s) {
            float a[8];
            x[s].get(a);
            shift(a, by);
            sum = squares(a, sum);
        }
        __syncthreads();  // before the sums are written again
        mean = mean_of(total(sum), p) + mul_keep(mul_keep(p.eps, by), by);
    }
    const InverseRoot inv(mean);
#pragma unroll
    for (int s = 0; s < kPieces; ++s) {
        const int i = tid + s * threads;
        float a[8], w[8];
        Raw8<T> wt;
        wt.zero();
        if (i < row_pieces) wt.load(reinterpret_cast<const T*>(p.weight) + i * 8);
        x[s].get(a);
        wt.get(w);
        if (by != 1.f) shift(a, by);
        inv.scale(a, w);
        uint32_t byte;
        const uint2 q = quantize_group(a, mask, byte);
        if (i < row_pieces) {
            reinterpret_cast<uint2*>(p.out)[r * row_pieces + i] = q;
            if ((tid & (kLanes - 1)) == 0)
                p.scales[r * ((row_pieces + kLanes - 1) / kLanes) + i / kLanes] = (uint8_t)byte;
        }
    }
}

// ------------------------------------------------------- any width, any alignment
// A CTA a row, a warp a group, element by element; the norm reads its rows twice. Bounded
// by the instructions that an element takes (16000 x 3001 bf16: plain 50 us, gated 65, norm
// with residual 127; by pieces, at 3000 values a row, 28, 43 and 58). Four groups of a warp
// at once were slower (124, 183, 232: too many registers). Left to itself the compiler gives
// the norm 56 registers and the gated form 38: 173 and 68 us.
constexpr int any_ctas(int op) {
    return op == TLB_ROWS_RMS_NORM ? 5 : op == TLB_ROWS_SILU_AND_MUL ? 8 : 1;
}
template <typename T, int kOp>
__global__ void __launch_bounds__(256, any_ctas(kOp))
    quantize_rows_any_kernel(const RowQuantParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    constexpr bool kNorm = kOp == TLB_ROWS_RMS_NORM, kSilu = kOp == TLB_ROWS_SILU_AND_MUL;
    __shared__ float sums[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = p.width;
    const int groups = (K + kGroup - 1) / kGroup;
    // a lane's values of a group are 32 apart; element i is the same thread's every time,
    // so that it reads back what it stored
    auto load = [&](const T* from, int first, float (&to)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            to[j] = first + 32 * j < K ? Elem<T>::to_f(from[first + 32 * j]) : 0.f;
    };
    for (long long r = blockIdx.x; r < p.num_rows; r += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(p.x) + r * p.x_stride;
        InverseRoot inv(1.f);
        float by = 1.f;
        if constexpr (kNorm) {
            const T* res = reinterpret_cast<const T*>(p.residual);
            T* h = nullptr;
            if (res) {
                res += r * p.residual_stride;
                h = reinterpret_cast<T*>(p.residual_out) + r * p.residual_out_stride;
            }
            float sum = 0.f;
            for (int g = warp; g < groups; g += 8) {
                const int first = g * kGroup + lane;
                float f[4];
                load(x, first, f);
                if (h) {
                    float y[4];
                    load(res, first, y);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const T e = Elem<T>::from_f(add_keep(f[j], y[j]));
                        if (first + 32 * j < K) h[first + 32 * j] = e;
                        f[j] = Elem<T>::to_f(e);
                    }
                }
                sum = squares(f, sum);
            }
            auto total = [&](float v) {
                v = group_sum<32>(v, 0xffffffffu);
                if (lane == 0) sums[warp] = v;
                __syncthreads();
                v = group_sum<32>(lane < 8 ? sums[lane] : 0.f, 0xffffffffu);
                __syncthreads();  // before the next sums
                return v;
            };
            if (h) x = h;
            float mean = mean_of(total(sum), p) + p.eps;
            by = range_shift<T>(mean);
            if (by != 1.f) {
                sum = 0.f;
                for (int g = warp; g < groups; g += 8) {
                    float f[4];
                    load(x, g * kGroup + lane, f);
                    shift(f, by);
                    sum = squares(f, sum);
                }
                mean = mean_of(total(sum), p) + mul_keep(mul_keep(p.eps, by), by);
            }
            inv = InverseRoot(mean);
        }
        for (int g = warp; g < groups; g += 8) {
            const int first = g * kGroup + lane;
            float f[4];
            load(x, first, f);
            if constexpr (kNorm || kSilu) {
                float y[4];
                load(kNorm ? reinterpret_cast<const T*>(p.weight) : x + K, first, y);
                // values past the row's end count neither for a scale (0, or NaN where the
                // root is infinite) nor are they written
                if constexpr (kSilu) {
                    silu_mul(f, y);
                } else {
                    if (by != 1.f) shift(f, by);
                    inv.scale(f, y);
                }
            }
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) m = max(m, finite_abs_bits(f[j]));
            const uint32_t byte = scale_byte<E4M3>(group_max<32>(m, 0xffffffffu));
            const uint32_t q =
                quantize4<E4M3, false>(f[0], f[1], f[2], f[3], inverse_scale(byte));
            uint8_t* out = reinterpret_cast<uint8_t*>(p.out) + r * K;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (first + 32 * j < K) out[first + 32 * j] = (uint8_t)(q >> (8 * j));
            if (lane == 0) p.scales[r * groups + g] = (uint8_t)byte;
        }
    }
}

template <typename T, bool kResidual>
cudaError_t launch_norm(const RowQuantParams& p, int sms, cudaStream_t st) {
    const int pieces = p.width / 8;
    const dim3 grid((unsigned)p.num_rows);
    auto threads = [&](int each) { return ((pieces + each - 1) / each + 31) / 32 * 32; };
    // Many rows of 16 bits: more pieces a lane and fewer lanes a row (16383 x 4096 with
    // residual 83.1 us, 85.2 with two pieces; 16384 x 2048 26.1 and 31.9 with one); fewer
    // rows are better spread (2000 x 4096: 12.0 with two, 12.7 with four), fp32 gains
    // nothing. CTAs that go through several rows took 92 us for the first of these.
    const bool many = sizeof(T) == 2 && p.num_rows >= 24ll * sms;
    if (many && pieces >= 256 && pieces <= 2048)
        return launch_early(rms_norm_kernel<T, kResidual, 4>, grid, threads(4), 0, st, p);
    if (pieces <= 64 || (pieces <= 256 && !many))
        return launch_early(rms_norm_kernel<T, kResidual, 1>, grid, threads(1), 0, st, p);
    if (pieces <= 1024)
        return launch_early(rms_norm_kernel<T, kResidual, 2>, grid, threads(2), 0, st, p);
    return launch_early(rms_norm_kernel<T, kResidual, 4>, grid, threads(4), 0, st, p);
}

// Eight-value pieces of a row's groups, the last of them filled up.
long long padded_pieces(int width) { return (width + kGroup - 1ll) / kGroup * kLanes; }

template <typename T, bool kSilu, int kSteps>
cudaError_t launch_pieces(const RowQuantParams& p, int sms, cudaStream_t st) {
    const long long padded = padded_pieces(p.width), pieces = p.num_rows * padded;
    const long long want = (pieces + 256 * kSteps - 1) / (256 * kSteps), cap = 8ll * sms;
    return launch_early(quantize_pieces_kernel<T, kSilu, kSteps>,
                        dim3((unsigned)(want < cap ? want : cap)), 256, 0, st, p,
                        FastDivisor((uint32_t)padded), (uint32_t)pieces);
}

template <typename T>
cudaError_t launch(int op, const RowQuantParams& p, int sms, bool vec, cudaStream_t st) {
    // rows of the norm that a CTA holds in registers: 4 pieces of up to 512 threads;
    // pieces of the others that 32-bit indexes count
    const bool held = op == TLB_ROWS_RMS_NORM
                          ? p.width <= 16384 && p.num_rows < (1ll << 31)
                          : p.num_rows * padded_pieces(p.width) < (1ll << 31) - (1 << 24);
    if (!vec || !held) {
        const long long rows = p.num_rows < 32ll * sms ? p.num_rows : 32ll * sms;
        return launch_early(op == TLB_ROWS_RMS_NORM ? quantize_rows_any_kernel<T, TLB_ROWS_RMS_NORM>
                            : op == TLB_ROWS_SILU_AND_MUL
                                ? quantize_rows_any_kernel<T, TLB_ROWS_SILU_AND_MUL>
                                : quantize_rows_any_kernel<T, TLB_ROWS_PLAIN>,
                            dim3((unsigned)rows), 256, 0, st, p);
    }
    if (op == TLB_ROWS_RMS_NORM)
        return p.residual ? launch_norm<T, true>(p, sms, st) : launch_norm<T, false>(p, sms, st);
    // 64 bytes of a lane in flight where there are enough pieces (16381 x 4096 fp16 rows
    // 33.1 us, 38.3 with 32 bytes), one piece where more CTAs are worth more (64 x 2048:
    // 1.3 us, 2.0 with four).
    constexpr int kSteps = sizeof(T) == 2 ? 4 : 1, kSiluSteps = (kSteps + 1) / 2;
    const bool few = p.num_rows * padded_pieces(p.width) <= 256ll * 4 * sms;
    if (op == TLB_ROWS_SILU_AND_MUL)
        return few ? launch_pieces<T, true, 1>(p, sms, st)
                   : launch_pieces<T, true, kSiluSteps>(p, sms, st);
    return few ? launch_pieces<T, false, 1>(p, sms, st)
               : launch_pieces<T, false, kSteps>(p, sms, st);
}

}  // namespace

cudaError_t launch_quantize_rows(int dtype, int op, const RowQuantParams& p, int sms, bool vec,
                                 cudaStream_t st) {
    switch (dtype) {
        case TLB_FLOAT16: return launch<__half>(op, p, sms, vec, st);
        case TLB_BFLOAT16: return launch<__nv_bfloat16>(op, p, sms, vec, st);
        default: return launch<float>(op, p, sms, vec, st);
    }
}

}  // namespace tlb
