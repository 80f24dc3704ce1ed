// Product of 8-bit rows with 8-bit weights for any shape and alignment, on the CUDA
// cores: what the tensor-core kernel's copies cannot fetch (rows off 16-byte
// boundaries). A CTA takes a tile of 64 tokens x 64 features, 16 sums a thread;
// the tiles of both operands are widened to fp32 on their way into shared memory,
// and a group's sum is scaled by both exponents at once, so that one scale may be
// far up and the other far down. Its speed was not worked on.
#include "kernels.h"
#include "quant.cuh"

namespace tlb {

namespace {

constexpr int kTile = 64, kDepth = 32, kGroup = 128;

// v * 2^(a + b - 254), NaN where a or b is 255.
__device__ __forceinline__ float scaled(float v, uint32_t a, uint32_t b) {
    return a == 255u || b == 255u ? __uint_as_float(0x7fffffffu) : ldexpf(v, (int)(a + b) - 254);
}

template <typename T>
__global__ void __launch_bounds__(256) product_any_kernel(const ProductParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    __shared__ float xs[kDepth][kTile + 1], ws[kDepth][kTile + 1];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const long long tiles_n = (p.features + kTile - 1) / kTile;
    const long long tiles = (p.num_tokens + kTile - 1) / kTile * tiles_n;
    for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const long long t0 = tile / tiles_n * kTile, n0 = tile % tiles_n * kTile;
        float total[4][4] = {}, acc[4][4] = {};
        for (int k0 = 0; k0 < p.width; k0 += kDepth) {
            for (int i = tid; i < kTile * kDepth; i += 256) {
                const int row = i / kDepth, kk = i % kDepth, k = k0 + kk;
                const long long t = t0 + row, n = n0 + row;
                float a = 0.f, b = 0.f;
                if (k < p.width && t < p.num_tokens)
                    a = dequantize1<E4M3>(p.x[t * p.x_stride + k]);
                if (k < p.width && n < p.features)
                    b = dequantize1<E4M3>(p.weight[n * p.weight_stride + k]);
                xs[kk][row] = a;
                ws[kk][row] = b;
            }
            __syncthreads();
#pragma unroll 4
            for (int kk = 0; kk < kDepth; ++kk) {
                float a[4], b[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[i] = xs[kk][ty + 16 * i];
                    b[i] = ws[kk][tx + 16 * i];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
            }
            __syncthreads();
            if ((k0 + kDepth) % kGroup != 0 && k0 + kDepth < p.width) continue;
            const int g = k0 / kGroup;  // ends here
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const long long t = t0 + ty + 16 * i;
                const uint32_t a = t < p.num_tokens ? p.x_scales[t * p.x_scales_stride + g] : 127u;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const long long n = n0 + tx + 16 * j;
                    const uint32_t b =
                        n < p.features ? p.weight_scales[n / kGroup * p.weight_scales_stride + g]
                                       : 127u;
                    total[i][j] += scaled(acc[i][j], a, b);
                    acc[i][j] = 0.f;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long t = t0 + ty + 16 * i;
            if (t >= p.num_tokens) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const long long n = n0 + tx + 16 * j;
                if (n >= p.features) continue;
                float v = total[i][j];
                if (p.bias) v += Elem<T>::to_f(reinterpret_cast<const T*>(p.bias)[n]);
                reinterpret_cast<T*>(p.out)[t * p.out_stride + n] = Elem<T>::from_f(v);
            }
        }
    }
}

}  // namespace

cudaError_t launch_product_any(int out_dtype, const ProductParams& p, cudaStream_t st) {
    const long long tiles = ((p.num_tokens + kTile - 1) / kTile) * ((p.features + kTile - 1) / kTile);
    const dim3 grid((unsigned)(tiles < (1 << 20) ? tiles : (1 << 20)));
    switch (out_dtype) {
        case TLB_FLOAT16: return launch_early(product_any_kernel<__half>, grid, 256, 0, st, p);
        case TLB_BFLOAT16:
            return launch_early(product_any_kernel<__nv_bfloat16>, grid, 256, 0, st, p);
        default: return launch_early(product_any_kernel<float>, grid, 256, 0, st, p);
    }
}

}  // namespace tlb
