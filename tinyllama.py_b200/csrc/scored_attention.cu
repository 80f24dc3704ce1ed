// Decode attention with scored tokens: the path choice's helpers and the kernel
// for the shapes and types that the tensor-core kernel does not serve (fp32,
// head dims other than 64 and 128, block sizes that are no multiple of eight,
// unaligned tensors).
#include "scored_attention.cuh"

namespace tlb {
namespace scored {

namespace {

constexpr int kWarps = 8, kThreads = 256;

// One CTA per (sequence, query head): eight warps take tokens in turn, a lane
// holds the dims lane + 32 i, everything in fp32. Same scores as the tensor-core
// kernel (scored_attention.cuh).
template <typename QT, typename CT, int NPL>
__global__ void __launch_bounds__(kThreads) generic_kernel(const Params p) {
    extern __shared__ float gsm[];
    __shared__ float m_s[kWarps], l_s[kWarps];
    const int D = p.head_dim, s = blockIdx.x, h = blockIdx.y;
    const int kvh = h / p.group;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    grid_dependency_wait();
    grid_launch_dependents();
    const Span sp = span_of(s, p);
    if (p.seq_lens[s] > p.max_tokens && tid == 0) flag_status(TLB_STATUS_SEQ_TOO_LONG);
    const QT* query = reinterpret_cast<const QT*>(p.query) + (long long)s * p.query_stride +
                      (long long)h * D;
    const CT* kc = reinterpret_cast<const CT*>(p.key_cache);
    const CT* vc = reinterpret_cast<const CT*>(p.value_cache);
    const ScoreMod mod{p.cap_log2, p.inv_cap, p.alibi_slopes != nullptr};
    const float slope = mod.alibi ? p.alibi_slopes[h] * kLog2e : 0.f;
    auto read = [](const CT* c, long long i) -> float {
        if constexpr (sizeof(CT) == 1)
            return dequantize1<CT>(reinterpret_cast<const uint8_t*>(c)[i]);
        else
            return Elem<CT>::to_f(c[i]);
    };
    float q[NPL], acc[NPL], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
        const int d = lane + 32 * i;
        q[i] = d < D ? Elem<QT>::to_f(query[d]) : 0.f;
        acc[i] = 0.f;
    }
    for (int t = sp.first + warp; t < sp.len; t += kWarps) {
        const int b = p.block_of(t);
        const int bid = p.block_tables[(long long)s * p.max_blocks + b];
        if (bid < 0) continue;
        if (bid >= p.num_blocks) {
            if (lane == 0) flag_status(TLB_STATUS_BAD_BLOCK_ID);
            continue;
        }
        const long long row = ((long long)bid * p.num_kv_heads + kvh) * p.block_size +
                              (t - b * p.block_size);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            const int d = lane + 32 * i;
            if (d < D) dot += q[i] * read(kc, row * D + d);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        float ks = 1.f, vs = 1.f;
        if constexpr (sizeof(CT) == 1) {
            ks = scale_value(p.key_scales[row]);
            vs = scale_value(p.value_scales[row]);
        }
        float x = dot * (ks * p.scale);
        x = p.cap_log2 > 0.f ? mod.cap(x) : x * kLog2e;
        x = fmaf(slope, (float)(t - (sp.len - 1)), x);
        const float M = fmaxf(m, x), al = piece_weight(m, M);
        const float w = x == -INFINITY ? 0.f : ex2(x - M);
        l = l * al + w;
        m = M;
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            const int d = lane + 32 * i;
            if (d < D) acc[i] = acc[i] * al + w * (read(vc, row * D + d) * vs);
        }
    }
    if (lane == 0) {
        m_s[warp] = m;
        l_s[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
        const int d = lane + 32 * i;
        if (d < D) gsm[warp * D + d] = acc[i];
    }
    __syncthreads();
    float M = -INFINITY;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, m_s[w]);
    float L = 0.f;
    for (int w = 0; w < kWarps; ++w) L += piece_weight(m_s[w], M) * l_s[w];
    QT* out = reinterpret_cast<QT*>(p.out) + ((long long)s * p.num_heads + h) * D;
    for (int d = tid; d < D; d += kThreads) {
        float a = 0.f;
        for (int w = 0; w < kWarps; ++w) a += piece_weight(m_s[w], M) * gsm[w * D + d];
        out[d] = Elem<QT>::from_f(L > 0.f || L != L ? a / L : 0.f);
    }
}

template <typename QT, typename CT>
cudaError_t generic_tc(const Params& p, cudaStream_t st) {
    const dim3 grid(p.num_seqs, p.num_heads);
    const size_t smem = (size_t)kWarps * p.head_dim * sizeof(float);
    return p.head_dim <= 128 ? launch_early(generic_kernel<QT, CT, 4>, grid, kThreads, smem, st, p)
                             : launch_early(generic_kernel<QT, CT, 32>, grid, kThreads, smem, st, p);
}
template <typename QT>
cudaError_t generic_t(int cache_dtype, const Params& p, cudaStream_t st) {
    if (cache_dtype == TLB_INT8) return generic_tc<QT, int8_t>(p, st);
    if (cache_dtype == TLB_FLOAT8_E4M3) return generic_tc<QT, E4M3>(p, st);
    return generic_tc<QT, QT>(p, st);
}

}  // namespace

bool fast_supported(int dtype, int cache_dtype, int head_dim, int block_size) {
    return (dtype == TLB_FLOAT16 || dtype == TLB_BFLOAT16) &&
           (cache_dtype == dtype || cache_dtype == TLB_INT8 || cache_dtype == TLB_FLOAT8_E4M3) &&
           (head_dim == 64 || head_dim == 128) && block_size % 8 == 0;
}

// Units of 16 heads read a kv head's rows once for all of them, units of 8 run
// more warps with less to hold. 128 sequences of 500-3000 tokens, one kv head of
// 128, bf16 over e4m3: groups of 16 take 30.8 us as one unit and 30.9 us as two
// (fp16 over int8: 32.9 and 35.3), groups of 24 take 43.0 us as 16 + 8 and 39.0 us
// as 8 + 8 + 8.
int unit_heads_of(int group) {
    const int rest = group % 16;
    return group <= 8 ? group : rest > 0 && rest <= 8 ? 8 : group < 16 ? group : 16;
}

int box_shift_of(int block_size, int tile) {
    int n = 3;
    while ((2 << n) <= tile && block_size % (2 << n) == 0) ++n;
    return n;
}

int ctas_for(long long units, long long unit_tiles, int group, int sms) {
    const int warps = warps_for(unit_heads_of(group));
    const long long n = (units * unit_tiles + warps - 1) / warps;
    const long long cap = units < sms ? units * kMaxShares < sms ? units * kMaxShares : sms : sms;
    return (int)(n < 1 ? 1 : n < cap ? n : cap);
}

Workspace workspace_layout(int group, int head_dim, int ctas) {
    const int heads = unit_heads_of(group) <= 8 ? 8 : 16;
    const size_t frags = (size_t)heads / 8 * (head_dim / 16) * 32 * sizeof(float4);
    Workspace w;
    w.counters_end = ((size_t)ctas * sizeof(unsigned) + 255) / 256 * 256;
    w.warp_partials = w.counters_end;
    w.cta_partials = w.warp_partials + (size_t)ctas * warps_for(heads) * frags;
    w.cta_ml = w.cta_partials + 2 * (size_t)ctas * frags;
    w.total = w.cta_ml + 2 * (size_t)ctas * heads * sizeof(float2);
    return w;
}

cudaError_t launch_generic(int dtype, int cache_dtype, const Params& p, cudaStream_t stream) {
    switch (dtype) {
        case TLB_FLOAT32: return generic_t<float>(cache_dtype, p, stream);
        case TLB_FLOAT16: return generic_t<__half>(cache_dtype, p, stream);
        default: return generic_t<__nv_bfloat16>(cache_dtype, p, stream);
    }
}

}  // namespace scored
}  // namespace tlb
