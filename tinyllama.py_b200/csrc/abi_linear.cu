// C ABI of the 8-bit rows and their product: argument checks, path choice and
// launches (contract in tinyllama_b200.h).
#include <cstdarg>
#include <cstdio>
#include <initializer_list>

#include <cudaTypedefs.h>

#include "kernels.h"
#include "tinyllama_b200.h"

namespace {

int fail(int code, const char* fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    tlb::set_last_error(buf);
    return code;
}
int cuda_result(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return TLB_OK;
    return fail(TLB_ERR_CUDA, "launching %s: %s (%s)", what, cudaGetErrorString(e),
                cudaGetErrorName(e));
}

#define TLB_REQUIRE(cond, ...)                                           \
    do {                                                                 \
        if (!(cond)) return fail(TLB_ERR_INVALID_ARGUMENT, __VA_ARGS__); \
    } while (0)

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
bool is_float(int64_t dtype) {
    return dtype == TLB_FLOAT32 || dtype == TLB_FLOAT16 || dtype == TLB_BFLOAT16;
}
int elem_bytes(int64_t dtype) { return dtype == TLB_FLOAT32 ? 4 : 2; }

int sm_count(int* sms) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
    return cuda_result(e, "a device query");
}

// Whether a call that writes rows `out` (of one CTA each) while it reads rows `in` reads what
// it may have written: rows are the same ones, or have no byte in common. In bytes.
struct Rows {
    int64_t at, count, stride, width;
};
bool rows_clash(const Rows& in, const Rows& out) {
    using wide = __int128;
    if (in.at == out.at && in.count == out.count && in.width == out.width &&
        (in.count == 1 || in.stride == out.stride))
        return false;
    const wide in_last = in.at + (wide)(in.count - 1) * in.stride;
    const wide out_last = out.at + (wide)(out.count - 1) * out.stride;
    auto low = [](wide a, wide b) { return a < b ? a : b; };
    auto high = [](wide a, wide b) { return a < b ? b : a; };
    if (high(in.at, in_last) + in.width <= low(out.at, out_last) ||
        high(out.at, out_last) + out.width <= low(in.at, in_last))
        return false;
    const wide step = in.stride < 0 ? -(wide)in.stride : in.stride;
    if (in.count > 1 && out.count > 1 && in.stride == out.stride && step > 0) {
        // parts of the same wider rows: one place of the row decides
        const wide away = (((wide)out.at - in.at) % step + step) % step;
        return away < in.width || away > step - out.width;
    }
    // row by row of `out`: the first row of `in` (from its lowest) that ends behind its begin
    const wide first = low(in.at, in_last);
    for (int64_t r = 0; r < out.count; ++r) {
        const wide begin = out.at + (wide)r * out.stride;
        wide j = 0;
        if (step > 0 && begin - first >= in.width) j = (begin - first - in.width) / step + 1;
        if (j < in.count && first + j * step < begin + out.width &&
            first + j * step + in.width > begin)
            return true;
    }
    return false;
}

// Rows of bytes or 16-bit elements as a 2-D tensor {width, rows}, read or written in
// boxes of {box_width, box_rows}, swizzled by rows of a box, zeros past the ends.
// Encoded for each call (under a microsecond): nothing is kept by address.
int rows_map(const void* base, int64_t rows, int64_t width, int64_t stride_bytes, int bytes,
             int box_width, int box_rows, CUtensorMap* out) {
    auto fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tlb::tensor_map_encoder());
    if (fn == nullptr) return fail(TLB_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)stride_bytes};
    cuuint32_t box[2] = {(cuuint32_t)box_width, (cuuint32_t)box_rows};
    cuuint32_t steps[2] = {1, 1};
    CUresult r = fn(out, bytes == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16,
                    2, const_cast<void*>(base), dims, strides, box, steps,
                    CU_TENSOR_MAP_INTERLEAVE_NONE,
                    box_width * bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(TLB_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return TLB_OK;
}
}  // namespace

extern "C" {

int tlb_quantize_rows(const tlb_quantize_rows_args* args, void* stream) {
    TLB_REQUIRE(args != nullptr, "args must not be null");
    const tlb_quantize_rows_args& a = *args;
    TLB_REQUIRE(a.op == TLB_ROWS_PLAIN || a.op == TLB_ROWS_SILU_AND_MUL ||
                    a.op == TLB_ROWS_RMS_NORM,
                "unknown op");
    TLB_REQUIRE(is_float(a.dtype), "dtype must be float16, bfloat16 or float32");
    TLB_REQUIRE(a.num_rows >= 0, "num_rows must not be negative");
    TLB_REQUIRE(a.width > 0, "width must be positive");
    TLB_REQUIRE(a.width < (1ll << 30) && a.num_rows <= (1ll << 46) / a.width,
                "sizes exceed the supported range");
    const bool norm = a.op == TLB_ROWS_RMS_NORM;
    TLB_REQUIRE(norm || (!a.residual && !a.weight), "residual and weight belong to the norm");
    TLB_REQUIRE(!norm || a.eps >= 0, "eps must not be negative");
    if (a.num_rows == 0) return TLB_OK;
    TLB_REQUIRE(a.out && a.scales && a.x && (!norm || a.weight) && (!a.residual || a.residual_out),
                "tensor pointers must not be null");
    const int e = elem_bytes(a.dtype);
    bool vec = a.width % 8 == 0 && aligned(a.out, 8);
    const void* h = a.residual ? a.residual_out : nullptr;
    for (const void* p : {a.x, a.residual, a.weight, h}) {
        TLB_REQUIRE(!p || aligned(p, e), "tensor pointers must be aligned to the element size");
        vec = vec && (!p || aligned(p, 16));
    }
    vec = vec && a.x_stride * e % 16 == 0 &&
          (!a.residual || (a.residual_stride * e % 16 == 0 && a.residual_out_stride * e % 16 == 0));
    if (a.residual) {
        TLB_REQUIRE(a.num_rows < 2 || a.residual_out_stride >= a.width ||
                        a.residual_out_stride <= -a.width,
                    "residual_out's rows overlap");
        const int64_t w = a.width * e;
        auto at = [](const void* ptr) { return (int64_t)reinterpret_cast<uintptr_t>(ptr); };
        const Rows written{at(a.residual_out), a.num_rows, a.residual_out_stride * e, w};
        TLB_REQUIRE(!rows_clash({at(a.x), a.num_rows, a.x_stride * e, w}, written) &&
                        !rows_clash({at(a.residual), a.num_rows, a.residual_stride * e, w}, written) &&
                        !rows_clash({at(a.weight), 1, 0, w}, written),
                    "residual_out must be x or residual itself, or share no memory with the inputs");
    }
    tlb::RowQuantParams p{};
    p.out = a.out;
    p.scales = static_cast<uint8_t*>(a.scales);
    p.residual_out = a.residual_out;
    p.x = a.x;
    p.residual = a.residual;
    p.weight = a.weight;
    p.num_rows = a.num_rows;
    p.x_stride = a.x_stride;
    p.residual_stride = a.residual_stride;
    p.residual_out_stride = a.residual_out_stride;
    p.width = (int)a.width;
    p.eps = (float)a.eps;
    const double inverse = 1.0 / (double)a.width;
    p.inverse_width = (float)inverse;
    p.inverse_width_rest = (float)(inverse - p.inverse_width);
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    return cuda_result(tlb::launch_quantize_rows((int)a.dtype, (int)a.op, p, sms, vec,
                                                 reinterpret_cast<cudaStream_t>(stream)),
                       "quantize_rows");
}

int tlb_matmul_quantized(const tlb_matmul_quantized_args* args, void* stream) {
    TLB_REQUIRE(args != nullptr, "args must not be null");
    const tlb_matmul_quantized_args& a = *args;
    TLB_REQUIRE(is_float(a.out_dtype), "out dtype must be float16, bfloat16 or float32");
    TLB_REQUIRE(a.num_tokens >= 0 && a.features >= 0, "num_tokens and features must not be negative");
    TLB_REQUIRE(a.width > 0, "width must be positive");
    TLB_REQUIRE(a.num_tokens < (1ll << 31) - 1024 && a.features < (1ll << 31) - 1024 &&
                    a.width < (1ll << 30),
                "sizes exceed the supported range");
    if (a.num_tokens == 0 || a.features == 0) return TLB_OK;
    TLB_REQUIRE(a.out && a.x && a.x_scales && a.weight && a.weight_scales,
                "tensor pointers must not be null");
    TLB_REQUIRE(a.num_tokens < 2 || a.out_stride >= a.features || a.out_stride <= -a.features,
                "out's rows overlap");
    const int e = elem_bytes(a.out_dtype);
    TLB_REQUIRE(aligned(a.out, e) && (!a.bias || aligned(a.bias, e)),
                "tensor pointers must be aligned to the element size");
    tlb::ProductParams p{};
    p.out = a.out;
    p.x = static_cast<const uint8_t*>(a.x);
    p.x_scales = static_cast<const uint8_t*>(a.x_scales);
    p.weight = static_cast<const uint8_t*>(a.weight);
    p.weight_scales = static_cast<const uint8_t*>(a.weight_scales);
    p.bias = a.bias;
    p.num_tokens = a.num_tokens;
    p.features = a.features;
    p.x_stride = a.x_stride;
    p.x_scales_stride = a.x_scales_stride;
    p.weight_stride = a.weight_stride;
    p.weight_scales_stride = a.weight_scales_stride;
    p.out_stride = a.out_stride;
    p.width = (int)a.width;
    const auto st = reinterpret_cast<cudaStream_t>(stream);
    // A row's stride only counts where there is a second row.
    const int64_t x_stride = a.num_tokens > 1 ? a.x_stride : (a.width + 15) / 16 * 16;
    const int64_t w_stride = a.features > 1 ? a.weight_stride : (a.width + 15) / 16 * 16;
    // wider rows would take a tile longer than the bound of its waits (10 ms at 2^22)
    const bool tiled = a.width <= (1 << 22) && aligned(a.x, 16) && aligned(a.weight, 16) && x_stride % 16 == 0 &&
                       w_stride % 16 == 0 && x_stride >= a.width && w_stride >= a.width;
    if (tiled) {
        int sms = 0;
        if (int rc = sm_count(&sms)) return rc;
        const int64_t out_stride = a.num_tokens > 1 ? a.out_stride : (a.features + 7) / 8 * 8;
        const tlb::ProductPlan plan =
            tlb::plan_product(a.num_tokens, a.features, a.width, e == 2, sms);
        const bool tma_out = plan.pieces && aligned(a.out, 16) && out_stride % 8 == 0 &&
                             out_stride >= a.features;
        CUtensorMap map_w, map_x, map_out{};
        if (int rc = rows_map(a.weight, a.features, a.width, w_stride, 1, 128, 128, &map_w)) return rc;
        if (int rc = rows_map(a.x, a.num_tokens, a.width, x_stride, 1, 128,
                              plan.pair ? plan.tile_tokens / 2 : plan.tile_tokens, &map_x))
            return rc;
        if (tma_out)
            if (int rc = rows_map(a.out, a.num_tokens, a.features, out_stride * 2, 2, 32,
                                  plan.tile_tokens % 32 == 0 ? 32 : 16, &map_out))
                return rc;
        return cuda_result(
            tlb::launch_product((int)a.out_dtype, p, plan, map_w, map_x, map_out, tma_out,
                                tlb::attention_wait_limit(), st),
            "matmul_quantized");
    }
    return cuda_result(
        tlb::launch_product_any((int)a.out_dtype, p, st), "matmul_quantized");
}

}  // extern "C"
