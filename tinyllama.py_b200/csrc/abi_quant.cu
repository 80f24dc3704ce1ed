// C ABI of the quantised-cache, query/key-norm and scored-attention operators:
// argument checks, path choice and launches (contract in tinyllama_b200.h).
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
bool is_float(int dtype) {
    return dtype == TLB_FLOAT32 || dtype == TLB_FLOAT16 || dtype == TLB_BFLOAT16;
}
bool is_8bit(int dtype) { return dtype == TLB_FLOAT8_E4M3 || dtype == TLB_INT8; }
bool is_index(int dtype) { return dtype == TLB_INT32 || dtype == TLB_INT64; }
int index_bytes(int dtype) { return dtype == TLB_INT64 ? 8 : 4; }
int elem_bytes(int dtype) { return dtype == TLB_FLOAT32 ? 4 : is_8bit(dtype) ? 1 : 2; }

// log2 of a power of two, -1 for other numbers.
int shift_of(int64_t x) {
    for (int i = 0; i < 24; ++i)
        if (x == (1ll << i)) return i;
    return -1;
}

// 16-byte accesses: every listed pointer aligned, every stride a multiple of
// 16 bytes.
bool vec_ok(int dtype, std::initializer_list<const void*> ptrs,
            std::initializer_list<int64_t> strides) {
    for (const void* p : ptrs)
        if (p && !aligned(p, 16)) return false;
    for (int64_t s : strides)
        if (s * elem_bytes(dtype) % 16) return false;
    return true;
}

int cache_checks(const void* key_cache, const void* value_cache, int64_t num_tokens,
                 int64_t num_kv_heads, int64_t head_size, int64_t num_blocks,
                 int64_t block_size) {
    TLB_REQUIRE(num_tokens >= 0, "num_tokens must not be negative");
    TLB_REQUIRE(num_kv_heads > 0 && head_size > 0 && num_blocks > 0 && block_size > 0,
                "cache sizes must be positive");
    TLB_REQUIRE(num_tokens < (1ll << 40) && num_kv_heads < (1 << 16) && head_size < (1 << 16) &&
                    block_size < (1 << 20) && num_blocks < (1ll << 31) &&
                    num_kv_heads * block_size * head_size < (1ll << 31),
                "sizes exceed the supported range");
    TLB_REQUIRE(key_cache && value_cache, "cache pointers must not be null");
    return TLB_OK;
}

}  // namespace

extern "C" {

int tlb_reshape_and_cache_quantized(const tlb_quantized_write_args* args, void* stream) {
    TLB_REQUIRE(args != nullptr, "args must not be null");
    const void* key = args->key;
    const void* value = args->value;
    void* key_cache = args->key_cache;
    void* value_cache = args->value_cache;
    void* key_scales = args->key_scales;
    void* value_scales = args->value_scales;
    const void* slots = args->slots;
    const int64_t num_tokens = args->num_tokens;
    const int64_t num_kv_heads = args->num_kv_heads;
    const int64_t head_size = args->head_size;
    const int64_t num_blocks = args->num_blocks;
    const int64_t block_size = args->block_size;
    const int64_t key_stride = args->key_stride;
    const int64_t value_stride = args->value_stride;
    const int slot_dtype = (int)args->slot_dtype;
    const int dtype = (int)args->dtype;
    const int cache_dtype = (int)args->cache_dtype;
    TLB_REQUIRE(is_float(dtype), "dtype must be float16, bfloat16 or float32");
    TLB_REQUIRE(is_8bit(cache_dtype), "cache dtype must be float8_e4m3 or int8");
    if (int rc = cache_checks(key_cache, value_cache, num_tokens, num_kv_heads, head_size,
                              num_blocks, block_size))
        return rc;
    TLB_REQUIRE(is_index(slot_dtype), "slot_mapping must be int32 or int64");
    TLB_REQUIRE(key_scales && value_scales, "scale pointers must not be null");
    if (num_tokens == 0) return TLB_OK;
    TLB_REQUIRE(key && value && slots, "tensor pointers must not be null");
    const int e = elem_bytes(dtype);
    TLB_REQUIRE(aligned(key, e) && aligned(value, e) && aligned(slots, index_bytes(slot_dtype)),
                "tensor pointers must be aligned to the element size");
    tlb::QuantCacheParams p{};
    p.key = key;
    p.value = value;
    p.key_cache = key_cache;
    p.value_cache = value_cache;
    p.key_scales = static_cast<uint8_t*>(key_scales);
    p.value_scales = static_cast<uint8_t*>(value_scales);
    p.slots = slots;
    p.slots64 = slot_dtype == TLB_INT64;
    p.num_tokens = num_tokens;
    p.key_stride = key_stride;
    p.value_stride = value_stride;
    p.num_blocks = num_blocks;
    p.num_kv_heads = (int)num_kv_heads;
    p.head_size = (int)head_size;
    p.block_size = (int)block_size;
    p.block_shift = shift_of(block_size);
    const bool vec = head_size % 16 == 0 && vec_ok(dtype, {key, value, key_cache, value_cache},
                                                  {key_stride, value_stride});
    return cuda_result(tlb::launch_quantize_write(dtype, cache_dtype, p, vec,
                                                  reinterpret_cast<cudaStream_t>(stream)),
                       "reshape_and_cache_quantized");
}

int tlb_dequantize_blocks(const tlb_dequantize_args* args, void* stream) {
    TLB_REQUIRE(args != nullptr, "args must not be null");
    void* key_out = args->key_out;
    void* value_out = args->value_out;
    const void* key_cache = args->key_cache;
    const void* value_cache = args->value_cache;
    const void* key_scales = args->key_scales;
    const void* value_scales = args->value_scales;
    const void* block_ids = args->block_ids;
    const int64_t num_ids = args->num_ids;
    const int64_t num_kv_heads = args->num_kv_heads;
    const int64_t head_size = args->head_size;
    const int64_t num_blocks = args->num_blocks;
    const int64_t block_size = args->block_size;
    const int id_dtype = (int)args->id_dtype;
    const int dtype = (int)args->dtype;
    const int cache_dtype = (int)args->cache_dtype;
    TLB_REQUIRE(is_float(dtype), "dtype must be float16, bfloat16 or float32");
    TLB_REQUIRE(is_8bit(cache_dtype), "cache dtype must be float8_e4m3 or int8");
    if (int rc = cache_checks(key_cache, value_cache, num_ids, num_kv_heads, head_size, num_blocks,
                              block_size))
        return rc;
    TLB_REQUIRE(is_index(id_dtype), "block_ids must be int32 or int64");
    TLB_REQUIRE(key_scales && value_scales, "scale pointers must not be null");
    if (num_ids == 0) return TLB_OK;
    TLB_REQUIRE(key_out && value_out && block_ids, "tensor pointers must not be null");
    const int e = elem_bytes(dtype);
    TLB_REQUIRE(aligned(key_out, e) && aligned(value_out, e) &&
                    aligned(block_ids, index_bytes(id_dtype)),
                "tensor pointers must be aligned to the element size");
    tlb::DequantParams p{};
    p.key_out = key_out;
    p.value_out = value_out;
    p.key_cache = key_cache;
    p.value_cache = value_cache;
    p.key_scales = static_cast<const uint8_t*>(key_scales);
    p.value_scales = static_cast<const uint8_t*>(value_scales);
    p.ids = block_ids;
    p.ids64 = id_dtype == TLB_INT64;
    p.num_ids = num_ids;
    p.num_blocks = num_blocks;
    p.rows_per_block = (int)(num_kv_heads * block_size);
    p.head_size = (int)head_size;
    const bool vec =
        head_size % 16 == 0 && vec_ok(dtype, {key_out, value_out, key_cache, value_cache}, {});
    return cuda_result(tlb::launch_dequantize_blocks(dtype, cache_dtype, p, vec,
                                                     reinterpret_cast<cudaStream_t>(stream)),
                       "dequantize_blocks");
}

int tlb_read_back_tables(const int32_t* block_tables, const int32_t* context_lens,
                         int64_t num_chunks, int64_t max_blocks, int64_t block_size,
                         int64_t num_blocks, int32_t* ids_out, int32_t* tables_out, void* stream) {
    TLB_REQUIRE(num_chunks >= 0 && max_blocks >= 0, "counts must not be negative");
    TLB_REQUIRE(block_size > 0 && num_blocks > 0, "cache sizes must be positive");
    TLB_REQUIRE(num_chunks < (1ll << 31) && max_blocks < (1ll << 31) && block_size < (1ll << 31) &&
                    num_chunks * max_blocks < (1ll << 31) - 1024 && num_blocks < (1ll << 31),
                "sizes exceed the supported range");
    if (num_chunks * max_blocks == 0) return TLB_OK;
    TLB_REQUIRE(block_tables && context_lens && ids_out && tables_out,
                "tensor pointers must not be null");
    for (const void* q : {(const void*)block_tables, (const void*)context_lens,
                          (const void*)ids_out, (const void*)tables_out})
        TLB_REQUIRE(aligned(q, 4), "tensor pointers must be aligned to the element size");
    return cuda_result(
        tlb::launch_read_back_tables(block_tables, context_lens, (int)num_chunks, (int)max_blocks,
                                     (int)block_size, num_blocks, ids_out, tables_out,
                                     reinterpret_cast<cudaStream_t>(stream)),
        "read_back_tables");
}

int tlb_qk_norm_rotary_embedding_neox(const tlb_qk_norm_rope_args* args, void* stream) {
    TLB_REQUIRE(args != nullptr, "args must not be null");
    void* query_out = args->query_out;
    void* key_out = args->key_out;
    const void* positions = args->positions;
    const void* query = args->query;
    const void* key = args->key;
    const void* value = args->value;
    const void* query_weight = args->query_weight;
    const void* key_weight = args->key_weight;
    void* key_cache = args->key_cache;
    void* value_cache = args->value_cache;
    void* key_scales = args->key_scales;
    void* value_scales = args->value_scales;
    const void* slots = args->slots;
    const int32_t* block_tables = args->block_tables;
    const void* cos_sin_cache = args->cos_sin_cache;
    const int64_t max_blocks_per_seq = args->max_blocks_per_seq;
    const int64_t num_tokens = args->num_tokens;
    const int64_t num_heads = args->num_heads;
    const int64_t num_kv_heads = args->num_kv_heads;
    const int64_t head_size = args->head_size;
    const int64_t cache_rows = args->cache_rows;
    const int64_t rot_dim = args->rot_dim;
    const int64_t num_blocks = args->num_blocks;
    const int64_t block_size = args->block_size;
    const int64_t query_stride = args->query_stride;
    const int64_t key_stride = args->key_stride;
    const int64_t value_stride = args->value_stride;
    const int64_t flags = args->flags;
    const int pos_dtype = (int)args->pos_dtype;
    const int slot_dtype = (int)args->slot_dtype;
    const int dtype = (int)args->dtype;
    const int cache_dtype = (int)args->cache_dtype;
    const float eps = (float)args->eps;
    TLB_REQUIRE(is_float(dtype), "dtype must be float16, bfloat16 or float32");
    TLB_REQUIRE(is_index(pos_dtype), "positions must be int32 or int64");
    TLB_REQUIRE((flags & ~(int64_t)TLB_ROPE_OVERLAP_PREVIOUS) == 0, "unknown flags");
    TLB_REQUIRE(num_tokens >= 0 && num_heads > 0 && num_kv_heads > 0 && head_size > 0,
                "sizes must be positive");
    TLB_REQUIRE(num_tokens < (1ll << 40) && num_heads < (1 << 16) && num_kv_heads < (1 << 16) &&
                    head_size < (1 << 16) && (num_heads + num_kv_heads) * head_size < (1ll << 30),
                "sizes exceed the supported range");
    TLB_REQUIRE(rot_dim > 0 && rot_dim % 2 == 0, "rotary dimension must be even and positive");
    TLB_REQUIRE(rot_dim <= head_size, "rotary dimension must not exceed head_size");
    TLB_REQUIRE(cache_rows > 0, "cos_sin_cache must have at least one row");
    TLB_REQUIRE(eps >= 0.f, "eps must not be negative");
    const bool with_cache = key_cache != nullptr;
    if (with_cache) {
        TLB_REQUIRE(cache_dtype == dtype || is_8bit(cache_dtype),
                    "the caches must have the query dtype, or be float8_e4m3 or int8");
        if (int rc = cache_checks(key_cache, value_cache, num_tokens, num_kv_heads, head_size,
                                  num_blocks, block_size))
            return rc;
        TLB_REQUIRE(!is_8bit(cache_dtype) || (key_scales && value_scales),
                    "8-bit caches need key_scales and value_scales");
        if (slots) {
            TLB_REQUIRE(is_index(slot_dtype), "slot_mapping must be int32 or int64");
        } else {
            TLB_REQUIRE(block_tables && max_blocks_per_seq > 0,
                        "either slots or block_tables must be given");
            TLB_REQUIRE(max_blocks_per_seq < (1ll << 31), "sizes exceed the supported range");
        }
    }
    if (num_tokens == 0) return TLB_OK;
    TLB_REQUIRE(query_out && query && key && positions && cos_sin_cache && query_weight &&
                    key_weight && (with_cache ? value != nullptr : key_out != nullptr),
                "tensor pointers must not be null");
    const int e = elem_bytes(dtype);
    for (const void* q : {(const void*)query_out, (const void*)key_out, query, key, value,
                          query_weight, key_weight, cos_sin_cache})
        TLB_REQUIRE(aligned(q, e), "tensor pointers must be aligned to the element size");
    const int ce = elem_bytes(cache_dtype);
    TLB_REQUIRE(aligned(positions, index_bytes(pos_dtype)) &&
                    (!with_cache || (aligned(key_cache, ce) && aligned(value_cache, ce) &&
                                     (slots ? aligned(slots, index_bytes(slot_dtype))
                                            : aligned(block_tables, 4)))),
                "tensor pointers must be aligned to the element size");
    tlb::QuantCacheParams p{};
    p.out = query_out;
    p.key_out = key_out;
    p.positions = positions;
    p.positions64 = pos_dtype == TLB_INT64;
    p.query = query;
    p.key = key;
    p.value = value;
    p.query_weight = query_weight;
    p.key_weight = key_weight;
    p.cos_sin = cos_sin_cache;
    p.key_cache = key_cache;
    p.value_cache = value_cache;
    p.key_scales = static_cast<uint8_t*>(key_scales);
    p.value_scales = static_cast<uint8_t*>(value_scales);
    p.slots = slots;
    p.slots64 = slot_dtype == TLB_INT64;
    p.block_tables = block_tables;
    p.max_blocks = (int)max_blocks_per_seq;
    p.cache_rows = cache_rows;
    p.num_tokens = num_tokens;
    p.query_stride = query_stride;
    p.key_stride = key_stride;
    p.value_stride = value_stride;
    p.num_blocks = num_blocks;
    p.num_heads = (int)num_heads;
    p.num_kv_heads = (int)num_kv_heads;
    p.head_size = (int)head_size;
    p.rot_dim = (int)rot_dim;
    p.block_size = with_cache ? (int)block_size : 1;
    p.block_shift = shift_of(p.block_size);
    p.eps = eps;
    const bool vec = head_size % 16 == 0 && rot_dim % 16 == 0 &&
                     vec_ok(dtype,
                            {query_out, key_out, query, key, value, query_weight, key_weight,
                             cos_sin_cache, key_cache, value_cache},
                            {query_stride, key_stride, with_cache ? value_stride : 0});
    return cuda_result(tlb::launch_qk_norm_rope(dtype, with_cache ? cache_dtype : dtype, p, vec,
                                                reinterpret_cast<cudaStream_t>(stream)),
                       "qk_norm_rotary_embedding_neox");
}

}  // extern "C"

namespace {

// A cache as a 2-D tensor of bytes-or-halves {head_dim, rows}, read in boxes of
// {128 bytes or a whole shorter row, 2^box_shift rows}. Encoded for each call
// (under a microsecond): nothing is kept by address.
int cache_map(const void* base, int64_t rows, int head_dim, int bytes, int box_shift,
              CUtensorMap* out) {
    auto fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tlb::tensor_map_encoder());
    if (fn == nullptr) return fail(TLB_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const int row = head_dim * bytes, column = row < 128 ? row : 128;
    cuuint64_t dims[2] = {(cuuint64_t)head_dim, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)row};
    cuuint32_t box[2] = {(cuuint32_t)(column / bytes), 1u << box_shift};
    cuuint32_t steps[2] = {1, 1};
    CUresult r = fn(out, bytes == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16,
                    2, const_cast<void*>(base), dims, strides, box, steps,
                    CU_TENSOR_MAP_INTERLEAVE_NONE,
                    column == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(TLB_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return TLB_OK;
}

int sm_count(int* sms) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
    return cuda_result(e, "paged attention (device query)");
}

}  // namespace

extern "C" {

int tlb_paged_attention_scored_workspace_size(int64_t num_heads, int64_t num_kv_heads,
                                              int64_t head_dim, int64_t block_size, int dtype,
                                              int cache_dtype, size_t* bytes_out,
                                              size_t* zeroed_out) {
    TLB_REQUIRE(bytes_out != nullptr && zeroed_out != nullptr,
                "bytes_out and zeroed_out must not be null");
    TLB_REQUIRE(num_heads > 0 && num_kv_heads > 0 && head_dim > 0 && block_size > 0,
                "sizes must be positive");
    TLB_REQUIRE(num_heads % num_kv_heads == 0, "num_heads must be divisible by num_kv_heads");
    *bytes_out = *zeroed_out = 0;
    if (!tlb::scored::fast_supported(dtype, cache_dtype, (int)head_dim, (int)block_size))
        return TLB_OK;
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    const tlb::scored::Workspace w =
        tlb::scored::workspace_layout((int)(num_heads / num_kv_heads), (int)head_dim, sms);
    *bytes_out = w.total;
    *zeroed_out = w.counters_end;
    return TLB_OK;
}

int tlb_paged_attention_scored(const tlb_scored_attention_args* args, void* stream) {
    TLB_REQUIRE(args != nullptr, "args must not be null");
    void* out = args->out;
    const void* query = args->query;
    const void* key_cache = args->key_cache;
    const void* value_cache = args->value_cache;
    const void* key_scales = args->key_scales;
    const void* value_scales = args->value_scales;
    const int32_t* block_tables = args->block_tables;
    const int32_t* seq_lens = args->seq_lens;
    const float* alibi_slopes = args->alibi_slopes;
    void* workspace = args->workspace;
    const int64_t num_seqs = args->num_seqs;
    const int64_t num_heads = args->num_heads;
    const int64_t num_kv_heads = args->num_kv_heads;
    const int64_t head_dim = args->head_dim;
    const int64_t num_blocks = args->num_blocks;
    const int64_t block_size = args->block_size;
    const int64_t max_blocks_per_seq = args->max_blocks_per_seq;
    const int64_t query_stride = args->query_stride;
    const int64_t window = args->window;
    const int64_t flags = args->flags;
    const int dtype = (int)args->dtype;
    const int cache_dtype = (int)args->cache_dtype;
    const float scale = (float)args->scale;
    const float softcap = (float)args->softcap;
    TLB_REQUIRE(is_float(dtype), "dtype must be float16, bfloat16 or float32");
    TLB_REQUIRE(cache_dtype == dtype || is_8bit(cache_dtype),
                "the caches must have the query dtype, or be float8_e4m3 or int8");
    TLB_REQUIRE((flags & ~(int64_t)TLB_ATTN_OVERLAP_PROLOGUE) == 0, "unknown flags");
    TLB_REQUIRE(num_seqs > 0, "query must contain at least one sequence");
    TLB_REQUIRE(num_heads > 0 && num_kv_heads > 0 && head_dim > 0 && num_blocks > 0 &&
                    block_size > 0 && max_blocks_per_seq > 0,
                "sizes must be positive");
    TLB_REQUIRE(num_heads % num_kv_heads == 0, "num_heads must be divisible by num_kv_heads");
    TLB_REQUIRE(head_dim <= 1024, "head_dim must not exceed 1024");
    TLB_REQUIRE(num_heads < (1 << 16) && num_seqs * num_heads < (1ll << 31) &&
                    block_size < (1ll << 24) && max_blocks_per_seq < (1ll << 31) &&
                    max_blocks_per_seq * block_size < (1ll << 31) - 64 && num_blocks < (1ll << 31),
                "sizes exceed the supported range");
    TLB_REQUIRE(window >= 0, "window must not be negative");
    // beyond these its reciprocal or its product with a score leaves fp32
    TLB_REQUIRE(softcap == 0.f || (softcap >= 1e-30f && softcap <= 1e30f),
                "softcap must be 0 or between 1e-30 and 1e30");
    TLB_REQUIRE(out && query && key_cache && value_cache && block_tables && seq_lens,
                "tensor pointers must not be null");
    TLB_REQUIRE(!is_8bit(cache_dtype) || (key_scales && value_scales),
                "8-bit caches need key_scales and value_scales");
    const int e = elem_bytes(dtype), ce = elem_bytes(cache_dtype);
    TLB_REQUIRE(aligned(query, e) && aligned(out, e) && aligned(key_cache, ce) &&
                    aligned(value_cache, ce) && aligned(block_tables, 4) && aligned(seq_lens, 4) &&
                    aligned(alibi_slopes, 4),
                "tensor pointers must be aligned to the element size");
    const size_t workspace_bytes = args->workspace_bytes > 0 ? (size_t)args->workspace_bytes : 0;
    namespace sc = tlb::scored;
    sc::Params p{};
    p.out = out;
    p.query = query;
    p.key_cache = key_cache;
    p.value_cache = value_cache;
    p.key_scales = static_cast<const uint8_t*>(key_scales);
    p.value_scales = static_cast<const uint8_t*>(value_scales);
    p.block_tables = block_tables;
    p.seq_lens = seq_lens;
    p.alibi_slopes = alibi_slopes;
    p.num_blocks = num_blocks;
    p.query_stride = query_stride;
    p.num_seqs = (int)num_seqs;
    p.num_heads = (int)num_heads;
    p.num_kv_heads = (int)num_kv_heads;
    p.group = (int)(num_heads / num_kv_heads);
    p.unit_heads = sc::unit_heads_of(p.group);
    p.head_chunks = (p.group + p.unit_heads - 1) / p.unit_heads;
    p.units_per_seq = p.num_kv_heads * p.head_chunks;
    p.head_dim = (int)head_dim;
    p.block_size = (int)block_size;
    p.block_shift = shift_of(block_size);
    p.max_blocks = (int)max_blocks_per_seq;
    p.max_tokens = (int)(max_blocks_per_seq * block_size);
    p.window = window < p.max_tokens ? (int)window : 0;
    p.overlap = (flags & TLB_ATTN_OVERLAP_PROLOGUE) != 0;
    p.scale = scale;
    p.cap_log2 = softcap * 1.4426950408889634f;
    p.inv_cap = softcap > 0.f ? 1.f / softcap : 0.f;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    // The tensor-core kernel copies rows by TMA, whose coordinates are 32-bit
    // and whose base is 16-byte aligned, and scales four bytes at a time, stores
    // pairs of outputs, and numbers the tiles of a call (with their charges) in
    // 31 bits.
    const int tt = sc::tile_tokens((int)head_dim * ce);
    const long long seen = p.window > 0 ? (long long)p.window + tt : p.max_tokens;
    const long long tiles = (seen + tt - 1) / tt * p.units_per_seq * num_seqs;
    const bool fast =
        sc::fast_supported(dtype, cache_dtype, (int)head_dim, (int)block_size) &&
        aligned(out, 4) && aligned(query, 16) && query_stride % 8 == 0 &&
        aligned(key_cache, 16) && aligned(value_cache, 16) && aligned(key_scales, 4) &&
        aligned(value_scales, 4) &&
        num_blocks * num_kv_heads < (1ll << 31) / block_size && tiles < (1ll << 30);
    if (!fast)
        return cuda_result(sc::launch_generic(dtype, cache_dtype, p, st), "paged attention");
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    const long long units = (long long)p.units_per_seq * num_seqs;
    const long long unit_tiles = tiles / units;
    const int warps = sc::warps_for(p.unit_heads);
    p.aligned = units <= sms && unit_tiles <= (long long)sc::kAlignedTiles * warps;
    const int ctas = p.aligned ? (int)units : sc::ctas_for(units, unit_tiles, p.group, sms);
    // ceil(2^64 / warps)
    p.inv_warps = ~0ull / (unsigned long long)(ctas * warps) + 1;
    // laid out for the whole device whatever the grid: the counters' place, which
    // is zero between calls, is the same for every call
    const sc::Workspace w = sc::workspace_layout(p.group, p.head_dim, sms);
    if (workspace == nullptr || workspace_bytes < w.total || !aligned(workspace, 16))
        return fail(TLB_ERR_WORKSPACE,
                    "this call needs a 16-byte aligned workspace of %zu bytes (got %zu)", w.total,
                    workspace_bytes);
    char* ws = static_cast<char*>(workspace);
    p.counters = reinterpret_cast<unsigned*>(ws);
    p.warp_partials = reinterpret_cast<float4*>(ws + w.warp_partials);
    p.cta_partials = reinterpret_cast<float4*>(ws + w.cta_partials);
    p.cta_ml = reinterpret_cast<float2*>(ws + w.cta_ml);
    p.box_shift = sc::box_shift_of(p.block_size, tt);
    p.wait_limit = tlb::attention_wait_limit();
    CUtensorMap tk, tv;
    const int64_t rows = num_blocks * num_kv_heads * block_size;
    if (int rc = cache_map(key_cache, rows, p.head_dim, ce, p.box_shift, &tk)) return rc;
    if (int rc = cache_map(value_cache, rows, p.head_dim, ce, p.box_shift, &tv)) return rc;
    auto launch = cache_dtype == TLB_FLOAT8_E4M3 ? sc::launch_e4m3
                  : cache_dtype == TLB_INT8      ? sc::launch_int8
                                                 : sc::launch_16bit;
    const cudaError_t err = launch(dtype, p, tk, tv, ctas, st);
    return cuda_result(err, "paged attention");
}

}  // extern "C"
