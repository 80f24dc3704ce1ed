// Internal launch interface between the C ABI (abi.cu) and the kernel files.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace tlb {

// Message returned by tlb_last_error() on this thread (defined in abi.cu).
void set_last_error(const char* msg);

// The driver's tensor-map encoder (null when it has none) and the probe limit
// that tlb_attention_set_wait_limit holds (abi.cu).
void* tensor_map_encoder();
unsigned attention_wait_limit();

// The argument checks and path choice of tlb_paged_attention, without
// launching (abi.cu). On TLB_OK, `total` is the workspace the call will use
// and `zeroed` the prefix that must be zero when it starts; both are 0 when
// the kernel that serves the call needs no workspace. No CUDA call beyond
// device and occupancy queries.
int attention_workspace_plan(const void* out, const void* query, const void* key_cache,
                             const void* value_cache, const int32_t* block_tables,
                             const int32_t* seq_lens, int64_t num_seqs, int64_t num_heads,
                             int64_t num_kv_heads, int64_t head_dim, int64_t num_blocks,
                             int64_t block_size, int64_t max_blocks_per_seq, int dtype,
                             unsigned flags, size_t* total, size_t* zeroed);

// Marks the allocation-free entry point's static scratch on `dev` as not
// known to be zero (static_scratch.cu), so its next call clears it.
void no_alloc_scratch_dirty(int dev);

// ------------------------------------------------------------ attention
namespace attn {

constexpr int kConsumerWarps = 4;   // warps that run the mma / softmax
constexpr int kTileRows = 16;       // tokens per warp tile (mma k / n extent)
constexpr int kStageRows = kConsumerWarps * kTileRows;  // tokens per pipeline stage
constexpr int kGMax = 16;           // largest query-head group on the tensor-core path
#ifndef TLB_ATTN_CTAS_PER_SM
#define TLB_ATTN_CTAS_PER_SM 2
#endif
// Persistent grid: at most this many CTAs per SM (also sizes the workspace).
constexpr int kMaxCtasPerSm = TLB_ATTN_CTAS_PER_SM;
constexpr int kWorkspaceHeader = 256;
// Fewest context tokens (per kv head) a CTA of the tensor-core path is given
// before another CTA joins: below this, a split's merge costs more than the
// parallelism saves.
#ifndef TLB_ATTN_MIN_TOKENS
#define TLB_ATTN_MIN_TOKENS 128
#endif
// Work items per CTA of the grid the partial-result slots are sized for: one
// static range per CTA plus at most two tail chunks per CTA.
constexpr int kItemsPerCta = 3;

struct TcParams {
    void* out;
    const void* query;
    const int32_t* block_tables;
    const int32_t* seq_lens;
    float* ws_o;              // [2 * grid][gpad][head_dim] unnormalised partial outputs
    float* ws_ml;             // [2 * grid][gpad][2] (running max, running sum) per partial
    unsigned int* counters;   // [num_seqs * num_kv_heads] arrival counters (self-resetting)
    unsigned int* sched;      // [2] tail-chunk counter, finished-CTA counter (self-resetting)
    long long num_blocks;
    int num_seqs;
    int num_heads;
    int num_kv_heads;
    int group;                // num_heads / num_kv_heads
    int block_size;
    int max_blocks;
    int min_tokens;           // fewest tokens (per kv head) a CTA is given before more join
    float scale_log2;         // softmax scale * log2(e)
    unsigned wait_limit;      // mbarrier probes before a pipeline wait gives up
    // Fused decode step (cos_sin != nullptr): the new token of sequence s sits
    // at position seq_lens[s] - 1. `query` is then the raw query, rotated in
    // the kernel (NeoX, rot_dim == head_dim); the CTA that reads a sequence's
    // last block first writes that kv head's rotated key and its value into
    // the caches there (and the rotated key back into `key_new`).
    const void* cos_sin;      // [cache_rows, head_dim]: cos | sin halves
    long long cache_rows;
    void* key_new;            // [num_seqs, key_stride] raw key, rotated in place
    const void* value_new;    // [num_seqs, value_stride]
    long long key_stride;     // elements between tokens
    long long value_stride;
    void* key_cache;          // the caches, for the new rows' stores
    void* value_cache;
};

struct GenericParams {
    void* out;
    const void* query;
    const void* key_cache;
    const void* value_cache;
    const int32_t* block_tables;
    const int32_t* seq_lens;
    long long num_blocks;
    int num_seqs;
    int num_heads;
    int num_kv_heads;
    int group;
    int head_dim;
    int block_size;
    int max_blocks;
    float scale_log2;
};

// Returns true when the tensor-core path serves this shape / dtype.
bool tc_supported(int dtype, int head_dim, int group, int block_size);
// Heads per partial slot in the workspace for a group size.
int tc_gpad(int group);
// Number of CTAs the tensor-core kernel launches on `device` (persistent grid).
int tc_grid(int device, int dtype, int head_dim, int group, cudaError_t* err);

// `overlap`: launch with programmatic stream serialization (the kernel reads
// metadata before griddepcontrol.wait; see TLB_ATTN_OVERLAP_PROLOGUE).
cudaError_t launch_tc(int dtype, int head_dim, int group, const TcParams& p,
                      const CUtensorMap& tm_k, const CUtensorMap& tm_v, int grid, bool overlap,
                      cudaStream_t stream);
cudaError_t launch_generic(int dtype, const GenericParams& p, cudaStream_t stream);

}  // namespace attn

// ---------------------------------------------------- rope + cache writes
struct RopeCacheParams {
    void* out;                 // rotated query (may be null when no query work)
    const void* positions;
    const void* query;
    void* key;
    const void* value;
    void* key_cache;
    void* value_cache;
    const void* slots;         // slot mapping, or null with block_tables
    const int32_t* block_tables;
    const void* cos_sin;
    long long cache_rows;
    long long num_tokens;
    long long query_stride, key_stride, value_stride, out_stride;
    long long num_blocks;
    int max_blocks;
    int num_heads;
    int num_kv_heads;
    int head_size;
    int rot_dim;
    int block_size;
    int overlap;               // launched with programmatic stream serialization
};

// Rope only (query -> out, key in place).
cudaError_t launch_rope(int dtype, int pos_dtype, int vec, const RopeCacheParams& p,
                        cudaStream_t stream);
// Rope + write rotated key and value into the cache through `slots`, or
// through block_tables[t, pos / block_size] when by_block_table is set.
cudaError_t launch_rope_cache(int dtype, int pos_dtype, int slot_dtype, bool by_block_table,
                              int vec, const RopeCacheParams& p, cudaStream_t stream);
// Cache write only: `slots` (slot_dtype) or positions + block_tables.
cudaError_t launch_cache_write(int dtype, int index_dtype, bool by_block_table, int vec,
                               const RopeCacheParams& p, cudaStream_t stream);
cudaError_t launch_decode_metadata(const int32_t* context_lens, const int32_t* block_tables,
                                   long long num_seqs, int max_blocks, int block_size,
                                   int64_t* positions, int64_t* slots, cudaStream_t stream);

// Positions and slots of a packed step: prompts' tokens, then one token per
// decode sequence, padded to `num_padded` entries (step_metadata.cu).
constexpr int kStepMaxPrompts = 4096;
cudaError_t launch_step_metadata(const int32_t* prompt_lens, const int32_t* prompt_tables,
                                 int num_prompts, int prompt_max_blocks,
                                 const int32_t* context_lens, const int32_t* decode_tables,
                                 long long num_decode, int decode_max_blocks, int block_size,
                                 long long num_padded, int64_t* positions, int64_t* slots,
                                 cudaStream_t stream);

// Ids to read back and the table over what is read (step_metadata.cu).
cudaError_t launch_read_back_tables(const int32_t* tables, const int32_t* context_lens,
                                    int num_chunks, int max_blocks, int block_size,
                                    long long num_blocks, int32_t* ids, int32_t* places,
                                    cudaStream_t stream);

// Causal paged attention of prompt chunks (prefill_attention.cu).
cudaError_t launch_prefill_attention(int dtype, int head_dim, void* out, const void* query,
                                     const void* key_cache, const void* value_cache,
                                     const int32_t* block_tables, const int32_t* query_start,
                                     const int32_t* context_lens, long long num_blocks,
                                     int num_chunks, int num_heads, int num_kv_heads,
                                     int block_size, int max_blocks, int max_query_len,
                                     float scale_log2, const CUtensorMap* tm_k,
                                     const CUtensorMap* tm_v, cudaStream_t stream);
// Cache rows per TMA copy of the prefill kernel for this block size (a block,
// or a 64-row part of one), 0 when the block size needs the cp.async loader.
int prefill_box_rows(int block_size);

// ------------------------------------------------- quantised cache rows
// Arguments of the quantising cache write and of the query / key norm with
// rotation (the fields its name does not need stay null).
struct QuantCacheParams {
    void* out;                 // normed, rotated query [tokens, heads, D]
    void* key_out;             // the key likewise, when no cache is written
    const void* positions;
    const void* query;
    const void* key;
    const void* value;
    const void* query_weight;  // [D]
    const void* key_weight;
    const void* cos_sin;
    void* key_cache;
    void* value_cache;
    uint8_t* key_scales;       // exponent bytes [blocks, kv_heads, block_size] (8-bit caches)
    uint8_t* value_scales;
    const void* slots;         // slot mapping, or null with block_tables
    const int32_t* block_tables;
    long long cache_rows;
    long long num_tokens;
    long long query_stride, key_stride, value_stride;
    long long num_blocks;
    int max_blocks;
    int num_heads;
    int num_kv_heads;
    int head_size;
    int rot_dim;
    int block_size;
    int block_shift;           // log2(block_size), -1 when it is no power of two
    float eps;
    bool positions64, slots64;
};
struct DequantParams {
    void* key_out;
    void* value_out;
    const void* key_cache;
    const void* value_cache;
    const uint8_t* key_scales;
    const uint8_t* value_scales;
    const void* ids;
    long long num_ids;
    long long num_blocks;
    int rows_per_block;        // kv_heads * block_size
    int head_size;
    bool ids64;
};
// `vec`: pointers, strides and row widths allow 16-byte accesses.
cudaError_t launch_quantize_write(int dtype, int cache_dtype, const QuantCacheParams& p, bool vec,
                                  cudaStream_t stream);
cudaError_t launch_dequantize_blocks(int out_dtype, int cache_dtype, const DequantParams& p,
                                     bool vec, cudaStream_t stream);
// cache_dtype: an 8-bit type, or the dtype itself (also when no cache is written).
cudaError_t launch_qk_norm_rope(int dtype, int cache_dtype, const QuantCacheParams& p, bool vec,
                                cudaStream_t stream);

// ------------------------------------------------- scored decode attention
namespace scored {

// Warps of a CTA for units of up to `heads` (8 or 16) query heads: their output
// and query fragments take 168 registers a thread for 8 heads, 255 for 16.
constexpr int warps_for(int heads) { return heads <= 8 ? 12 : 8; }
// Tokens of a tile for rows of `bytes`: 4 KB of keys.
constexpr int tile_tokens(int bytes) { return 4096 / bytes; }

// CTAs that share a unit on average, at most: the last of them sums all their
// partials.
constexpr int kMaxShares = 32;
// Most tiles of a unit for each warp of a CTA that takes it whole.
constexpr int kAlignedTiles = 2;

struct Params {
    void* out;
    const void* query;
    const void* key_cache;
    const void* value_cache;
    const uint8_t* key_scales;    // exponent bytes, null for 16-bit / fp32 caches
    const uint8_t* value_scales;
    const int32_t* block_tables;
    const int32_t* seq_lens;
    const float* alibi_slopes;    // [num_heads] or null
    float4* warp_partials;        // [ctas][warps][fragments]
    float4* cta_partials;         // [2 * ctas][fragments]
    float2* cta_ml;               // [2 * ctas][unit heads padded] (reference, sum)
    unsigned* counters;           // [ctas] arrivals at the unit that begins in a CTA, zero at rest
    long long num_blocks;
    long long query_stride;       // elements between sequences' query rows
    int num_seqs;
    int num_heads;
    int num_kv_heads;
    int group;                    // query heads per kv head
    int unit_heads;               // query heads of a unit, 16 at most (unit_heads_of)
    int head_chunks;              // units per kv head
    int units_per_seq;
    int head_dim;
    int block_size;
    int block_shift;              // log2(block_size), -1 when it is no power of two
    int max_blocks;
    int max_tokens;               // max_blocks * block_size
    int window;                   // tokens the query sees, 0: all
    bool overlap;                 // the kernel before writes neither lengths nor tables
    unsigned long long inv_warps; // ceil(2^64 / warps of the grid)
    bool aligned;                 // a CTA takes one whole unit
    int box_shift;                // log2 of the cache rows a TMA box holds
    unsigned wait_limit;          // mbarrier probes before a wait gives up
    float scale;
    float cap_log2;               // softcap * log2(e), 0: none
    float inv_cap;

    __host__ __device__ int block_of(int pos) const {
        return block_shift >= 0 ? pos >> block_shift : pos / block_size;
    }
};

// Whether the tensor-core kernel serves these (aligned tensors assumed).
bool fast_supported(int dtype, int cache_dtype, int head_dim, int block_size);
// Offsets of the workspace arrays for `ctas` CTAs; the counters come first.
struct Workspace {
    size_t counters_end, warp_partials, cta_partials, cta_ml, total;
};
Workspace workspace_layout(int group, int head_dim, int ctas);
int unit_heads_of(int group);
// CTAs worth launching for `units` units with at most `unit_tiles` tiles each.
int ctas_for(long long units, long long unit_tiles, int group, int sms);
// log2 of the rows of a TMA box: the largest power of two that divides a block
// and a tile.
int box_shift_of(int block_size, int tile);

cudaError_t launch_e4m3(int dtype, const Params& p, const CUtensorMap& map_k,
                        const CUtensorMap& map_v, int ctas, cudaStream_t stream);
cudaError_t launch_int8(int dtype, const Params& p, const CUtensorMap& map_k,
                        const CUtensorMap& map_v, int ctas, cudaStream_t stream);
cudaError_t launch_16bit(int dtype, const Params& p, const CUtensorMap& map_k,
                         const CUtensorMap& map_v, int ctas, cudaStream_t stream);
// Any shape and type, one CTA per (sequence, query head).
cudaError_t launch_generic(int dtype, int cache_dtype, const Params& p, cudaStream_t stream);

}  // namespace scored

// ------------------------------------------------------------ block copies
constexpr int kCopyMaxCaches = 128;
constexpr int kCopyMaxPairs = 1024;
struct CopyParams {
    long long block_bytes;
    int num_caches;
    int num_pairs;
    char* dst[kCopyMaxCaches];
    const char* src[kCopyMaxCaches];
    long long pairs[2 * kCopyMaxPairs];
};
cudaError_t launch_copy_blocks(const CopyParams& p, bool vec16, cudaStream_t stream);

}  // namespace tlb
