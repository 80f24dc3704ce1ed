// Decode attention over e4m3 caches (scored_attention.cuh).
#include "scored_attention.cuh"

namespace tlb {
namespace scored {

cudaError_t launch_e4m3(int dtype, const Params& p, const CUtensorMap& map_k,
                         const CUtensorMap& map_v, int ctas, cudaStream_t stream) {
    return dtype == TLB_BFLOAT16
               ? launch_fast_shape<__nv_bfloat16, E4M3>(p, map_k, map_v, ctas, stream)
               : launch_fast_shape<__half, E4M3>(p, map_k, map_v, ctas, stream);
}

}  // namespace scored
}  // namespace tlb
