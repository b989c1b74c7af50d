// Gathered top-K attention forward without score modifiers.
#include "gather_attn_kernels.cuh"

namespace ossa {

cudaError_t launch_gather_attn(const GatherArgs& a, cudaStream_t stream) {
    if (a.dtype == kF32) {
        return a.idx_is_64 ? launch_typed<float, int64_t, false>(a, stream)
                           : launch_typed<float, int32_t, false>(a, stream);
    }
    return a.idx_is_64 ? launch_typed<__nv_bfloat16, int64_t, false>(a, stream)
                       : launch_typed<__nv_bfloat16, int32_t, false>(a, stream);
}

}  // namespace ossa
