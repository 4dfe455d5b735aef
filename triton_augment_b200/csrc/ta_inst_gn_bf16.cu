#include "ta_group_norm.cuh"
namespace ta {
cudaError_t launch_group_norm_bf16(const GnArgs &a, bool backward, cudaStream_t stream) { return gn_launch<__nv_bfloat16>(a, backward, stream); }
size_t scratch_group_norm_bf16(const GnArgs &a, bool backward) { return gn_scratch_bytes<__nv_bfloat16>(a, backward); }
}
