#include "ta_group_norm.cuh"
namespace ta {
cudaError_t launch_group_norm_f16(const GnArgs &a, bool backward, cudaStream_t stream) { return gn_launch<__half>(a, backward, stream); }
size_t scratch_group_norm_f16(const GnArgs &a, bool backward) { return gn_scratch_bytes<__half>(a, backward); }
}
