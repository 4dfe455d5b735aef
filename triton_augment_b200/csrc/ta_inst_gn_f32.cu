#include "ta_group_norm.cuh"
namespace ta {
cudaError_t launch_group_norm_f32(const GnArgs &a, bool backward, cudaStream_t stream) { return gn_launch<float>(a, backward, stream); }
}
namespace ta {
size_t group_norm_scratch_bytes(const GnArgs &a, int elem_bytes, bool backward)
{
    const GnShape s = gn_shape(a, gn_vector(a, elem_bytes));
    const size_t rows = (size_t)a.n * (backward ? s.chunks + 1 : s.chunks);
    return (rows * a.channels + (backward ? (size_t)a.n * a.groups : 0)) * sizeof(float2);
}
}
