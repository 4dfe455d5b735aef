#include "ta_group_norm.cuh"
namespace ta {
cudaError_t launch_group_norm_f32(const GnArgs &a, bool backward, cudaStream_t stream) { return gn_launch<float>(a, backward, stream); }

size_t group_norm_scratch_bytes(const GnArgs &all, int elem_bytes, bool backward)
{
    GnPlan plan;
    if (gn_plan(all, gn_vector(all, elem_bytes), elem_bytes, backward, plan))
        return backward && (all.dweight || all.dbias) ? (size_t)all.n * all.channels * sizeof(float2) : 0;
    const GnShape s = gn_shape(all, gn_vector(all, elem_bytes), backward);
    const size_t groups = (size_t)all.n * all.groups * s.chunks * s.split;
    const size_t channels = backward && (all.dweight || all.dbias) ? (size_t)all.n * s.chunks * all.channels : 0;
    return (groups + channels) * sizeof(float2);
}
}
