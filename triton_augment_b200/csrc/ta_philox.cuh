// Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", SC'11): a
// counter-based generator, so whatever it decides is a pure function of (key, counter) and can be
// computed again anywhere instead of being stored.
#pragma once
#include <stdint.h>

namespace ta {

// N counters at once, in place: they share the round keys.  (One 64-bit
// product instead of the two 32-bit halves is slower here: dropout of 201 M bfloat16 142 against 135 us.)
template <int N> __device__ __forceinline__ void philox4x32_10(uint2 key, uint4 (&ctr)[N])
{
#pragma unroll
    for (int r = 0; r < 10; ++r) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t hi0 = __umulhi(0xD2511F53u, ctr[i].x), lo0 = 0xD2511F53u * ctr[i].x;
            const uint32_t hi1 = __umulhi(0xCD9E8D57u, ctr[i].z), lo1 = 0xCD9E8D57u * ctr[i].z;
            ctr[i] = make_uint4(hi1 ^ ctr[i].y ^ key.x, lo1, hi0 ^ ctr[i].w ^ key.y, lo0);
        }
        key.x += 0x9E3779B9u;
        key.y += 0xBB67AE85u;
    }
}
__device__ __forceinline__ uint4 philox4x32_10(uint2 key, uint4 ctr)
{
    uint4 one[1] = {ctr};
    philox4x32_10(key, one);
    return one[0];
}

}  // namespace ta
