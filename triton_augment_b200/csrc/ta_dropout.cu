// Dropout whose mask is a function of (seed, mask entry) and is never stored.
//
//   y = residual + keep(i) * x / (1 - p).  Mask entry i belongs to block i / 8 of a counter-based generator:
//   Philox4x32-10 with key = seed and counter = (block lo, block hi, offset, tag) gives eight 16-bit
//   numbers, entry i the (i % 8)-th, low half of a word first.  They are the upper halves of 32-bit
//   numbers whose lower halves come from the same counter with tag + 1, and an entry is kept when its
//   32-bit number is not below round(p 2^32).  The lower halves decide for one entry in 65536 only, so
//   they are computed where an upper half equals the threshold's and nowhere else: eight decisions per
//   generator call at 32-bit resolution.
#include "ta_features.h"
#include "ta_pack.cuh"
#include "ta_philox.cuh"

namespace ta {

constexpr uint32_t kDropoutTag = 0x64726F70u;
constexpr int kDropoutThreads = 256;

__device__ __forceinline__ uint4 mask_words(uint2 key, unsigned long long block, uint32_t offset, uint32_t tag)
{
    return philox4x32_10(key, make_uint4((uint32_t)block, (uint32_t)(block >> 32), offset, tag));
}

__device__ __forceinline__ uint32_t half_of(const uint4 &w, int slot)
{
    const uint32_t word = slot < 4 ? (slot < 2 ? w.x : w.y) : (slot < 6 ? w.z : w.w);
    return slot & 1 ? word >> 16 : word & 0xFFFFu;
}

// One mask entry on its own
__device__ __forceinline__ bool keep_entry(const DropoutArgs &a, uint2 key, unsigned long long entry)
{
    const int slot = (int)(entry & 7);
    const uint32_t hi = half_of(mask_words(key, entry >> 3, a.offset, kDropoutTag), slot);
    if (hi != a.thr_hi) return hi > a.thr_hi;
    return half_of(mask_words(key, entry >> 3, a.offset, kDropoutTag + 1), slot) >= a.thr_lo;
}

__device__ __forceinline__ unsigned long long mask_index(const DropoutArgs &a, unsigned long long e)
{
    unsigned long long m = 0;
#pragma unroll
    for (int d = 3; d >= 0; --d) {
        const unsigned long long q = e / (unsigned long long)a.size[d];
        m += (e - q * a.size[d]) * a.mstride[d];
        e = q;
    }
    return m;
}

template <typename T>
__global__ void __launch_bounds__(kDropoutThreads) dropout_kernel(const DropoutArgs a)
{
    const uint64_t seed = a.seed_ptr ? *a.seed_ptr : a.seed;
    const uint2 key = make_uint2((uint32_t)seed, (uint32_t)(seed >> 32));
    const long long step = (long long)gridDim.x * kDropoutThreads;
    for (long long e = (long long)blockIdx.x * kDropoutThreads + threadIdx.x; e < a.numel; e += step) {
        const float x = FeatElem<T>::to_f(((const T *)a.x)[e]);
        float y = keep_entry(a, key, mask_index(a, e)) ? x * a.scale : 0.0f;
        if (a.residual) y += FeatElem<T>::to_f(((const T *)a.residual)[e]);
        ((T *)a.y)[e] = FeatElem<T>::from_f(y);
    }
}

template <typename T> static cudaError_t dropout_launch(const DropoutArgs &a, cudaStream_t stream)
{
    long long blocks = (a.numel + kDropoutThreads - 1) / kDropoutThreads;
    if (blocks > 8LL * a.sm_count) blocks = 8LL * a.sm_count;
    dropout_kernel<T><<<(unsigned)blocks, kDropoutThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_dropout(const DropoutArgs &a, int dtype, cudaStream_t stream)
{
    return dtype == 0 ? dropout_launch<float>(a, stream) : dtype == 1 ? dropout_launch<__half>(a, stream)
                                                                     : dropout_launch<__nv_bfloat16>(a, stream);
}

}  // namespace ta
