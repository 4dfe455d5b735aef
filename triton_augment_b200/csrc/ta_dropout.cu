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

__device__ __forceinline__ uint32_t word_of(const uint4 &w, int i) { return i < 2 ? (i == 0 ? w.x : w.y) : (i == 2 ? w.z : w.w); }

// Bit j: entry 8 block + j is kept
__device__ __forceinline__ uint32_t keep_bits(const DropoutArgs &a, uint2 key, unsigned long long block)
{
    const uint4 w = mask_words(key, block, a.offset, kDropoutTag);
    const uint32_t upper = a.thr_hi << 16;
    uint32_t bits = 0, equal = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t v = word_of(w, i);
        if ((v << 16) >= upper) bits |= 1u << (2 * i);
        if (v >= upper) bits |= 2u << (2 * i);
        // a half of v equal to the threshold (or, harmlessly, its neighbour): the test for zero bytes, on halves
        const uint32_t t = v ^ (upper | a.thr_hi);
        equal |= (t - 0x00010001u) & ~t & 0x80008000u;
    }
    if (a.thr_lo != 0 && equal != 0) {
        const uint4 lo = mask_words(key, block, a.offset, kDropoutTag + 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t v = word_of(w, i), l = word_of(lo, i);
            if ((v & 0xFFFFu) == a.thr_hi && (l & 0xFFFFu) < a.thr_lo) bits &= ~(1u << (2 * i));
            if ((v >> 16) == a.thr_hi && (l >> 16) < a.thr_lo) bits &= ~(2u << (2 * i));
        }
    }
    return bits;
}

// Bit j: mask entry m + j is kept (eight entries in a row, from one block or two)
__device__ __forceinline__ uint32_t keep_run(const DropoutArgs &a, uint2 key, unsigned long long m)
{
    const int shift = (int)(m & 7);
    uint32_t bits = keep_bits(a, key, m >> 3);
    if (shift) bits = (bits | keep_bits(a, key, (m >> 3) + 1) << 8) >> shift;
    return bits & 0xFFu;
}

__device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDiv &f)
{
    const uint32_t t = __umulhi(n, f.m);
    return (t + ((n - t) >> f.s1)) >> f.s2;
}

// Mask entry of element e; with `rest`, how many elements follow in the innermost dimension
__device__ __forceinline__ unsigned long long mask_index(const DropoutArgs &a, unsigned long long e, long long *rest = nullptr)
{
    unsigned long long m = 0;
#pragma unroll
    for (int d = 3; d >= 0; --d) {
        const unsigned long long q = e / (unsigned long long)a.size[d], c = e - q * a.size[d];
        if (d == 3 && rest) *rest = a.size[3] - (long long)c;
        m += c * a.mstride[d];
        e = q;
    }
    return m;
}
__device__ __forceinline__ unsigned long long mask_index32(const DropoutArgs &a, uint32_t e, long long *rest)
{
    unsigned long long m = 0;
#pragma unroll
    for (int d = 3; d >= 0; --d) {
        if (d < 3 && a.size[d] == 1) continue;
        const uint32_t q = d == 0 ? 0 : fast_div(e, a.div[d]), c = d == 0 ? e : e - q * a.div[d].d;
        if (d == 3) *rest = a.size[3] - (long long)c;
        m += (unsigned long long)c * a.mstride[d];
        e = q;
    }
    return m;
}

enum { kMaskLinear = 0, kMask32 = 1, kMask64 = 2 };       // entry = element; dimensions of fewer than 2^32 elements; any

// Bit j: element e + j is kept, j < 8
template <int KIND> __device__ __forceinline__ uint32_t keep_elements(const DropoutArgs &a, uint2 key, long long e, int valid)
{
    if (a.drop_all) return 0;
    if constexpr (KIND == kMaskLinear) return keep_bits(a, key, (unsigned long long)e >> 3);
    long long rest;
    const unsigned long long m = KIND == kMask32 ? mask_index32(a, (uint32_t)e, &rest) : mask_index(a, e, &rest);
    if (rest >= 8) {                                      // eight neighbours in a row: one entry for all, or eight in a row
        if (a.mstride[3] != 0) return keep_run(a, key, m);
        return (keep_bits(a, key, m >> 3) >> (m & 7)) & 1u ? 0xFFu : 0u;
    }
    uint32_t out = 0, bits = 0;
    unsigned long long have = ~0ull;
    for (int j = 0; j < valid; ++j) {
        long long r;
        const unsigned long long mj = KIND == kMask32 ? mask_index32(a, (uint32_t)(e + j), &r) : mask_index(a, e + j, &r);
        if (mj >> 3 != have) {
            have = mj >> 3;
            bits = keep_bits(a, key, have);
        }
        out |= ((bits >> (mj & 7)) & 1u) << j;
    }
    return out;
}

// Every thread: U times eight elements, their loads first; the generator's work hides the loads' latency.
// WIDE: all tensors on 16-byte boundaries.
template <typename T, int KIND, bool WIDE, bool RESIDUAL>
__global__ void __launch_bounds__(kDropoutThreads) dropout_kernel(const __grid_constant__ DropoutArgs a)
{
    constexpr int V = 16 / sizeof(T), N = 8 / V, U = sizeof(T) == 2 ? 2 : 1;      // N vectors of 16 bytes are eight elements
    const uint64_t seed = a.seed_ptr ? *a.seed_ptr : a.seed;
    const uint2 key = make_uint2((uint32_t)seed, (uint32_t)(seed >> 32));
    const T *px = (const T *)a.x, *pr = (const T *)a.residual;
    T *py = (T *)a.y;
    const long long first = ((long long)blockIdx.x * U * kDropoutThreads + threadIdx.x) * 8;
    Pack<T, V> x[U][N], r[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long e = first + (long long)u * kDropoutThreads * 8;
        if (WIDE && e + 8 <= a.numel) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x[u][i].load_stream(px + e + i * V);
                if (RESIDUAL) r[u][i].load_stream(pr + e + i * V);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long e = first + (long long)u * kDropoutThreads * 8;
        if (e >= a.numel) break;
        const int valid = (int)min(8LL, a.numel - e);
        const uint32_t keep = keep_elements<KIND>(a, key, e, valid);
        if (WIDE && valid == 8) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float2 f[V / 2], g[V / 2];
                x[u][i].unpack(f);
                if (RESIDUAL) r[u][i].unpack(g);
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    const uint32_t b = keep >> (i * V + 2 * j);
                    // a dropped element contributes 0 whatever it holds: selected, not multiplied
                    f[j] = make_float2(b & 1u ? f[j].x * a.scale : 0.0f, b & 2u ? f[j].y * a.scale : 0.0f);
                    if (RESIDUAL) f[j] = add2(f[j], g[j]);
                }
                x[u][i].pack(f);
                x[u][i].store(py + e + i * V);
            }
        } else {
            for (int j = 0; j < valid; ++j) {
                float f = (keep >> j) & 1u ? FeatElem<T>::to_f(px[e + j]) * a.scale : 0.0f;
                if (RESIDUAL) f += FeatElem<T>::to_f(pr[e + j]);
                py[e + j] = FeatElem<T>::from_f(f);
            }
        }
    }
}

template <typename T, int KIND> static cudaError_t dropout_launch_kind(const DropoutArgs &a, cudaStream_t stream)
{
    constexpr int per_block = kDropoutThreads * 8 * (sizeof(T) == 2 ? 2 : 1);
    const unsigned blocks = (unsigned)((a.numel + per_block - 1) / per_block);
    const bool wide = (((uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.residual) % 16) == 0;
    if (a.residual) {
        if (wide) dropout_kernel<T, KIND, true, true><<<blocks, kDropoutThreads, 0, stream>>>(a);
        else dropout_kernel<T, KIND, false, true><<<blocks, kDropoutThreads, 0, stream>>>(a);
    } else {
        if (wide) dropout_kernel<T, KIND, true, false><<<blocks, kDropoutThreads, 0, stream>>>(a);
        else dropout_kernel<T, KIND, false, false><<<blocks, kDropoutThreads, 0, stream>>>(a);
    }
    return cudaGetLastError();
}

template <typename T> static cudaError_t dropout_launch(const DropoutArgs &a, cudaStream_t stream)
{
    if (a.size[3] == a.numel && a.mstride[3] == 1) return dropout_launch_kind<T, kMaskLinear>(a, stream);
    return a.numel < (1LL << 32) ? dropout_launch_kind<T, kMask32>(a, stream) : dropout_launch_kind<T, kMask64>(a, stream);
}

cudaError_t launch_dropout(const DropoutArgs &a, int dtype, cudaStream_t stream)
{
    return dtype == 0 ? dropout_launch<float>(a, stream) : dtype == 1 ? dropout_launch<__half>(a, stream)
                                                                     : dropout_launch<__nv_bfloat16>(a, stream);
}

}  // namespace ta
