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
    // runs of neighbours: one entry for all of a run, or as many entries in a row; a row shorter than eight has several
    uint32_t out = 0;
    for (int j = 0; j < valid;) {
        long long rest;
        const unsigned long long m = KIND == kMask32 ? mask_index32(a, (uint32_t)(e + j), &rest) : mask_index(a, e + j, &rest);
        const uint32_t run = a.mstride[3] != 0 ? keep_run(a, key, m) : 0u - ((keep_bits(a, key, m >> 3) >> (m & 7)) & 1u);
        out = (out & ((1u << j) - 1u)) | run << j;
        j += (int)min(rest, 8LL);
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

// The common case - entry = element, all tensors on 16-byte boundaries, a threshold that has a next smaller 16-bit
// number - straight from the generator's words to the result.  Bound by instruction issue for 16-bit types without
// residual (about 18 instructions an element), by the memory otherwise.  201 M bfloat16, sets of eight per thread 1 / 2 / 3 / 4:
// 160 / 149 / 135 / 140 us (floor 123), with residual 178 / 175 / 175 / 175; 101 M float32 (one set) 120 us.
template <typename T> constexpr int kLinearSets = sizeof(T) == 2 ? 3 : 1;
template <typename T, bool RESIDUAL>
__global__ void __launch_bounds__(kDropoutThreads, sizeof(T) == 2 ? 4 : 6) dropout_linear_kernel(const __grid_constant__ DropoutArgs a)
{
    constexpr int V = 16 / sizeof(T), N = 8 / V, U = kLinearSets<T>;
    const uint64_t seed = a.seed_ptr ? *a.seed_ptr : a.seed;
    const uint2 key = make_uint2((uint32_t)seed, (uint32_t)(seed >> 32));
    const long long block0 = (long long)blockIdx.x * (U * kDropoutThreads) + threadIdx.x, blocks = a.numel >> 3;
    const T *px = (const T *)a.x + block0 * 8, *pr = (const T *)a.residual + block0 * 8;
    T *py = (T *)a.y + block0 * 8;
    Pack<T, V> x[U][N], r[U][N];
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long block = block0 + u * kDropoutThreads;
        w[u] = make_uint4((uint32_t)block, (uint32_t)(block >> 32), a.offset, kDropoutTag);
        if (block < blocks) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x[u][i].load_stream(px + u * kDropoutThreads * 8 + i * V);
                if (RESIDUAL) r[u][i].load_stream(pr + u * kDropoutThreads * 8 + i * V);
            }
        }
    }
    philox4x32_10<U>(key, w);
    const uint32_t upper = a.thr_hi << 16, pair = upper | a.thr_hi;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long block = block0 + u * kDropoutThreads;
        if (block < blocks) {
            uint32_t equal = 0;                           // the test for zero bytes, on halves
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t t = word_of(w[u], i) ^ pair;
                equal |= (t - 0x00010001u) & ~t;
            }
            if (a.thr_lo != 0 && (equal & 0x80008000u) != 0) {
                // an upper half that equals the threshold's and whose lower half says drop becomes the next smaller number
                const uint4 lo = mask_words(key, block, a.offset, kDropoutTag + 1);
                const auto refine = [&](uint32_t v, uint32_t l) {
                    const uint32_t a0 = (v & 0xFFFFu) == a.thr_hi && (l & 0xFFFFu) < a.thr_lo, a1 = (v >> 16) == a.thr_hi && (l >> 16) < a.thr_lo;
                    return v - a0 - (a1 << 16);
                };
                w[u] = make_uint4(refine(w[u].x, lo.x), refine(w[u].y, lo.y), refine(w[u].z, lo.z), refine(w[u].w, lo.w));
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float2 f[V / 2], g[V / 2];
                x[u][i].unpack(f);
                if (RESIDUAL) r[u][i].unpack(g);
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    const uint32_t v = word_of(w[u], i * V / 2 + j);
                    // a dropped element contributes 0 whatever it holds: selected, not multiplied
                    f[j] = make_float2((v << 16) >= upper ? f[j].x * a.scale : 0.0f, v >= upper ? f[j].y * a.scale : 0.0f);
                    if (RESIDUAL) f[j] = make_float2(f[j].x + g[j].x, f[j].y + g[j].y);
                }
                x[u][i].pack(f);
                x[u][i].store(py + u * kDropoutThreads * 8 + i * V);
            }
        }
    }
    // the last elements, fewer than eight
    if (blockIdx.x == 0 && threadIdx.x < (a.numel & 7)) {
        const long long e = blocks * 8 + threadIdx.x;
        float f = (keep_bits(a, key, blocks) >> threadIdx.x) & 1u ? FeatElem<T>::to_f(((const T *)a.x)[e]) * a.scale : 0.0f;
        if (RESIDUAL) f += FeatElem<T>::to_f(((const T *)a.residual)[e]);
        ((T *)a.y)[e] = FeatElem<T>::from_f(f);
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

// One entry for a whole row of neighbours (planes of a channel, channels of a pixel, samples): a block makes the
// decisions of the rows that it touches once, in shared memory.  16-byte boundaries, indices of 32 bits.
// 64 x 256 x 56^2 float16, channels: a decision per eight elements 65 us, per row with sets of eight per thread 1 / 2 / 3 / 4:
// 53 / 43 / 42 / 35.5 us (floor 31).
//
// PERIODIC: the other way round, a row of entries that all rows of a plane share (the channels of channels-last features).  A
// block touches at most two planes and keeps a bit per entry of either's row; rows of up to half the block's elements
// pay for their table.  25 M float16 channels last, a decision per eight elements / from the table: 3 channels 141 / 27 us,
// 255: 77 / 24, 256: 36 / 21.5, 4095: 50 / 35, 4096: 37 / 29 (floor 15.4); 64 x 255 x 55^2 144 / 41 us (floor 30).
template <typename T> constexpr int kRowSets = sizeof(T) == 2 ? 4 : 2;
template <typename T> constexpr int kRowSpan = kDropoutThreads * 8 * kRowSets<T>;       // elements of a block
template <typename T, bool RESIDUAL, bool PERIODIC>
__global__ void __launch_bounds__(kDropoutThreads, 4) dropout_rows_kernel(const __grid_constant__ DropoutArgs a)
{
    constexpr int V = 16 / sizeof(T), N = 8 / V, U = kRowSets<T>, SPAN = kRowSpan<T>;
    __shared__ uint8_t kept[SPAN + 1];
    const uint64_t seed = a.seed_ptr ? *a.seed_ptr : a.seed;
    const uint2 key = make_uint2((uint32_t)seed, (uint32_t)(seed >> 32));
    const uint32_t numel = (uint32_t)a.numel, begin = blockIdx.x * (uint32_t)SPAN, size = (uint32_t)a.size[3];
    const uint32_t end = numel - begin > SPAN ? begin + SPAN : numel, first = begin + threadIdx.x * 8u;
    const T *px = (const T *)a.x, *pr = (const T *)a.residual;
    T *py = (T *)a.y;
    Pack<T, V> x[U][N], r[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t e = first + u * kDropoutThreads * 8u;
        if (e < end && end - e >= 8) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x[u][i].load_stream(px + e + i * V);
                if (RESIDUAL) r[u][i].load_stream(pr + e + i * V);
            }
        }
    }
    const uint32_t row0 = fast_div(begin, a.div[3]), rows = fast_div(end - 1, a.div[3]) - row0 + 1;
    // the rows from `turn` on belong to the second plane; a table is followed by a byte that may be read but does not count
    const uint32_t bytes = (size + 7) / 8, table = bytes + 1;
    const uint32_t turn = PERIODIC ? (fast_div(row0, a.div[2]) + 1) * (uint32_t)a.size[2] : 0;
    if constexpr (PERIODIC) {
        const bool two = row0 + rows > turn;
        for (uint32_t i = threadIdx.x; i < (two ? 2 * bytes : bytes); i += kDropoutThreads) {
            const uint32_t second = i >= bytes, at = i - second * bytes;
            long long rest;
            const unsigned long long m = mask_index32(a, (second ? turn : turn - (uint32_t)a.size[2]) * size, &rest) + 8 * at;
            kept[second * table + at] = a.drop_all ? 0 : keep_run(a, key, m);
        }
    } else {
        for (uint32_t i = threadIdx.x; i < rows; i += kDropoutThreads) {
            long long rest;
            const unsigned long long m = mask_index32(a, (row0 + i) * size, &rest);
            kept[i] = a.drop_all ? 0 : (keep_bits(a, key, m >> 3) >> (m & 7)) & 1u;
        }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t e = first + u * kDropoutThreads * 8u;
        if (e >= end) break;
        const int valid = (int)min(8u, end - e);
        uint32_t row = fast_div(e, a.div[3]), keep = 0;
        uint32_t rest = size - (e - row * size);
        if (!PERIODIC) row -= row0;
        for (uint32_t j = 0; j < (uint32_t)valid;) {
            uint32_t run;
            if constexpr (PERIODIC) {
                const uint32_t c = size - rest;
                const uint8_t *bits = kept + (row >= turn ? table : 0) + (c >> 3);
                run = (bits[0] | (uint32_t)bits[1] << 8) >> (c & 7) & 0xFFu;
            } else {
                run = 0u - (uint32_t)kept[row];
            }
            keep = (keep & ((1u << j) - 1u)) | run << j;
            j += min(rest, 8u);
            rest = size;
            ++row;
        }
        if (valid == 8) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float2 f[V / 2], g[V / 2];
                x[u][i].unpack(f);
                if (RESIDUAL) r[u][i].unpack(g);
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    const uint32_t b = keep >> (i * V + 2 * j);
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

template <typename T> static cudaError_t dropout_launch(const DropoutArgs &a, cudaStream_t stream)
{
    const bool wide = (((uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.residual) % 16) == 0;
    if (wide && a.numel <= (1LL << 32) - (1 << 15)) {       // (indices up to a block past the end fit 32 bits)
        const unsigned blocks = (unsigned)((a.numel + kRowSpan<T> - 1) / kRowSpan<T>);
        if (a.mstride[3] == 0) {
            if (a.residual) dropout_rows_kernel<T, true, false><<<blocks, kDropoutThreads, 0, stream>>>(a);
            else dropout_rows_kernel<T, false, false><<<blocks, kDropoutThreads, 0, stream>>>(a);
            return cudaGetLastError();
        }
        if (a.size[2] > 1 && 2 * a.size[3] <= kRowSpan<T> && a.size[2] * a.size[3] >= kRowSpan<T>) {
            if (a.residual) dropout_rows_kernel<T, true, true><<<blocks, kDropoutThreads, 0, stream>>>(a);
            else dropout_rows_kernel<T, false, true><<<blocks, kDropoutThreads, 0, stream>>>(a);
            return cudaGetLastError();
        }
    }
    if (a.size[3] == a.numel && a.mstride[3] == 1) {
        if (wide && !a.drop_all && (a.thr_hi != 0 || a.thr_lo == 0)) {
            constexpr int per_block = kDropoutThreads * 8 * kLinearSets<T>;
            const unsigned blocks = (unsigned)((a.numel + per_block - 1) / per_block);
            if (a.residual) dropout_linear_kernel<T, true><<<blocks, kDropoutThreads, 0, stream>>>(a);
            else dropout_linear_kernel<T, false><<<blocks, kDropoutThreads, 0, stream>>>(a);
            return cudaGetLastError();
        }
        return dropout_launch_kind<T, kMaskLinear>(a, stream);
    }
    return a.numel < (1LL << 32) ? dropout_launch_kind<T, kMask32>(a, stream) : dropout_launch_kind<T, kMask64>(a, stream);
}

cudaError_t launch_dropout(const DropoutArgs &a, int dtype, cudaStream_t stream)
{
    return dtype == 0 ? dropout_launch<float>(a, stream) : dtype == 1 ? dropout_launch<__half>(a, stream)
                                                                     : dropout_launch<__nv_bfloat16>(a, stream);
}

}  // namespace ta
