// Vectors of V elements of a feature tensor: one memory access each, converted to and from float.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "ta_features.h"

namespace ta {

template <typename T> struct FeatElem;
template <> struct FeatElem<float> {
    static __device__ __forceinline__ float to_f(float v) { return v; }
    static __device__ __forceinline__ float from_f(float v) { return v; }
    static __device__ __forceinline__ float2 to_f2(float2 v) { return v; }
    static __device__ __forceinline__ float2 from_f2(float a, float b) { return make_float2(a, b); }
    using Pair = float2;
};
template <> struct FeatElem<__half> {
    static __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
    static __device__ __forceinline__ float plus(__half v, float c) { float r; asm("add.f32.f16 %0, %1, %2;" : "=f"(r) : "h"(__half_as_ushort(v)), "f"(c)); return r; }
    static __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ float2 to_f2(__half2 v) { return __half22float2(v); }
    static __device__ __forceinline__ __half2 from_f2(float a, float b) { return __floats2half2_rn(a, b); }
    using Pair = __half2;
};
template <> struct FeatElem<__nv_bfloat16> {
    static __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ float plus(__nv_bfloat16 v, float c) { float r; asm("add.f32.bf16 %0, %1, %2;" : "=f"(r) : "h"(__bfloat16_as_ushort(v)), "f"(c)); return r; }
    static __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ float2 to_f2(__nv_bfloat162 v) { return __bfloat1622float2(v); }
    static __device__ __forceinline__ __nv_bfloat162 from_f2(float a, float b) { return __floats2bfloat162_rn(a, b); }
    using Pair = __nv_bfloat162;
};

template <int BYTES> struct RawOf;
template <> struct RawOf<2> { using type = unsigned short; };
template <> struct RawOf<4> { using type = unsigned; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<16> { using type = uint4; };

// V elements, V * sizeof(T) in {2, 4, 8, 16} bytes and aligned to that
template <typename T, int V> struct Pack {
    using Raw = typename RawOf<V * sizeof(T)>::type;
    using Half = std::conditional_t<(V > 1), typename FeatElem<T>::Pair, T>;       // (a pair would make a single element as large as two)
    union { Raw raw; T v[V]; Half p[V > 1 ? V / 2 : 1]; };
    __device__ __forceinline__ Pack() { static_assert(sizeof(Pack) == V * sizeof(T), "a vector is its elements"); }
    __device__ __forceinline__ Pack(const Pack &o) : raw(o.raw) {}
    __device__ __forceinline__ Pack &operator=(const Pack &o) { raw = o.raw; return *this; }
    __device__ __forceinline__ void load(const T *ptr) { raw = *reinterpret_cast<const Raw *>(ptr); }
    // read once, by this thread only: does not stay in the L1 cache
    __device__ __forceinline__ void load_stream(const T *ptr) { raw = __ldcs(reinterpret_cast<const Raw *>(ptr)); }
    __device__ __forceinline__ void store(T *ptr) const { *reinterpret_cast<Raw *>(ptr) = raw; }
    // as pairs of floats, the form of the packed arithmetic; a single element leaves its pair's second half 0
    static constexpr int P = (V + 1) / 2;
    __device__ __forceinline__ void unpack(float2 (&f)[P]) const
    {
        if constexpr (V == 1) f[0] = make_float2(FeatElem<T>::to_f(v[0]), 0.0f);
        else {
#pragma unroll
            for (int i = 0; i < P; ++i) f[i] = FeatElem<T>::to_f2(p[i]);
        }
    }
    // each element plus its c: for 16-bit types one instruction converts (exactly), adds and rounds.  Group norm of
    // 32 x 256 x 56^2 bfloat16 32.3 -> 31.4 us, backward 60.0 -> 58.5 us, against unpack() and packed additions.
    __device__ __forceinline__ void unpack_plus(const float2 (&c)[P], float2 (&f)[P]) const
    {
        if constexpr (V == 1 || sizeof(T) == 4) {
            unpack(f);
#pragma unroll
            for (int i = 0; i < P; ++i) f[i] = __fadd2_rn(f[i], c[i]);
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i) f[i] = make_float2(FeatElem<T>::plus(v[2 * i], c[i].x), FeatElem<T>::plus(v[2 * i + 1], c[i].y));
        }
    }
    __device__ __forceinline__ void pack(const float2 (&f)[P])
    {
        if constexpr (V == 1) v[0] = FeatElem<T>::from_f(f[0].x);
        else {
#pragma unroll
            for (int i = 0; i < P; ++i) p[i] = FeatElem<T>::from_f2(f[i].x, f[i].y);
        }
    }
};

// Two independent round-to-nearest operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 neg2(float2 a) { return make_float2(-a.x, -a.y); }
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

__device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDiv &f)
{
    const uint32_t t = __umulhi(n, f.m);
    return (t + ((n - t) >> f.s1)) >> f.s2;
}

// Feature types by their TA_B200_* code (0 float32, 1 float16, 4 bfloat16), for operands that are read a few times per thread
__device__ __forceinline__ float load_code(const void *p, int code, long long i)
{
    return code == 0 ? static_cast<const float *>(p)[i]
         : code == 1 ? __half2float(static_cast<const __half *>(p)[i]) : __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void store_code(void *p, int code, long long i, float v)
{
    if (code == 0) static_cast<float *>(p)[i] = v;
    else if (code == 1) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

}  // namespace ta
