// Rotary positions with one to three axes on queries and keys.
//
//   Pair j of a token's head, (a, b), becomes (a cos t - b sin t, b cos t + a sin t), t = position of the
//   token on the pair's axis x the pair's frequency; the backward pass turns by -t.  t is kept in turns:
//   frequency / 2 pi is the sum of two floats, the product with the position is split into its rounded
//   part and the exact remainder, and whole turns are taken off before anything is rounded, so far
//   positions lose no digits of the angle (64-bit accuracy of the angle at 32-bit cost).
#include "ta_features.h"
#include "ta_pack.cuh"

namespace ta {

constexpr int kRotaryThreads = 256;

struct AxisPos { float hi, lo; };       // position = hi + lo

// fraction of a turn of position p at frequency (fh + fl) turns per unit, in [-1, 1]
__device__ __forceinline__ float turns_of(float p, float fh, float fl)
{
    const float t = p * fh, rest = fmaf(p, fh, -t);
    return (t - rintf(t)) + fmaf(p, fl, rest);
}

__device__ __forceinline__ void cos_sin_of(const AxisPos &p, float fh, float fl, int inverse, float &c, float &s)
{
    float t = turns_of(p.hi, fh, fl);
    if (p.lo != 0.0f) t += turns_of(p.lo, fh, fl);
    sincospif(2.0f * t, &s, &c);
    if (inverse) s = -s;
}

// position of token l (counted after the prefix) of sample n on axis `axis`
__device__ __forceinline__ AxisPos axis_position(const RotaryArgs &a, long long n, long long l, int axis)
{
    AxisPos r;
    r.lo = 0.0f;
    if (a.pos_kind == 0) {
        long long i = l;
        for (int d = a.axes - 1; d > axis; --d) i /= a.grid[d];
        i %= a.grid[axis];
        const bool column = axis == a.axes - 1;
        if (column && a.flip && a.flip[n]) i = a.grid[axis] - 1 - i;
        // in pixels (the frequencies are per pixel): offset of the window + patch x index, as an exact sum of two floats
        const float step = (float)i * a.patch;
        const float origin = column ? (a.left ? a.left[n] : 0.0f) : axis == a.axes - 2 && a.top ? a.top[n] : 0.0f;
        r.hi = origin + step;
        const float b = r.hi - origin;
        r.lo = (origin - (r.hi - b)) + (step - b);
        return r;
    }
    const long long at = n * a.pos_s[0] + (l + a.prefix) * a.pos_s[1] + axis * a.pos_s[2];
    if (a.pos_kind == 2) { r.hi = ((const float *)a.positions)[at]; return r; }
    const long long p = a.pos_kind == 1 ? ((const long long *)a.positions)[at] : (long long)((const int *)a.positions)[at];
    const long long low = p & 0xFFFFFF;                 // two exact floats up to 2^48
    r.hi = (float)(p - low);
    r.lo = (float)low;
    if (r.hi == 0.0f) { r.hi = r.lo; r.lo = 0.0f; }
    return r;
}

// One thread per (token, element pair or lone element), all heads
template <typename T>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryArgs a)
{
    const int lone = a.dim - 2 * a.pairs, units = a.pairs + lone;
    const long long total = a.n * a.tokens * units, step = (long long)gridDim.x * kRotaryThreads;
    for (long long id = (long long)blockIdx.x * kRotaryThreads + threadIdx.x; id < total; id += step) {
        const long long tok = id / units;
        const int u = (int)(id - tok * units);
        const long long n = tok / a.tokens, l = tok - n * a.tokens;
        const bool pair = u < a.pairs, turn = pair && l >= a.prefix;
        float c = 1.0f, s = 0.0f;
        if (turn) {
            const int axis = u < a.axis_end[0] ? 0 : u < a.axis_end[1] ? 1 : 2;
            cos_sin_of(axis_position(a, n, l - a.prefix, axis), a.freq_hi[u], a.freq_lo[u], a.inverse, c, s);
        }
        const int i0 = pair ? (a.halves ? u : 2 * u) : a.pairs + u, i1 = pair ? (a.halves ? u + a.pairs : 2 * u + 1) : i0;
        for (int h = 0; h < a.q_heads + a.k_heads; ++h) {
            const bool is_q = h < a.q_heads;
            const int hh = is_q ? h : h - a.q_heads;
            const T *in = is_q ? (const T *)a.q + n * a.qs[0] + l * a.qs[1] + hh * a.qs[2]
                               : (const T *)a.k + n * a.ks[0] + l * a.ks[1] + hh * a.ks[2];
            T *out = is_q ? (T *)a.q_out + n * a.qos[0] + l * a.qos[1] + hh * a.qos[2]
                          : (T *)a.k_out + n * a.kos[0] + l * a.kos[1] + hh * a.kos[2];
            if (!turn) {
                const T x0 = in[i0], x1 = in[i1];
                out[i0] = x0;
                out[i1] = x1;
            } else {
                const float x0 = FeatElem<T>::to_f(in[i0]), x1 = FeatElem<T>::to_f(in[i1]);
                out[i0] = FeatElem<T>::from_f(x0 * c - x1 * s);
                out[i1] = FeatElem<T>::from_f(x1 * c + x0 * s);
            }
        }
    }
}

template <typename T> static cudaError_t rotary_launch(const RotaryArgs &a, cudaStream_t stream)
{
    const long long total = a.n * a.tokens * (a.dim - a.pairs);
    long long blocks = (total + kRotaryThreads - 1) / kRotaryThreads;
    if (blocks > 8LL * a.sm_count) blocks = 8LL * a.sm_count;
    rotary_kernel<T><<<(unsigned)blocks, kRotaryThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_rotary(const RotaryArgs &a, int dtype, cudaStream_t stream)
{
    return dtype == 0 ? rotary_launch<float>(a, stream) : dtype == 1 ? rotary_launch<__half>(a, stream)
                                                                    : rotary_launch<__nv_bfloat16>(a, stream);
}

}  // namespace ta
