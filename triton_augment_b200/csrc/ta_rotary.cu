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

// positions of token l (counted after the prefix) of sample n on its axes
__device__ __forceinline__ void axis_positions(const RotaryArgs &a, long long n, int l, AxisPos (&pos)[3])
{
#pragma unroll
    for (int d = 0; d < 3; ++d) pos[d] = {0.0f, 0.0f};
    if (a.pos_kind == 0) {
        uint32_t left = (uint32_t)l;
#pragma unroll
        for (int d = 2; d >= 0; --d) {
            if (d >= a.axes) continue;
            const uint32_t q = d == 0 ? 0u : fast_div(left, a.grid_div[d]);
            int i = (int)(left - q * (uint32_t)a.grid[d]);
            left = q;
            float origin = 0.0f;
            if (d == a.axes - 1) {
                if (a.flip && a.flip[n]) i = a.grid[d] - 1 - i;
                if (a.left) origin = a.left[n];
            } else if (d == a.axes - 2 && a.top) origin = a.top[n];
            // in pixels (the frequencies are per pixel): offset of the window + patch x index, as an exact sum of two floats
            const float step = (float)i * a.patch, sum = origin + step, b = sum - origin;
            pos[d] = {sum, (origin - (sum - b)) + (step - b)};
        }
        return;
    }
    const long long at = n * a.pos_s[0] + (long long)(l + a.prefix) * a.pos_s[1];
#pragma unroll
    for (int d = 0; d < 3; ++d) {
        if (d >= a.axes) continue;
        const long long i = at + d * a.pos_s[2];
        if (a.pos_kind == 2) { pos[d].hi = ((const float *)a.positions)[i]; continue; }
        const long long p = a.pos_kind == 1 ? ((const long long *)a.positions)[i] : (long long)((const int *)a.positions)[i];
        const long long low = p & 0xFFFFFF;               // two exact floats up to 2^48
        pos[d] = {(float)(p - low), (float)low};
        if (pos[d].hi == 0.0f) pos[d] = {pos[d].lo, 0.0f};
    }
}

// ----------------------------------------------------------------------------- scalar kernel
// Any stride and alignment: one thread per (token, element pair or lone element), all heads.
template <typename T>
__global__ void __launch_bounds__(kRotaryThreads) rotary_scalar_kernel(const __grid_constant__ RotaryArgs a)
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
            AxisPos pos[3];
            axis_positions(a, n, (int)l - a.prefix, pos);
            cos_sin_of(axis == 0 ? pos[0] : axis == 1 ? pos[1] : pos[2], a.freq_hi[u], a.freq_lo[u], a.inverse, c, s);
        }
        const int i0 = pair ? (a.halves ? u : 2 * u) : a.pairs + u, i1 = pair ? (a.halves ? u + a.pairs : 2 * u + 1) : i0;
        for (int h = 0; h < a.q_heads + a.k_heads; ++h) {
            const bool is_q = h < a.q_heads;
            const int hh = is_q ? h : h - a.q_heads;
            const T *in = is_q ? (const T *)a.q + n * a.qs[0] + l * a.qs[1] + hh * a.qs[2]
                               : (const T *)a.k + n * a.ks[0] + l * a.ks[1] + hh * a.ks[2];
            T *out = is_q ? (T *)a.q_out + n * a.qos[0] + l * a.qos[1] + hh * a.qos[2]
                          : (T *)a.k_out + n * a.kos[0] + l * a.kos[1] + hh * a.kos[2];
            const T x0 = in[i0], x1 = in[i1];
            if (!turn) {
                out[i0] = x0;
                out[i1] = x1;
            } else {
                const float f0 = FeatElem<T>::to_f(x0), f1 = FeatElem<T>::to_f(x1);
                out[i0] = FeatElem<T>::from_f(f0 * c - f1 * s);
                out[i1] = FeatElem<T>::from_f(f1 * c + f0 * s);
            }
        }
    }
}

// ----------------------------------------------------------------------------- vector kernel
// Bound by the memory: 16 x 4096 tokens x 32 heads x 128 bfloat16 (1.07 GB) 181 us in halves, 177 us interleaved = 91, 93 % of the
// copy bandwidth; 8 x 1568 tokens x 24 heads x 64 (77 MB) 20 us = 59 %; single tokens 3.7 us, latency.
//
// A thread owns one vector of a token's head (two, half the rotated part apart, with HALVES), computes the
// cosines and sines of its pairs once and turns that vector in every `head_step`-th head of q and k,
// kRotaryBatch heads' loads in flight.  A block covers `block_units` of the head's vectors x head_step heads x
// `block_tokens` tokens and walks over the tokens, so that a thread's frequencies stay in registers.
constexpr int kRotaryBatch = 4;
struct RotaryPlan {
    int units, turned;              // vectors of a head (pairs of vectors with HALVES), those that are rotated
    int block_units, head_step, block_tokens, threads, unit_blocks;
};

template <typename T, int V, bool HALVES>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryArgs a, const __grid_constant__ RotaryPlan p)
{
    constexpr int PAIRS = HALVES ? V : V / 2, P = (V + 1) / 2;
    const int per_token = p.block_units * p.head_step;
    const int tl = threadIdx.x / (unsigned)per_token, rest = threadIdx.x - tl * per_token;
    const int hg = rest / (unsigned)p.block_units, u = blockIdx.y * p.block_units + rest - hg * p.block_units;
    if (tl >= p.block_tokens || u >= p.units) return;
    const bool turned = u < p.turned;
    // element offsets of the vector(s); behind the rotated part there is one vector to a unit
    const int i0 = !HALVES ? u * V : turned ? u * V : 2 * a.pairs + (u - p.turned) * V;
    float fh[PAIRS], fl[PAIRS];
    int axis_of[PAIRS];
    if (turned) {
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
            const int pair = u * PAIRS + j;
            fh[j] = a.freq_hi[pair];
            fl[j] = a.freq_lo[pair];
            axis_of[j] = pair < a.axis_end[0] ? 0 : pair < a.axis_end[1] ? 1 : 2;
        }
    }
    const int heads = a.q_heads + a.k_heads;
    const long long tokens = a.n * a.tokens;
    for (long long tok = (long long)blockIdx.x * p.block_tokens + tl; tok < tokens; tok += (long long)gridDim.x * p.block_tokens) {
        const long long n = tokens < (1LL << 32) ? fast_div((uint32_t)tok, a.token_div) : tok / a.tokens;
        const int l = (int)(tok - n * a.tokens);
        const bool turn = turned && l >= a.prefix;
        const T *q = (const T *)a.q + n * a.qs[0] + l * a.qs[1] + i0, *k = (const T *)a.k + n * a.ks[0] + l * a.ks[1] + i0;
        T *qo = (T *)a.q_out + n * a.qos[0] + l * a.qos[1] + i0, *ko = (T *)a.k_out + n * a.kos[0] + l * a.kos[1] + i0;
        float c[PAIRS], s[PAIRS];
        if (turn) {
            AxisPos pos[3];
            axis_positions(a, n, l - a.prefix, pos);
#pragma unroll
            for (int j = 0; j < PAIRS; ++j)
                cos_sin_of(axis_of[j] == 0 ? pos[0] : axis_of[j] == 1 ? pos[1] : pos[2], fh[j], fl[j], a.inverse, c[j], s[j]);
        }
        for (int h0 = hg; h0 < heads; h0 += kRotaryBatch * p.head_step) {
            Pack<T, V> x[kRotaryBatch], y[HALVES ? kRotaryBatch : 1];
#pragma unroll
            for (int b = 0; b < kRotaryBatch; ++b) {
                const int h = h0 + b * p.head_step;
                if (h >= heads) continue;
                const T *in = h < a.q_heads ? q + h * a.qs[2] : k + (h - a.q_heads) * a.ks[2];
                x[b].load_stream(in);
                if (HALVES && turned) y[b].load_stream(in + a.pairs);
            }
#pragma unroll
            for (int b = 0; b < kRotaryBatch; ++b) {
                const int h = h0 + b * p.head_step;
                if (h >= heads) continue;
                if (turn) {
                    float2 f[P], g[P];
                    x[b].unpack(f);
                    if constexpr (HALVES) {
                        y[b].unpack(g);
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            float &lo = j % 2 ? f[j / 2].y : f[j / 2].x, &hi = j % 2 ? g[j / 2].y : g[j / 2].x;
                            const float t0 = lo, t1 = hi;
                            lo = t0 * c[j] - t1 * s[j];
                            hi = t1 * c[j] + t0 * s[j];
                        }
                        y[b].pack(g);
                    } else {
#pragma unroll
                        for (int j = 0; j < PAIRS; ++j) f[j] = make_float2(f[j].x * c[j] - f[j].y * s[j], f[j].y * c[j] + f[j].x * s[j]);
                    }
                    x[b].pack(f);
                }
                T *out = h < a.q_heads ? qo + h * a.qos[2] : ko + (h - a.q_heads) * a.kos[2];
                x[b].store(out);
                if (HALVES && turned) y[b].store(out + a.pairs);
            }
        }
    }
}

template <typename T, int V, bool HALVES> static cudaError_t rotary_launch_vector(const RotaryArgs &a, cudaStream_t stream)
{
    RotaryPlan p;
    const int tail = (a.dim - 2 * a.pairs) / V, heads = a.q_heads + a.k_heads;
    p.turned = HALVES ? a.pairs / V : 2 * a.pairs / V;
    p.units = p.turned + tail;
    p.block_units = p.units < kRotaryThreads ? p.units : kRotaryThreads;
    p.unit_blocks = (p.units + p.block_units - 1) / p.block_units;
    const long long tokens = a.n * a.tokens;
    // As few threads per token as still fill the GPU, so that a thread's cosines serve many heads: they cost as much
    // as about five heads' rotations (16 x 4096 tokens x 32 heads x 128, 4 / 8 / 16 / 32 heads to a thread: 217 / 189 /
    // 182 / 190 us).  Single tokens get a thread per head.
    const long long fill = (long long)a.sm_count * 512;
    int step = (heads + 15) / 16;
    while (step < heads && tokens * p.units * step < fill) step = step * 2 < heads ? step * 2 : heads;
    if (step > kRotaryThreads / p.block_units) step = kRotaryThreads / p.block_units;
    p.head_step = step < 1 ? 1 : step;
    const int per_token = p.block_units * p.head_step;
    p.block_tokens = kRotaryThreads / per_token;
    if (p.block_tokens > tokens) p.block_tokens = (int)tokens;
    p.threads = (p.block_tokens * per_token + 31) / 32 * 32;
    long long blocks = (tokens + p.block_tokens - 1) / p.block_tokens;
    const long long most = 16LL * a.sm_count;
    if (blocks > most) blocks = most;
    rotary_kernel<T, V, HALVES><<<dim3((unsigned)blocks, p.unit_blocks), p.threads, 0, stream>>>(a, p);
    return cudaGetLastError();
}

template <typename T> static cudaError_t rotary_launch(const RotaryArgs &a, cudaStream_t stream)
{
    // the widest vector that all offsets are multiples of
    unsigned long long bits = (a.halves ? a.pairs : 2 * a.pairs) | a.dim;
    const auto add = [&](const void *in, const void *out, const long long *is, const long long *os, long long heads) {
        bits |= (uintptr_t)in / sizeof(T) | (uintptr_t)out / sizeof(T);
        if (a.n > 1) bits |= (unsigned long long)(is[0] | os[0]);
        if (a.tokens > 1) bits |= (unsigned long long)(is[1] | os[1]);
        if (heads > 1) bits |= (unsigned long long)(is[2] | os[2]);
    };
    if (a.q_heads) add(a.q, a.q_out, a.qs, a.qos, a.q_heads);
    if (a.k_heads) add(a.k, a.k_out, a.ks, a.kos, a.k_heads);
    int v = 16 / (int)sizeof(T);
    while (v > 1 && bits % v) v /= 2;
    if (a.halves) {
        if constexpr (sizeof(T) == 2) if (v == 8) return rotary_launch_vector<T, 8, true>(a, stream);
        if (v >= 4) return rotary_launch_vector<T, 4, true>(a, stream);
        if (v == 2) return rotary_launch_vector<T, 2, true>(a, stream);
    } else {
        if constexpr (sizeof(T) == 2) if (v == 8) return rotary_launch_vector<T, 8, false>(a, stream);
        if (v >= 4) return rotary_launch_vector<T, 4, false>(a, stream);
        if (v == 2) return rotary_launch_vector<T, 2, false>(a, stream);
    }
    const long long total = a.n * a.tokens * (a.dim - a.pairs);
    long long blocks = (total + kRotaryThreads - 1) / kRotaryThreads;
    if (blocks > 8LL * a.sm_count) blocks = 8LL * a.sm_count;
    rotary_scalar_kernel<T><<<(unsigned)blocks, kRotaryThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_rotary(const RotaryArgs &a, int dtype, cudaStream_t stream)
{
    return dtype == 0 ? rotary_launch<float>(a, stream) : dtype == 1 ? rotary_launch<__half>(a, stream)
                                                                    : rotary_launch<__nv_bfloat16>(a, stream);
}

}  // namespace ta
