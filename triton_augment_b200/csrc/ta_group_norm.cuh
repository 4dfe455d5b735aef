// Group normalisation with an activation on channels-last features, forward and backward.
//
//   z = (x - mean) * rstd * weight + bias, y = act(z); mean and rstd over the rows x (C / G) elements of a
//   sample's group.  With g = dy * act'(z) and u = g * weight:
//   dweight = sum g * xhat, dbias = sum g, dx = rstd * (u - mean(u) - xhat * mean(u * xhat)).
#pragma once
#include "ta_features.h"
#include "ta_pack.cuh"

namespace ta {

// ----------------------------------------------------------------------------- activations
// FAST (results of 16 bits): the hardware's approximations, a few units of 2^-23 off, 2^-8 of half a
// step of float16; float32 results take the library functions.
template <bool FAST> __device__ __forceinline__ float exp_of(float x) { return FAST ? __expf(x) : expf(x); }
template <bool FAST> __device__ __forceinline__ float sigmoid_of(float z)
{
    const float d = 1.0f + exp_of<FAST>(-z);
    return FAST ? __fdividef(1.0f, d) : 1.0f / d;
}

template <bool FAST, int V> __device__ __forceinline__ void activate(int act, float (&z)[V])
{
    if (act == kActSilu) {
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = z[i] * sigmoid_of<FAST>(z[i]);
    } else if (act == kActRelu) {
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = z[i] < 0.0f ? 0.0f : z[i];          // a NaN stays
    } else if (act == kActGelu) {
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = z[i] * normcdff(z[i]);
    }
}

// g = dy * act'(z), in place of dy
template <bool FAST, int V> __device__ __forceinline__ void activate_grad(int act, const float (&z)[V], float (&g)[V])
{
    if (act == kActSilu) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float s = sigmoid_of<FAST>(z[i]);
            g[i] *= s * (1.0f + z[i] * (1.0f - s));
        }
    } else if (act == kActRelu) {
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] = z[i] > 0.0f ? g[i] : 0.0f;
    } else if (act == kActGelu) {
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] *= normcdff(z[i]) + z[i] * 0.3989422804014327f * exp_of<FAST>(-0.5f * z[i] * z[i]);
    }
}

// ----------------------------------------------------------------------------- shape of the streaming kernels
// A block covers `tile` vectors of the channel axis (all of them up to kGnThreads) and a chunk of
// rows; thread t holds channel vector t % tile and rows t / tile, + rows_per_step, ...
constexpr int kGnThreads = 256;
struct GnShape { int vecs, tile, tiles, rows_per_step, chunks; long long chunk_rows; };

__host__ inline GnShape gn_shape(const GnArgs &a, int v)
{
    GnShape s;
    s.vecs = a.channels / v;
    s.tile = s.vecs < kGnThreads ? s.vecs : kGnThreads;
    s.tiles = (s.vecs + s.tile - 1) / s.tile;
    s.rows_per_step = kGnThreads / s.tile;
    // about eight blocks per SM, at least eight steps each, at most 512 chunks per sample
    const long long want = (8LL * a.sm_count + a.n * s.tiles - 1) / (a.n * s.tiles);
    const long long most = (a.rows + 8LL * s.rows_per_step - 1) / (8LL * s.rows_per_step);
    long long chunks = want < most ? want : most;
    chunks = chunks > 512 ? 512 : chunks < 1 ? 1 : chunks;
    s.chunk_rows = (a.rows + chunks - 1) / chunks;
    s.chunks = (int)((a.rows + s.chunk_rows - 1) / s.chunk_rows);
    return s;
}

// ----------------------------------------------------------------------------- streaming kernels
// Per (sample, chunk, channel): mean and sum of squared deviations.  A thread sums differences to the
// first value it sees, so that a mean far from zero cancels nothing; threads are joined by Chan's rule.
template <typename T, int V>
__global__ void __launch_bounds__(kGnThreads) gn_stats_kernel(const GnArgs a, const GnShape s)
{
    const int v = threadIdx.x % s.tile, r = threadIdx.x / s.tile, vec = blockIdx.y * s.tile + v;
    const long long item = blockIdx.x, n = item / s.chunks;
    const int chunk = (int)(item - n * s.chunks);
    const long long row0 = chunk * s.chunk_rows, row1 = min(row0 + s.chunk_rows, a.rows);
    float pivot[V], sum[V], sq[V];
    int count = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) pivot[i] = sum[i] = sq[i] = 0.0f;
    if (r < s.rows_per_step && vec < s.vecs) {
        const T *base = (const T *)a.x + (n * a.rows) * a.channels + (long long)vec * V;
        for (long long row = row0 + r; row < row1; row += s.rows_per_step) {
            Pack<T, V> p;
            p.load(base + row * a.channels);
            float f[V];
            p.unpack(f);
            if (count == 0) {
#pragma unroll
                for (int i = 0; i < V; ++i) pivot[i] = f[i];
            }
            ++count;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = f[i] - pivot[i];
                sum[i] += d;
                sq[i] = fmaf(d, d, sq[i]);
            }
        }
    }
    __shared__ float2 acc[kGnThreads * V];      // [row slot][channel of the tile]
    const float inv = count > 0 ? 1.0f / (float)count : 0.0f;
    if (r < s.rows_per_step) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            acc[(r * s.tile + v) * V + i] = make_float2(pivot[i] + sum[i] * inv, fmaxf(sq[i] - sum[i] * sum[i] * inv, 0.0f));
    }
    __syncthreads();
    const long long rows = row1 - row0;
    for (int c = threadIdx.x; c < s.tile * V; c += kGnThreads) {
        const int channel = blockIdx.y * s.tile * V + c;
        if (channel >= a.channels) continue;
        float mean = 0.0f, m2 = 0.0f, total = 0.0f;
        for (int j = 0; j < s.rows_per_step; ++j) {
            const long long have = rows > j ? (rows - j + s.rows_per_step - 1) / s.rows_per_step : 0;
            if (have == 0) break;
            const float2 b = acc[j * s.tile * V + c];
            const float nb = (float)have, delta = b.x - mean, tot = total + nb;
            mean += delta * (nb / tot);
            m2 += b.y + delta * delta * (total * nb / tot);
            total = tot;
        }
        a.part[item * a.channels + channel] = make_float2(mean, m2);
    }
}

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// One warp per (sample, group): the partial means and deviations of its channels and chunks become mean and rstd.
static __global__ void gn_stats_finish_kernel(const GnArgs a, const int chunks, const long long chunk_rows)
{
    const long long id = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    if (id >= a.n * a.groups) return;
    const int lane = threadIdx.x % 32;
    const long long n = id / a.groups;
    const int first = (int)(id - n * a.groups) * a.cpg;
    const long long entries = (long long)chunks * a.cpg;
    const float total = (float)a.rows * (float)a.cpg;
    float s = 0.0f;
    for (long long e = lane; e < entries; e += 32) {
        const long long chunk = e / a.cpg;
        const float rows = (float)min(chunk_rows, a.rows - chunk * chunk_rows);
        s = fmaf(rows, a.part[(n * chunks + chunk) * a.channels + first + (e - chunk * a.cpg)].x, s);
    }
    // the mean in two steps: the second, around the first estimate, removes its rounding
    float mean = warp_sum(s) / total;
    s = 0.0f;
    for (long long e = lane; e < entries; e += 32) {
        const long long chunk = e / a.cpg;
        const float rows = (float)min(chunk_rows, a.rows - chunk * chunk_rows);
        s = fmaf(rows, a.part[(n * chunks + chunk) * a.channels + first + (e - chunk * a.cpg)].x - mean, s);
    }
    mean += warp_sum(s) / total;
    s = 0.0f;
    for (long long e = lane; e < entries; e += 32) {
        const long long chunk = e / a.cpg;
        const float rows = (float)min(chunk_rows, a.rows - chunk * chunk_rows);
        const float2 p = a.part[(n * chunks + chunk) * a.channels + first + (e - chunk * a.cpg)];
        const float d = p.x - mean;
        s += p.y + rows * d * d;
    }
    const float var = warp_sum(s) / total;
    if (lane == 0) {
        a.mean[id] = mean;
        a.rstd[id] = rsqrtf(var + a.eps);
    }
}

// Per-thread constants of V channels of one sample
template <int V> struct GnChannels {
    float mean[V], scale[V], bias[V];       // z = (x - mean) * scale + bias
    __device__ __forceinline__ void load(const GnArgs &a, long long n, int c0)
    {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = c0 + i;
            const long long g = n * a.groups + c / a.cpg;
            mean[i] = a.mean[g];
            scale[i] = a.rstd[g] * (a.weight ? load_code(a.weight, a.param_code, c) : 1.0f);
            bias[i] = a.bias ? load_code(a.bias, a.param_code, c) : 0.0f;
        }
    }
};

template <typename T, int V>
__global__ void __launch_bounds__(kGnThreads) gn_apply_kernel(const GnArgs a, const GnShape s)
{
    const int v = threadIdx.x % s.tile, r = threadIdx.x / s.tile, vec = blockIdx.y * s.tile + v;
    if (r >= s.rows_per_step || vec >= s.vecs) return;
    const long long item = blockIdx.x, n = item / s.chunks;
    const long long row0 = (item - n * s.chunks) * s.chunk_rows, row1 = min(row0 + s.chunk_rows, a.rows);
    GnChannels<V> ch;
    ch.load(a, n, vec * V);
    const long long base = n * a.rows * a.channels + (long long)vec * V;
    for (long long row = row0 + r; row < row1; row += s.rows_per_step) {
        Pack<T, V> p;
        p.load((const T *)a.x + base + row * a.channels);
        float f[V];
        p.unpack(f);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = fmaf(f[i] - ch.mean[i], ch.scale[i], ch.bias[i]);
        activate<sizeof(T) == 2, V>(a.act, f);
        p.pack(f);
        p.store((T *)a.y + base + row * a.channels);
    }
}

// Per (sample, chunk, channel): sums of g * xhat and of g.
template <typename T, int V>
__global__ void __launch_bounds__(kGnThreads) gn_grad_sums_kernel(const GnArgs a, const GnShape s)
{
    const int v = threadIdx.x % s.tile, r = threadIdx.x / s.tile, vec = blockIdx.y * s.tile + v;
    const long long item = blockIdx.x, n = item / s.chunks;
    const long long row0 = (item - n * s.chunks) * s.chunk_rows, row1 = min(row0 + s.chunk_rows, a.rows);
    float sum_gx[V], sum_g[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum_gx[i] = sum_g[i] = 0.0f;
    if (r < s.rows_per_step && vec < s.vecs) {
        GnChannels<V> ch;
        ch.load(a, n, vec * V);
        float rstd[V];
#pragma unroll
        for (int i = 0; i < V; ++i) rstd[i] = a.rstd[n * a.groups + (vec * V + i) / a.cpg];
        const long long base = n * a.rows * a.channels + (long long)vec * V;
        for (long long row = row0 + r; row < row1; row += s.rows_per_step) {
            Pack<T, V> px, pd;
            px.load((const T *)a.x + base + row * a.channels);
            pd.load((const T *)a.dy + base + row * a.channels);
            float x[V], z[V], g[V];
            px.unpack(x);
            pd.unpack(g);
#pragma unroll
            for (int i = 0; i < V; ++i) { x[i] -= ch.mean[i]; z[i] = fmaf(x[i], ch.scale[i], ch.bias[i]); }
            activate_grad<sizeof(T) == 2, V>(a.act, z, g);
#pragma unroll
            for (int i = 0; i < V; ++i) { sum_g[i] += g[i]; sum_gx[i] = fmaf(g[i], x[i] * rstd[i], sum_gx[i]); }
        }
    }
    __shared__ float2 acc[kGnThreads * V];
    if (r < s.rows_per_step) {
#pragma unroll
        for (int i = 0; i < V; ++i) acc[(r * s.tile + v) * V + i] = make_float2(sum_gx[i], sum_g[i]);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < s.tile * V; c += kGnThreads) {
        const int channel = blockIdx.y * s.tile * V + c;
        if (channel >= a.channels) continue;
        float2 t = make_float2(0.0f, 0.0f);
        for (int j = 0; j < s.rows_per_step; ++j) { t.x += acc[j * s.tile * V + c].x; t.y += acc[j * s.tile * V + c].y; }
        a.part[item * a.channels + channel] = t;
    }
}

// Scratch of the backward pass: [n, chunks, C] partial sums, then [n, C] their sums over chunks, then
// [n, G] means of (u * xhat, u) over the group.
__device__ __forceinline__ float2 *gn_channel_sums(const GnArgs &a, int chunks) { return a.part + a.n * chunks * a.channels; }
__device__ __forceinline__ float2 *gn_group_means(const GnArgs &a, int chunks) { return a.part + a.n * (chunks + 1) * a.channels; }

// One warp per (sample, group)
static __global__ void gn_grad_finish_kernel(const GnArgs a, const int chunks)
{
    const long long id = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    if (id >= a.n * a.groups) return;
    const int lane = threadIdx.x % 32;
    const long long n = id / a.groups;
    const int first = (int)(id - n * a.groups) * a.cpg;
    float2 *sums = gn_channel_sums(a, chunks);
    float s_ux = 0.0f, s_u = 0.0f;
    for (int i = 0; i < a.cpg; ++i) {
        const int c = first + i;
        float gx = 0.0f, g = 0.0f;
        for (int chunk = lane; chunk < chunks; chunk += 32) {
            const float2 p = a.part[(n * chunks + chunk) * a.channels + c];
            gx += p.x; g += p.y;
        }
        gx = warp_sum(gx); g = warp_sum(g);
        if (lane == 0) sums[n * a.channels + c] = make_float2(gx, g);
        const float w = a.weight ? load_code(a.weight, a.param_code, c) : 1.0f;
        s_ux = fmaf(w, gx, s_ux); s_u = fmaf(w, g, s_u);
    }
    const float inv = 1.0f / ((float)a.rows * (float)a.cpg);
    if (lane == 0) gn_group_means(a, chunks)[id] = make_float2(s_ux * inv, s_u * inv);
}

template <typename T, int V>
__global__ void __launch_bounds__(kGnThreads) gn_grad_input_kernel(const GnArgs a, const GnShape s)
{
    const int v = threadIdx.x % s.tile, r = threadIdx.x / s.tile, vec = blockIdx.y * s.tile + v;
    if (r >= s.rows_per_step || vec >= s.vecs) return;
    const long long item = blockIdx.x, n = item / s.chunks;
    const long long row0 = (item - n * s.chunks) * s.chunk_rows, row1 = min(row0 + s.chunk_rows, a.rows);
    GnChannels<V> ch;
    ch.load(a, n, vec * V);
    float rstd[V], m_ux[V], m_u[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const long long g = n * a.groups + (vec * V + i) / a.cpg;
        rstd[i] = a.rstd[g];
        const float2 m = gn_group_means(a, s.chunks)[g];
        m_ux[i] = m.x; m_u[i] = m.y;
    }
    const long long base = n * a.rows * a.channels + (long long)vec * V;
    for (long long row = row0 + r; row < row1; row += s.rows_per_step) {
        Pack<T, V> px, pd;
        px.load((const T *)a.x + base + row * a.channels);
        pd.load((const T *)a.dy + base + row * a.channels);
        float x[V], z[V], g[V];
        px.unpack(x);
        pd.unpack(g);
#pragma unroll
        for (int i = 0; i < V; ++i) { x[i] -= ch.mean[i]; z[i] = fmaf(x[i], ch.scale[i], ch.bias[i]); }
        activate_grad<sizeof(T) == 2, V>(a.act, z, g);
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] = fmaf(g[i], ch.scale[i], -rstd[i] * fmaf(x[i] * rstd[i], m_ux[i], m_u[i]));
        px.pack(g);
        px.store((T *)a.dx + base + row * a.channels);
    }
}

// dweight and dbias: the per-sample channel sums added over the samples, in sample order per lane row
static __global__ void gn_grad_params_kernel(const GnArgs a, const int chunks)
{
    const int c = blockIdx.x * 32 + threadIdx.x;
    const float2 *sums = gn_channel_sums(a, chunks);
    float gx = 0.0f, g = 0.0f;
    if (c < a.channels)
        for (long long n = threadIdx.y; n < a.n; n += blockDim.y) {
            const float2 p = sums[n * a.channels + c];
            gx += p.x; g += p.y;
        }
    __shared__ float2 acc[32][33];
    acc[threadIdx.y][threadIdx.x] = make_float2(gx, g);
    __syncthreads();
    if (threadIdx.y == 0 && c < a.channels) {
        gx = g = 0.0f;
        for (int j = 0; j < (int)blockDim.y; ++j) { gx += acc[j][threadIdx.x].x; g += acc[j][threadIdx.x].y; }
        if (a.dweight) store_code(a.dweight, a.param_code, c, gx);
        if (a.dbias) store_code(a.dbias, a.param_code, c, g);
    }
}

// ----------------------------------------------------------------------------- launches
template <typename T, int V> cudaError_t gn_launch_streaming(const GnArgs &a, bool backward, cudaStream_t stream)
{
    const GnShape s = gn_shape(a, V);
    const dim3 grid((unsigned)(a.n * s.chunks), s.tiles);
    const unsigned warps = (unsigned)((a.n * a.groups + 7) / 8);
    if (!backward) {
        gn_stats_kernel<T, V><<<grid, kGnThreads, 0, stream>>>(a, s);
        gn_stats_finish_kernel<<<warps, 256, 0, stream>>>(a, s.chunks, s.chunk_rows);
        gn_apply_kernel<T, V><<<grid, kGnThreads, 0, stream>>>(a, s);
    } else {
        gn_grad_sums_kernel<T, V><<<grid, kGnThreads, 0, stream>>>(a, s);
        gn_grad_finish_kernel<<<warps, 256, 0, stream>>>(a, s.chunks);
        if (a.dx) gn_grad_input_kernel<T, V><<<grid, kGnThreads, 0, stream>>>(a, s);
        if (a.dweight || a.dbias)
            gn_grad_params_kernel<<<(a.channels + 31) / 32, dim3(32, a.n >= 32 ? 32 : 8), 0, stream>>>(a, s.chunks);
    }
    return cudaGetLastError();
}

// Widest vector that divides the channels and that the pointers are aligned to
__host__ inline int gn_vector(const GnArgs &a, int elem_bytes)
{
    uintptr_t bits = (uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.dy | (uintptr_t)a.dx;
    int v = 16 / elem_bytes;
    while (v > 1 && (a.channels % v != 0 || bits % (v * elem_bytes) != 0)) v /= 2;
    return v;
}

template <typename T> cudaError_t gn_launch(const GnArgs &a, bool backward, cudaStream_t stream)
{
    switch (gn_vector(a, sizeof(T))) {
    case 8: if constexpr (sizeof(T) == 2) return gn_launch_streaming<T, 8>(a, backward, stream);
    case 4: return gn_launch_streaming<T, 4>(a, backward, stream);
    case 2: return gn_launch_streaming<T, 2>(a, backward, stream);
    default: return gn_launch_streaming<T, 1>(a, backward, stream);
    }
}

}  // namespace ta
