// Group normalisation with an activation on channels-last features, forward and backward.
//
//   z = (x - mean) * rstd * weight + bias, y = act(z); mean and rstd over the rows x (C / G) elements of a
//   sample's group.  With g = dy * act'(z) and u = g * weight:
//   dweight = sum g * xhat, dbias = sum g, dx = rstd * (u - mean(u) - xhat * mean(u * xhat)).
#pragma once
#include <atomic>

#include "ta_features.h"
#include "ta_pack.cuh"

namespace ta {

// ----------------------------------------------------------------------------- activations
// FAST (results of 16 bits): the hardware's exponential and reciprocal, each within 2^-22, a sixteenth
// of a float16's half step at most after three of them; float32 results take the library functions.
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float rcp_fast(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
constexpr float kLog2E = 1.4426950408889634f;

// 1 / (1 + e^-z).  (One reciprocal for two values, 1 / (d0 d1) times the other factor, is worth 2 % forward and costs 1 %
// backward: 4 x 128 x 224^2 bfloat16 36.5 -> 35.5 us, 64 x 320 x 28^2 bfloat16 backward 49.5 -> 50.1 us.  The product needs
// e^-z held to 2^60, so that results below z = -41 are wrong by orders of magnitude: not taken.)
template <bool FAST> __device__ __forceinline__ float2 sigmoid2(float2 z)
{
    if constexpr (!FAST) return make_float2(1.0f / (1.0f + expf(-z.x)), 1.0f / (1.0f + expf(-z.y)));
    const float2 e = mul2(z, both(-kLog2E)), d = add2(make_float2(exp2_fast(e.x), exp2_fast(e.y)), both(1.0f));
    return make_float2(rcp_fast(d.x), rcp_fast(d.y));
}

// Normal distribution function, and its density through `density`.  FAST: Abramowitz and Stegun 7.1.26,
// erf(x) = 1 - (a1 t + ... + a5 t^5) e^-x^2 with t = 1 / (1 + p x), off by 1.5e-7 at most, which shares its exponential with the density.
template <bool FAST> __device__ __forceinline__ float normal_cdf(float z, float &density)
{
    if constexpr (!FAST) {
        density = 0.3989422804014327f * expf(-0.5f * z * z);
        return fmaf(0.5f, erff(z * 0.7071067811865476f), 0.5f);
    }
    const float x = fabsf(z) * 0.7071067811865476f, e = exp2_fast(-kLog2E * x * x), t = rcp_fast(fmaf(0.3275911f, x, 1.0f));
    density = 0.3989422804014327f * e;
    const float poly = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
    const float upper = 0.5f * poly * e;                  // 1 - cdf(|z|)
    return z < 0.0f ? upper : 1.0f - upper;
}

template <int ACT, bool FAST, int P> __device__ __forceinline__ void activate(float2 (&z)[P])
{
    if constexpr (ACT == kActSilu) {
#pragma unroll
        for (int i = 0; i < P; ++i) z[i] = mul2(z[i], sigmoid2<FAST>(z[i]));
    } else if constexpr (ACT == kActRelu) {
#pragma unroll
        for (int i = 0; i < P; ++i) z[i] = make_float2(z[i].x < 0.0f ? 0.0f : z[i].x, z[i].y < 0.0f ? 0.0f : z[i].y);          // a NaN stays
    } else if constexpr (ACT == kActGelu) {
        float density;
#pragma unroll
        for (int i = 0; i < P; ++i) z[i] = make_float2(z[i].x * normal_cdf<FAST>(z[i].x, density), z[i].y * normal_cdf<FAST>(z[i].y, density));
    }
}

// g = dy * act'(z), in place of dy
template <int ACT, bool FAST, int P> __device__ __forceinline__ void activate_grad(const float2 (&z)[P], float2 (&g)[P])
{
    if constexpr (ACT == kActSilu) {
#pragma unroll
        for (int i = 0; i < P; ++i) {                     // s (1 + z (1 - s)) = s + z s - z s s
            const float2 s = sigmoid2<FAST>(z[i]), t = mul2(z[i], s);
            g[i] = mul2(g[i], fma2(neg2(t), s, add2(s, t)));
        }
    } else if constexpr (ACT == kActRelu) {
#pragma unroll
        for (int i = 0; i < P; ++i) g[i] = make_float2(z[i].x > 0.0f ? g[i].x : 0.0f, z[i].y > 0.0f ? g[i].y : 0.0f);
    } else if constexpr (ACT == kActGelu) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float dx, dy;
            const float cx = normal_cdf<FAST>(z[i].x, dx), cy = normal_cdf<FAST>(z[i].y, dy);
            g[i] = mul2(g[i], fma2(z[i], make_float2(dx, dy), make_float2(cx, cy)));
        }
    }
}

// f(activation as a type): the choice is made once, outside the loops over the data
template <int N> struct ActTag { static constexpr int value = N; };
template <typename F> __device__ __forceinline__ void with_activation(int act, F f)
{
    if (act == kActSilu) f(ActTag<kActSilu>());
    else if (act == kActGelu) f(ActTag<kActGelu>());
    else if (act == kActRelu) f(ActTag<kActRelu>());
    else f(ActTag<kActNone>());
}

// V values of a parameter vector as pairs; `value` where there is no vector.  `wide`: float32 on 16-byte boundaries.
template <int V> __device__ __forceinline__ void load_params(const void *ptr, int code, bool wide, int first, bool active, float value, float2 (&out)[(V + 1) / 2])
{
#pragma unroll
    for (int i = 0; i < (V + 1) / 2; ++i) out[i] = both(value);
    if (!ptr || !active) return;
    if constexpr (V >= 4) if (wide) {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const float4 q = reinterpret_cast<const float4 *>(static_cast<const float *>(ptr) + first)[i];
            out[2 * i] = make_float2(q.x, q.y);
            out[2 * i + 1] = make_float2(q.z, q.w);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float t = load_code(ptr, code, first + j);
        if (j % 2) out[j / 2].y = t;
        else out[j / 2].x = t;
    }
}

// (x, y) of the groups of a thread's V channels as pairs; get(group).  `group` is the group of the first
// channel, `left` how many channels of it follow.
template <int V, typename Get> __device__ __forceinline__ void spread_groups(int group, int left, int cpg, Get get, float2 (&x)[(V + 1) / 2], float2 (&y)[(V + 1) / 2])
{
    float2 t = get(group);
    if (left >= V) {
#pragma unroll
        for (int i = 0; i < (V + 1) / 2; ++i) { x[i] = both(t.x); y[i] = both(t.y); }
        return;
    }
    if (V >= 4 && cpg >= V) {                             // two groups, and the threads of a warp cut at different places: selected
        const float2 next = get(group + 1);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float2 s = j < left ? t : next;
            if (j % 2) { x[j / 2].y = s.x; y[j / 2].y = s.y; }
            else { x[j / 2].x = s.x; y[j / 2].x = s.y; }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (left == 0) { t = get(++group); left = cpg; }
        --left;
        if (j % 2) { x[j / 2].y = t.x; y[j / 2].y = t.y; }
        else { x[j / 2].x = t.x; y[j / 2].x = t.y; }
    }
}

__device__ __forceinline__ float half_of_pair(float2 v, int j) { return j % 2 ? v.y : v.x; }

// Pairs of values of V channels added up over neighbours of one group, `fold` at a time, into dst[]
template <int V> __device__ __forceinline__ void store_folded(float2 *dst, const float2 (&a)[(V + 1) / 2], const float2 (&b)[(V + 1) / 2], int fold)
{
    float2 s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = make_float2(half_of_pair(a[i / 2], i), half_of_pair(b[i / 2], i));
#pragma unroll
    for (int w = 1; w < V; w *= 2)
        if (w < fold) {
#pragma unroll
            for (int i = 0; i < V; i += 2 * w) s[i] = add2(s[i], s[i + w]);
        }
#pragma unroll
    for (int w = 1; w <= V; w *= 2)                       // (constants: a division by `fold` costs more than all else here)
        if (w == fold) {
#pragma unroll
            for (int i = 0; i < V; i += w) dst[i / w] = s[i];
        }
}

// How a block adds up its groups: `lanes` lanes each, the same order every time.  A group's entries are
// `width` neighbouring values in each of a number of rows.
struct GnLanes {
    int lanes, shift, per_pass, width, row_step, entry_step;      // lanes = 1 << shift, groups of a pass; a lane's next entry: row_step rows and entry_step values on
    FastDiv width_div;
};
__host__ inline GnLanes gn_lanes(int groups, int threads, int width)
{
    GnLanes l;
    l.lanes = 32;
    while (l.lanes > 1 && groups * l.lanes > threads) l.lanes >>= 1;
    l.shift = 0;
    while ((1 << l.shift) < l.lanes) ++l.shift;
    l.per_pass = threads >> l.shift;
    l.width = width;
    l.row_step = l.lanes / width;
    l.entry_step = l.lanes % width;
    l.width_div = fast_div_of(width);
    return l;
}
__device__ __forceinline__ float2 lane_sum(float2 v, int lanes)
{
    const auto add = [&](int o) { v = add2(v, make_float2(__shfl_down_sync(0xffffffffu, v.x, o), __shfl_down_sync(0xffffffffu, v.y, o))); };
    if (lanes > 16) add(16);
    if (lanes > 8) add(8);
    if (lanes > 4) add(4);
    if (lanes > 2) add(2);
    if (lanes > 1) add(1);
    return v;
}
__device__ __forceinline__ float lane_sum(float v, int lanes)
{
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_down_sync(0xffffffffu, v, o);
    return v;
}
// Sum of a group's entries in its lane 0 (all threads of the block call it together)
__device__ __forceinline__ float2 group_sum(const GnLanes &l, const float2 *red, int stride, int rows, int width, int g, bool valid)
{
    float2 s = make_float2(0.0f, 0.0f);
    if (valid) {
        const int lane = threadIdx.x & (l.lanes - 1);
        int r = (int)fast_div(lane, l.width_div), e = lane - r * l.width;
        while (r < rows) {
            if (e < width) s = add2(s, red[r * stride + g * l.width + e]);
            r += l.row_step;
            e += l.entry_step;
            if (e >= l.width) { e -= l.width; ++r; }
        }
    }
    return lane_sum(s, l.lanes);
}

// ----------------------------------------------------------------------------- work split
// Two launches a pass: the first reduces chunks of rows, the second reads the same rows again, last ones first
// since those are still in the L2 cache, and writes the result.  (Ranges of samples that fit the cache, one pair
// of launches each, were slower for all that the gaps between launches cost: 16 x 128 x 224^2 float16 in
// 64 MB ranges 162 us against 116 in one pair, both with rows held in registers.)
//
// A block covers a tile of channel vectors and a chunk of rows; thread t holds vector t % tile of rows
// t / tile + i rows_per_step.  Tiles hold whole groups (groups_per_tile); a group wider than a block is
// cut into `split` tiles.  Each block leaves one partial result per group of its tile:
// part[((n groups + g) chunks + chunk) split + piece].
//
// What bounds it: the memory for large tensors, three passes over the features forward and five backward
// (16 x 128 x 224^2 float16 with SiLU, 617 MB, 111 us = 5.5 TB/s); instruction issue where the second pass reads the L2 cache
// (4 x 128 x 224^2 bfloat16 35 us forward, 58 us backward).  Rows held in registers instead of the ring: 122, 44, 73 us.
constexpr int kGnThreads = 256;
constexpr int kGnBlocksForward = 4, kGnBlocksBackward = 3;       // blocks per SM (64 and 80 registers a thread)
struct GnShape {
    int vecs, tile, tiles, rows_per_step, groups_per_tile, split, unit, chunks, fold, per_vec;      // per_vec: folded values of a vector
    float inv;                          // 1 / (values of a group in the sample)
    long long chunk_rows;
    GnLanes columns;                    // sums over a tile's columns
};

__host__ __device__ inline int gn_gcd(int a, int b) { while (b) { const int t = a % b; a = b; b = t; } return a; }

// vectors of the smallest run of whole vectors that is made of whole groups
__host__ inline int gn_unit(const GnArgs &a, int v) { return a.cpg / gn_gcd(a.cpg, v); }

__host__ inline GnShape gn_shape(const GnArgs &a, int v, bool backward)
{
    GnShape s;
    s.vecs = a.channels / v;
    s.unit = gn_unit(a, v);
    if (s.unit <= kGnThreads) {
        const int units = s.vecs / s.unit, most = kGnThreads / s.unit;
        s.tiles = (units + most - 1) / most;
        s.tile = (units + s.tiles - 1) / s.tiles * s.unit;
        s.tiles = (s.vecs + s.tile - 1) / s.tile;
        s.groups_per_tile = s.tile * v / a.cpg;
        s.split = 1;
    } else {                                              // gn_vector() saw to it that v divides cpg
        s.split = (s.unit + kGnThreads - 1) / kGnThreads;
        s.tile = (s.unit + s.split - 1) / s.split;
        s.tiles = a.groups * s.split;
        s.groups_per_tile = 1;
    }
    s.rows_per_step = kGnThreads / s.tile;
    s.fold = v;
    while (a.cpg % s.fold) s.fold /= 2;
    s.columns = gn_lanes(s.groups_per_tile, kGnThreads, (s.split == 1 ? a.cpg : s.tile * v) / s.fold);
    s.per_vec = v / s.fold;
    s.inv = 1.0f / ((float)a.rows * (float)a.cpg);
    // one wave of blocks where the samples allow it, at least four steps a thread
    const long long want = (long long)(backward ? kGnBlocksBackward : kGnBlocksForward) * a.sm_count / (a.n * s.tiles);
    const long long most = (a.rows + 4LL * s.rows_per_step - 1) / (4LL * s.rows_per_step);
    long long chunks = want < most ? want : most;
    chunks = chunks > 512 ? 512 : chunks < 1 ? 1 : chunks;
    s.chunk_rows = (a.rows + chunks - 1) / chunks;
    s.chunks = (int)((a.rows + s.chunk_rows - 1) / s.chunk_rows);
    return s;
}

// Where a thread works
struct GnPlace {
    int v, r, vec, vec_end, group0, piece, chunk, rows;
    unsigned n, item;
    long long row0;
    bool active;
    __device__ __forceinline__ GnPlace(const GnArgs &a, const GnShape &s, unsigned block)
    {
        r = threadIdx.x / s.tile;
        v = threadIdx.x - r * s.tile;
        const int tile = blockIdx.y;
        group0 = s.split == 1 ? tile * s.groups_per_tile : tile / s.split;
        piece = s.split == 1 ? 0 : tile - group0 * s.split;
        const int start = s.split == 1 ? tile * s.tile : group0 * s.unit + piece * s.tile;
        vec_end = s.split == 1 ? s.vecs : (group0 + 1) * s.unit;
        vec = start + v;
        n = block / (unsigned)s.chunks;
        chunk = (int)(block - n * s.chunks);
        item = block;
        row0 = chunk * s.chunk_rows;
        rows = (int)min(s.chunk_rows, a.rows - row0);
        active = r < s.rows_per_step && vec < vec_end;
    }
    // vectors of the tile that exist
    __device__ __forceinline__ int width(const GnShape &s) const { return min(s.tile, vec_end - (vec - v)); }
    __device__ __forceinline__ int groups(const GnArgs &a, const GnShape &s) const { return min(s.groups_per_tile, a.groups - group0); }
    __device__ __forceinline__ int count(const GnShape &s) const { return active && rows > r ? (rows - r + s.rows_per_step - 1) / s.rows_per_step : 0; }
};

// The cluster's barrier in two halves: every thread of every block arrives once and waits once per phase.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// *ptr of the block with cluster rank `rank`
__device__ __forceinline__ float2 load_rank(const float2 *ptr, int rank)
{
    uint32_t remote;
    float2 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(ptr)), "r"(rank));
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(remote) : "memory");
    return v;
}

template <int BYTES> __device__ __forceinline__ void copy_async(void *shared, const void *global)
{
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(shared)), "l"(global) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(shared)), "l"(global), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// The second launch of a pass may start while the first one ends (programmatic dependent launch): what
// does not depend on the first is fetched before gn_wait_first().
__device__ __forceinline__ void gn_allow_second() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void gn_wait_first() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Rows on their way into a thread's own ring in shared memory: N tensors, D rows ahead.  Nothing but the thread's own
// cp.async groups orders the copies, so every thread has D rows in flight all the time and no registers hold them.
template <typename T, int V, int N, int D> struct GnStream {
    using Vec = Pack<T, V>;
    static constexpr int kBytes = N * D * kGnThreads * (int)sizeof(Vec);
    Vec *ring;
    const T *src[N];
    long long step;
    int count, next;
    static constexpr bool kAsync = sizeof(Vec) >= 4;      // cp.async moves four bytes at least; two-byte vectors are loaded four rows at a time
    __device__ __forceinline__ void fetch()
    {
        if (next < count) {
#pragma unroll
            for (int t = 0; t < N; ++t) {
                copy_async<sizeof(Vec)>(ring + ((next & (D - 1)) * N + t) * kGnThreads, src[t]);
                src[t] += step;
            }
        }
        ++next;
        copy_commit();
    }
    __device__ __forceinline__ void start(void *shared, long long row_step, int rows)
    {
        ring = static_cast<Vec *>(shared) + threadIdx.x;
        step = row_step;
        count = rows;
        next = 0;
        if constexpr (kAsync) {
#pragma unroll
            for (int i = 0; i < D; ++i) fetch();
        } else if (count > 0) ring[0].load(src[0]);       // (the first row, for those who look at it)
    }
    // the first row has arrived
    __device__ __forceinline__ void wait() const { if constexpr (kAsync) asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory"); }
    // f(the row's vectors), row by row
    template <typename F> __device__ __forceinline__ void run(F f)
    {
        if constexpr (kAsync) {
            for (int i = 0; i < count; ++i) {
                wait();
                Vec v[N];
#pragma unroll
                for (int t = 0; t < N; ++t) v[t] = ring[((i & (D - 1)) * N + t) * kGnThreads];
                fetch();
                f(v);
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        } else {
            for (int i = 0; i < count; i += 4) {
                Vec v[4][N];
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (i + u < count) {
#pragma unroll
                        for (int t = 0; t < N; ++t) v[u][t].load(src[t] + (i + u) * step);
                    }
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (i + u < count) f(v[u]);
            }
        }
    }
};
constexpr int kGnAhead = 8, kGnAheadGrad = 4;

// ----------------------------------------------------------------------------- forward
// Sums of differences to the group's pivot (negated in pv) and of their squares, per channel
template <int P, typename Vec> __device__ __forceinline__ void add_moments(const Vec &p, const float2 (&pv)[P], float2 (&sm)[P], float2 (&s2)[P])
{
    float2 f[P];
    p.unpack_plus(pv, f);
#pragma unroll
    for (int j = 0; j < P; ++j) {
        sm[j] = add2(sm[j], f[j]);
        s2[j] = fma2(f[j], f[j], s2[j]);
    }
}
// (mean, sum of squared deviations) from the pivot and the sums of differences to it and of their squares
__device__ __forceinline__ float2 moments_of(float pivot, float2 t, float inv)
{
    const float q = fmaf(-t.x * inv, t.x, t.y);
    return make_float2(fmaf(t.x, inv, pivot), q < 0.0f ? 0.0f : q);       // (a NaN stays)
}
// Per (sample, group, chunk): mean and sum of squared deviations from it.
//
// The pivot of a group: the mean of its first channel in the block's first rows, up to eight.  However far from zero the
// values lie, the sums of differences to it and of their squares lose a few 2^-24 of the variance as a rule.  At the very
// worst, a pivot made of nothing but outliers d away from the block's other rows, the squares add up to rows x d^2 where
// their deviations are 8 d^2: chains of L additions then lose up to 3 (L + 3) rows / 8 x 2^-24 of the block's variance.
template <typename T, int V>
__global__ void __launch_bounds__(kGnThreads, kGnBlocksForward) gn_stats_kernel(const __grid_constant__ GnArgs a, const __grid_constant__ GnShape s)
{
    gn_allow_second();
    extern __shared__ __align__(16) unsigned char smem[];  // the ring; afterwards [row slot][folded channel]
    constexpr int P = Pack<T, V>::P;
    const GnPlace at(a, s, blockIdx.x);
    const int count = at.count(s);
    GnStream<T, V, 1, kGnAhead> rows;
    rows.src[0] = (const T *)a.x + (at.n * a.rows + at.row0 + at.r) * a.channels + at.vec * V;
    rows.start(smem, (long long)s.rows_per_step * a.channels, count);
    const int per_vec = s.per_vec, stride = s.tile * per_vec, groups = at.groups(a, s);
    const int width = s.split == 1 ? s.columns.width : at.width(s) * per_vec;
    const int sample_rows = min(min(8, s.rows_per_step), at.rows);
    const float sample_inv = 1.0f / (float)sample_rows;
    const auto pivot_of = [&](int g) {                    // (the first row slots lie side by side: thread t has vector t)
        const T *first = reinterpret_cast<const T *>(smem) + g * a.cpg;
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < sample_rows) t += FeatElem<T>::to_f(first[k * s.tile * V]);
        return t * sample_inv;
    };
    float2 pv[P], sm[P], s2[P];
    rows.wait();
    __syncthreads();
    const int group = at.active ? (at.vec * V) / a.cpg - at.group0 : 0;
    spread_groups<V>(group, at.active ? a.cpg - (at.vec * V) % a.cpg : V, a.cpg, [&](int g) { return make_float2(-pivot_of(g), 0.0f); }, pv, sm);
    const int lanes = s.columns.lanes, per_pass = s.columns.per_pass, lane = threadIdx.x & (lanes - 1), mine = threadIdx.x >> s.columns.shift;
    constexpr int kSums = kGnThreads * V * (int)sizeof(float2), kRing = GnStream<T, V, 1, kGnAhead>::kBytes;
    float *pivots = reinterpret_cast<float *>(smem + (kRing > kSums ? kRing : kSums));          // [groups]
    for (int g = threadIdx.x; g < groups; g += kGnThreads) pivots[g] = pivot_of(g);
#pragma unroll
    for (int j = 0; j < P; ++j) s2[j] = both(0.0f);
    __syncthreads();                                      // the first row may be overwritten now
    rows.run([&](Pack<T, V> (&x)[1]) { add_moments<P>(x[0], pv, sm, s2); });
    __syncthreads();
    float2 *red = reinterpret_cast<float2 *>(smem);
    if (at.r < s.rows_per_step) store_folded<V>(red + at.r * stride + at.v * per_vec, sm, s2, s.fold);
    __syncthreads();
    const float inv = 1.0f / ((float)at.rows * (float)(width * s.fold));
    for (int base = 0; base < groups; base += per_pass) {
        const int g = base + mine;
        const float2 t = group_sum(s.columns, red, stride, s.rows_per_step, width, g, g < groups);
        if (g < groups && lane == 0)
            a.part[(((long long)at.n * a.groups + at.group0 + g) * s.chunks + at.chunk) * s.split + at.piece] = moments_of(pivots[g], t, inv);
    }
}

// Mean and rstd of the tile's groups from their chunks, into stat[]
__device__ __forceinline__ void gn_finish_stats(const GnArgs &a, const GnShape &s, const GnPlace &at, int v, float2 *stat)
{
    const int groups = at.groups(a, s), lanes = s.columns.lanes, lane = threadIdx.x & (lanes - 1), entries = s.chunks * s.split;
    const float inv = s.inv;
    const auto values = [&](int e) {
        if (s.split == 1) return (float)min(s.chunk_rows, a.rows - e * s.chunk_rows) * (float)a.cpg;
        const int chunk = e / s.split;
        return (float)min(s.chunk_rows, a.rows - chunk * s.chunk_rows) * (float)(min(s.tile, s.unit - (e - chunk * s.split) * s.tile) * v);
    };
    for (int base = 0; base < groups; base += s.columns.per_pass) {
        const int g = base + (threadIdx.x >> s.columns.shift);
        const bool valid = g < groups;
        const long long id = (long long)at.n * a.groups + at.group0 + g;
        const float2 *part = a.part + id * entries;
        // Sums of the distances to the first chunk's mean and of their squares: it holds at least 1 / 1024 of the values, so its
        // mean is at most 32 spreads off, and as a rule a fraction of one.
        float2 t = make_float2(0.0f, 0.0f);
        float ref = 0.0f;
        if (valid) {
            ref = __ldcg(part).x;
#pragma unroll 4
            for (int e = lane; e < entries; e += lanes) {
                const float2 p = __ldcg(part + e);
                const float n = values(e), d = p.x - ref;
                t = add2(t, make_float2(n * d, fmaf(n * d, d, p.y)));
            }
        }
        t = lane_sum(t, lanes);
        const float2 mq = moments_of(ref, t, inv);
        if (valid && lane == 0) {
            const float rstd = rsqrtf(mq.y * inv + a.eps);
            stat[g] = make_float2(mq.x, rstd);
            if (at.chunk == 0 && at.piece == 0) { a.mean[id] = mq.x; a.rstd[id] = rstd; }
        }
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kGnThreads, kGnBlocksForward) gn_apply_kernel(const __grid_constant__ GnArgs a, const __grid_constant__ GnShape s)
{
    extern __shared__ __align__(16) unsigned char smem[];  // the ring, then
    using Rows = GnStream<T, V, 1, kGnAhead>;
    float2 *stat = reinterpret_cast<float2 *>(smem + Rows::kBytes);       // [groups_per_tile] (mean, rstd)
    const GnPlace at(a, s, gridDim.x - 1 - blockIdx.x);        // what was read last comes first: it is in L2
    const int count = at.count(s), c0 = at.vec * V;
    const long long first = (at.n * a.rows + at.row0 + at.r) * a.channels + c0, step = (long long)s.rows_per_step * a.channels;
    T *dst = (T *)a.y + first;
    Rows rows;                                            // (x is not written by the first launch)
    rows.src[0] = (const T *)a.x + first;
    rows.start(smem, step, count);
    constexpr int P = Pack<T, V>::P;
    float2 mean[P], scale[P], bias[P], rstd[P];
    load_params<V>(a.weight, a.param_code, a.wide_params, c0, at.active, 1.0f, scale);
    load_params<V>(a.bias, a.param_code, a.wide_params, c0, at.active, 0.0f, bias);
    const int group = at.active ? c0 / a.cpg : at.group0, left = at.active ? (group + 1) * a.cpg - c0 : V;
    gn_wait_first();
    gn_finish_stats(a, s, at, V, stat);
    __syncthreads();
    spread_groups<V>(group - at.group0, left, a.cpg, [&](int g) { return make_float2(-stat[g].x, stat[g].y); }, mean, rstd);
#pragma unroll
    for (int j = 0; j < P; ++j) scale[j] = mul2(scale[j], rstd[j]);
    with_activation(a.act, [&](auto act) {
        rows.run([&](Pack<T, V> (&x)[1]) {
            float2 f[P];
            x[0].unpack_plus(mean, f);
#pragma unroll
            for (int j = 0; j < P; ++j) f[j] = fma2(f[j], scale[j], bias[j]);
            activate<decltype(act)::value, sizeof(T) == 2, P>(f);
            x[0].pack(f);
            x[0].store(dst);
            dst += step;
        });
    });
}

// ----------------------------------------------------------------------------- backward
// Scratch: [n, groups, chunks, split] sums of (u xhat, u), then [n, chunks, C] sums of (g xhat, g).
__host__ __device__ inline float2 *gn_channel_part(const GnArgs &a, const GnShape &s) { return a.part + a.n * a.groups * s.chunks * s.split; }

// acc[rows][stride]: every column's rows into its first one, by all threads: part p adds rows p, p + parts, ...
// and then the parts are added.  Ends with the block synchronised.
__device__ __forceinline__ void sum_columns(float2 *acc, int stride, int columns, int rows, int threads)
{
    int parts = 2 * columns > threads ? 1 : threads / columns;
    parts = parts > rows ? rows : parts;
    for (int i = threadIdx.x; i < columns * parts; i += threads) {
        const int part = parts == 1 ? 0 : i / columns, c = i - part * columns;
        float2 t = acc[part * stride + c];
#pragma unroll 4
        for (int k = part + parts; k < rows; k += parts) { const float2 e = acc[k * stride + c]; t = add2(t, e); }
        acc[part * stride + c] = t;
    }
    __syncthreads();
    if (parts > 1) {
        for (int c = threadIdx.x; c < columns; c += threads) {
            float2 t = acc[c];
            for (int k = 1; k < parts; ++k) t = add2(t, acc[k * stride + c]);
            acc[c] = t;
        }
        __syncthreads();
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kGnThreads, kGnBlocksBackward) gn_grad_sums_kernel(const __grid_constant__ GnArgs a, const __grid_constant__ GnShape s)
{
    gn_allow_second();
    const GnPlace at(a, s, blockIdx.x);
    const int count = at.count(s), c0 = at.vec * V;
    constexpr int P = Pack<T, V>::P;
    extern __shared__ __align__(16) unsigned char smem[];  // the ring; afterwards
    float2 *acc = reinterpret_cast<float2 *>(smem);       // [row slot][folded channel], then [row slot][channel]
    {
        const long long g0 = (long long)at.n * a.groups;
        float2 mean[P], scale[P], bias[P], rstd[P], sgx[P], sg[P];
        load_params<V>(a.weight, a.param_code, a.wide_params, c0, at.active, 1.0f, scale);
        load_params<V>(a.bias, a.param_code, a.wide_params, c0, at.active, 0.0f, bias);
        const int group = at.active ? c0 / a.cpg : at.group0, left = at.active ? (group + 1) * a.cpg - c0 : V;
        spread_groups<V>(group, left, a.cpg, [&](int g) { return make_float2(-a.mean[g0 + g], a.rstd[g0 + g]); }, mean, rstd);
#pragma unroll
        for (int j = 0; j < P; ++j) { scale[j] = mul2(scale[j], rstd[j]); sgx[j] = sg[j] = both(0.0f); }
        const long long first = (at.n * a.rows + at.row0 + at.r) * a.channels + c0, step = (long long)s.rows_per_step * a.channels;
        GnStream<T, V, 2, kGnAheadGrad> rows;
        rows.src[0] = (const T *)a.x + first;
        rows.src[1] = (const T *)a.dy + first;
        rows.start(smem, step, count);
        with_activation(a.act, [&](auto act) {
            rows.run([&](Pack<T, V> (&x)[2]) {
                float2 f[P], z[P], g[P];
                x[0].unpack_plus(mean, f);
                x[1].unpack(g);
#pragma unroll
                for (int j = 0; j < P; ++j) z[j] = fma2(f[j], scale[j], bias[j]);
                activate_grad<decltype(act)::value, sizeof(T) == 2, P>(z, g);
#pragma unroll
                for (int j = 0; j < P; ++j) { sg[j] = add2(sg[j], g[j]); sgx[j] = fma2(g[j], f[j], sgx[j]); }
            });
        });
        __syncthreads();
        // sums of (u xhat, rstd u) of the groups: u xhat = g scale (x - mean)
        const int per_vec = s.per_vec, stride = s.tile * per_vec, groups = at.groups(a, s), lanes = s.columns.lanes, lane = threadIdx.x & (lanes - 1);
        const int width = s.split == 1 ? s.columns.width : at.width(s) * per_vec;
        if (at.r < s.rows_per_step) {
            float2 ux[P], u[P];
#pragma unroll
            for (int j = 0; j < P; ++j) { ux[j] = mul2(scale[j], sgx[j]); u[j] = mul2(scale[j], sg[j]); }
            store_folded<V>(acc + at.r * stride + at.v * per_vec, ux, u, s.fold);
        }
        __syncthreads();
        for (int base = 0; base < groups; base += s.columns.per_pass) {
            const int g = base + (threadIdx.x >> s.columns.shift);
            const float2 t = group_sum(s.columns, acc, stride, s.rows_per_step, width, g, g < groups);
            if (g < groups && lane == 0)
                a.part[(((long long)at.n * a.groups + at.group0 + g) * s.chunks + at.chunk) * s.split + at.piece] = t;
        }
        if (!a.dweight && !a.dbias) return;
        __syncthreads();
        if (at.r < s.rows_per_step) {
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const float2 gx = mul2(sgx[j], rstd[j]);
                float2 *to = acc + (at.r * s.tile + at.v) * V + 2 * j;
                to[0] = make_float2(gx.x, sg[j].x);
                if (V > 1) to[V > 1 ? 1 : 0] = make_float2(gx.y, sg[j].y);
            }
        }
    }
    __syncthreads();
    const int tile_c0 = (at.vec - at.v) * V, channels = at.width(s) * V;
    float2 *chan = a.channel_part + (long long)at.item * a.channels + tile_c0;
    sum_columns(acc, s.tile * V, channels, s.rows_per_step, kGnThreads);
    for (int c = threadIdx.x; c < channels; c += kGnThreads) chan[c] = acc[c];
}

// dweight and dbias of 32 channels by a cluster: the channel sums of all samples and chunks, a share of the rows to
// each block, always added in the same order.  Launched while the last blocks in front of it run, and waits for them: half
// a microsecond less per backward pass (64 x 14^2 float16 9.3 -> 8.8 us).  Latency: 64 samples x 320 channels are 1 MB of sums.
constexpr int kGnParamRanks = 8;
static __global__ void __launch_bounds__(kGnThreads) gn_grad_params_kernel(const GnArgs a, const float2 *sums, const long long rows)
{
    __shared__ float2 acc[kGnThreads / 32][33], share[32];
    const int x = threadIdx.x % 32, y = threadIdx.x / 32, lanes = kGnThreads / 32, c = blockIdx.y * 32 + x;
    const int ranks = gridDim.x, rank = blockIdx.x;
    float2 t = make_float2(0.0f, 0.0f);
    gn_wait_first();
    if (c < a.channels) {
#pragma unroll 8
        for (long long i = rank * lanes + y; i < rows; i += lanes * ranks) t = add2(t, sums[i * a.channels + c]);
    }
    acc[y][x] = t;
    __syncthreads();
    if (y == 0) {
        t = acc[0][x];
        for (int j = 1; j < lanes; ++j) t = add2(t, acc[j][x]);
        share[x] = t;
    }
    if (ranks > 1) { cluster_arrive(); cluster_wait(); }
    else __syncthreads();
    if (rank == 0 && y == 0 && c < a.channels) {
        for (int k = 1; k < ranks; ++k) t = add2(t, load_rank(share + x, k));
        if (a.dweight) store_code(a.dweight, a.param_code, c, t.x);
        if (a.dbias) store_code(a.dbias, a.param_code, c, t.y);
    }
    if (ranks > 1) { cluster_arrive(); cluster_wait(); }
}

template <typename T, int V>
__global__ void __launch_bounds__(kGnThreads, kGnBlocksBackward) gn_grad_input_kernel(const __grid_constant__ GnArgs a, const __grid_constant__ GnShape s)
{
    gn_allow_second();
    extern __shared__ __align__(16) unsigned char smem[];  // the ring, then
    using Rows = GnStream<T, V, 2, kGnAheadGrad>;
    float2 *stat = reinterpret_cast<float2 *>(smem + Rows::kBytes);       // [groups_per_tile] means of (u xhat, rstd u)
    const GnPlace at(a, s, gridDim.x - 1 - blockIdx.x);
    const int count = at.count(s), c0 = at.vec * V;
    constexpr int P = Pack<T, V>::P;
    const long long first = (at.n * a.rows + at.row0 + at.r) * a.channels + c0, step = (long long)s.rows_per_step * a.channels;
    Rows rows;                                            // (x and dy are not written by the first launch)
    rows.src[0] = (const T *)a.x + first;
    rows.src[1] = (const T *)a.dy + first;
    rows.start(smem, step, count);
    const long long g0 = (long long)at.n * a.groups;
    float2 mean[P], scale[P], bias[P], rstd[P], m_ux[P], m_u[P];
    load_params<V>(a.weight, a.param_code, a.wide_params, c0, at.active, 1.0f, scale);
    load_params<V>(a.bias, a.param_code, a.wide_params, c0, at.active, 0.0f, bias);
    const int group = at.active ? c0 / a.cpg : at.group0, left = at.active ? (group + 1) * a.cpg - c0 : V;
    spread_groups<V>(group, left, a.cpg, [&](int g) { return make_float2(-a.mean[g0 + g], a.rstd[g0 + g]); }, mean, rstd);
#pragma unroll
    for (int j = 0; j < P; ++j) scale[j] = mul2(scale[j], rstd[j]);
    gn_wait_first();
    const int groups = at.groups(a, s), lanes = s.columns.lanes, lane = threadIdx.x & (lanes - 1), entries = s.chunks * s.split;
    const float inv = s.inv;
    for (int base = 0; base < groups; base += s.columns.per_pass) {
        const int g = base + (threadIdx.x >> s.columns.shift);
        float ux = 0.0f, u = 0.0f;
        if (g < groups) {
            const float2 *part = a.part + ((long long)at.n * a.groups + at.group0 + g) * entries;
#pragma unroll 4
            for (int e = lane; e < entries; e += lanes) { const float2 p = __ldcg(part + e); ux += p.x; u += p.y; }
        }
        ux = lane_sum(ux, lanes);
        u = lane_sum(u, lanes);
        if (g < groups && lane == 0) stat[g] = make_float2(ux * inv, u * inv);
    }
    __syncthreads();
    spread_groups<V>(group - at.group0, left, a.cpg, [&](int g) { return make_float2(-stat[g].x, -stat[g].y); }, m_ux, m_u);
#pragma unroll
    for (int j = 0; j < P; ++j) m_ux[j] = mul2(m_ux[j], mul2(rstd[j], rstd[j]));       // dx = g scale - ((x - mean) m_ux + m_u)
    T *out = (T *)a.dx + first;
    with_activation(a.act, [&](auto act) {
        rows.run([&](Pack<T, V> (&x)[2]) {
            float2 f[P], z[P], g[P];
            x[0].unpack_plus(mean, f);
            x[1].unpack(g);
#pragma unroll
            for (int j = 0; j < P; ++j) z[j] = fma2(f[j], scale[j], bias[j]);
            activate_grad<decltype(act)::value, sizeof(T) == 2, P>(z, g);
#pragma unroll
            for (int j = 0; j < P; ++j) g[j] = fma2(g[j], scale[j], fma2(f[j], m_ux[j], m_u[j]));
            x[1].pack(g);
            x[1].store(out);
            out += step;
        });
    });
}

// ----------------------------------------------------------------------------- launches
// Shared memory and cluster sizes beyond the defaults, once per device (twice does no harm)
template <auto kernel, bool CLUSTER> cudaError_t gn_prepare(int bytes)
{
    static std::atomic<unsigned> ready{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    if (device < 32 && (ready.load(std::memory_order_acquire) >> device) & 1u) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && CLUSTER) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && device < 32) ready.fetch_or(1u << device, std::memory_order_release);
    return e;
}

template <typename Kernel, typename... Args>
cudaError_t gn_launch_kernel(Kernel kernel, dim3 grid, size_t smem, bool dependent, cudaStream_t stream, Args... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kGnThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

inline cudaError_t gn_launch_params(const GnArgs &a, const float2 *sums, long long rows, cudaStream_t stream)
{
    cudaLaunchConfig_t cfg = {};
    const int ranks = rows >= 64 ? kGnParamRanks : 1;    // (fewer rows are one block's work)
    cfg.gridDim = dim3(ranks, (a.channels + 31) / 32);
    cfg.blockDim = dim3(kGnThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ranks > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, gn_grad_params_kernel, a, sums, rows);
}

template <typename T, int V> cudaError_t gn_launch_streaming(const GnArgs &all, bool backward, cudaStream_t stream)
{
    GnArgs a = all;
    const GnShape s = gn_shape(a, V, backward);
    const size_t stat = s.groups_per_tile * sizeof(float2), sums = kGnThreads * V * sizeof(float2);
    constexpr size_t ring = GnStream<T, V, 1, kGnAhead>::kBytes, grad_ring = GnStream<T, V, 2, kGnAheadGrad>::kBytes;
    const dim3 grid((unsigned)(a.n * s.chunks), s.tiles);
    cudaError_t e;
    if (!backward) {
        e = gn_launch_kernel(gn_stats_kernel<T, V>, grid, (ring > sums ? ring : sums) + stat, false, stream, a, s);
        return e != cudaSuccess ? e : gn_launch_kernel(gn_apply_kernel<T, V>, grid, ring + stat, true, stream, a, s);
    }
    a.channel_part = gn_channel_part(a, s);
    // A quarter of an SM's shared memory keeps a fourth block off it: kernels with narrow vectors need so few registers that
    // the second launch's blocks would crowd on the SMs that are free first (32 x 33 x 112^2 float32 132 us against 104,
    // 16 x 130 x 96^2 bfloat16 81 against 67; forward, where up to four blocks fit, no difference).
    // (A tile has kGnThreads V channels at most, and no more groups.)
    constexpr int grad_bytes = 57 * 1024;
    static_assert(kGnBlocksBackward == 3 && grad_ring + kGnThreads * V * sizeof(float2) <= grad_bytes);
    e = gn_prepare<gn_grad_sums_kernel<T, V>, false>(grad_bytes);
    if (e == cudaSuccess) e = gn_launch_kernel(gn_grad_sums_kernel<T, V>, grid, grad_bytes, false, stream, a, s);
    if (e == cudaSuccess && a.dx) e = gn_prepare<gn_grad_input_kernel<T, V>, false>(grad_bytes);
    if (e == cudaSuccess && a.dx) e = gn_launch_kernel(gn_grad_input_kernel<T, V>, grid, grad_bytes, true, stream, a, s);
    if (e == cudaSuccess && (a.dweight || a.dbias)) e = gn_launch_params(a, a.channel_part, a.n * s.chunks, stream);
    return e;
}

// Widest vector that divides the channels and that the pointers are aligned to
__host__ inline int gn_vector(const GnArgs &a, int elem_bytes)
{
    uintptr_t bits = (uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.dy | (uintptr_t)a.dx;
    int v = 16 / elem_bytes;
    while (v > 1 && (a.channels % v != 0 || bits % (v * elem_bytes) != 0)) v /= 2;
    while (v > 1 && gn_unit(a, v) > kGnThreads && a.cpg % v) v /= 2;
    return v;
}

}  // namespace ta

#include "ta_group_norm_cluster.cuh"

namespace ta {

template <typename T> cudaError_t gn_launch(const GnArgs &a, bool backward, cudaStream_t stream)
{
    const int v = gn_vector(a, sizeof(T));
    GnPlan plan;
    if (gn_plan<T>(a, v, backward, plan)) return gn_launch_planned<T>(a, plan, backward, stream);
    switch (v) {
    case 8: if constexpr (sizeof(T) == 2) return gn_launch_streaming<T, 8>(a, backward, stream);
    case 4: return gn_launch_streaming<T, 4>(a, backward, stream);
    case 2: return gn_launch_streaming<T, 2>(a, backward, stream);
    default: return gn_launch_streaming<T, 1>(a, backward, stream);
    }
}

// scratch of a call, bytes
template <typename T> size_t gn_scratch_bytes(const GnArgs &a, bool backward)
{
    const int v = gn_vector(a, sizeof(T));
    const bool params = backward && (a.dweight || a.dbias);
    GnPlan plan;
    if (gn_plan<T>(a, v, backward, plan)) return params ? (size_t)a.n * plan.ranks * a.channels * sizeof(float2) : 0;
    const GnShape s = gn_shape(a, v, backward);
    return ((size_t)a.n * a.groups * s.chunks * s.split + (params ? (size_t)a.n * s.chunks * a.channels : 0)) * sizeof(float2);
}

}  // namespace ta
