// Group norm in one pass over the data: a cluster of thread blocks holds a slab of whole groups of one
// sample in shared memory, agrees on its statistics through distributed shared memory, and writes
// the result from there - one read and one write of the features, one launch.
//
// Every thread copies with cp.async exactly the vectors that it works on later, all of them before it waits for
// the first, so a block's whole share is in flight at once and nothing but cp.async.wait_group orders
// the copies.  The share is loaded in four parts and reduced part by part as they arrive.
#pragma once
#include <atomic>

namespace ta {

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

__device__ __forceinline__ void copy_async16(void *shared, const void *global)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(shared)), "l"(global) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the last `left` of four parts have arrived
__device__ __forceinline__ void copy_wait(int left)
{
    if (left >= 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
    else if (left == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (left == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// A cluster of `ranks` blocks covers a slab of `vecs` channel vectors; block k holds rows [k rows_per_block, ...),
// thread t channel vector t % vecs of rows t / vecs + i rows_per_step, i < steps.
struct GnPlan {
    int threads, ranks, vecs, slabs, rows_per_step, groups, fold, steps, smem, rows_per_block;
    GnLanes columns;                    // sums over the slab's columns
};

// grid: (samples x ranks, slabs), clusters along x
struct GnClusterPlace {
    int rank, r, v, c0, slab_c0, slab_channels, groups, rows, count, group, left;
    unsigned n;
    bool active;
    long long first, step;              // element offset of the thread's first vector, distance to the next
    __device__ __forceinline__ GnClusterPlace(const GnArgs &a, const GnPlan &p, int v_elems)
    {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm("mov.u32 %0, %%clusterid.x;" : "=r"(n));
        r = threadIdx.x / (unsigned)p.vecs;
        v = threadIdx.x - r * p.vecs;
        slab_c0 = blockIdx.y * p.vecs * v_elems;
        c0 = slab_c0 + v * v_elems;
        slab_channels = min(p.vecs * v_elems, a.channels - slab_c0);
        groups = min(p.groups, a.groups - (int)blockIdx.y * p.groups);
        const int row0 = rank * p.rows_per_block;
        rows = max(0, min(p.rows_per_block, (int)a.rows - row0));
        active = r < p.rows_per_step && c0 < a.channels;
        count = active && rows > r ? (rows - r + p.rows_per_step - 1) / (unsigned)p.rows_per_step : 0;
        first = (n * a.rows + row0 + r) * a.channels + c0;
        step = (long long)p.rows_per_step * a.channels;
        group = active ? (unsigned)(v * v_elems) / (unsigned)a.cpg : 0;                   // within the slab
        left = active ? (group + 1) * a.cpg - v * v_elems : v_elems;
    }
};

template <typename T, int THREADS, int PER_SM>
__global__ void __launch_bounds__(THREADS, PER_SM) gn_cluster_kernel(const GnArgs a, const GnPlan p)
{
    constexpr int V = 16 / sizeof(T), P = V / 2;
    extern __shared__ __align__(16) unsigned char smem[];
    const int slots = p.rows_per_step * p.vecs, per_vec = V / p.fold, stride = p.vecs * per_vec;
    Pack<T, V> *data = reinterpret_cast<Pack<T, V> *>(smem) + threadIdx.x;             // [steps][slots]
    float2 *pub = reinterpret_cast<float2 *>(smem + (size_t)p.steps * slots * 16);    // [groups] this block's (mean, squared deviations), read by the cluster
    float2 *stat = pub + p.groups;                      // [groups] the sample's (mean, rstd)
    float *block_mean = reinterpret_cast<float *>(stat + p.groups);                    // [groups]
    float *red = block_mean + p.groups;                 // [rows_per_step][folded channels of the slab]
    const GnClusterPlace at(a, p, V);
    const T *src = (const T *)a.x + at.first;
    const int quarter = (p.steps + 3) / 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int end = min((q + 1) * quarter, at.count);
        for (int i = q * quarter; i < end; ++i, src += at.step) copy_async16(data + i * slots, src);
        copy_commit();
    }
    float2 scale[P], bias[P];
    load_params<V>(a.weight, a.param_code, a.wide_params, at.c0, at.active, 1.0f, scale);
    load_params<V>(a.bias, a.param_code, a.wide_params, at.c0, at.active, 0.0f, bias);

    // mean and squared deviations, as in gn_stats_kernel
    float2 pv[P], sm[P], s2[P];
#pragma unroll
    for (int j = 0; j < P; ++j) pv[j] = sm[j] = s2[j] = both(0.0f);
    for (int q = 0; q < 4; ++q) {
        copy_wait(3 - q);
        const int end = min((q + 1) * quarter, at.count);
        if (q == 0 && end > 0) {
            data[0].unpack(pv);
#pragma unroll
            for (int j = 0; j < P; ++j) pv[j] = neg2(pv[j]);
        }
#pragma unroll 2
        for (int i = q * quarter; i < end; ++i) add_moments<P>(data[i * slots], pv, sm, s2);
    }
    float *slot = red + at.r * stride + at.v * per_vec;
    const bool holds = at.r < p.rows_per_step;
    float t[V];
#pragma unroll
    for (int j = 0; j < V; ++j) t[j] = fmaf((float)-at.count, half_of_pair(pv[j / 2], j), half_of_pair(sm[j / 2], j));
    if (holds) store_folded<V>(slot, t, p.fold);
    __syncthreads();
    const int lanes = p.columns.lanes, lane = threadIdx.x & (lanes - 1), per_pass = THREADS / lanes, mine = threadIdx.x / (unsigned)lanes;
    const float block_inv = 1.0f / ((float)max(at.rows, 1) * (float)a.cpg);
    for (int base = 0; base < at.groups; base += per_pass) {
        const int g = base + mine;
        const float m = group_sum(p.columns, red, stride, p.rows_per_step, p.columns.width, g, g < at.groups) * block_inv;
        if (g < at.groups && lane == 0) block_mean[g] = m;
    }
    __syncthreads();
    deviations<V>(at.group, at.left, a.cpg, at.count, pv, sm, s2, block_mean, t);
    if (holds) store_folded<V>(slot, t, p.fold);
    __syncthreads();
    for (int base = 0; base < at.groups; base += per_pass) {
        const int g = base + mine;
        const float q = group_sum(p.columns, red, stride, p.rows_per_step, p.columns.width, g, g < at.groups);
        if (g < at.groups && lane == 0) pub[g] = make_float2(block_mean[g], q);
    }
    if (p.ranks > 1) { cluster_arrive(); cluster_wait(); }
    else __syncthreads();
    const float inv = 1.0f / ((float)a.rows * (float)a.cpg);
    for (int base = 0; base < at.groups; base += per_pass) {
        const int g = base + mine;
        const bool valid = g < at.groups;
        // at most sixteen blocks: a lane has one of them, or lanes / 16 times as many
        float m = 0.0f, q = 0.0f;
        for (int k = lane; k < p.ranks; k += lanes) {
            const float n = (float)max(0, min(p.rows_per_block, (int)a.rows - k * p.rows_per_block)) * (float)a.cpg;
            if (valid) m = fmaf(n, p.ranks > 1 ? load_rank(pub + g, k).x : pub[g].x, m);
        }
        m = __shfl_sync(0xffffffffu, lane_sum(m, lanes) * inv, 0, lanes);
        for (int k = lane; k < p.ranks; k += lanes) {
            const float n = (float)max(0, min(p.rows_per_block, (int)a.rows - k * p.rows_per_block)) * (float)a.cpg;
            if (valid && n > 0.0f) {
                const float2 b = p.ranks > 1 ? load_rank(pub + g, k) : pub[g];
                q += fmaf(n * (b.x - m), b.x - m, b.y);
            }
        }
        q = lane_sum(q, lanes);
        if (valid && lane == 0) {
            const float rstd = rsqrtf(q * inv + a.eps);
            stat[g] = make_float2(m, rstd);
            if (at.rank == 0) {
                const long long id = (long long)at.n * a.groups + blockIdx.y * p.groups + g;
                a.mean[id] = m;
                a.rstd[id] = rstd;
            }
        }
    }
    if (p.ranks > 1) cluster_arrive();                  // done with the others' memory
    __syncthreads();
    {
        float2 mean[P], rstd[P];
        spread_groups<V>(at.group, at.left, a.cpg, [&](int g) { return make_float2(-stat[g].x, stat[g].y); }, mean, rstd);
#pragma unroll
        for (int j = 0; j < P; ++j) scale[j] = mul2(scale[j], rstd[j]);
        T *dst = (T *)a.y + at.first;
        with_activation(a.act, [&](auto act) {
#pragma unroll 2
            for (int i = 0; i < at.count; ++i, dst += at.step) {
                float2 f[P];
                Pack<T, V> x = data[i * slots];
                x.unpack(f);
#pragma unroll
                for (int j = 0; j < P; ++j) f[j] = fma2(add2(f[j], mean[j]), scale[j], bias[j]);
                activate<decltype(act)::value, sizeof(T) == 2, P>(f);
                x.pack(f);
                x.store(dst);
            }
        });
    }
    if (p.ranks > 1) cluster_wait();                    // no block leaves while others read it
}

// Backward: x and dy side by side in shared memory.
template <typename T, int THREADS, int PER_SM>
__global__ void __launch_bounds__(THREADS, PER_SM) gn_cluster_grad_kernel(const GnArgs a, const GnPlan p, float2 *channel_sums)
{
    constexpr int V = 16 / sizeof(T), P = V / 2;
    extern __shared__ __align__(16) unsigned char smem[];
    const int slots = p.rows_per_step * p.vecs, columns = p.vecs * V;
    Pack<T, V> *xs = reinterpret_cast<Pack<T, V> *>(smem) + threadIdx.x, *ds = xs + (size_t)p.steps * slots;      // [steps][slots] each
    float2 *chan = reinterpret_cast<float2 *>(smem + (size_t)p.steps * slots * 32);    // [rows_per_step][channels of the slab], then in the first row
                                                        // this block's sums of (g xhat, g), read by the cluster
    float2 *pub = chan + p.rows_per_step * columns;                       // [groups] sums of (u xhat, u), read by the cluster
    float2 *stat = pub + p.groups;                      // [groups] the sample's means of (u xhat, u)
    const GnClusterPlace at(a, p, V);
    const int quarter = (p.steps + 3) / 4;
    {
        const T *px = (const T *)a.x + at.first, *pd = (const T *)a.dy + at.first;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int end = min((q + 1) * quarter, at.count);
            for (int i = q * quarter; i < end; ++i, px += at.step, pd += at.step) {
                copy_async16(xs + i * slots, px);
                copy_async16(ds + i * slots, pd);
            }
            copy_commit();
        }
    }
    const long long g0 = (long long)at.n * a.groups + blockIdx.y * p.groups;
    float2 mean[P], scale[P], bias[P], rstd[P];
    load_params<V>(a.weight, a.param_code, a.wide_params, at.c0, at.active, 1.0f, scale);
    load_params<V>(a.bias, a.param_code, a.wide_params, at.c0, at.active, 0.0f, bias);
    spread_groups<V>(at.group, at.left, a.cpg, [&](int g) { return make_float2(-a.mean[g0 + g], a.rstd[g0 + g]); }, mean, rstd);
#pragma unroll
    for (int j = 0; j < P; ++j) scale[j] = mul2(scale[j], rstd[j]);
    {
        float2 sgx[P], sg[P];
#pragma unroll
        for (int j = 0; j < P; ++j) sgx[j] = sg[j] = both(0.0f);
        with_activation(a.act, [&](auto act) {
            for (int q = 0; q < 4; ++q) {
                copy_wait(3 - q);
                const int end = min((q + 1) * quarter, at.count);
                for (int i = q * quarter; i < end; ++i) {
                    float2 f[P], z[P], g[P];
                    xs[i * slots].unpack(f);
                    ds[i * slots].unpack(g);
#pragma unroll
                    for (int j = 0; j < P; ++j) { f[j] = add2(f[j], mean[j]); z[j] = fma2(f[j], scale[j], bias[j]); }
                    activate_grad<decltype(act)::value, sizeof(T) == 2, P>(z, g);
#pragma unroll
                    for (int j = 0; j < P; ++j) { sg[j] = add2(sg[j], g[j]); sgx[j] = fma2(g[j], f[j], sgx[j]); }
                }
            }
        });
        if (at.r < p.rows_per_step) {
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const float2 gx = mul2(sgx[j], rstd[j]);
                reinterpret_cast<float4 *>(chan + (at.r * p.vecs + at.v) * V)[j] = make_float4(gx.x, sg[j].x, gx.y, sg[j].y);
            }
        }
        __syncthreads();
        sum_columns(chan, columns, at.slab_channels, p.rows_per_step, THREADS);
    }
    const int lanes = p.columns.lanes, lane = threadIdx.x & (lanes - 1);
    for (int base = 0; base < at.groups; base += THREADS / lanes) {
        const int g = base + threadIdx.x / lanes;
        float ux = 0.0f, u = 0.0f;
        if (g < at.groups)
            for (int e = lane; e < a.cpg; e += lanes) {
                const int c = g * a.cpg + e;
                const float w = a.weight ? load_code(a.weight, a.param_code, at.slab_c0 + c) : 1.0f;
                ux = fmaf(w, chan[c].x, ux);
                u = fmaf(w, chan[c].y, u);
            }
        ux = lane_sum(ux, lanes);
        u = lane_sum(u, lanes);
        if (g < at.groups && lane == 0) pub[g] = make_float2(ux, u);
    }
    if (p.ranks > 1) { cluster_arrive(); cluster_wait(); }
    else __syncthreads();
    const float inv = 1.0f / ((float)a.rows * (float)a.cpg);
    for (int base = 0; base < at.groups; base += THREADS / lanes) {
        const int g = base + threadIdx.x / lanes;
        float ux = 0.0f, u = 0.0f;
        if (g < at.groups)
            for (int k = lane; k < p.ranks; k += lanes) {
                const float2 e = p.ranks > 1 ? load_rank(pub + g, k) : pub[g];
                ux += e.x; u += e.y;
            }
        ux = lane_sum(ux, lanes);
        u = lane_sum(u, lanes);
        if (g < at.groups && lane == 0) stat[g] = make_float2(ux * inv, u * inv);
    }
    if (channel_sums)                                   // each block adds up a share of the channels
        for (int c = at.rank + (int)threadIdx.x * p.ranks; c < at.slab_channels; c += THREADS * p.ranks) {
            float2 t = make_float2(0.0f, 0.0f);
#pragma unroll 8
            for (int k = 0; k < p.ranks; ++k) {
                const float2 e = p.ranks > 1 ? load_rank(chan + c, k) : chan[c];
                t.x += e.x; t.y += e.y;
            }
            channel_sums[(long long)at.n * a.channels + at.slab_c0 + c] = t;
        }
    if (p.ranks > 1) cluster_arrive();
    __syncthreads();
    if (a.dx) {
        float2 m_ux[P], m_u[P];
        spread_groups<V>(at.group, at.left, a.cpg, [&](int g) { return make_float2(-stat[g].x, -stat[g].y); }, m_ux, m_u);
#pragma unroll
        for (int j = 0; j < P; ++j) {
            m_ux[j] = mul2(m_ux[j], mul2(rstd[j], rstd[j]));
            m_u[j] = mul2(m_u[j], rstd[j]);
        }
        T *dst = (T *)a.dx + at.first;
        with_activation(a.act, [&](auto act) {
            for (int i = 0; i < at.count; ++i, dst += at.step) {
                float2 f[P], z[P], g[P];
                xs[i * slots].unpack(f);
                Pack<T, V> d = ds[i * slots];
                d.unpack(g);
#pragma unroll
                for (int j = 0; j < P; ++j) { f[j] = add2(f[j], mean[j]); z[j] = fma2(f[j], scale[j], bias[j]); }
                activate_grad<decltype(act)::value, sizeof(T) == 2, P>(z, g);
#pragma unroll
                for (int j = 0; j < P; ++j) g[j] = fma2(g[j], scale[j], fma2(f[j], m_ux[j], m_u[j]));
                d.pack(g);
                d.store(dst);
            }
        });
    }
    if (p.ranks > 1) cluster_wait();
}

// ----------------------------------------------------------------------------- choice of the plan
// false: a slab of whole groups does not fit a cluster's shared memory
__host__ inline bool gn_plan(const GnArgs &a, int v, int elem_bytes, bool backward, GnPlan &p)
{
    if (v * elem_bytes != 16 || a.rows >= (1LL << 30)) return false;
    const int all = a.channels / v, unit = gn_unit(a, v);
    // blocks per SM, their threads (64 registers each forward, 80 backward), their shared memory
    struct Class { int per_sm, threads, bytes; };
    static const Class forward_classes[] = {{4, 256, 56 * 1024}, {3, 320, 75 * 1024}, {2, 512, 113 * 1024}};
    static const Class backward_classes[] = {{4, 192, 56 * 1024}, {3, 256, 75 * 1024}, {2, 384, 113 * 1024}};
    for (int max_ranks = 8; max_ranks <= 16; max_ranks *= 2)
        for (int i = 0; i < 3; ++i)
            for (int seg = all < 32 ? all : 32; seg >= 1; seg = seg == 1 ? 0 : (seg + 1) / 2) {
                const Class &c = backward ? backward_classes[i] : forward_classes[i];
                const int vecs = (seg + unit - 1) / unit * unit;
                if (vecs * 16 < 64 && vecs < all) break;
                if (vecs > c.threads) continue;
                p.threads = c.threads;
                p.vecs = vecs;
                p.slabs = (all + vecs - 1) / vecs;
                p.rows_per_step = c.threads / vecs;
                p.groups = vecs * v / a.cpg;
                p.fold = v;
                while (a.cpg % p.fold) p.fold /= 2;
                const int slots = p.rows_per_step * vecs;
                const int extra = backward ? slots * v * 8 + 2 * p.groups * 8 : slots * (v / p.fold) * 4 + p.groups * 20;
                const int steps = (c.bytes - 1024 - extra) / (slots * (backward ? 32 : 16));
                if (steps < 1) continue;
                const long long ranks = (a.rows + (long long)p.rows_per_step * steps - 1) / ((long long)p.rows_per_step * steps);
                if (ranks > max_ranks) continue;
                p.ranks = (int)ranks;
                p.rows_per_block = (int)((a.rows + ranks - 1) / ranks);
                p.steps = (p.rows_per_block + p.rows_per_step - 1) / p.rows_per_step;
                p.smem = p.steps * slots * (backward ? 32 : 16) + extra;
                p.columns = gn_lanes(p.groups, p.threads, backward ? a.cpg : a.cpg / p.fold);
                return a.n * ranks < (1LL << 31) && p.slabs <= 65535;
            }
    return false;
}

template <auto kernel, typename... Args>
cudaError_t gn_launch_cluster( const GnPlan &p, long long samples, cudaStream_t stream, Args... args)
{
    // once per device: shared memory and cluster size beyond the defaults (setting them twice does no harm)
    static std::atomic<unsigned> ready{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    if (device > 31 || !((ready.load(std::memory_order_acquire) >> device) & 1u)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 113 * 1024);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        if (device <= 31) ready.fetch_or(1u << device, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(samples * p.ranks), p.slabs);
    cfg.blockDim = dim3(p.threads);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.ranks > 1 ? 1 : 0;                 // (a cluster of one needs no attribute: 1 us less on the host)
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T> cudaError_t gn_launch_planned(const GnArgs &a, const GnPlan &p, bool backward, cudaStream_t stream)
{
    if (!backward)
        return p.threads == 256   ? gn_launch_cluster<gn_cluster_kernel<T, 256, 4>>(p, a.n, stream, a, p)
               : p.threads == 320 ? gn_launch_cluster<gn_cluster_kernel<T, 320, 3>>(p, a.n, stream, a, p)
                                  : gn_launch_cluster<gn_cluster_kernel<T, 512, 2>>(p, a.n, stream, a, p);
    float2 *sums = a.dweight || a.dbias ? a.part : nullptr;
    const cudaError_t e = p.threads == 192   ? gn_launch_cluster<gn_cluster_grad_kernel<T, 192, 4>>(p, a.n, stream, a, p, sums)
                          : p.threads == 256 ? gn_launch_cluster<gn_cluster_grad_kernel<T, 256, 3>>(p, a.n, stream, a, p, sums)
                                             : gn_launch_cluster<gn_cluster_grad_kernel<T, 384, 2>>(p, a.n, stream, a, p, sums);
    if (e != cudaSuccess || !sums) return e;
    return gn_launch_kernel(gn_grad_params_kernel, dim3((a.channels + 31) / 32), 0, false, stream, a, (const float2 *)sums, a.n);
}

}  // namespace ta
