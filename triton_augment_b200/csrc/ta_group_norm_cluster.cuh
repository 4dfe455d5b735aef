// Group norm in one pass over the data: a cluster of thread blocks holds a slab of whole groups of one
// sample in shared memory, agrees on its statistics through distributed shared memory, and writes the
// result from there - one read and one write of the features, one launch.
//
// Every thread copies with cp.async exactly the vectors that it works on later, all of them before it waits for
// the first, so a block's whole share is in flight at once and nothing but cp.async.wait_group orders
// the copies.  The share is loaded in four parts and added up part by part as they arrive.
//
// What bounds it: the time a block lives, of which the copies take a third and the arithmetic another; about 200 KB
// per SM are in flight.  32 x 256 x 56^2 bfloat16 with SiLU 31.4 us forward, 58.5 us backward; 64 x 320 x 28^2 25.0 and 44.6 us.
// (Divisions by powers of two in the kernels, and groups looked up in branches, cost 2.2 and 3.5 us of the latter.)
// (Clusters that stay and fetch the next sample into a second buffer meanwhile have half the blocks
// per SM to hide the latency of the sums: 32 x 256 x 56^2 bfloat16 37 us against 34, both before the pivot's one reduction.
// Clusters that start up to 3 us apart, so that copies and arithmetic of different ones overlap: 3 % faster there, 2 % slower
// on 64 x 320 x 28^2, 14 % on 64 x 1024 x 7^2.)
#pragma once

namespace ta {

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
    int threads, ranks, vecs, slabs, rows_per_step, groups, fold, per_vec, steps, smem, rows_per_block;      // per_vec: folded values of a vector
    float inv, block_inv;               // 1 / (values of a group in the sample), in a full block
    int data_bytes;                     // of the features, in front of everything else in shared memory
    FastDiv vecs_div, step_div, cpg_div, slab_div;
    GnLanes columns;                    // sums over the slab's columns
};

// One cluster per (sample, slab), the slabs of a sample side by side
struct GnClusterPlace {
    int rank, slab, r, v, c0, slab_c0, slab_channels, groups, rows, count, group, left;
    unsigned n;
    bool active, holds;
    long long first, step;              // element offset of the thread's first vector, distance to the next
    __device__ __forceinline__ GnClusterPlace(const GnArgs &a, const GnPlan &p, int v_elems)
    {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        unsigned item;
        asm("mov.u32 %0, %%clusterid.x;" : "=r"(item));
        n = fast_div(item, p.slab_div);
        slab = item - n * p.slabs;
        r = (int)fast_div(threadIdx.x, p.vecs_div);
        v = threadIdx.x - r * p.vecs;
        slab_c0 = slab * p.vecs * v_elems;
        c0 = slab_c0 + v * v_elems;
        slab_channels = min(p.vecs * v_elems, a.channels - slab_c0);
        groups = min(p.groups, a.groups - slab * p.groups);
        const int row0 = rank * p.rows_per_block;
        rows = max(0, min(p.rows_per_block, (int)a.rows - row0));
        holds = r < p.rows_per_step;
        active = holds && c0 < a.channels;
        count = active && rows > r ? (int)fast_div(rows - r + p.rows_per_step - 1, p.step_div) : 0;
        first = (n * a.rows + row0 + r) * a.channels + c0;
        step = (long long)p.rows_per_step * a.channels;
        group = active ? (int)fast_div(v * v_elems, p.cpg_div) : 0;                       // within the slab
        left = active ? (group + 1) * a.cpg - v * v_elems : v_elems;
    }
};

template <typename T, int THREADS, int PER_SM>
__global__ void __launch_bounds__(THREADS, PER_SM) gn_cluster_kernel(const __grid_constant__ GnArgs a, const __grid_constant__ GnPlan p)
{
    constexpr int V = 16 / sizeof(T), P = V / 2;
    extern __shared__ __align__(16) unsigned char smem[];
    const int slots = p.rows_per_step * p.vecs, per_vec = p.per_vec, stride = p.vecs * per_vec;
    Pack<T, V> *data = reinterpret_cast<Pack<T, V> *>(smem) + threadIdx.x;             // [steps][slots]
    float2 *pub = reinterpret_cast<float2 *>(smem + p.data_bytes);                     // [groups] this block's (mean, squared deviations), read by the cluster
    float2 *stat = pub + p.groups;                      // [groups] the sample's (mean, rstd)
    float2 *red = stat + p.groups;                      // [rows_per_step][folded channels of the slab]
    const GnClusterPlace at(a, p, V);
    const int quarter = (p.steps + 3) / 4;
    {
        const T *src = (const T *)a.x + at.first;
        Pack<T, V> *to = data;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int end = min((q + 1) * quarter, at.count);
            for (int i = q * quarter; i < end; ++i, src += at.step, to += slots) copy_async<16>(to, src);
            copy_commit();
        }
    }
    float2 scale[P], bias[P];
    load_params<V>(a.weight, a.param_code, a.wide_params, at.c0, at.active, 1.0f, scale);
    load_params<V>(a.bias, a.param_code, a.wide_params, at.c0, at.active, 0.0f, bias);
    // The pivot of a group: the mean of its first channel over the block's first rows, up to eight, with the loss
    // that gn_stats_kernel states.
    const int sample_rows = min(min(8, p.rows_per_step), at.rows);
    const float sample_inv = sample_rows == 8 ? 0.125f : sample_rows > 0 ? 1.0f / (float)sample_rows : 0.0f;
    const auto pivot_of = [&](int g) {
        const T *first = reinterpret_cast<const T *>(smem) + g * a.cpg;
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < sample_rows) s += FeatElem<T>::to_f(first[k * p.vecs * V]);
        return s * sample_inv;
    };
    float2 pv[P], sm[P], s2[P];
    copy_wait(3);
    __syncthreads();
    spread_groups<V>(at.group, at.left, a.cpg, [&](int g) { return make_float2(-pivot_of(g), 0.0f); }, pv, sm);
#pragma unroll
    for (int j = 0; j < P; ++j) s2[j] = both(0.0f);
    for (int q = 0; q < 4; ++q) {
        copy_wait(3 - q);
        const int end = min((q + 1) * quarter, at.count);
#pragma unroll 2
        for (int i = q * quarter; i < end; ++i) add_moments<P>(data[i * slots], pv, sm, s2);
    }
    if (at.holds) store_folded<V>(red + at.r * stride + at.v * per_vec, sm, s2, p.fold);
    const int lanes = p.columns.lanes, lane = threadIdx.x & (lanes - 1), per_pass = p.columns.per_pass, mine = threadIdx.x >> p.columns.shift;
    const float block_inv = at.rows == p.rows_per_block ? p.block_inv : 1.0f / ((float)max(at.rows, 1) * (float)a.cpg);
    const float full = (float)p.rows_per_block * (float)a.cpg;
    const auto values = [&](int k) { return k < p.ranks - 1 && (k + 1) * p.rows_per_block <= (int)a.rows ? full : (float)max(0, min(p.rows_per_block, (int)a.rows - k * p.rows_per_block)) * (float)a.cpg; };
    __syncthreads();
    for (int base = 0; base < at.groups; base += per_pass) {
        const int g = base + mine;
        const float2 t = group_sum(p.columns, red, stride, p.rows_per_step, p.columns.width, g, g < at.groups);
        if (g < at.groups && lane == 0) pub[g] = moments_of(pivot_of(g), t, block_inv);
    }
    if (p.ranks > 1) { cluster_arrive(); cluster_wait(); }
    else __syncthreads();
    for (int base = 0; base < at.groups; base += per_pass) {
        const int g = base + mine;
        const bool valid = g < at.groups;
        const auto block = [&](int k) { return p.ranks > 1 ? load_rank(pub + g, k) : pub[g]; };
        // sums of the distances to the first block's mean, and of their squares: that block holds at least a sixteenth
        // of the values, so its mean is at most four spreads off
        float2 t = make_float2(0.0f, 0.0f);
        float ref = 0.0f;
        if (valid) {
            ref = block(0).x;
            for (int k = lane; k < p.ranks; k += lanes) {
                const float n = values(k);
                const float2 b = block(k);
                const float d = b.x - ref;
                if (n > 0.0f) t = add2(t, make_float2(n * d, fmaf(n * d, d, b.y)));
            }
        }
        t = lane_sum(t, lanes);
        if (valid && lane == 0) {
            const float2 m = moments_of(ref, t, p.inv);
            const float rstd = rsqrtf(m.y * p.inv + a.eps);
            stat[g] = make_float2(m.x, rstd);
            if (at.rank == 0) {
                const long long id = (long long)at.n * a.groups + at.slab * p.groups + g;
                a.mean[id] = m.x;
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
                x.unpack_plus(mean, f);
#pragma unroll
                for (int j = 0; j < P; ++j) f[j] = fma2(f[j], scale[j], bias[j]);
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
__global__ void __launch_bounds__(THREADS, PER_SM) gn_cluster_grad_kernel(const __grid_constant__ GnArgs a, const __grid_constant__ GnPlan p, float2 *channel_sums)
{
    gn_allow_second();                                  // the parameters' gradients
    constexpr int V = 16 / sizeof(T), P = V / 2;
    extern __shared__ __align__(16) unsigned char smem[];
    const int slots = p.rows_per_step * p.vecs, columns = p.vecs * V, per_vec = p.per_vec, stride = p.vecs * per_vec;
    Pack<T, V> *xs = reinterpret_cast<Pack<T, V> *>(smem) + threadIdx.x, *ds = xs + (size_t)p.steps * slots;      // [steps][slots] each
    float2 *pub = reinterpret_cast<float2 *>(smem + p.data_bytes);                     // [groups] sums of (u xhat, rstd u), read by the cluster
    float2 *stat = pub + p.groups;                      // [groups] the sample's means of (u xhat, rstd u)
    float2 *red = stat + p.groups;                      // [rows_per_step][folded channels of the slab]; at the end, from the
                                                        // start of the memory, [rows_per_step][channels]
    const GnClusterPlace at(a, p, V);
    const int quarter = (p.steps + 3) / 4, lanes = p.columns.lanes, lane = threadIdx.x & (lanes - 1);
    {
        const T *px = (const T *)a.x + at.first, *pd = (const T *)a.dy + at.first;
        Pack<T, V> *tx = xs, *td = ds;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int end = min((q + 1) * quarter, at.count);
            for (int i = q * quarter; i < end; ++i, px += at.step, pd += at.step, tx += slots, td += slots) {
                copy_async<16>(tx, px);
                copy_async<16>(td, pd);
            }
            copy_commit();
        }
    }
    const long long g0 = (long long)at.n * a.groups + at.slab * p.groups;
    float2 mean[P], scale[P], bias[P], rstd[P], sgx[P], sg[P];
    load_params<V>(a.weight, a.param_code, a.wide_params, at.c0, at.active, 1.0f, scale);
    load_params<V>(a.bias, a.param_code, a.wide_params, at.c0, at.active, 0.0f, bias);
    spread_groups<V>(at.group, at.left, a.cpg, [&](int g) { return make_float2(-a.mean[g0 + g], a.rstd[g0 + g]); }, mean, rstd);
#pragma unroll
    for (int j = 0; j < P; ++j) { scale[j] = mul2(scale[j], rstd[j]); sgx[j] = sg[j] = both(0.0f); }
    with_activation(a.act, [&](auto act) {
        for (int q = 0; q < 4; ++q) {
            copy_wait(3 - q);
            const int end = min((q + 1) * quarter, at.count);
            for (int i = q * quarter; i < end; ++i) {
                float2 f[P], z[P], g[P];
                xs[i * slots].unpack_plus(mean, f);
                ds[i * slots].unpack(g);
#pragma unroll
                for (int j = 0; j < P; ++j) z[j] = fma2(f[j], scale[j], bias[j]);
                activate_grad<decltype(act)::value, sizeof(T) == 2, P>(z, g);
#pragma unroll
                for (int j = 0; j < P; ++j) { sg[j] = add2(sg[j], g[j]); sgx[j] = fma2(g[j], f[j], sgx[j]); }
            }
        }
    });
    if (at.holds) {
        float2 ux[P], u[P];
#pragma unroll
        for (int j = 0; j < P; ++j) { ux[j] = mul2(scale[j], sgx[j]); u[j] = mul2(scale[j], sg[j]); }
        store_folded<V>(red + at.r * stride + at.v * per_vec, ux, u, p.fold);
    }
    __syncthreads();
    for (int base = 0; base < at.groups; base += p.columns.per_pass) {
        const int g = base + (threadIdx.x >> p.columns.shift);
        const float2 t = group_sum(p.columns, red, stride, p.rows_per_step, p.columns.width, g, g < at.groups);
        if (g < at.groups && lane == 0) pub[g] = t;
    }
    if (p.ranks > 1) { cluster_arrive(); cluster_wait(); }
    else __syncthreads();
    for (int base = 0; base < at.groups; base += p.columns.per_pass) {
        const int g = base + (threadIdx.x >> p.columns.shift);
        float2 t = make_float2(0.0f, 0.0f);
        if (g < at.groups)
            for (int k = lane; k < p.ranks; k += lanes) t = add2(t, p.ranks > 1 ? load_rank(pub + g, k) : pub[g]);
        t = lane_sum(t, lanes);
        if (g < at.groups && lane == 0) stat[g] = make_float2(t.x * p.inv, t.y * p.inv);
    }
    if (p.ranks > 1) cluster_arrive();                  // done with the others' memory
    __syncthreads();
    if (a.dx) {
        float2 m_ux[P], m_u[P];
        spread_groups<V>(at.group, at.left, a.cpg, [&](int g) { return make_float2(-stat[g].x, -stat[g].y); }, m_ux, m_u);
#pragma unroll
        for (int j = 0; j < P; ++j) m_ux[j] = mul2(m_ux[j], mul2(rstd[j], rstd[j]));       // dx = g scale - ((x - mean) m_ux + m_u)
        T *dst = (T *)a.dx + at.first;
        with_activation(a.act, [&](auto act) {
            for (int i = 0; i < at.count; ++i, dst += at.step) {
                float2 f[P], z[P], g[P];
                xs[i * slots].unpack_plus(mean, f);
                Pack<T, V> d = ds[i * slots];
                d.unpack(g);
#pragma unroll
                for (int j = 0; j < P; ++j) z[j] = fma2(f[j], scale[j], bias[j]);
                activate_grad<decltype(act)::value, sizeof(T) == 2, P>(z, g);
#pragma unroll
                for (int j = 0; j < P; ++j) g[j] = fma2(g[j], scale[j], fma2(f[j], m_ux[j], m_u[j]));
                d.pack(g);
                d.store(dst);
            }
        });
    }
    if (channel_sums) {                                 // this block's sums of (g xhat, g) per channel, after the result: nothing waits for them
        float2 *sums = reinterpret_cast<float2 *>(smem);  // the features have been used up; pub, which others may still read, lies behind
        __syncthreads();
        if (at.holds) {
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const float2 gx = mul2(sgx[j], rstd[j]);
                reinterpret_cast<float4 *>(sums + (at.r * p.vecs + at.v) * V)[j] = make_float4(gx.x, sg[j].x, gx.y, sg[j].y);
            }
        }
        __syncthreads();
        sum_columns(sums, columns, at.slab_channels, p.rows_per_step, THREADS);
        float2 *to = channel_sums + ((long long)at.n * p.ranks + at.rank) * a.channels + at.slab_c0;
        for (int c = threadIdx.x; c < at.slab_channels; c += THREADS) to[c] = sums[c];
    }
    if (p.ranks > 1) cluster_wait();                    // no block leaves while others read it
}

// ----------------------------------------------------------------------------- choice of the plan
// false: a slab of whole groups does not fit a cluster's shared memory
template <typename T> bool gn_plan(const GnArgs &a, int v, bool backward, GnPlan &p)
{
    if (v * sizeof(T) != 16 || a.rows >= (1LL << 30)) return false;
    const int all = a.channels / v, unit = gn_unit(a, v), vector_bytes = backward ? 32 : 16;
    // blocks per SM, their threads (64 registers each forward, 128 backward), their shared memory
    struct Class { int per_sm, threads, bytes; };
    static const Class forward_classes[] = {{4, 256, 55 * 1024}, {3, 320, 74 * 1024}, {2, 512, 113 * 1024}};
    static const Class backward_classes[] = {{4, 128, 55 * 1024}, {3, 160, 74 * 1024}, {2, 256, 113 * 1024}};
    for (int max_ranks = 8; max_ranks <= 16; max_ranks *= 2)
        for (int i = 0; i < 3; ++i)
            for (int seg = all < 32 ? all : 32; seg >= 1; seg = seg == 1 ? 0 : (seg + 1) / 2) {
                const Class &c = backward ? backward_classes[i] : forward_classes[i];
                // slabs of whole units, alike but for one unit: 40 vectors in units of 5 are 20 + 20, not 35 + 5 (half the
                // blocks would hold next to nothing: 256 x 320 x 14^2 bfloat16 40.4 us against 26.9, backward 78 against 50)
                const int units = all / unit, most_units = (seg + unit - 1) / unit, slabs = (units + most_units - 1) / most_units;
                const int vecs = (units + slabs - 1) / slabs * unit;
                if (vecs * 16 < 64 && vecs < all) break;                // row segments of at least 64 bytes (32: 187 us against 122 on 16 x 128 x 224^2)
                if (vecs > c.threads) continue;
                p.threads = c.threads;
                p.vecs = vecs;
                p.slabs = (all + vecs - 1) / vecs;
                p.rows_per_step = c.threads / vecs;
                p.groups = vecs * v / a.cpg;
                p.fold = v;
                while (a.cpg % p.fold) p.fold /= 2;
                const int slots = p.rows_per_step * vecs;
                const int extra = slots * (v / p.fold) * 8 + 2 * p.groups * 8;
                const int most = (c.bytes - extra) / (slots * vector_bytes);
                if (most < 1) continue;
                const long long ranks = (a.rows + (long long)p.rows_per_step * most - 1) / ((long long)p.rows_per_step * most);
                if (ranks > max_ranks) continue;
                p.ranks = (int)ranks;
                p.rows_per_block = (int)((a.rows + ranks - 1) / ranks);
                p.steps = (p.rows_per_block + p.rows_per_step - 1) / p.rows_per_step;
                p.data_bytes = p.steps * slots * vector_bytes;
                if (backward && p.data_bytes < slots * v * 8) p.data_bytes = slots * v * 8;        // the channel sums at the end
                p.smem = p.data_bytes + extra;
                p.vecs_div = fast_div_of(p.vecs);
                p.step_div = fast_div_of(p.rows_per_step);
                p.cpg_div = fast_div_of(a.cpg);
                p.slab_div = fast_div_of(p.slabs);
                p.per_vec = v / p.fold;
                p.inv = 1.0f / ((float)a.rows * (float)a.cpg);
                p.block_inv = 1.0f / ((float)p.rows_per_block * (float)a.cpg);
                p.columns = gn_lanes(p.groups, p.threads, a.cpg / p.fold);
                return p.smem <= c.bytes && a.n * p.slabs * ranks < (1LL << 31);
            }
    return false;
}

template <auto kernel, typename... Args>
cudaError_t gn_launch_cluster(const GnPlan &p, long long samples, cudaStream_t stream, Args... args)
{
    const cudaError_t e = gn_prepare<kernel, true>(113 * 1024);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(samples * p.slabs * p.ranks));
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
    const cudaError_t e = p.threads == 128   ? gn_launch_cluster<gn_cluster_grad_kernel<T, 128, 4>>(p, a.n, stream, a, p, sums)
                          : p.threads == 160 ? gn_launch_cluster<gn_cluster_grad_kernel<T, 160, 3>>(p, a.n, stream, a, p, sums)
                                             : gn_launch_cluster<gn_cluster_grad_kernel<T, 256, 2>>(p, a.n, stream, a, p, sums);
    if (e != cudaSuccess || !sums) return e;
    return gn_launch_params(a, sums, a.n * p.ranks, stream);
}

}  // namespace ta
