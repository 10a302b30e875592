// Group norm and its gradient in one pass over memory, for point sets that a
// cluster holds: the CTAs of a cluster copy the points of one instance and a
// tile of whole groups into their shared memory, exchange their sums through
// distributed shared memory, and write the result from what they hold.
//
// Each thread copies the vectors that it computes on, into slots of its own, so
// that the data needs no barrier and no registers while it is under way.
#pragma once
#include <cooperative_groups.h>

#include "kernels_norm.cuh"

namespace cpde::ops {

namespace cg = cooperative_groups;

constexpr int SLAB_THREADS = 128;
constexpr int SLAB_WARPS = SLAB_THREADS / 32;
constexpr int SLAB_BLOCKS = 6;  // CTAs of an SM

template <int BYTES>
__device__ __forceinline__ void copy_async(void* shared, const void* global) {
    const uint32_t to = uint32_t(__cvta_generic_to_shared(shared));
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(global) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(global), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_done() {
    asm volatile("cp.async.commit_group;\ncp.async.wait_all;" ::: "memory");
}

// What a launch fixes: the cluster, and reciprocals for the places' divisions,
// which else would be a third of a short slab's instructions.
struct SlabShape {
    NormShape norm;
    int32_t cluster, slots;  // CTAs of a cluster; vectors of a thread, and array
    int32_t ys;              // points that the block's threads cover at once
    int32_t group_vectors;   // vectors of a group
    int32_t tile_channels, tile_groups;
    Divisor by_cluster, by_tiles, by_tile, by_ys, by_group_vectors;
    bool wide_parameters;    // weight and bias allow vector loads
};

// A thread's place: its vector of channels and its points p = lo + ty + i ys.
template <int V>
struct Place {
    int32_t rank, n, lo, hi, length, ty, tx, channel, count;
    int32_t first_channel, channels, first_group, groups;  // the tile's
    bool active;
    __device__ __forceinline__ explicit Place(const SlabShape& s) {
        const int32_t cluster = s.by_cluster.quotient(blockIdx.x);
        rank = blockIdx.x - cluster * s.cluster;
        n = s.by_tiles.quotient(cluster);
        const int32_t tile = cluster - n * s.norm.tiles;
        first_channel = tile * s.tile_channels;
        channels = min(s.tile_channels, s.norm.channels - first_channel);
        first_group = tile * s.tile_groups;
        groups = min(s.tile_groups, s.norm.groups - first_group);
        length = length_of(s.norm, n);
        share(s, length, lo, hi);
        ty = s.by_tile.quotient(threadIdx.x);
        tx = threadIdx.x - ty * s.norm.tile;
        channel = first_channel + tx * V;
        active = ty < s.ys && tx * V < channels;
        count = active && hi - lo > ty ? int32_t(s.by_ys.quotient(hi - lo - ty - 1)) + 1 : 0;
    }
    // This CTA's part of `points` points.
    __device__ __forceinline__ void share(const SlabShape& s, int32_t points, int32_t& from, int32_t& to) const {
        const int32_t per = s.by_cluster.quotient(points + s.cluster - 1);
        from = min(rank * per, points);
        to = min(from + per, points);
    }
};

template <class T, int V>
__device__ __forceinline__ void copy_points(Vector<T, V>* slots, const T* from, int64_t step, int32_t count) {
#pragma unroll 4
    for (int32_t i = 0; i < count; ++i, from += step, slots += SLAB_THREADS) copy_async<sizeof(T) * V>(slots, from);
}

// Weights or biases of a thread's channels; `none` where there are none.
template <class P, int V>
__device__ __forceinline__ Pairs<V> load_parameters(const P* p, int32_t channel, bool wide, float none) {
    Pairs<V> f;
    if (!p) {
        f.fill(none);
    } else if (wide) {
        f = unpack_pairs<P, V>(load<P, V>(p + channel));
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) f.set(j, to_float(p[channel + j]));
    }
    return f;
}

// Zeros behind an instance's points, shared by the cluster's CTAs.
template <class T, int V>
__device__ __forceinline__ void clear_tail(T* out, const Place<V>& at, const SlabShape& s) {
    if (!at.active || at.length == s.norm.points) return;
    int32_t lo, hi;
    at.share(s, s.norm.points - at.length, lo, hi);
    for (int32_t p = at.length + lo + at.ty; p < at.length + hi; p += s.ys)
        store<T, V>(out + (int64_t(at.n) * s.norm.points + p) * s.norm.channels + at.channel, zeros<T, V>());
}

// Shared memory behind the slots: each thread's sums, the CTA's moments by
// group, (-mean, rstd) by group.
struct SlabMoments {
    float2 threads[SLAB_THREADS];
    Moments groups[SLAB_THREADS];
    float2 statistics[SLAB_THREADS];
};

// Sums over a warp's lanes of moments, by deviations from one of the means.
__device__ __forceinline__ Moments warp_sum(const Moments& m, float pivot) {
    float count = m.count, d = m.mean - pivot, s1 = count * d, s2 = count > 0.0f ? fmaf(s1, d, m.m2) : 0.0f;
#pragma unroll
    for (int i = 16; i; i /= 2) {
        count += __shfl_xor_sync(~0u, count, i);
        s1 += __shfl_xor_sync(~0u, s1, i);
        s2 += __shfl_xor_sync(~0u, s2, i);
    }
    if (count == 0.0f) return {0.0f, 0.0f, 0.0f};
    d = s1 / count;
    return {count, pivot + d, fmaxf(s2 - s1 * d, 0.0f)};
}

template <class T, class P, int V>
__global__ void __launch_bounds__(SLAB_THREADS, SLAB_BLOCKS) k_norm_slab(const T* __restrict__ x,
                                                                          const P* __restrict__ weight,
                                                                          const P* __restrict__ bias,
                                                                          T* __restrict__ y, float* __restrict__ mean,
                                                                          float* __restrict__ rstd, SlabShape s) {
    extern __shared__ __align__(16) unsigned char slab[];
    using Slot = Vector<T, V>;
    Slot* data = reinterpret_cast<Slot*>(slab) + threadIdx.x;
    auto& shared = *reinterpret_cast<SlabMoments*>(slab + size_t(s.slots) * SLAB_THREADS * sizeof(Slot));
    const Place<V> at(s);
    const int32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int32_t tg = s.by_group_vectors.quotient(at.tx);  // the thread's group in the tile
    const T* from = x + at.n * s.norm.x_instance + at.lo * s.norm.x_point + at.channel;
    copy_points<T, V>(data, from + at.ty * s.norm.x_point, s.ys * s.norm.x_point, at.count);
    // Deviations from a pivot, the mean of the group's first vector of values:
    // what their squares lose to cancellation is bounded by the number of values
    // over V^2 however far off that vector lies.
    float pivot = 0.0f;
    Terms<V, true> k;
    if (at.active) {
        if (at.hi > at.lo) {
            const Pairs<V> f =
                unpack_pairs<T, V>(load<T, V>(from + (tg * s.group_vectors - at.tx) * V));
            float2 sum = f.p[0];
#pragma unroll
            for (int j = 1; j < Pairs<V>::N; ++j) sum = __fadd2_rn(sum, f.p[j]);
            pivot = (sum.x + sum.y) * (1.0f / V);
        }
        k.gain = load_parameters<P, V>(weight, at.channel, s.wide_parameters, 1.0f);
        k.bias = load_parameters<P, V>(bias, at.channel, s.wide_parameters, 0.0f);
    }
    clear_tail<T, V>(y, at, s);
    copies_done();
    {
        const float2 shift = both(-pivot);
        float2 s1 = both(0.0f), s2 = both(0.0f);
        const Slot* slot = data;
#pragma unroll 2
        for (int32_t i = 0; i < at.count; ++i, slot += SLAB_THREADS) {
            const Pairs<V> f = unpack_pairs<T, V>(*slot);
#pragma unroll
            for (int j = 0; j < Pairs<V>::N; ++j) {
                const float2 d = __fadd2_rn(f.p[j], shift);
                s1 = __fadd2_rn(s1, d);
                s2 = __ffma2_rn(d, d, s2);
            }
        }
        shared.threads[threadIdx.x] = make_float2(s1.x + s1.y, s2.x + s2.y);
        if (at.active && at.ty == 0 && at.tx == tg * s.group_vectors) shared.groups[tg].mean = pivot;
    }
    __syncthreads();
    const float inverse = at.hi > at.lo ? 1.0f / (float(at.hi - at.lo) * float(s.norm.width)) : 0.0f;
    for (int32_t g = warp; g < at.groups; g += SLAB_WARPS) {
        const float2* sums = shared.threads + g * s.group_vectors;
        float s1 = 0.0f, s2 = 0.0f;
        for (int32_t i = lane; i < s.group_vectors * s.ys; i += 32) {
            const int32_t ty = s.by_group_vectors.quotient(i);
            const float2 v = sums[ty * (s.norm.tile - s.group_vectors) + i];
            s1 += v.x;
            s2 += v.y;
        }
#pragma unroll
        for (int i = 16; i; i /= 2) {
            s1 += __shfl_xor_sync(~0u, s1, i);
            s2 += __shfl_xor_sync(~0u, s2, i);
        }
        if (lane == 0) {
            const float d = s1 * inverse;
            Moments& m = shared.groups[g];
            m.count = float(at.hi - at.lo) * float(s.norm.width);
            m.mean += d;
            m.m2 = fmaxf(s2 - s1 * d, 0.0f);
        }
    }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int32_t g = warp; g < at.groups; g += SLAB_WARPS) {
        Moments m = {0.0f, 0.0f, 0.0f};
        if (lane < s.cluster) m = cluster.map_shared_rank(&shared, lane)->groups[g];
        m = warp_sum(m, __shfl_sync(~0u, m.mean, 0));
        if (lane == 0) {
            const float r = at.length ? 1.0f / sqrtf(m.m2 / m.count + s.norm.eps) : 0.0f;
            shared.statistics[g] = make_float2(-m.mean, r);
            if (at.rank == 0) {
                mean[int64_t(at.n) * s.norm.groups + at.first_group + g] = m.mean;
                rstd[int64_t(at.n) * s.norm.groups + at.first_group + g] = r;
            }
        }
    }
    __syncthreads();
    auto token = cluster.barrier_arrive();  // done with the other CTAs' memory
    if (at.active) {
        const float2 m = shared.statistics[tg];
        k.minus_mean.set(0, m.x);
        scale<V>(k.gain, m.y);
        int64_t to = (int64_t(at.n) * s.norm.points + at.lo + at.ty) * s.norm.channels + at.channel;
        const int64_t step = int64_t(s.ys) * s.norm.channels;
        const Slot* slot = data;
#pragma unroll 2
        for (int32_t i = 0; i < at.count; ++i, to += step, slot += SLAB_THREADS) {
            Pairs<V> f = unpack_pairs<T, V>(*slot);
            norm_value<V, true>(f, k, uint64_t(to), s.norm);
            store<T, V>(y + to, pack_pairs<T, V>(f));
        }
    }
    cluster.barrier_wait(std::move(token));
}

// Shared memory of the gradient behind the slots: [row][channel] partial sums,
// then the CTA's and the cluster's sums by channel, then the means by group.
// Where a power of two of lanes covers the tile, a row is a warp's, joined by
// shuffles first; else it is a ty's.
__host__ __device__ inline bool slab_rows_are_warps(int32_t tile) { return tile <= 32 && (tile & (tile - 1)) == 0; }

template <class T, class P, int V>
__global__ void __launch_bounds__(SLAB_THREADS, SLAB_BLOCKS) k_norm_slab_gradient(
    const T* __restrict__ grad, const T* __restrict__ x, const float* __restrict__ mean,
    const float* __restrict__ rstd, const P* __restrict__ weight, const P* __restrict__ bias, T* __restrict__ dx,
    float2* __restrict__ channel_sums, SlabShape s) {
    extern __shared__ __align__(16) unsigned char slab[];
    using Slot = Vector<T, V>;
    Slot* data = reinterpret_cast<Slot*>(slab) + threadIdx.x;
    Slot* grads = data + size_t(s.slots) * SLAB_THREADS;
    const int32_t width = s.tile_channels;
    const bool warps = slab_rows_are_warps(s.norm.tile);
    const int32_t rows = warps ? SLAB_WARPS : s.ys;
    float2* parts = reinterpret_cast<float2*>(slab + size_t(s.slots) * SLAB_THREADS * 2 * sizeof(Slot));
    float2* sums = parts + rows * width;
    float2* totals = sums + width;
    float2* means = totals + width;
    const Place<V> at(s);
    const int32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int32_t tg = s.by_group_vectors.quotient(at.tx);
    copy_points<T, V>(data, x + at.n * s.norm.x_instance + (at.lo + at.ty) * s.norm.x_point + at.channel,
                      s.ys * s.norm.x_point, at.count);
    copy_points<T, V>(grads, grad + at.n * s.norm.grad_instance + (at.lo + at.ty) * s.norm.grad_point + at.channel,
                      s.ys * s.norm.grad_point, at.count);
    AdjointTerms<V, true> k;
    if (at.active) {
        const int64_t g = int64_t(at.n) * s.norm.groups + at.first_group + tg;
        k.minus_mean.set(0, -mean[g]);
        k.rstd.set(0, rstd[g]);
        k.weight = load_parameters<P, V>(weight, at.channel, s.wide_parameters, 1.0f);
        k.bias = load_parameters<P, V>(bias, at.channel, s.wide_parameters, 0.0f);
    }
    clear_tail<T, V>(dx, at, s);
    copies_done();
    const int64_t first = (int64_t(at.n) * s.norm.points + at.lo + at.ty) * s.norm.channels + at.channel;
    const int64_t step = int64_t(s.ys) * s.norm.channels;
    Pairs<V> sh, sx;
    sh.fill(0.0f);
    sx.fill(0.0f);
    {
        int64_t index = first;
        Slot *slot = data, *gslot = grads;
#pragma unroll 2
        for (int32_t i = 0; i < at.count; ++i, index += step, slot += SLAB_THREADS, gslot += SLAB_THREADS) {
            Pairs<V> xhat = unpack_pairs<T, V>(*slot), h = unpack_pairs<T, V>(*gslot);
            if (s.norm.rule.threshold) {
                drop_at<V>(h, uint64_t(index), s.norm.rule);
                *gslot = pack_pairs<T, V>(h);  // exact; the second pass finds the zeros and need not draw again
            }
            norm_adjoint<V, true>(xhat, h, k, s.norm.activation);
#pragma unroll
            for (int j = 0; j < Pairs<V>::N; ++j) {
                sh.p[j] = __fadd2_rn(sh.p[j], h.p[j]);
                sx.p[j] = __ffma2_rn(h.p[j], xhat.p[j], sx.p[j]);
            }
        }
    }
    if (warps) {
        for (int32_t d = 16; d >= s.norm.tile; d /= 2) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                sh.set(j, sh.get(j) + __shfl_xor_sync(~0u, sh.get(j), d));
                sx.set(j, sx.get(j) + __shfl_xor_sync(~0u, sx.get(j), d));
            }
        }
    }
    if (warps ? lane < s.norm.tile : at.ty < rows) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            parts[(warps ? warp : at.ty) * width + at.tx * V + j] = make_float2(sh.get(j), sx.get(j));
    }
    __syncthreads();
    for (int32_t c = threadIdx.x; c < at.channels; c += SLAB_THREADS) {
        float2 v = parts[c];
        for (int32_t r = 1; r < rows; ++r) v = __fadd2_rn(v, parts[r * width + c]);
        sums[c] = v;
    }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int32_t c = threadIdx.x; c < at.channels; c += SLAB_THREADS) {
        float2 v = make_float2(0.0f, 0.0f);
#pragma unroll 4
        for (int32_t r = 0; r < s.cluster; ++r) v = __fadd2_rn(v, cluster.map_shared_rank(sums, r)[c]);
        v = __fmul2_rn(v, both(s.norm.rule.factor));
        if (at.rank == 0) channel_sums[int64_t(at.n) * s.norm.channels + at.first_channel + c] = v;
        totals[c] = __fmul2_rn(v, both(parameter(weight, at.first_channel + c, 1.0f)));
    }
    __syncthreads();
    auto token = cluster.barrier_arrive();  // done with the other CTAs' memory
    const float inverse = at.length ? 1.0f / (float(at.length) * float(s.norm.width)) : 0.0f;
    for (int32_t g = warp; g < at.groups; g += SLAB_WARPS) {
        float2 v = make_float2(0.0f, 0.0f);
        for (int32_t c = g * s.norm.width + lane; c < (g + 1) * s.norm.width; c += 32) v = __fadd2_rn(v, totals[c]);
#pragma unroll
        for (int d = 16; d; d /= 2) {
            v.x += __shfl_down_sync(~0u, v.x, d);
            v.y += __shfl_down_sync(~0u, v.y, d);
        }
        if (lane == 0) means[g] = __fmul2_rn(v, both(inverse));
    }
    __syncthreads();
    if (at.active) {
        InputTerms<V, true> to_input;
#pragma unroll
        for (int j = 0; j < V; ++j) to_input.set(k, j, means[tg], s.norm.rule.factor);
        int64_t to = first;
        const Slot *slot = data, *gslot = grads;
#pragma unroll 2
        for (int32_t i = 0; i < at.count; ++i, to += step, slot += SLAB_THREADS, gslot += SLAB_THREADS) {
            Pairs<V> xhat = unpack_pairs<T, V>(*slot), h = unpack_pairs<T, V>(*gslot);
            norm_adjoint<V, true>(xhat, h, k, s.norm.activation);
            to_input.apply(h, xhat);
            store<T, V>(dx + to, pack_pairs<T, V>(h));
        }
    }
    cluster.barrier_wait(std::move(token));
}

// dw and db from the channels' sums by instance.
template <class P>
__global__ void __launch_bounds__(NORM_THREADS) k_norm_parameters(P* __restrict__ dweight, P* __restrict__ dbias,
                                                                   const float2* __restrict__ channel_sums,
                                                                   int32_t rows, int32_t channels) {
    sum_parameters<P>(dweight, dbias, channel_sums, rows, channels, blockIdx.x);
}

}  // namespace cpde::ops
