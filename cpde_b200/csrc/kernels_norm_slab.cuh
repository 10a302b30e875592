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

// A thread's place: its vector of channels and its points p = lo + ty + i ys.
template <int V>
struct Place {
    int32_t n, lo, hi, length, ys, ty, tx, channel, count;
    Tile tile;
    bool active;
    __device__ Place(const NormShape& s, uint32_t rank, uint32_t size) {
        const int32_t cluster = blockIdx.x / size;
        n = cluster / s.tiles;
        tile = tile_of<V>(s, cluster - n * s.tiles);
        length = length_of(s, n);
        split_range(length, rank, size, lo, hi);
        ys = NORM_THREADS / s.tile;
        ty = threadIdx.x / s.tile;
        tx = threadIdx.x - ty * s.tile;
        channel = tile.first + tx * V;
        active = ty < ys && tx * V < tile.count;
        count = active ? points(ty) : 0;
    }
    __device__ int32_t points(int32_t y) const { return hi - lo > y ? (hi - lo - y - 1) / ys + 1 : 0; }
};

// Zeros behind an instance's points, shared by the cluster's CTAs.
template <class T, int V>
__device__ __forceinline__ void clear_tail(T* out, const Place<V>& at, const NormShape& s, uint32_t rank, uint32_t size) {
    if (!at.active || at.length == s.points) return;
    int32_t lo, hi;
    split_range(s.points - at.length, rank, size, lo, hi);
    for (int32_t p = at.length + lo + at.ty; p < at.length + hi; p += at.ys)
        store<T, V>(out + (int64_t(at.n) * s.points + p) * s.channels + at.channel, zeros<T, V>());
}

// Shared memory behind the slots: a thread's moments, the CTA's moments by
// group, the statistics by group.
struct SlabMoments {
    float2 threads[NORM_THREADS];
    Moments groups[NORM_THREADS];
    float2 statistics[NORM_THREADS];
};

// Sums of moments by deviations from one of the means, `pivot`.
__device__ __forceinline__ Moments warp_sum(float count, float mean, float m2, float pivot) {
    float d = mean - pivot, s1 = count * d, s2 = count > 0.0f ? fmaf(s1, d, m2) : 0.0f;
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
__global__ void __launch_bounds__(NORM_THREADS, 3) k_norm_slab(const T* __restrict__ x, const P* __restrict__ weight,
                                                                const P* __restrict__ bias, T* __restrict__ y,
                                                                float* __restrict__ mean, float* __restrict__ rstd,
                                                                NormShape s, int32_t slots) {
    extern __shared__ __align__(16) unsigned char slab[];
    using Slot = Vector<T, V>;
    Slot* data = reinterpret_cast<Slot*>(slab);
    auto& shared = *reinterpret_cast<SlabMoments*>(slab + size_t(slots) * NORM_THREADS * sizeof(Slot));
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t size = cluster.num_blocks(), rank = cluster.block_rank();
    const int32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const Place<V> at(s, rank, size);
    const T* from = x + at.n * s.x_instance + (at.lo + at.ty) * s.x_point + at.channel;
    for (int32_t i = 0; i < at.count; ++i)
        copy_async<sizeof(Slot)>(&data[i * NORM_THREADS + threadIdx.x], from + int64_t(i) * at.ys * s.x_point);
    Terms<V, true> k;
    if (at.active) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            k.gain.set(j, parameter(weight, at.channel + j, 1.0f));
            k.bias.set(j, parameter(bias, at.channel + j, 0.0f));
        }
    }
    clear_tail<T, V>(y, at, s, rank, size);
    copies_done();
    if (at.active) {
        // Deviations from the thread's first value: their squares cancel by no
        // more than the number of the thread's values.
        float2 shift = both(0.0f), t1 = both(0.0f), t2 = both(0.0f);
#pragma unroll 2
        for (int32_t i = 0; i < at.count; ++i) {
            const Pairs<V> f = unpack_pairs<T, V>(data[i * NORM_THREADS + threadIdx.x]);
            if (i == 0) shift = both(-f.p[0].x);
#pragma unroll
            for (int j = 0; j < Pairs<V>::N; ++j) {
                const float2 d = __fadd2_rn(f.p[j], shift);
                t1 = __fadd2_rn(t1, d);
                t2 = __ffma2_rn(d, d, t2);
            }
        }
        const float s1 = t1.x + t1.y, s2 = t2.x + t2.y;
        const float m = at.count ? s1 / float(at.count * V) : 0.0f;
        shared.threads[threadIdx.x] = make_float2(m - shift.x, fmaxf(s2 - s1 * m, 0.0f));
    }
    __syncthreads();
    const int32_t per_group = s.width / V;  // vectors of a group
    for (int32_t g = warp; g < at.tile.groups; g += NORM_WARPS) {
        const float pivot = shared.threads[g * per_group].x;
        float count = 0.0f, s1 = 0.0f, s2 = 0.0f;
        for (int32_t i = lane; i < per_group * at.ys; i += 32) {
            const int32_t ty = i / per_group, tx = g * per_group + i - ty * per_group;
            const float points = float(at.points(ty) * V);
            const float2 v = shared.threads[ty * s.tile + tx];
            const float d = v.x - pivot;
            count += points;
            s1 = fmaf(points, d, s1);
            if (points > 0.0f) s2 += fmaf(points * d, d, v.y);
        }
        const float d = count > 0.0f ? s1 / count : 0.0f;
        const Moments m = warp_sum(count, pivot + d, fmaxf(s2 - s1 * d, 0.0f), pivot);
        if (lane == 0) shared.groups[g] = m;
    }
    cluster.sync();
    for (int32_t g = warp; g < at.tile.groups; g += NORM_WARPS) {
        Moments m = {0.0f, 0.0f, 0.0f};
        if (lane < int32_t(size)) m = cluster.map_shared_rank(&shared, lane)->groups[g];
        m = warp_sum(m.count, m.mean, m.m2, __shfl_sync(~0u, m.mean, 0));
        if (lane == 0) {
            const float r = at.length ? 1.0f / sqrtf(m.m2 / m.count + s.eps) : 0.0f;
            shared.statistics[g] = make_float2(m.mean, r);
            if (rank == 0) {
                mean[int64_t(at.n) * s.groups + at.tile.group + g] = m.mean;
                rstd[int64_t(at.n) * s.groups + at.tile.group + g] = r;
            }
        }
    }
    __syncthreads();
    auto token = cluster.barrier_arrive();  // done with the other CTAs' memory
    if (at.active) {
        const float2 m = shared.statistics[at.tx / per_group];
        k.minus_mean.set(0, -m.x);
        scale<V>(k.gain, m.y);
        int64_t to = (int64_t(at.n) * s.points + at.lo + at.ty) * s.channels + at.channel;
        const int64_t step = int64_t(at.ys) * s.channels;
#pragma unroll 2
        for (int32_t i = 0; i < at.count; ++i, to += step) {
            Pairs<V> f = unpack_pairs<T, V>(data[i * NORM_THREADS + threadIdx.x]);
            norm_value<V, true>(f, k, uint64_t(to), s);
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
__global__ void __launch_bounds__(NORM_THREADS, 3) k_norm_slab_gradient(
    const T* __restrict__ grad, const T* __restrict__ x, const float* __restrict__ mean,
    const float* __restrict__ rstd, const P* __restrict__ weight, const P* __restrict__ bias, T* __restrict__ dx,
    float2* __restrict__ channel_sums, NormShape s, int32_t slots) {
    extern __shared__ __align__(16) unsigned char slab[];
    using Slot = Vector<T, V>;
    Slot* data = reinterpret_cast<Slot*>(slab);
    Slot* grads = data + size_t(slots) * NORM_THREADS;
    const int32_t width = s.tile * V;
    const bool warps = slab_rows_are_warps(s.tile);
    const int32_t rows = warps ? NORM_WARPS : NORM_THREADS / s.tile;
    float2* parts = reinterpret_cast<float2*>(grads + size_t(slots) * NORM_THREADS);
    float2* sums = parts + rows * width;
    float2* totals = sums + width;
    float2* means = totals + width;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t size = cluster.num_blocks(), rank = cluster.block_rank();
    const int32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const Place<V> at(s, rank, size);
    const T* from = x + at.n * s.x_instance + (at.lo + at.ty) * s.x_point + at.channel;
    const T* gfrom = grad + at.n * s.grad_instance + (at.lo + at.ty) * s.grad_point + at.channel;
    for (int32_t i = 0; i < at.count; ++i) {
        copy_async<sizeof(Slot)>(&data[i * NORM_THREADS + threadIdx.x], from + int64_t(i) * at.ys * s.x_point);
        copy_async<sizeof(Slot)>(&grads[i * NORM_THREADS + threadIdx.x], gfrom + int64_t(i) * at.ys * s.grad_point);
    }
    AdjointTerms<V, true> k;
    if (at.active) load_terms<P, V, true>(k, s, at.n, at.channel, mean, rstd, weight, bias);
    clear_tail<T, V>(dx, at, s, rank, size);
    copies_done();
    const int64_t first = (int64_t(at.n) * s.points + at.lo + at.ty) * s.channels + at.channel;
    const int64_t step = int64_t(at.ys) * s.channels;
    Pairs<V> sh, sx;
    sh.fill(0.0f);
    sx.fill(0.0f);
#pragma unroll 2
    for (int32_t i = 0; i < at.count; ++i) {
        Slot& slot = grads[i * NORM_THREADS + threadIdx.x];
        Pairs<V> xhat = unpack_pairs<T, V>(data[i * NORM_THREADS + threadIdx.x]), h = unpack_pairs<T, V>(slot);
        if (s.rule.threshold) {
            drop_at<V>(h, uint64_t(first + i * step), s.rule);
            slot = pack_pairs<T, V>(h);  // exact; the second pass finds the zeros and need not draw again
        }
        norm_adjoint<V, true>(xhat, h, k, s.activation);
#pragma unroll
        for (int j = 0; j < Pairs<V>::N; ++j) {
            sh.p[j] = __fadd2_rn(sh.p[j], h.p[j]);
            sx.p[j] = __ffma2_rn(h.p[j], xhat.p[j], sx.p[j]);
        }
    }
    scale<V>(sh, s.rule.factor);
    scale<V>(sx, s.rule.factor);
    float2 sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = make_float2(sh.get(j), sx.get(j));
    if (warps) {
        for (int32_t d = 16; d >= s.tile; d /= 2) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                sum[j].x += __shfl_xor_sync(~0u, sum[j].x, d);
                sum[j].y += __shfl_xor_sync(~0u, sum[j].y, d);
            }
        }
    }
    if (warps ? lane < s.tile : at.ty < rows) {
#pragma unroll
        for (int j = 0; j < V; ++j) parts[(warps ? warp : at.ty) * width + at.tx * V + j] = sum[j];
    }
    __syncthreads();
    for (int32_t c = threadIdx.x; c < at.tile.count; c += NORM_THREADS) {
        float2 v = parts[c];
        for (int32_t r = 1; r < rows; ++r) {
            v.x += parts[r * width + c].x;
            v.y += parts[r * width + c].y;
        }
        sums[c] = v;
    }
    cluster.sync();
    for (int32_t c = threadIdx.x; c < at.tile.count; c += NORM_THREADS) {
        float2 v = make_float2(0.0f, 0.0f);
        for (uint32_t r = 0; r < size; ++r) {
            const float2 o = cluster.map_shared_rank(sums, r)[c];
            v.x += o.x;
            v.y += o.y;
        }
        if (rank == 0) channel_sums[int64_t(at.n) * s.channels + at.tile.first + c] = v;
        const float w = parameter(weight, at.tile.first + c, 1.0f);
        totals[c] = make_float2(v.x * w, v.y * w);
    }
    __syncthreads();
    auto token = cluster.barrier_arrive();  // done with the other CTAs' memory
    const float inverse = at.length ? 1.0f / (float(at.length) * float(s.width)) : 0.0f;
    for (int32_t g = warp; g < at.tile.groups; g += NORM_WARPS) {
        float2 v = make_float2(0.0f, 0.0f);
        for (int32_t c = g * s.width + lane; c < (g + 1) * s.width; c += 32) {
            v.x += totals[c].x;
            v.y += totals[c].y;
        }
#pragma unroll
        for (int d = 16; d; d /= 2) {
            v.x += __shfl_down_sync(~0u, v.x, d);
            v.y += __shfl_down_sync(~0u, v.y, d);
        }
        if (lane == 0) means[g] = make_float2(v.x * inverse, v.y * inverse);
    }
    __syncthreads();
    if (at.active) {
        InputTerms<V, true> to_input;
#pragma unroll
        for (int j = 0; j < V; ++j) to_input.set(k, j, means[at.tx * V / s.width], s.rule.factor);
        int64_t to = first;
#pragma unroll 2
        for (int32_t i = 0; i < at.count; ++i, to += step) {
            Pairs<V> xhat = unpack_pairs<T, V>(data[i * NORM_THREADS + threadIdx.x]);
            Pairs<V> h = unpack_pairs<T, V>(grads[i * NORM_THREADS + threadIdx.x]);
            norm_adjoint<V, true>(xhat, h, k, s.activation);
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
