// Group norm and its gradient in one pass over memory, for point sets that a
// cluster holds: the CTAs of a cluster copy the points of one instance and a
// tile of whole groups into their shared memory, exchange their sums through
// distributed shared memory, and write the result from what they hold.
//
// Measured on 32 instances of 4096 points and 512 bf16 channels in 32 groups, SiLU:
// forward 65 us for 268 MB (two passes: 131; the copies alone, without sums and
// arithmetic, 48), where the special function unit's two operations an element
// are busy for 30 us; the gradient with dropout and half of the points 106 us for
// 268 MB (two passes: 177), bound by issue at 10 to 11 warps an SM, the most that
// the slabs leave room for. A tile is 64 bytes of a point: with 128, a cluster has
// twice the CTAs to wait for (76 us forward), with 32 memory is read in half lines.
//
// Each thread copies the vectors that it computes on, into slots of its own, so
// that the data needs no barrier and no registers while it is under way. A
// cluster takes one item (an instance and a tile) after the other: as a thread
// has written a slot's results it starts the next item's copy into that slot, so
// that memory is read while it is written and while sums are joined. Where there
// are more items than clusters, a counter deals them out: point counts, and with
// them times, differ, and even equal items went faster so than in turn (64.2
// against 65.4 us for 67M bf16).
#pragma once
#include <cooperative_groups.h>

#include "kernels_norm.cuh"

namespace cpde::ops {

namespace cg = cooperative_groups;

constexpr int SLAB_THREADS = 128;
constexpr int SLAB_WARPS = SLAB_THREADS / 32;
constexpr int SLAB_BLOCKS = 6, SLAB_GRADIENT_BLOCKS = 3;  // CTAs of an SM

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

// Halves of a cluster barrier: what was written before any CTA arrived is seen
// after the wait.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// The most groups of a tile: a tile is SLAB_TILE_BYTES of vectors of at least
// eight bytes, or one group.
constexpr int SLAB_TILE_BYTES = 64;
constexpr int SLAB_GROUPS = SLAB_TILE_BYTES / 8;
constexpr int SLAB_CLUSTER = 16;  // the most CTAs of a cluster

// What a launch fixes: the cluster, and reciprocals for the places' divisions,
// which else would be a third of a short slab's instructions.
struct SlabShape {
    NormShape norm;
    int32_t cluster, slots;  // CTAs of a cluster; vectors of a thread, and array
    int32_t clusters, items;
    uint32_t* counter;       // items dealt out behind the first of each cluster; null if there are none
    int32_t ys;              // points that the block's threads cover at once
    int32_t group_vectors;   // vectors of a group
    int32_t tile_channels, tile_groups;
    Divisor by_cluster, by_tiles, by_tile, by_ys, by_group_vectors;
    bool wide_parameters;    // weight and bias allow vector loads
};

// A thread's place in the cluster: CTA, row of points, vector and group of the tile.
struct Seat {
    int32_t cluster, rank, ty, tx, group;
    __device__ __forceinline__ explicit Seat(const SlabShape& s) {
        cluster = s.by_cluster.quotient(blockIdx.x);
        rank = blockIdx.x - cluster * s.cluster;
        ty = s.by_tile.quotient(threadIdx.x);
        tx = threadIdx.x - ty * s.norm.tile;
        group = s.by_group_vectors.quotient(tx);
    }
};

__device__ __forceinline__ int32_t item_length(const SlabShape& s, int32_t item) {
    return item < s.items ? length_of(s.norm, s.by_tiles.quotient(item)) : 0;
}

// An item and a thread's share of it: its channels, and its points
// p = lo + ty + i ys, i < count.
template <int V>
struct Item {
    int32_t n, lo, hi, length, channel, count;
    int32_t first_channel, channels, first_group, groups;  // the tile's
    bool active;
    __device__ __forceinline__ Item(const SlabShape& s, const Seat& seat, int32_t item, int32_t points) {
        n = s.by_tiles.quotient(item);
        length = points;
        const int32_t tile = item - n * s.norm.tiles;
        first_channel = tile * s.tile_channels;
        channels = min(s.tile_channels, s.norm.channels - first_channel);
        first_group = tile * s.tile_groups;
        groups = min(s.tile_groups, s.norm.groups - first_group);
        share(s, seat, length, lo, hi);
        channel = first_channel + seat.tx * V;
        active = seat.ty < s.ys && seat.tx * V < channels;
        count = active && hi - lo > seat.ty ? int32_t(s.by_ys.quotient(hi - lo - seat.ty - 1)) + 1 : 0;
    }
    // This CTA's part of `points` points.
    __device__ __forceinline__ static void share(const SlabShape& s, const Seat& seat, int32_t points, int32_t& from,
                                                 int32_t& to) {
        const int32_t per = s.by_cluster.quotient(points + s.cluster - 1);
        from = min(seat.rank * per, points);
        to = min(from + per, points);
    }
    // The thread's first vector in an array.
    template <class T>
    __device__ __forceinline__ const T* in(const T* array, const Seat& seat, int64_t instance, int64_t point) const {
        return array + n * instance + (lo + seat.ty) * point + channel;
    }
    __device__ __forceinline__ int64_t index(const SlabShape& s, const Seat& seat) const {
        return (int64_t(n) * s.norm.points + lo + seat.ty) * s.norm.channels + channel;
    }
};

template <class T, int V, int ARRAYS = 1>
__device__ __forceinline__ void copy_points(Vector<T, V>* slots, const T* from, int64_t step, int32_t count) {
#pragma unroll 4
    for (int32_t i = 0; i < count; ++i, from += step, slots += ARRAYS * SLAB_THREADS)
        copy_async<sizeof(T) * V>(slots, from);
}

// The tile's weights and biases in shared memory, and for the gradient its means
// and reciprocal deviations. They are copied with the points: a load of its own
// would wait behind the points' in the queue to memory, once more an item.
__host__ __device__ constexpr size_t tile_parameter_array(int64_t channels, size_t parameter) {
    return (size_t(channels) * parameter + 15) / 16 * 16;
}
__host__ __device__ constexpr size_t tile_parameter_bytes(int64_t channels, size_t parameter) {
    return 2 * tile_parameter_array(channels, parameter) + 2 * SLAB_GROUPS * sizeof(float);
}
template <class P>
struct TileParameters {
    P *weight, *bias;
    float *mean, *rstd;
    __device__ __forceinline__ TileParameters(unsigned char* at, int32_t channels) {
        const size_t array = tile_parameter_array(channels, sizeof(P));
        weight = reinterpret_cast<P*>(at);
        bias = reinterpret_cast<P*>(at + array);
        mean = reinterpret_cast<float*>(at + 2 * array);
        rstd = mean + SLAB_GROUPS;
    }
};

template <class P, int V>
__device__ __forceinline__ void copy_parameters(P* to, const P* from, bool wide) {
    if (!from) return;
    if (wide && sizeof(P) * V >= 8) {
        constexpr int BYTES = sizeof(P) * V >= 16 ? 16 : 8;
#pragma unroll
        for (int i = 0; i < int(sizeof(P)) * V / BYTES; ++i)
            copy_async<BYTES>(reinterpret_cast<unsigned char*>(to) + i * BYTES,
                              reinterpret_cast<const unsigned char*>(from) + i * BYTES);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) to[j] = from[j];
    }
}

// Weights or biases of V channels; `none` where the call has none.
template <class P, int V>
__device__ __forceinline__ Pairs<V> stored_parameters(const P* stored, const P* given, float none) {
    Pairs<V> f;
    if (given) {
        Vector<P, V> v;
        memcpy(&v, __builtin_assume_aligned(stored, sizeof(v) < 16 ? sizeof(v) : 16), sizeof(v));
        f = unpack_pairs<P, V>(v);
    } else {
        f.fill(none);
    }
    return f;
}

// Zeros behind an instance's points, shared by the cluster's CTAs.
template <class T, int V>
__device__ __forceinline__ void clear_tail(T* out, const Item<V>& at, const Seat& seat, const SlabShape& s) {
    if (!at.active || at.length == s.norm.points) return;
    int32_t lo, hi;
    at.share(s, seat, s.norm.points - at.length, lo, hi);
    for (int32_t p = at.length + lo + seat.ty; p < at.length + hi; p += s.ys)
        store<T, V>(out + (int64_t(at.n) * s.norm.points + p) * s.norm.channels + at.channel, zeros<T, V>());
}

// What the CTAs of a cluster tell one another: each writes its sums by group into
// every CTA's memory before the cluster's barrier, so that after it all is
// local; the first also writes the next item and its length. Two of these
// alternate from item to item: one barrier an item keeps a CTA from writing over
// what another still reads.
struct SlabExchange {
    float4* groups;  // [group of the tile][CTA]
    int2* next;
    __host__ __device__ static constexpr size_t bytes(int32_t tile_groups, int32_t cluster) {
        return (size_t(tile_groups) * cluster + 1) * sizeof(float4);
    }
    __device__ __forceinline__ SlabExchange(const SlabShape& s, unsigned char* at, int32_t turn)
        : groups(reinterpret_cast<float4*>(at + turn * bytes(s.tile_groups, s.cluster))),
          next(reinterpret_cast<int2*>(groups + s.tile_groups * s.cluster)) {}
};

// Joins the values of the cluster's CTAs for a group, on the 32 / cluster first
// groups' lanes at once (lane (g, r) has CTA r's value for group g), for the
// tile's groups in turn; each lane gets the result of its group `mine`.
template <class J>
__device__ __forceinline__ float2 over_cluster(const SlabShape& s, const SlabExchange& e, int32_t groups, int32_t mine,
                                               J&& join) {
    const int32_t lane = threadIdx.x % 32, per = 32 / s.cluster;
    float2 got = both(0.0f);
    for (int32_t base = 0; base < groups; base += per) {
        const int32_t g = base + lane / s.cluster;
        const float2 v = join(e.groups[(g < groups ? g : groups - 1) * s.cluster + lane % s.cluster]);
        const int32_t from = ((mine - base) * s.cluster) & 31;
        const float2 one = make_float2(__shfl_sync(~0u, v.x, from), __shfl_sync(~0u, v.y, from));
        if (mine >= base && mine < base + per) got = one;
    }
    return got;
}

// The dealer (CTA 0's first thread) writes the next item to the cluster's CTAs.
__device__ __forceinline__ void deal(const SlabShape& s, cg::cluster_group& cluster, const SlabExchange& exchange,
                                     const Seat& seat, int32_t next, int32_t length) {
    if (!s.counter || seat.rank != 0 || threadIdx.x >= 32) return;
    const int2 v = make_int2(__shfl_sync(~0u, next, 0), __shfl_sync(~0u, length, 0));
    if (threadIdx.x < s.cluster) *cluster.map_shared_rank(exchange.next, threadIdx.x) = v;
}

__device__ __forceinline__ float2 shuffle_xor(const float2& v, int32_t d) {
    return make_float2(__shfl_xor_sync(~0u, v.x, d), __shfl_xor_sync(~0u, v.y, d));
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
    unsigned char* behind = slab + size_t(s.slots) * SLAB_THREADS * sizeof(Slot);
    float2* thread_sums = reinterpret_cast<float2*>(behind + 2 * SlabExchange::bytes(s.tile_groups, s.cluster));
    const TileParameters<P> tile(reinterpret_cast<unsigned char*>(thread_sums + SLAB_THREADS), s.tile_channels);
    cg::cluster_group cluster = cg::this_cluster();
    const Seat seat(s);
    const int32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t read_step = s.ys * s.norm.x_point, step = int64_t(s.ys) * s.norm.channels;
    auto fetch_parameters = [&](const Item<V>& item) {
        if (seat.ty != 0 || !item.active) return;
        copy_parameters<P, V>(tile.weight + seat.tx * V, weight ? weight + item.channel : nullptr, s.wide_parameters);
        copy_parameters<P, V>(tile.bias + seat.tx * V, bias ? bias + item.channel : nullptr, s.wide_parameters);
    };
    Item<V> at(s, seat, seat.cluster, item_length(s, seat.cluster));
    fetch_parameters(at);
    copy_points<T, V>(data, at.in(x, seat, s.norm.x_instance, s.norm.x_point), read_step, at.count);
    cluster_arrive();
    bool started = false;
    for (int32_t turn = 0;; turn ^= 1) {
        const SlabExchange exchange(s, behind, turn);
        const bool dealer = s.counter && seat.rank == 0 && threadIdx.x == 0;
        int32_t next = s.items;
        if (dealer) next = s.clusters + atomicAdd(s.counter, 1u);
        clear_tail<T, V>(y, at, seat, s);
        copies_done();
        __syncthreads();
        const int32_t next_length = dealer ? item_length(s, next) : 0;
        Terms<V, true> k;
        k.gain = stored_parameters<P, V>(tile.weight + seat.tx * V, weight, 1.0f);
        k.bias = stored_parameters<P, V>(tile.bias + seat.tx * V, bias, 0.0f);
        // Deviations from a pivot, the mean of the group's first vector of values:
        // however far off that vector lies, its own share of the variance bounds what the
        // squares' sum loses to cancellation by the number of values over V.
        auto pivot_of = [&](int32_t g) {
            if (at.hi <= at.lo) return 0.0f;
            const Pairs<V> f = unpack_pairs<T, V>(reinterpret_cast<const Slot*>(slab)[g * s.group_vectors]);
            float2 sum = f.p[0];
#pragma unroll
            for (int j = 1; j < Pairs<V>::N; ++j) sum = __fadd2_rn(sum, f.p[j]);
            return finite_or_zero((sum.x + sum.y) * (1.0f / V));
        };
        {
            const float2 shift = both(at.active ? -pivot_of(seat.group) : 0.0f);
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
            thread_sums[threadIdx.x] = make_float2(s1.x + s1.y, s2.x + s2.y);
        }
        __syncthreads();
        if (!started) cluster_wait();  // every CTA runs, and its memory can be written
        started = true;
        for (int32_t g = warp; g < at.groups; g += SLAB_WARPS) {
            const float2* sums = thread_sums + g * s.group_vectors;
            float2 v = both(0.0f);
            for (int32_t i = lane; i < s.group_vectors * s.ys; i += 32) {
                const int32_t ty = s.by_group_vectors.quotient(i);
                v = __fadd2_rn(v, sums[ty * (s.norm.tile - s.group_vectors) + i]);
            }
#pragma unroll
            for (int i = 16; i; i /= 2) v = __fadd2_rn(v, shuffle_xor(v, i));
            const float count = float(at.hi - at.lo) * float(s.norm.width), d = count > 0.0f ? v.x / count : 0.0f;
            if (lane < s.cluster)
                cluster.map_shared_rank(exchange.groups, lane)[g * s.cluster + seat.rank] =
                    make_float4(count, pivot_of(g) + d, not_negative(v.y - v.x * d), 0.0f);
        }
        deal(s, cluster, exchange, seat, next, next_length);
        cluster_arrive();
        cluster_wait();
        const float2 statistics = over_cluster(s, exchange, at.groups, seat.group, [&](const float4& m) {
            // (count, mean, m2): sums by deviations from the first CTA's mean.
            const float pivot = finite_or_zero(__shfl_sync(~0u, m.y, (lane / s.cluster) * s.cluster));
            float count = m.x, d = m.y - pivot;
            float2 v = make_float2(count * d, count > 0.0f ? fmaf(count * d, d, m.z) : 0.0f);
            for (int32_t i = s.cluster / 2; i; i /= 2) {
                count += __shfl_xor_sync(~0u, count, i);
                v = __fadd2_rn(v, shuffle_xor(v, i));
            }
            d = count > 0.0f ? v.x / count : 0.0f;
            const float var = not_negative(v.y - v.x * d) / count;
            return make_float2(pivot + d, count > 0.0f ? 1.0f / sqrtf(var + s.norm.eps) : 0.0f);
        });
        const int2 coming = s.counter ? *exchange.next : make_int2(s.items, 0);
        const bool more = coming.x < s.items;
        const Item<V> then(s, seat, more ? coming.x : 0, more ? coming.y : 0);
        if (more) fetch_parameters(then);
        const T* from = then.in(x, seat, s.norm.x_instance, s.norm.x_point);
        Slot* slot = data;
        if (at.active) {
            if (seat.rank == 0 && seat.ty == 0 && seat.tx == seat.group * s.group_vectors) {
                mean[int64_t(at.n) * s.norm.groups + at.first_group + seat.group] = statistics.x;
                rstd[int64_t(at.n) * s.norm.groups + at.first_group + seat.group] = statistics.y;
            }
            k.minus_mean.set(0, -statistics.x);
            scale<V>(k.gain, statistics.y);
            with_tail(s.norm, [&](auto activation, auto drops) {
                constexpr int32_t ACTIVATION = decltype(activation)::value;
                if constexpr (argument_scale<ACTIVATION, false>() != 1.0f) {
                    scale<V>(k.gain, argument_scale<ACTIVATION, false>());
                    scale<V>(k.bias, argument_scale<ACTIVATION, false>());
                }
                const int64_t index = at.index(s, seat);
                T* to = y + index;
#pragma unroll 2
                for (int32_t i = 0; i < at.count; ++i, to += step, slot += SLAB_THREADS) {
                    Pairs<V> f = unpack_pairs<T, V>(*slot);
                    norm_value<ACTIVATION, decltype(drops)::value, V, true>(f, k, uint64_t(to - y), s.norm.rule);
                    store<T, V>(to, pack_pairs<T, V>(f));
                    if (i < then.count) {
                        copy_async<sizeof(Slot)>(slot, from);
                        from += read_step;
                    }
                }
            });
        }
        if (!more) break;
        copy_points<T, V>(slot, from, read_step, then.count - at.count);
        at = then;
    }
}

// The gradient's sums by channel go through [row][channel] partial sums.
// Where a power of two of lanes covers the tile, a row is a warp's, joined by
// shuffles first; else it is a ty's.
__host__ __device__ inline bool slab_rows_are_warps(int32_t tile) { return tile <= 32 && (tile & (tile - 1)) == 0; }

template <class T, class P, int V>
__global__ void __launch_bounds__(SLAB_THREADS, SLAB_GRADIENT_BLOCKS) k_norm_slab_gradient(
    const T* __restrict__ grad, const T* __restrict__ x, const float* __restrict__ mean,
    const float* __restrict__ rstd, const P* __restrict__ weight, const P* __restrict__ bias, T* __restrict__ dx,
    float2* __restrict__ channel_sums, SlabShape s) {
    extern __shared__ __align__(16) unsigned char slab[];
    next_launch_may_begin();
    using Slot = Vector<T, V>;
    // A slot of x and one of the gradient in turn.
    Slot* data = reinterpret_cast<Slot*>(slab) + threadIdx.x;
    Slot* grads = data + SLAB_THREADS;
    constexpr int32_t NEXT = 2 * SLAB_THREADS;
    const int32_t width = s.tile_channels;
    const bool warps = slab_rows_are_warps(s.norm.tile);
    const int32_t rows = warps ? SLAB_WARPS : s.ys;
    unsigned char* behind = slab + size_t(s.slots) * SLAB_THREADS * 2 * sizeof(Slot);
    float2* parts = reinterpret_cast<float2*>(behind + 2 * SlabExchange::bytes(s.tile_groups, s.cluster));
    float2* sums = parts + rows * width;
    const TileParameters<P> tile(reinterpret_cast<unsigned char*>(sums + width), width);
    cg::cluster_group cluster = cg::this_cluster();
    const Seat seat(s);
    const int32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t x_step = s.ys * s.norm.x_point, grad_step = s.ys * s.norm.grad_point;
    const int64_t step = int64_t(s.ys) * s.norm.channels;
    auto fetch_parameters = [&](const Item<V>& item) {
        if (seat.ty != 0 || !item.active) return;
        copy_parameters<P, V>(tile.weight + seat.tx * V, weight ? weight + item.channel : nullptr, s.wide_parameters);
        copy_parameters<P, V>(tile.bias + seat.tx * V, bias ? bias + item.channel : nullptr, s.wide_parameters);
        if (seat.tx == seat.group * s.group_vectors) {
            const int64_t g = int64_t(item.n) * s.norm.groups + item.first_group + seat.group;
            copy_async<4>(tile.mean + seat.group, mean + g);
            copy_async<4>(tile.rstd + seat.group, rstd + g);
        }
    };
    Item<V> at(s, seat, seat.cluster, item_length(s, seat.cluster));
    fetch_parameters(at);
    copy_points<T, V, 2>(data, at.in(x, seat, s.norm.x_instance, s.norm.x_point), x_step, at.count);
    copy_points<T, V, 2>(grads, at.in(grad, seat, s.norm.grad_instance, s.norm.grad_point), grad_step, at.count);
    cluster_arrive();
    bool started = false;
    for (int32_t turn = 0;; turn ^= 1) {
        const SlabExchange exchange(s, behind, turn);
        const bool dealer = s.counter && seat.rank == 0 && threadIdx.x == 0;
        int32_t next = s.items;
        if (dealer) next = s.clusters + atomicAdd(s.counter, 1u);
        clear_tail<T, V>(dx, at, seat, s);
        copies_done();
        __syncthreads();
        AdjointTerms<V, true> k;
        k.minus_mean.set(0, at.active ? -tile.mean[seat.group] : 0.0f);
        k.rstd.set(0, at.active ? tile.rstd[seat.group] : 0.0f);
        k.set_gain(stored_parameters<P, V>(tile.weight + seat.tx * V, weight, 1.0f));
        k.bias = stored_parameters<P, V>(tile.bias + seat.tx * V, bias, 0.0f);
        const int32_t next_length = dealer ? item_length(s, next) : 0;
        AdjointSums<V, true> sums_of;
        with_tail(s.norm, [&](auto activation, auto drops) {
            constexpr int32_t ACTIVATION = decltype(activation)::value;
            const auto scaled = k.template scaled<ACTIVATION>();
            uint64_t index = uint64_t(at.index(s, seat));
            Slot* slot = data;
#pragma unroll 1  // two vectors at once spill: 111 against 105 us
            for (int32_t i = 0; i < at.count; ++i, index += step, slot += NEXT) {
                Pairs<V> d = unpack_pairs<T, V>(slot[0]), h = unpack_pairs<T, V>(slot[SLAB_THREADS]);
                if constexpr (decltype(drops)::value) {
                    drop_at<V>(h, index, s.norm.rule);
                    // Exact; the second pass finds the zeros and need not draw again.
                    slot[SLAB_THREADS] = pack_pairs<T, V>(h);
                }
                norm_adjoint<ACTIVATION, V, true>(d, h, scaled);
                sums_of.add(d, h);
            }
        });
        // Sums over the points, by channel: within a warp where its lanes repeat the
        // tile's vectors (each step halves the values that a lane keeps), then over
        // the rows that are left.
        float2 sum[V];
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] = sums_of.of(j, k, s.norm.rule.factor);
        if (warps) {
            int32_t kept = 0;  // the first of the channels that the lane keeps
            int32_t d = 16;
#pragma unroll
            for (int half = V / 2; half; half /= 2) {
                if (d >= s.norm.tile) {
                    const bool upper = lane & d;
#pragma unroll
                    for (int j = 0; j < half; ++j) {
                        const float2 send = upper ? sum[j] : sum[j + half], keep = upper ? sum[j + half] : sum[j];
                        sum[j] = __fadd2_rn(keep, shuffle_xor(send, d));
                    }
                    if (upper) kept += half;
                    d /= 2;
                } else {
#pragma unroll
                    for (int j = 0; j < half; ++j) parts[warp * width + seat.tx * V + kept + half + j] = sum[j + half];
                }
            }
            for (; d >= s.norm.tile; d /= 2)
                sum[0] = __fadd2_rn(sum[0], shuffle_xor(sum[0], d));
            parts[warp * width + seat.tx * V + kept] = sum[0];
        } else if (seat.ty < rows) {
#pragma unroll
            for (int j = 0; j < V; ++j) parts[seat.ty * width + seat.tx * V + j] = sum[j];
        }
        __syncthreads();
        for (int32_t c = threadIdx.x; c < at.channels; c += SLAB_THREADS) {
            float2 v = parts[c];
            for (int32_t r = 1; r < rows; ++r) v = __fadd2_rn(v, parts[r * width + c]);
            channel_sums[(int64_t(at.n) * s.cluster + seat.rank) * s.norm.channels + at.first_channel + c] = v;
            sums[c] = __fmul2_rn(v, both(weight ? to_float(tile.weight[c]) : 1.0f));
        }
        __syncthreads();
        if (!started) cluster_wait();  // every CTA runs, and its memory can be written
        started = true;
        for (int32_t g = warp; g < at.groups; g += SLAB_WARPS) {
            float2 v = make_float2(0.0f, 0.0f);
            for (int32_t c = g * s.norm.width + lane; c < (g + 1) * s.norm.width; c += 32) v = __fadd2_rn(v, sums[c]);
#pragma unroll
            for (int d = 16; d; d /= 2) v = __fadd2_rn(v, shuffle_xor(v, d));
            if (lane < s.cluster)
                cluster.map_shared_rank(exchange.groups, lane)[g * s.cluster + seat.rank] = make_float4(v.x, v.y, 0.0f, 0.0f);
        }
        deal(s, cluster, exchange, seat, next, next_length);
        cluster_arrive();
        cluster_wait();
        float2 means = over_cluster(s, exchange, at.groups, seat.group, [&](const float4& m) {
            float2 v = make_float2(m.x, m.y);
            for (int32_t i = s.cluster / 2; i; i /= 2) v = __fadd2_rn(v, shuffle_xor(v, i));
            return v;
        });
        const int2 coming = s.counter ? *exchange.next : make_int2(s.items, 0);
        const bool more = coming.x < s.items;
        const Item<V> then(s, seat, more ? coming.x : 0, more ? coming.y : 0);
        if (more) fetch_parameters(then);
        const T* from = then.in(x, seat, s.norm.x_instance, s.norm.x_point);
        const T* gfrom = then.in(grad, seat, s.norm.grad_instance, s.norm.grad_point);
        Slot* slot = data;
        if (at.active) {
            const float inverse = at.length ? 1.0f / (float(at.length) * float(s.norm.width)) : 0.0f;
            means = __fmul2_rn(means, both(inverse));
            InputTerms<V, true> to_input;
#pragma unroll
            for (int j = 0; j < V; ++j)
                to_input.set(j, input_gain(k.gain.get(j), s.norm.rule.factor), -k.rstd_of(j) * means.x,
                             -k.rstd_of(j) * k.rstd_of(j) * means.y);
            with_activation(s.norm.activation, [&](auto activation) {
                constexpr int32_t ACTIVATION = decltype(activation)::value;
                const auto scaled = k.template scaled<ACTIVATION>();
                T* to = dx + at.index(s, seat);
#pragma unroll 1
                for (int32_t i = 0; i < at.count; ++i, to += step, slot += NEXT) {
                    Pairs<V> d = unpack_pairs<T, V>(slot[0]), h = unpack_pairs<T, V>(slot[SLAB_THREADS]);
                    norm_adjoint<ACTIVATION, V, true>(d, h, scaled);
                    to_input.apply(h, d);
                    store<T, V>(to, pack_pairs<T, V>(h));
                    if (i < then.count) {
                        copy_async<sizeof(Slot)>(slot, from);
                        copy_async<sizeof(Slot)>(slot + SLAB_THREADS, gfrom);
                        from += x_step;
                        gfrom += grad_step;
                    }
                }
            });
        }
        if (!more) break;
        copy_points<T, V, 2>(slot, from, x_step, then.count - at.count);
        copy_points<T, V, 2>(slot + SLAB_THREADS, gfrom, grad_step, then.count - at.count);
        at = then;
    }
}

// dw and db from the channels' sums by instance.
template <class P>
__global__ void __launch_bounds__(1024) k_norm_parameters(P* __restrict__ dweight, P* __restrict__ dbias,
                                                                   const float2* channel_sums, int32_t rows, int32_t channels) {
    after_previous_launch();
    sum_parameters<P, 32>(dweight, dbias, channel_sums, rows, channels, blockIdx.x);
}

}  // namespace cpde::ops
