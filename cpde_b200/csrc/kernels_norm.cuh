// Group norm with an activation over (instance, point, channel) arrays,
// channels last, and its gradient.
//
//   mean, var over the points and the channels of a group; rstd = 1/sqrt(var + eps)
//   xhat = (x - mean) rstd; z = w xhat + b; y = drop(act(z))
//   h = drop(dy) act'(z); db = sum h; dw = sum h xhat
//   dx = rstd (w h - (mean_g(w h) + xhat mean_g(w h xhat)))
//
// Points at or behind lengths[n] count nowhere, are never read, and their
// outputs are zeros.
//
// The kernels of this file take two passes over memory, for point sets that no
// cluster holds (kernels_norm_slab.cuh). Both directions are bound by memory: a
// million points of 64 f32 channels take 160 us forward (805 MB in two passes, 5.0
// TB/s) and 238 us for the gradient (1.34 GB, 5.6 TB/s). The second pass goes from the back
// because the first leaves the ends of the blocks' ranges in L2. FP32 arithmetic
// is in packed pairs: an issue slot then has two operations, and issue slots are
// what an activation and a generator run short of.
#pragma once
#include "device_vector.cuh"
#include "kernels_dropout.cuh"
#include "point_range.hpp"

namespace cpde::ops {

enum Activation : int32_t { SIGMOID = 0, LINEAR = 1, TANH = 2, SILU = 3 };

constexpr int NORM_THREADS = 256;
constexpr int NORM_WARPS = NORM_THREADS / 32;
constexpr int NORM_BLOCKS = 4;  // CTAs of an SM; a launch has as many as the GPU holds at once

struct NormShape {
    int64_t x_point, x_instance, grad_point, grad_instance;  // strides in elements
    int32_t instances, points, channels, groups, width;      // width: channels of a group
    int32_t vectors;                                         // channels / V
    int32_t tile, tiles;                                     // vectors of a block, blocks across the channels
    int32_t pieces;                                          // most groups that a tile meets
    int32_t splits;                                          // blocks along the points
    int32_t activation;
    float eps;
    const int32_t* lengths;
    DropoutRule rule;
};

template <class P>
__device__ __forceinline__ float parameter(const P* p, int32_t i, float none) {
    return p ? to_float(p[i]) : none;
}

__device__ __forceinline__ int32_t length_of(const NormShape& s, int32_t n) {
    if (!s.lengths) return s.points;
    const int32_t l = s.lengths[n];
    return l < 0 ? 0 : l < s.points ? l : s.points;
}

// Calls f with the activation as a compile-time constant: the loops over points
// hold no branch on it.
template <class F>
__device__ __forceinline__ void with_activation(int32_t activation, F&& f) {
    if (activation == SILU) f(std::integral_constant<int32_t, SILU>{});
    else if (activation == SIGMOID) f(std::integral_constant<int32_t, SIGMOID>{});
    else if (activation == TANH) f(std::integral_constant<int32_t, TANH>{});
    else f(std::integral_constant<int32_t, LINEAR>{});
}

constexpr float LOG2_E = 1.4426950408889634f;

// 1 / (1 + 2^t) of V values, a sigmoid of z for t = -log2(e) z, from the special
// function unit's exponential and reciprocal (a few 2^-23 off): an IEEE
// reciprocal alone would take as many instructions as the rest of an element.
template <int V>
__device__ __forceinline__ Pairs<V> sigmoid2(const Pairs<V>& t) {
    Pairs<V> f;
    f.fill(0.0f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t.get(j)));
        f.set(j, e);
    }
#pragma unroll
    for (int i = 0; i < Pairs<V>::N; ++i) f.p[i] = __fadd2_rn(f.p[i], both(1.0f));
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(f.get(j)));
        f.set(j, r);
    }
    return f;
}

// What the weights and biases of z are scaled by, so that the activation's
// argument comes out of the normalisation's own multiply-add: the forward's
// sigmoid, and the gradients of both, want t.
template <int32_t ACTIVATION, bool GRADIENT>
__device__ constexpr float argument_scale() {
    return ACTIVATION == SIGMOID || (GRADIENT && ACTIVATION == SILU) ? -LOG2_E : 1.0f;
}

// act(z) of z argument_scale.
template <int32_t ACTIVATION, int V>
__device__ __forceinline__ void activate(Pairs<V>& z) {
    if constexpr (ACTIVATION == SILU) {
        Pairs<V> t = z;
        scale<V>(t, -LOG2_E);
        t = sigmoid2<V>(t);
#pragma unroll
        for (int i = 0; i < Pairs<V>::N; ++i) z.p[i] = __fmul2_rn(z.p[i], t.p[i]);
    } else if constexpr (ACTIVATION == SIGMOID) {
        z = sigmoid2<V>(z);
    } else if constexpr (ACTIVATION == TANH) {
#pragma unroll
        for (int j = 0; j < V; ++j) z.set(j, tanhf(z.get(j)));
    }
}

// h *= act'(z), from t = z argument_scale: f + f (1 - f) z, f (1 - f) or 1 - tanh(z)^2.
template <int32_t ACTIVATION, int V>
__device__ __forceinline__ void activate_gradient(Pairs<V>& h, const Pairs<V>& t) {
    if constexpr (ACTIVATION == SILU || ACTIVATION == SIGMOID) {
        const Pairs<V> f = sigmoid2<V>(t);
        constexpr float by = ACTIVATION == SILU ? -1.0f / LOG2_E : 1.0f;
#pragma unroll
        for (int i = 0; i < Pairs<V>::N; ++i) {
            const float2 back = __ffma2_rn(f.p[i], both(-by), both(by));
            const float2 slope = ACTIVATION == SILU ? __ffma2_rn(f.p[i], __fmul2_rn(t.p[i], back), f.p[i])
                                                    : __fmul2_rn(f.p[i], back);
            h.p[i] = __fmul2_rn(h.p[i], slope);
        }
    } else if constexpr (ACTIVATION == TANH) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float y = tanhf(t.get(j));
            h.set(j, h.get(j) * fmaf(-y, y, 1.0f));
        }
    }
}

// (count, mean, sum of squared deviations) of two sets together (Chan, Golub
// and LeVeque, 1979).
struct Moments {
    float count, mean, m2;
};
__device__ __forceinline__ Moments merged(const Moments& a, const Moments& b) {
    const float count = a.count + b.count;
    if (b.count == 0.0f) return a;
    if (a.count == 0.0f) return b;
    const float delta = b.mean - a.mean, share = b.count / count;
    return {count, finite(delta) ? a.mean + delta * share : a.mean + b.mean, a.m2 + b.m2 + delta * delta * a.count * share};
}
__device__ __forceinline__ Moments warp_merged(Moments m) {
#pragma unroll
    for (int d = 16; d; d /= 2) {
        const Moments o = {__shfl_down_sync(~0u, m.count, d), __shfl_down_sync(~0u, m.mean, d),
                           __shfl_down_sync(~0u, m.m2, d)};
        m = merged(m, o);
    }
    return m;
}

// Channels [first, first + count) of the tile, and the groups they meet.
struct Tile {
    int32_t first, count, group, groups;
};
template <int V>
__device__ __forceinline__ Tile tile_of(const NormShape& s, int32_t tile) {
    const int32_t first = tile * s.tile * V, count = min(s.tile * V, s.channels - first);
    const int32_t group = first / s.width;
    return {first, count, group, (first + count - 1) / s.width - group + 1};
}

// Moments of each piece of a group in a block's points and channels.
// pieces[instance][split][tile][piece] = (count, mean, m2).
template <class T, int V>
__global__ void __launch_bounds__(NORM_THREADS, NORM_BLOCKS) k_norm_moments(const T* __restrict__ x, NormShape s,
                                                                Moments* __restrict__ pieces) {
    extern __shared__ float norm_shared[];  // [ty][channel of the tile] x (mean, m2)
    next_launch_may_begin();
    const int32_t split = blockIdx.x % s.splits, n = blockIdx.x / s.splits;
    const Tile t = tile_of<V>(s, blockIdx.y);
    const int32_t ys = NORM_THREADS / s.tile;
    const int32_t ty = threadIdx.x / s.tile, tx = threadIdx.x % s.tile;
    const int32_t width = s.tile * V;
    int32_t lo, hi;
    split_range(length_of(s, n), split, s.splits, lo, hi);
    const bool active = ty < ys && tx * V < t.count;
    if (active) {
        // Deviations from the thread's own first value: their squares cancel by
        // no more than the number of the thread's points.
        constexpr int N = Pairs<V>::N;
        Pairs<V> shift, s1, s2;
        shift.fill(0.0f);
        s1.fill(0.0f);
        s2.fill(0.0f);
        int32_t count = 0;
        // Points are counted from lo: a thread's last step goes beyond hi, which may be
        // 2^31 - 2.
        const T* base = x + n * s.x_instance + lo * s.x_point + t.first + tx * V;
        const int32_t points = hi - lo;
        if (ty < points) {
            shift = unpack_pairs<T, V>(load<T, V>(base + ty * s.x_point));
#pragma unroll
            for (int j = 0; j < V; ++j) shift.set(j, -finite_or_zero(shift.get(j)));
        }
#pragma unroll 4
        for (int32_t p = ty; p < points; p += ys) {
            const Pairs<V> f = unpack_pairs<T, V>(load<T, V>(base + p * s.x_point));
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float2 d = __fadd2_rn(f.p[i], shift.p[i]);
                s1.p[i] = __fadd2_rn(s1.p[i], d);
                s2.p[i] = __ffma2_rn(d, d, s2.p[i]);
            }
            ++count;
        }
        const float inverse = count ? 1.0f / float(count) : 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float mean = s1.get(j) * inverse;
            float* to = norm_shared + 2 * (ty * width + tx * V + j);
            to[0] = mean - shift.get(j);
            to[1] = not_negative(s2.get(j) - s1.get(j) * mean);
        }
    }
    __syncthreads();
    // A warp joins a group's piece: its channels' and threads' moments.
    const int32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int32_t g = warp; g < t.groups; g += NORM_WARPS) {
        const int32_t c0 = max((t.group + g) * s.width - t.first, 0);
        const int32_t c1 = min((t.group + g + 1) * s.width - t.first, t.count);
        Moments m = {0.0f, 0.0f, 0.0f};
        const int32_t cs = c1 - c0;
        for (int32_t i = lane; i < cs * ys; i += 32) {
            const int32_t y = i / cs, c = c0 + i - y * cs;
            const int32_t points = hi - lo > y ? (hi - lo - y - 1) / ys + 1 : 0;
            const float* from = norm_shared + 2 * (y * width + c);
            m = merged(m, {float(points), from[0], from[1]});
        }
        m = warp_merged(m);
        if (lane == 0) pieces[(int64_t(blockIdx.x) * s.tiles + blockIdx.y) * s.pieces + g] = m;
    }
}

// Terms of a thread's vector by channel. ONE: its channels are of one group, so
// that what belongs to the group is two registers and not V.
template <int V, bool ONE>
struct GroupTerms {
    static constexpr int N = ONE ? 1 : Pairs<V>::N;
    float2 p[N];
    __device__ __forceinline__ const float2& of(int i) const { return p[ONE ? 0 : i]; }
    __device__ __forceinline__ void set(int j, float v) {
        if (ONE) p[0] = both(v);
        else (j % 2 ? p[ONE ? 0 : j / 2].y : p[ONE ? 0 : j / 2].x) = v;
    }
};

// z = (x - mean) gain + bias, gain = weight rstd.
template <int V, bool ONE>
struct Terms {
    GroupTerms<V, ONE> minus_mean;
    Pairs<V> gain, bias;
};

// factor drop(act(z)) of a vector of x.
template <int32_t ACTIVATION, bool DROPS, int V, bool ONE>
__device__ __forceinline__ void norm_value(Pairs<V>& f, const Terms<V, ONE>& k, uint64_t at, const DropoutRule& rule) {
#pragma unroll
    for (int i = 0; i < Pairs<V>::N; ++i)
        f.p[i] = __ffma2_rn(__fadd2_rn(f.p[i], k.minus_mean.of(i)), k.gain.p[i], k.bias.p[i]);
    activate<ACTIVATION, V>(f);
    if constexpr (DROPS) {
        drop_at<V>(f, at, rule);
        scale<V>(f, rule.factor);
    }
}

// Calls f(activation, whether there is dropout), both as constants.
template <class F>
__device__ __forceinline__ void with_tail(const NormShape& s, F&& f) {
    with_activation(s.activation, [&](auto activation) {
        if (s.rule.threshold) f(activation, std::true_type{});
        else f(activation, std::false_type{});
    });
}

// y = drop(act(norm(x))). The block first joins the moments of its groups'
// pieces; the first split of the tile that holds a group's first channel also
// writes mean and rstd.
template <class T, class P, int V, bool ONE>
__global__ void __launch_bounds__(NORM_THREADS, NORM_BLOCKS) k_norm_apply(const T* __restrict__ x, const P* __restrict__ weight,
                                                              const P* __restrict__ bias, T* __restrict__ y,
                                                              float* __restrict__ mean, float* __restrict__ rstd,
                                                              const Moments* pieces, NormShape s) {
    extern __shared__ float norm_shared[];  // [group of the tile] x (mean, rstd)
    after_previous_launch();
    const int32_t split = blockIdx.x % s.splits, n = blockIdx.x / s.splits;
    const Tile t = tile_of<V>(s, blockIdx.y);
    const int32_t length = length_of(s, n);
    const int32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int32_t g = warp; g < t.groups; g += NORM_WARPS) {
        const int32_t group = t.group + g, per = s.tile * V;
        const int32_t first_tile = group * s.width / per, last_tile = ((group + 1) * s.width - 1) / per;
        const int32_t spans = last_tile - first_tile + 1;
        Moments m = {0.0f, 0.0f, 0.0f};
        for (int32_t i = lane; i < spans * s.splits; i += 32) {
            const int32_t sp = i / spans, tile = first_tile + i - sp * spans;
            const int32_t piece = group - tile * per / s.width;
            m = merged(m, pieces[((int64_t(n) * s.splits + sp) * s.tiles + tile) * s.pieces + piece]);
        }
        m = warp_merged(m);
        if (lane == 0) {
            const float r = length ? 1.0f / sqrtf(m.m2 / m.count + s.eps) : 0.0f;
            norm_shared[2 * g] = m.mean;
            norm_shared[2 * g + 1] = r;
            if (split == 0 && first_tile == int32_t(blockIdx.y)) {
                mean[int64_t(n) * s.groups + group] = m.mean;
                rstd[int64_t(n) * s.groups + group] = r;
            }
        }
    }
    __syncthreads();
    const int32_t ys = NORM_THREADS / s.tile;
    const int32_t ty = threadIdx.x / s.tile, tx = threadIdx.x % s.tile;
    if (ty >= ys || tx * V >= t.count) return;
    const int32_t channel = t.first + tx * V;
    Terms<V, ONE> k;
    k.gain.fill(0.0f);
    k.bias.fill(0.0f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int32_t g = (channel + j) / s.width - t.group;
        k.minus_mean.set(j, -norm_shared[2 * g]);
        k.gain.set(j, parameter(weight, channel + j, 1.0f) * norm_shared[2 * g + 1]);
        k.bias.set(j, parameter(bias, channel + j, 0.0f));
    }
    int32_t lo, hi;
    split_range(s.points, split, s.splits, lo, hi);
    const T* from = x + n * s.x_instance + channel;
    const int64_t row = int64_t(n) * s.points;
    // From the back: the moments' pass has left the ends of the ranges in L2.
    with_tail(s, [&](auto activation, auto drops) {
        constexpr int32_t ACTIVATION = decltype(activation)::value;
        Terms<V, ONE> scaled = k;
        if constexpr (argument_scale<ACTIVATION, false>() != 1.0f) {
            scale<V>(scaled.gain, argument_scale<ACTIVATION, false>());
            scale<V>(scaled.bias, argument_scale<ACTIVATION, false>());
        }
#pragma unroll 4
        for (int32_t p = hi - 1 - ty; p >= lo; p -= ys) {
            const int64_t at = (row + p) * s.channels + channel;
            if (p >= length) {
                store<T, V>(y + at, zeros<T, V>());
                continue;
            }
            Pairs<V> f = unpack_pairs<T, V>(load<T, V>(from + p * s.x_point));
            norm_value<ACTIVATION, decltype(drops)::value, V, ONE>(f, scaled, uint64_t(at), s.rule);
            store<T, V>(y + at, pack_pairs<T, V>(f));
        }
    });
}

// Terms of the gradient. With d = x - mean: z = d gain + bias, gain = weight rstd,
// and xhat = d rstd stays unformed: rstd goes into what multiplies d.
template <int V, bool ONE>
struct AdjointTerms {
    GroupTerms<V, ONE> minus_mean, rstd;
    Pairs<V> gain, bias;
    __device__ __forceinline__ float rstd_of(int j) const { return j % 2 ? rstd.of(j / 2).y : rstd.of(j / 2).x; }
    __device__ __forceinline__ void set_gain(const Pairs<V>& weight) {
#pragma unroll
        for (int i = 0; i < Pairs<V>::N; ++i) gain.p[i] = __fmul2_rn(weight.p[i], rstd.of(i));
    }
    // For an activation's argument.
    template <int32_t ACTIVATION>
    __device__ __forceinline__ AdjointTerms scaled() const {
        AdjointTerms k = *this;
        if constexpr (argument_scale<ACTIVATION, true>() != 1.0f) {
            scale<V>(k.gain, argument_scale<ACTIVATION, true>());
            scale<V>(k.bias, argument_scale<ACTIVATION, true>());
        }
        return k;
    }
};

template <class P, int V, bool ONE>
__device__ __forceinline__ void load_terms(AdjointTerms<V, ONE>& k, const NormShape& s, int32_t n, int32_t channel,
                                           const float* mean, const float* rstd, const P* weight, const P* bias) {
    Pairs<V> w;
    w.fill(0.0f);
    k.bias.fill(0.0f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int64_t g = int64_t(n) * s.groups + (channel + j) / s.width;
        if (!ONE || j == 0) {
            k.minus_mean.set(j, -mean[g]);
            k.rstd.set(j, rstd[g]);
        }
        w.set(j, parameter(weight, channel + j, 1.0f));
        k.bias.set(j, parameter(bias, channel + j, 0.0f));
    }
    k.set_gain(w);
}

// From x and the kept gradients in h: d, and h act'(z), not yet scaled by the
// dropout's factor. `k` is scaled for the activation.
template <int32_t ACTIVATION, int V, bool ONE>
__device__ __forceinline__ void norm_adjoint(Pairs<V>& d, Pairs<V>& h, const AdjointTerms<V, ONE>& k) {
    Pairs<V> t;
#pragma unroll
    for (int i = 0; i < Pairs<V>::N; ++i) {
        d.p[i] = __fadd2_rn(d.p[i], k.minus_mean.of(i));
        if constexpr (ACTIVATION != LINEAR) t.p[i] = __ffma2_rn(d.p[i], k.gain.p[i], k.bias.p[i]);
    }
    if constexpr (ACTIVATION != LINEAR) activate_gradient<ACTIVATION, V>(h, t);
}

// A thread's sums of h and of h xhat by channel.
template <int V, bool ONE>
struct AdjointSums {
    Pairs<V> h, hd;
    __device__ __forceinline__ AdjointSums() {
        h.fill(0.0f);
        hd.fill(0.0f);
    }
    __device__ __forceinline__ void add(const Pairs<V>& d, const Pairs<V>& values) {
#pragma unroll
        for (int i = 0; i < Pairs<V>::N; ++i) {
            h.p[i] = __fadd2_rn(h.p[i], values.p[i]);
            hd.p[i] = __ffma2_rn(values.p[i], d.p[i], hd.p[i]);
        }
    }
    __device__ __forceinline__ float2 of(int j, const AdjointTerms<V, ONE>& k, float factor) const {
        return make_float2(h.get(j) * factor, hd.get(j) * factor * k.rstd_of(j));
    }
};

// dx = rstd (factor w h - (m1 + xhat m2)) as products and sums.
template <int V, bool ONE>
struct InputTerms {
    Pairs<V> gain;              // factor w rstd
    GroupTerms<V, ONE> m1, m2;  // -rstd m1, -rstd^2 m2
    __device__ __forceinline__ void set(int j, float channel_gain, float minus_m1, float minus_m2) {
        gain.set(j, channel_gain);
        if (!ONE || j == 0) {
            m1.set(j, minus_m1);
            m2.set(j, minus_m2);
        }
    }
    __device__ __forceinline__ void apply(Pairs<V>& h, const Pairs<V>& d) const {
#pragma unroll
        for (int i = 0; i < Pairs<V>::N; ++i)
            h.p[i] = __ffma2_rn(h.p[i], gain.p[i], __ffma2_rn(d.p[i], m2.of(i), m1.of(i)));
    }
    // With the product rounded by itself, as it is in m1: a group of one value, whose
    // m1 is that product, then gives exactly zero. (A compiler joins a packed product
    // and sum, the products of single values it leaves apart.)
    __device__ __forceinline__ void apply_apart(Pairs<V>& h, const Pairs<V>& d) const {
#pragma unroll
        for (int j = 0; j < V; ++j) h.set(j, __fmul_rn(h.get(j), gain.get(j)));
#pragma unroll
        for (int i = 0; i < Pairs<V>::N; ++i) h.p[i] = __fadd2_rn(h.p[i], __ffma2_rn(d.p[i], m2.of(i), m1.of(i)));
    }
};

// factor w rstd, rounded in one order wherever it is needed.
__device__ __forceinline__ float input_gain(float weight_rstd, float factor) { return factor * weight_rstd; }

// Sums of h and h d over a block's points: per channel as h and h xhat for dw and
// db (channel_sums[instance][split][channel]), and times factor w rstd per piece of
// a group for dx (pieces[instance][split][tile][piece]).
template <class T, class P, int V, bool ONE>
__global__ void __launch_bounds__(NORM_THREADS, NORM_BLOCKS) k_norm_sums(const T* __restrict__ grad, const T* __restrict__ x,
                                                             const float* __restrict__ mean,
                                                             const float* __restrict__ rstd,
                                                             const P* __restrict__ weight, const P* __restrict__ bias,
                                                             NormShape s, float2* __restrict__ channel_sums,
                                                             float2* __restrict__ pieces) {
    extern __shared__ float norm_shared[];  // [ty][channel of the tile] x (h, h d)
    next_launch_may_begin();
    float2* shared = reinterpret_cast<float2*>(norm_shared);
    const int32_t split = blockIdx.x % s.splits, n = blockIdx.x / s.splits;
    const Tile t = tile_of<V>(s, blockIdx.y);
    const int32_t ys = NORM_THREADS / s.tile;
    const int32_t ty = threadIdx.x / s.tile, tx = threadIdx.x % s.tile;
    const int32_t width = s.tile * V;
    int32_t lo, hi;
    split_range(length_of(s, n), split, s.splits, lo, hi);
    if (ty < ys && tx * V < t.count) {
        const int32_t channel = t.first + tx * V;
        AdjointTerms<V, ONE> k;
        load_terms<P, V, ONE>(k, s, n, channel, mean, rstd, weight, bias);
        AdjointSums<V, ONE> sums;
        const T* from = x + n * s.x_instance + lo * s.x_point + channel;
        const T* gfrom = grad + n * s.grad_instance + lo * s.grad_point + channel;
        const int64_t row = int64_t(n) * s.points + lo;
        const int32_t points = hi - lo;  // counted from lo, as the moments
        with_tail(s, [&](auto activation, auto drops) {
            constexpr int32_t ACTIVATION = decltype(activation)::value;
            const auto scaled = k.template scaled<ACTIVATION>();
#pragma unroll 2
            for (int32_t p = ty; p < points; p += ys) {
                Pairs<V> d = unpack_pairs<T, V>(load<T, V>(from + p * s.x_point));
                Pairs<V> h = unpack_pairs<T, V>(load<T, V>(gfrom + p * s.grad_point));
                if constexpr (decltype(drops)::value)
                    drop_at<V>(h, uint64_t((row + p) * s.channels + channel), s.rule);
                norm_adjoint<ACTIVATION, V, ONE>(d, h, scaled);
                sums.add(d, h);
            }
        });
#pragma unroll
        for (int j = 0; j < V; ++j) shared[ty * width + tx * V + j] = make_float2(sums.h.get(j), sums.hd.get(j));
    }
    __syncthreads();
    for (int32_t c = threadIdx.x; c < t.count; c += NORM_THREADS) {
        float2 sum = make_float2(0.0f, 0.0f);
        for (int32_t y = 0; y < ys; ++y) {
            const float2 v = shared[y * width + c];
            sum.x += v.x;
            sum.y += v.y;
        }
        const int32_t channel = t.first + c;
        const float r = rstd[int64_t(n) * s.groups + channel / s.width];
        channel_sums[int64_t(blockIdx.x) * s.channels + channel] = make_float2(sum.x * s.rule.factor, sum.y * s.rule.factor * r);
        const float gain = input_gain(parameter(weight, channel, 1.0f) * r, s.rule.factor);
        shared[c] = make_float2(sum.x * gain, sum.y * gain);  // only this thread reads column c
    }
    __syncthreads();
    const int32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int32_t g = warp; g < t.groups; g += NORM_WARPS) {
        const int32_t c0 = max((t.group + g) * s.width - t.first, 0);
        const int32_t c1 = min((t.group + g + 1) * s.width - t.first, t.count);
        float2 sum = make_float2(0.0f, 0.0f);
        for (int32_t c = c0 + lane; c < c1; c += 32) {
            sum.x += shared[c].x;
            sum.y += shared[c].y;
        }
#pragma unroll
        for (int d = 16; d; d /= 2) {
            sum.x += __shfl_down_sync(~0u, sum.x, d);
            sum.y += __shfl_down_sync(~0u, sum.y, d);
        }
        if (lane == 0) pieces[(int64_t(blockIdx.x) * s.tiles + blockIdx.y) * s.pieces + g] = sum;
    }
}

// dw and db of 32 channels: sums over the rows of channel_sums in a fixed order.
template <class P, int WARPS>
__device__ __forceinline__ void sum_parameters(P* __restrict__ dweight, P* __restrict__ dbias,
                                               const float2* channel_sums, int32_t rows,
                                               int32_t channels, int32_t block) {
    __shared__ float2 shared[WARPS][32];
    const int32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, channel = block * 32 + lane;
    float2 sum = make_float2(0.0f, 0.0f);
    if (channel < channels) {
#pragma unroll 8
        for (int32_t i = warp; i < rows; i += WARPS) sum = __fadd2_rn(sum, channel_sums[int64_t(i) * channels + channel]);
    }
    shared[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && channel < channels) {
        for (int w = 1; w < WARPS; ++w) sum = __fadd2_rn(sum, shared[w][lane]);
        if (dbias) dbias[channel] = from_float<P>(sum.x);
        if (dweight) dweight[channel] = from_float<P>(sum.y);
    }
}

// dx, and in the blocks behind those of the last instance dw and db: 32
// channels each, summed over instances and splits in a fixed order.
template <class T, class P, int V, bool ONE>
__global__ void __launch_bounds__(NORM_THREADS, NORM_BLOCKS) k_norm_input_gradient(
    const T* __restrict__ grad, const T* __restrict__ x, const float* __restrict__ mean,
    const float* __restrict__ rstd, const P* __restrict__ weight, const P* __restrict__ bias, T* __restrict__ dx,
    P* __restrict__ dweight, P* __restrict__ dbias, const float2* channel_sums, const float2* pieces, NormShape s) {
    extern __shared__ float norm_shared[];
    after_previous_launch();
    float2* shared = reinterpret_cast<float2*>(norm_shared);
    const int32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int32_t n = blockIdx.x / s.splits;
    if (n >= s.instances) {
        if (blockIdx.y == 0)
            sum_parameters<P, NORM_WARPS>(dweight, dbias, channel_sums, s.instances * s.splits, s.channels,
                              blockIdx.x - s.instances * s.splits);
        return;
    }
    const int32_t split = blockIdx.x % s.splits;
    const Tile t = tile_of<V>(s, blockIdx.y);
    const int32_t length = length_of(s, n);
    for (int32_t g = warp; g < t.groups; g += NORM_WARPS) {
        const int32_t group = t.group + g, per = s.tile * V;
        const int32_t first_tile = group * s.width / per, last_tile = ((group + 1) * s.width - 1) / per;
        const int32_t spans = last_tile - first_tile + 1;
        float2 sum = make_float2(0.0f, 0.0f);
        for (int32_t i = lane; i < spans * s.splits; i += 32) {
            const int32_t sp = i / spans, tile = first_tile + i - sp * spans;
            const int32_t piece = group - tile * per / s.width;
            const float2 v = pieces[((int64_t(n) * s.splits + sp) * s.tiles + tile) * s.pieces + piece];
            sum.x += v.x;
            sum.y += v.y;
        }
#pragma unroll
        for (int d = 16; d; d /= 2) {
            sum.x += __shfl_down_sync(~0u, sum.x, d);
            sum.y += __shfl_down_sync(~0u, sum.y, d);
        }
        const float inverse = length ? 1.0f / (float(length) * float(s.width)) : 0.0f;
        if (lane == 0) shared[g] = make_float2(sum.x * inverse, sum.y * inverse);
    }
    __syncthreads();
    const int32_t ys = NORM_THREADS / s.tile;
    const int32_t ty = threadIdx.x / s.tile, tx = threadIdx.x % s.tile;
    if (ty >= ys || tx * V >= t.count) return;
    const int32_t channel = t.first + tx * V;
    AdjointTerms<V, ONE> k;
    load_terms<P, V, ONE>(k, s, n, channel, mean, rstd, weight, bias);
    InputTerms<V, ONE> to_input;
    to_input.gain.fill(0.0f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 m = shared[(channel + j) / s.width - t.group];
        const float r = k.rstd_of(j);
        to_input.set(j, input_gain(k.gain.get(j), s.rule.factor), -m.x, -r * r * m.y);
    }
    int32_t lo, hi;
    split_range(s.points, split, s.splits, lo, hi);
    const T* from = x + n * s.x_instance + channel;
    const T* gfrom = grad + n * s.grad_instance + channel;
    // From the back, as the forward.
    with_tail(s, [&](auto activation, auto drops) {
        constexpr int32_t ACTIVATION = decltype(activation)::value;
        const auto scaled = k.template scaled<ACTIVATION>();
#pragma unroll 2
        for (int32_t p = hi - 1 - ty; p >= lo; p -= ys) {
            const int64_t at = (int64_t(n) * s.points + p) * s.channels + channel;
            if (p >= length) {
                store<T, V>(dx + at, zeros<T, V>());
                continue;
            }
            Pairs<V> d = unpack_pairs<T, V>(load<T, V>(from + p * s.x_point));
            Pairs<V> h = unpack_pairs<T, V>(load<T, V>(gfrom + p * s.grad_point));
            if constexpr (decltype(drops)::value) drop_at<V>(h, uint64_t(at), s.rule);
            norm_adjoint<ACTIVATION, V, ONE>(d, h, scaled);
            to_input.apply_apart(h, d);
            store<T, V>(dx + at, pack_pairs<T, V>(h));
        }
    });
}

}  // namespace cpde::ops
