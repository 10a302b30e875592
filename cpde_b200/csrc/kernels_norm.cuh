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
#pragma once
#include "device_vector.cuh"
#include "kernels_dropout.cuh"

namespace cpde::ops {

enum Activation : int32_t { SIGMOID = 0, LINEAR = 1, TANH = 2, SILU = 3 };

constexpr int NORM_THREADS = 256;
constexpr int NORM_WARPS = NORM_THREADS / 32;

struct NormShape {
    int64_t x_point, x_instance, grad_point, grad_instance;  // strides in elements
    int32_t instances, points, channels, groups, width;      // width: channels of a group
    int32_t vectors;                                         // channels / V
    int32_t tile, tiles;                                     // vectors of a block, blocks across the channels
    int32_t pieces;                                          // most groups that a tile meets
    int32_t splits, apply_splits;                            // blocks along the points
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

// 1 / (1 + e^-z) from the special function unit's exponential and reciprocal
// (a few 2^-23 off): an IEEE reciprocal alone would take as many instructions
// as the rest of an element.
__device__ __forceinline__ float sigmoid(float z) {
    float e, f;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(f) : "f"(1.0f + e));
    return f;
}

template <int V>
__device__ __forceinline__ void activate(float (&z)[V], int32_t activation) {
    if (activation == SILU) {
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] *= sigmoid(z[i]);
    } else if (activation == SIGMOID) {
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = sigmoid(z[i]);
    } else if (activation == TANH) {
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = tanhf(z[i]);
    }
}

// h *= act'(z).
template <int V>
__device__ __forceinline__ void activate_gradient(float (&h)[V], const float (&z)[V], int32_t activation) {
    if (activation == SILU) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float f = sigmoid(z[i]);
            h[i] *= f * (1.0f + z[i] * (1.0f - f));
        }
    } else if (activation == SIGMOID) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float f = sigmoid(z[i]);
            h[i] *= f * (1.0f - f);
        }
    } else if (activation == TANH) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float t = tanhf(z[i]);
            h[i] *= 1.0f - t * t;
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
    return {count, a.mean + delta * share, a.m2 + b.m2 + delta * delta * a.count * share};
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

// The points [lo, hi) of split `split` of `splits`.
__device__ __forceinline__ void split_range(int32_t length, int32_t split, int32_t splits, int32_t& lo, int32_t& hi) {
    const int32_t per = (length + splits - 1) / splits;
    const int64_t first = int64_t(split) * per;
    lo = int32_t(first < length ? first : length);
    hi = int32_t(first + per < length ? first + per : length);
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
__global__ void __launch_bounds__(NORM_THREADS) k_norm_moments(const T* __restrict__ x, NormShape s,
                                                                Moments* __restrict__ pieces) {
    extern __shared__ float norm_shared[];  // [ty][channel of the tile] x (mean, m2)
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
        float shift[V], s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) shift[j] = s1[j] = s2[j] = 0.0f;
        int32_t count = 0;
        const T* base = x + n * s.x_instance + t.first + tx * V;
        if (lo + ty < hi) unpack<T, V>(load<T, V>(base + (lo + ty) * s.x_point), shift);
#pragma unroll 4
        for (int32_t p = lo + ty; p < hi; p += ys) {
            float f[V];
            unpack<T, V>(load<T, V>(base + p * s.x_point), f);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = f[j] - shift[j];
                s1[j] += d;
                s2[j] = fmaf(d, d, s2[j]);
            }
            ++count;
        }
        const float inverse = count ? 1.0f / float(count) : 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float mean = s1[j] * inverse;
            float* to = norm_shared + 2 * (ty * width + tx * V + j);
            to[0] = shift[j] + mean;
            to[1] = fmaxf(s2[j] - s1[j] * mean, 0.0f);
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

// Terms of a thread's vector by channel; ONE: its channels are of one group, so
// that the statistics are two registers and not 2 V.
template <int V, bool ONE>
struct Terms {
    static constexpr int M = ONE ? 1 : V;
    float mean[M], rstd[M], weight[V], bias[V];
    __device__ __forceinline__ float mean_of(int j) const { return mean[ONE ? 0 : j]; }
    __device__ __forceinline__ float rstd_of(int j) const { return rstd[ONE ? 0 : j]; }
};

// drop(act((f - mean) weight + bias)), with rstd in the weight.
template <int V, bool ONE>
__device__ __forceinline__ void norm_value(float (&f)[V], const Terms<V, ONE>& k, uint64_t at, const NormShape& s) {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = fmaf(f[j] - k.mean_of(j), k.weight[j], k.bias[j]);
    activate<V>(f, s.activation);
    if (s.rule.threshold) drop_at<V>(f, at, s.rule);
}

// y = drop(act(norm(x))). The block first joins the moments of its groups'
// pieces; the first split of the tile that holds a group's first channel also
// writes mean and rstd.
template <class T, class P, int V, bool ONE>
__global__ void __launch_bounds__(NORM_THREADS) k_norm_apply(const T* __restrict__ x, const P* __restrict__ weight,
                                                              const P* __restrict__ bias, T* __restrict__ y,
                                                              float* __restrict__ mean, float* __restrict__ rstd,
                                                              const Moments* __restrict__ pieces, NormShape s) {
    extern __shared__ float norm_shared[];  // [group of the tile] x (mean, rstd)
    const int32_t split = blockIdx.x % s.apply_splits, n = blockIdx.x / s.apply_splits;
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
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int32_t g = (channel + j) / s.width - t.group;
        if (!ONE || j == 0) k.mean[j] = norm_shared[2 * g];
        k.weight[j] = parameter(weight, channel + j, 1.0f) * norm_shared[2 * g + 1];
        k.bias[j] = parameter(bias, channel + j, 0.0f);
    }
    int32_t lo, hi;
    split_range(s.points, split, s.apply_splits, lo, hi);
    const T* from = x + n * s.x_instance + channel;
    const int64_t row = int64_t(n) * s.points;
    // From the back: the moments' pass has left the ends of the ranges in L2.
#pragma unroll 4
    for (int32_t p = hi - 1 - ty; p >= lo; p -= ys) {
        const int64_t at = (row + p) * s.channels + channel;
        if (p >= length) {
            store<T, V>(y + at, zeros<T, V>());
            continue;
        }
        float f[V];
        unpack<T, V>(load<T, V>(from + p * s.x_point), f);
        norm_value<V, ONE>(f, k, uint64_t(at), s);
        store<T, V>(y + at, pack<T, V>(f));
    }
}

// xhat and h of a thread's vector at one point.
template <class T, int V, bool ONE>
__device__ __forceinline__ void norm_adjoint(const Vector<T, V>& vx, const Vector<T, V>& vg, const Terms<V, ONE>& k,
                                             uint64_t at, const NormShape& s, float (&xhat)[V], float (&h)[V]) {
    float z[V];
    unpack<T, V>(vx, xhat);
    unpack<T, V>(vg, h);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        xhat[j] = (xhat[j] - k.mean_of(j)) * k.rstd_of(j);
        z[j] = fmaf(xhat[j], k.weight[j], k.bias[j]);
    }
    if (s.rule.threshold) drop_at<V>(h, at, s.rule);
    activate_gradient<V>(h, z, s.activation);
}

template <class P, int V, bool ONE>
__device__ __forceinline__ void load_terms(Terms<V, ONE>& k, const NormShape& s, int32_t n, int32_t channel,
                                           const float* mean, const float* rstd, const P* weight, const P* bias) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int64_t g = int64_t(n) * s.groups + (channel + j) / s.width;
        if (!ONE || j == 0) {
            k.mean[j] = mean[g];
            k.rstd[j] = rstd[g];
        }
        k.weight[j] = parameter(weight, channel + j, 1.0f);
        k.bias[j] = parameter(bias, channel + j, 0.0f);
    }
}

// Sums of h and h xhat over a block's points: per channel for dw and db
// (channel_sums[instance][split][channel]), and times w per piece of a group
// for dx (pieces[instance][split][tile][piece]).
template <class T, class P, int V, bool ONE>
__global__ void __launch_bounds__(NORM_THREADS) k_norm_sums(const T* __restrict__ grad, const T* __restrict__ x,
                                                             const float* __restrict__ mean,
                                                             const float* __restrict__ rstd,
                                                             const P* __restrict__ weight, const P* __restrict__ bias,
                                                             NormShape s, float2* __restrict__ channel_sums,
                                                             float2* __restrict__ pieces) {
    extern __shared__ float norm_shared[];  // [ty][channel of the tile] x (h, h xhat)
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
        Terms<V, ONE> k;
        load_terms<P, V, ONE>(k, s, n, channel, mean, rstd, weight, bias);
        float sh[V], sx[V];
#pragma unroll
        for (int j = 0; j < V; ++j) sh[j] = sx[j] = 0.0f;
        const T* from = x + n * s.x_instance + channel;
        const T* gfrom = grad + n * s.grad_instance + channel;
#pragma unroll 2
        for (int32_t p = lo + ty; p < hi; p += ys) {
            float xhat[V], h[V];
            norm_adjoint<T, V, ONE>(load<T, V>(from + p * s.x_point), load<T, V>(gfrom + p * s.grad_point), k,
                               uint64_t((int64_t(n) * s.points + p) * s.channels + channel), s, xhat, h);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                sh[j] += h[j];
                sx[j] = fmaf(h[j], xhat[j], sx[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) shared[ty * width + tx * V + j] = make_float2(sh[j], sx[j]);
    }
    __syncthreads();
    for (int32_t c = threadIdx.x; c < t.count; c += NORM_THREADS) {
        float2 sum = make_float2(0.0f, 0.0f);
        for (int32_t y = 0; y < ys; ++y) {
            const float2 v = shared[y * width + c];
            sum.x += v.x;
            sum.y += v.y;
        }
        channel_sums[int64_t(blockIdx.x) * s.channels + t.first + c] = sum;
        const float w = parameter(weight, t.first + c, 1.0f);
        shared[c] = make_float2(sum.x * w, sum.y * w);  // only this thread reads column c
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
template <class P>
__device__ __forceinline__ void sum_parameters(P* __restrict__ dweight, P* __restrict__ dbias,
                                               const float2* __restrict__ channel_sums, int32_t rows,
                                               int32_t channels, int32_t block) {
    __shared__ float2 shared[NORM_WARPS][32];
    const int32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, channel = block * 32 + lane;
    float2 sum = make_float2(0.0f, 0.0f);
    if (channel < channels) {
#pragma unroll 4
        for (int32_t i = warp; i < rows; i += NORM_WARPS) {
            const float2 v = channel_sums[int64_t(i) * channels + channel];
            sum.x += v.x;
            sum.y += v.y;
        }
    }
    shared[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && channel < channels) {
        for (int w = 1; w < NORM_WARPS; ++w) {
            sum.x += shared[w][lane].x;
            sum.y += shared[w][lane].y;
        }
        if (dbias) dbias[channel] = from_float<P>(sum.x);
        if (dweight) dweight[channel] = from_float<P>(sum.y);
    }
}

// dx, and in the blocks behind those of the last instance dw and db: 32
// channels each, summed over instances and splits in a fixed order.
template <class T, class P, int V, bool ONE>
__global__ void __launch_bounds__(NORM_THREADS) k_norm_input_gradient(
    const T* __restrict__ grad, const T* __restrict__ x, const float* __restrict__ mean,
    const float* __restrict__ rstd, const P* __restrict__ weight, const P* __restrict__ bias, T* __restrict__ dx,
    P* __restrict__ dweight, P* __restrict__ dbias, const float2* __restrict__ channel_sums,
    const float2* __restrict__ pieces, NormShape s) {
    extern __shared__ float norm_shared[];
    float2* shared = reinterpret_cast<float2*>(norm_shared);
    const int32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int32_t n = blockIdx.x / s.apply_splits;
    if (n >= s.instances) {
        if (blockIdx.y == 0)
            sum_parameters<P>(dweight, dbias, channel_sums, s.instances * s.splits, s.channels,
                              blockIdx.x - s.instances * s.apply_splits);
        return;
    }
    const int32_t split = blockIdx.x % s.apply_splits;
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
    Terms<V, ONE> k;
    load_terms<P, V, ONE>(k, s, n, channel, mean, rstd, weight, bias);
    constexpr int M = Terms<V, ONE>::M;
    float m1[M], m2[M];
#pragma unroll
    for (int j = 0; j < M; ++j) {
        const float2 m = shared[(channel + j) / s.width - t.group];
        m1[j] = m.x;
        m2[j] = m.y;
    }
    int32_t lo, hi;
    split_range(s.points, split, s.apply_splits, lo, hi);
    const T* from = x + n * s.x_instance + channel;
    const T* gfrom = grad + n * s.grad_instance + channel;
    // From the back, as the forward.
#pragma unroll 2
    for (int32_t p = hi - 1 - ty; p >= lo; p -= ys) {
        const int64_t at = (int64_t(n) * s.points + p) * s.channels + channel;
        if (p >= length) {
            store<T, V>(dx + at, zeros<T, V>());
            continue;
        }
        float xhat[V], h[V];
        norm_adjoint<T, V, ONE>(load<T, V>(from + p * s.x_point), load<T, V>(gfrom + p * s.grad_point), k, uint64_t(at), s,
                           xhat, h);
#pragma unroll
        for (int j = 0; j < V; ++j)
            h[j] = (h[j] * k.weight[j] - fmaf(xhat[j], m2[ONE ? 0 : j], m1[ONE ? 0 : j])) * k.rstd_of(j);
        store<T, V>(dx + at, pack<T, V>(h));
    }
}

}  // namespace cpde::ops
