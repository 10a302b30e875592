// Linear layers: what stands before and behind the matrix products of
// kernels_gemm.cuh and kernels_gather.cuh.
//
// z = x W' + b, y = r + act(z); from dy: dz = dy act'(z), dx = dz W, dW = dz' x,
// db = sum of dz over the points.
#pragma once
#include "kernels_gather.cuh"

namespace cpde::ops {

// 1 / (1 + e^-z) from the special function unit's 2^x and 1/x.
__device__ __forceinline__ float layer_sigmoid(float z) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * z));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
}
// tanh z = 1 - 2 / (1 + e^2z), and its Taylor series below 0.35, where the difference would
// lose the digits that are left (the next term is 1e-8 of the value). Both without a
// branch: of a warp's values some are always on either side.
__device__ __forceinline__ float layer_tanh(float z) {
    const float a = fabsf(z), q = z * z;
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(2.885390081777927f * a));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    float s = fmaf(q, -1382.0f / 155925.0f, 62.0f / 2835.0f);
    s = fmaf(q, s, -17.0f / 315.0f);
    s = fmaf(q, s, 2.0f / 15.0f);
    s = fmaf(q, s, -1.0f / 3.0f);
    const float near = fmaf(z * q, s, z), far = copysignf(fmaf(-2.0f, r, 1.0f), z);
    return a < 0.35f ? near : far;
}
// The activations by their codes: 0 sigmoid, 1 linear, 2 tanh, 3 SiLU. FP32 arrays
// (EXACT) take the library's functions, good to an ulp or two, 16-bit ones those above.
template <bool EXACT>
__device__ __forceinline__ float layer_activation(float z, int32_t activation) {
    if (activation == 1) return z;
    if (activation == 2) return EXACT ? tanhf(z) : layer_tanh(z);
    const float f = EXACT ? 1.0f / (1.0f + expf(-z)) : layer_sigmoid(z);
    return activation == 3 ? z * f : f;
}
template <bool EXACT>
__device__ __forceinline__ float layer_slope(float z, int32_t activation) {
    if (activation == 1) return 1.0f;
    if (activation == 2) {
        const float t = EXACT ? tanhf(z) : layer_tanh(z);
        return fmaf(-t, t, 1.0f);
    }
    const float f = EXACT ? 1.0f / (1.0f + expf(-z)) : layer_sigmoid(z);
    return activation == 3 ? fmaf(f, z * (1.0f - f), f) : f * (1.0f - f);
}

template <bool EXACT, int V>
__device__ __forceinline__ void activate_all(float (&v)[V], int32_t activation) {
    if (activation == 1) return;
    if (activation == 2) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = layer_activation<EXACT>(v[i], 2);
    } else if (activation == 3) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = layer_activation<EXACT>(v[i], 3);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = layer_activation<EXACT>(v[i], 0);
    }
}

// Bias, activation and residual in the product's epilogue, or plain results, or the
// partial sums of a split contraction.
template <class T>
struct LinearEpilogue {
    const void* bias;       // of FP32 or T, or null
    const T* residual;      // or null
    T* z;                   // or null
    void* y;                // of FP32 or T
    float* partial;         // where the contraction is split: (split, row, column) sums, pitch n rounded up to 16
    int64_t residual_stride;
    int32_t activation;
    bool bias_wide, y_wide;
    bool whole;             // 16 elements at a time are there and in whole 32 bytes, in every array
    bool fours;             // four at a time are, for the joining of partial sums

    using Fetched = Sixteen<T>;  // the residual
    __device__ static int64_t partial_pitch(const GemmShape& s) { return (s.n + 15) / 16 * 16; }

    __device__ __forceinline__ void fetch(Fetched& f, int64_t row, int column, int, const GemmShape&) const {
        if (residual && !partial) f.load(residual + row * residual_stride + column);
    }
    __device__ __forceinline__ void whole_row(float (&v)[16], const Fetched& f, int64_t row, int column, int, int split, int, int,
                                         const GemmShape& s) const {
        if (partial) {
            Sixteen<float>::store(partial + (split * int64_t(s.m) + row) * partial_pitch(s) + column, v);
            return;
        }
        if (bias) {
            float b[16];
            if (bias_wide) load_some<float, 16>(static_cast<const float*>(bias) + column, b, 16, true);
            else load_some<T, 16>(static_cast<const T*>(bias) + column, b, 16, true);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] += b[i];
        }
        const int64_t at = row * s.n + column;
        if (z) Sixteen<T>::store(z + at, v);
        activate_all<sizeof(T) == 4, 16>(v, activation);
        if (residual) {
            float r[16];
            f.get(r);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] += r[i];
        }
        if (y_wide) Sixteen<float>::store(static_cast<float*>(y) + at, v);
        else Sixteen<T>::store(static_cast<T*>(y) + at, v);
    }
    // The same of `left` columns in arrays of any layout; what goes to z and to y.
    __device__ __forceinline__ void odd(float (&v)[16], float (&before)[16], int64_t row, int column, int left, int,
                                        const GemmShape&) const {
        float b[16];
        if (bias) {
            if (bias_wide) load_some<float, 16>(static_cast<const float*>(bias) + column, b, left, false);
            else load_some<T, 16>(static_cast<const T*>(bias) + column, b, left, false);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] += b[i];
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) before[i] = v[i];
        activate_all<sizeof(T) == 4, 16>(v, activation);
        if (residual) {
            load_some<T, 16>(residual + row * residual_stride + column, b, left, false);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] += b[i];
        }
    }
    __device__ __forceinline__ bool writes_z() const { return z; }
    template <int WHICH>
    __device__ __forceinline__ void write(float f, int64_t row, int column, int, const GemmShape& s) const {
        const int64_t at = row * s.n + column;
        if (WHICH == 0) z[at] = from_float<T>(f);
        else if (y_wide) static_cast<float*>(y)[at] = f;
        else static_cast<T*>(y)[at] = from_float<T>(f);
    }
    // V elements, whatever the arrays' alignment if V is 1.
    template <int V>
    __device__ __forceinline__ void some(float (&v)[V], int64_t row, int column, const GemmShape& s) const {
        const int64_t at = row * s.n + column;
        if (bias) {
            float b[V];
            if (bias_wide) load_some<float, V>(static_cast<const float*>(bias) + column, b, V, true);
            else load_some<T, V>(static_cast<const T*>(bias) + column, b, V, true);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] += b[i];
        }
        if (z) store<T, V>(z + at, pack<T, V>(v));
        activate_all<sizeof(T) == 4, V>(v, activation);
        if (residual) {
            float r[V];
            load_some<T, V>(residual + row * residual_stride + column, r, V, true);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] += r[i];
        }
        if (y_wide) store<float, V>(static_cast<float*>(y) + at, pack<float, V>(v));
        else store<T, V>(static_cast<T*>(y) + at, pack<T, V>(v));
    }
};

// Joins the partial sums of a split contraction and ends them as the epilogue does. A
// result's splits are shared by `share` neighbouring threads (1 or 8), each of which adds
// every share-th in order; their sums are added in order too.
template <class T, int V>
__global__ void __launch_bounds__(256) k_join(LinearEpilogue<T> epilogue, GemmShape s, int32_t share) {
    next_launch_may_begin();
    after_previous_launch();
    const float* partial = epilogue.partial;
    epilogue.partial = nullptr;
    const int64_t pitch = LinearEpilogue<T>::partial_pitch(s), across = (s.n + V - 1) / V, all = s.m * across;
    const int mine = threadIdx.x % share;
    // Whole warps go round together.
    const int64_t step = gridDim.x * int64_t(256 / share);
    for (int64_t begin = blockIdx.x * int64_t(256 / share); begin < all; begin += step) {
        const int64_t i = begin + threadIdx.x / share, row = min(i, all - 1) / across;
        const int column = int(min(i, all - 1) % across) * V;
        float sum[V] = {};
#pragma unroll 8
        for (int split = mine; split < s.splits; split += share) {
            float v[V];
            load_some<float, V>(partial + (split * int64_t(s.m) + row) * pitch + column, v, V, true);
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += v[j];
        }
        for (int o = 1; o < share; o *= 2)
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += __shfl_xor_sync(~0u, sum[j], o);
        if (mine == 0 && i < all) epilogue.template some<V>(sum, row, column, s);
    }
}

// An operand's parts from an array: part after part, rows of `pitch`. With z, the
// array is multiplied by the activation's slope there. `sums` takes the column sums
// of each chunk of rows.
template <class T>
struct PartsCall {
    const T* x;
    const T* z;
    void* out;         // or null: sums alone
    float* sums;       // (chunk, column), or null
    int64_t x_stride, z_stride, rows, chunk;
    int32_t columns, pitch, activation;
    int32_t lanes;     // threads of a row, eight columns each: a power of two up to 32
    int32_t strips, blocks;  // strips of columns; blocks, all strips of a chunk of rows in turn
    bool whole;        // x and z can be read in eights
    bool rest;         // what rounding to a 16-bit type leaves follows as a second array
};

// Up to three operands in one launch, block after block. Bound by memory: dz of 32,768 x
// 2048 bf16 with SiLU and its column sums takes 95 us (403 MB, 4.2 TB/s; the exponentials
// and divisions half of that).
constexpr int MOST_PARTS = 3;
template <class T>
struct PartsCalls {
    PartsCall<T> call[MOST_PARTS];
    int32_t count;
};

template <class T>
__global__ void __launch_bounds__(256) k_parts(const __grid_constant__ PartsCalls<T> calls) {
    __shared__ float shared[256 * 8];
    next_launch_may_begin();
    after_previous_launch();
    int which = 0, block = blockIdx.x;
    while (which + 1 < calls.count && block >= calls.call[which].blocks) block -= calls.call[which++].blocks;
    const PartsCall<T>& c = calls.call[which];
    const int strip = block % c.strips, chunk = block / c.strips;
    const int lane = threadIdx.x % c.lanes, high = 256 / c.lanes;
    const int column = (strip * c.lanes + lane) * 8;
    const int64_t from = chunk * c.chunk, to = min(c.rows, from + c.chunk);
    float sum[8] = {};
    if (column < c.columns) {
        const int left = c.columns - column;
        const bool whole = c.whole && left >= 8;
#pragma unroll 2
        for (int64_t row = from + threadIdx.x / c.lanes; row < to; row += high) {
            float v[8];
            load_some<T, 8>(c.x + row * c.x_stride + column, v, left, whole);
            if (c.z) {
                float z[8];
                load_some<T, 8>(c.z + row * c.z_stride + column, z, left, whole);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < left) v[i] *= layer_slope<sizeof(T) == 4>(z[i], c.activation);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += v[i];
            if (c.out) {
                auto* out = static_cast<typename Parts<T>::type*>(c.out) + row * c.pitch + column;
                uint4 part[Parts<T>::count];
                if constexpr (sizeof(T) == 2)
                    if (c.rest) {
                        float h[8], left_over[8];
                        unpack<T, 8>(pack<T, 8>(v), h);
#pragma unroll
                        for (int i = 0; i < 8; ++i) left_over[i] = finite(h[i]) ? v[i] - h[i] : 0.0f;
                        store<T, 8>(out + c.rows * c.pitch, pack<T, 8>(left_over));
                    }
                split_eight<T>(v, part);
#pragma unroll
                for (int p = 0; p < Parts<T>::count; ++p, out += c.rows * c.pitch) *reinterpret_cast<uint4*>(out) = part[p];
            }
        }
    }
    if (!c.sums) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) shared[(threadIdx.x * 8) + i] = sum[i];
    __syncthreads();
    // The rows of threads are added in their order.
    const int wide = c.lanes * 8;
    for (int i = threadIdx.x; i < wide; i += 256) {
        float total = 0.0f;
        for (int r = 0; r < high; ++r) total += shared[r * wide + i];
        const int at = strip * wide + i;
        if (at < c.columns) c.sums[chunk * int64_t(c.columns) + at] = total;
    }
}

// Column sums over the chunks: 32 columns a block, whose 32 warps take every 32nd chunk.
template <class O>
__global__ void __launch_bounds__(1024) k_column_sums(const float* sums, int32_t chunks, int32_t columns, O* out) {
    __shared__ float shared[32][33];
    next_launch_may_begin();
    after_previous_launch();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, column = blockIdx.x * 32 + lane;
    float sum = 0.0f;
    if (column < columns) {
#pragma unroll 8
        for (int i = warp; i < chunks; i += 32) sum += sums[i * int64_t(columns) + column];
    }
    shared[warp][lane] = sum;
    __syncthreads();
    // Warp w adds the 32 sums of column w.
    sum = shared[lane][warp];
    for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0 && blockIdx.x * 32 + warp < columns) out[blockIdx.x * 32 + warp] = from_float<O>(sum);
}

}  // namespace cpde::ops
