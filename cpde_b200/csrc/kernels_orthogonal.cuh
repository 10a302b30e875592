// Orthogonalised matrices by Newton-Schulz steps, on the products of
// kernels_gemm.cuh: X0 = G / (|G| + eps) with the Frobenius norm, then
//     A = X X',  Q = b A + c A^2,  X <- a X + Q X
// (or A = X' X and X <- a X + X Q where X is tall), an odd polynomial of the
// singular values. A and Q are symmetric: their tiles up to the diagonal are
// computed, the others are those mirrored.
//
// X, A and Q are held as FP16 parts of value * 2^s, s from the bound that the
// polynomials put on the singular values (no entry of a matrix is above its
// largest one). X always has two parts, 22 bits. For FP32 and FP16 matrices, and small
// ones, the products take both parts of everything. For larger BF16 ones, and optimiser
// steps of 16-bit weights, they take the first: what the steps amplify is an error of X itself in the directions of small singular
// values, and those come through a X, which the epilogue adds from both parts. In
// steps on bf16-like random matrices with a decaying spectrum the result is then
// within 2e-4 to 7e-4 of the exact one in norm (X in one part: 6e-3, all in bf16:
// 5e-2), below the 1.7e-3 of rounding it to bf16.
//
// A 2048 x 8192 bf16 matrix takes 0.72 ms, a step 16 us for A^2 (half of a wave of tiles), 38
// for A and 72 for X, whose tiles fill 3.5 waves; 2048 x 2048 FP32 0.62 ms.
#pragma once
#include "kernels_gemm.cuh"

namespace cpde::ops {

// One of the three products' epilogues: `scale_d` D + `scale_in` (parts in), to parts
// or to the result's type, the new weights of an optimiser step where `weight` is given.
template <bool MIRROR, int IN, int OUT, class T>
struct OrthogonalEpilogue {
    const __half* in;       // IN parts a batch
    __half* out;            // OUT parts a batch
    T* final;               // OUT == 0: contiguous
    const T* weight;        // or null
    int64_t pitch, plane;   // of the parts: rows of whole 32 bytes
    int in_planes, out_planes;
    float scale_d, scale_in, keep, rate;
    bool whole;             // the result has rows of whole 32 bytes, or there are parts alone

    struct Fetched {
        Sixteen<__half> in[IN ? IN : 1];
        Sixteen<T> weight;
    };
    __device__ __forceinline__ void fetch(Fetched& f, int64_t row, int column, int batch, const GemmShape& s) const {
        if constexpr (IN > 0) {
            const __half* from = in + int64_t(batch) * in_planes * plane + row * pitch + column;
#pragma unroll
            for (int p = 0; p < IN; ++p) f.in[p].load(from + p * plane);
        }
        if constexpr (OUT == 0)
            if (weight) f.weight.load(weight + (int64_t(batch) * s.m + row) * s.n + column);
    }
    __device__ __forceinline__ void whole_row(float (&v)[16], const Fetched& f, int64_t row, int column, int batch, int, int bm, int bn,
                                         const GemmShape& s) const {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] *= scale_d;
        if constexpr (IN > 0) {
            float x[16], rest[16];
            f.in[0].get(x);
            if constexpr (IN > 1) {
                f.in[1].get(rest);
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] += rest[i];
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = fmaf(scale_in, x[i], v[i]);
        }
        if constexpr (OUT > 0) {
            __half* to = out + int64_t(batch) * out_planes * plane;
            // The tile on the other side of the diagonal, where none is computed. Pieces lie in one tile.
            const bool mirror = MIRROR && int(row) / bn * bn >= (column / bm + 1) * bm;
#pragma unroll
            for (int p = 0; p < OUT; ++p, to += plane) {
                __half h[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    h[i] = __float2half_rn(v[i]);
                    v[i] -= __half2float(h[i]);
                }
                Wide w;
                memcpy(&w, h, sizeof(w));
                store_wide(to + row * pitch + column, w);
                if (MIRROR && mirror) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) to[(column + i) * pitch + row] = h[i];
                }
            }
        } else {
            if (weight) {
                float w[16];
                f.weight.get(w);
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = fmaf(-rate, v[i], keep * w[i]);
            }
            Sixteen<T>::store(final + (int64_t(batch) * s.m + row) * s.n + column, v);
        }
    }
    __device__ __forceinline__ void odd(float (&v)[16], float (&)[16], int64_t row, int column, int left, int batch,
                                        const GemmShape& s) const {
        if constexpr (OUT == 0) {
            const __half* from = in + int64_t(batch) * in_planes * plane + row * pitch + column;
            float x[16], rest[16];
            Sixteen<__half> part;
            part.load(from);
            part.get(x);
            part.load(from + plane);
            part.get(rest);
            if (weight) {
                float w[16];
                load_some<T, 16>(weight + (int64_t(batch) * s.m + row) * s.n + column, w, left, false);
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = fmaf(-rate, fmaf(scale_in, x[i] + rest[i], scale_d * v[i]), keep * w[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = fmaf(scale_in, x[i] + rest[i], scale_d * v[i]);
            }
        }
    }
    __device__ __forceinline__ bool writes_z() const { return false; }
    template <int WHICH>
    __device__ __forceinline__ void write(float f, int64_t row, int column, int batch, const GemmShape& s) const {
        if constexpr (OUT == 0 && WHICH == 1) final[(int64_t(batch) * s.m + row) * s.n + column] = from_float<T>(f);
    }
};

// The matrices' values: given, or an optimiser step's update u from the gradient g and
// the momentum m, m' = beta m + (1 - beta) g and u = m' or beta m' + (1 - beta) g.
template <class T, class M>
struct UpdateCall {
    const T* x;
    const M* momentum;     // null: x itself
    M* new_momentum;
    float* update;         // u in FP32, for the second pass
    double* sums;          // (matrix, block) sums of squares
    int64_t rows;
    int32_t columns, lanes, blocks;
    float beta, rest;      // 1 - beta, rounded by itself: the difference of rounded numbers would be off by more
    bool nesterov, whole;
};

// Sums of squares in FP64, which no FP32 value overflows. The first of two passes over
// the matrices; bound by memory.
template <class T, class M>
__global__ void __launch_bounds__(256) k_update_norm(const UpdateCall<T, M> c) {
    __shared__ double shared[8];
    next_launch_may_begin();
    after_previous_launch();
    const int lane = threadIdx.x % c.lanes, high = 256 / c.lanes, wide = c.lanes * 8;
    const int64_t base = blockIdx.y * c.rows * c.columns;
    double sum = 0.0;
    for (int64_t row = blockIdx.x * int64_t(high) + threadIdx.x / c.lanes; row < c.rows; row += int64_t(gridDim.x) * high)
        for (int column = lane * 8; column < c.columns; column += wide) {
            const int64_t at = base + row * c.columns + column;
            const int left = c.columns - column;
            float v[8];
            auto some = [&](auto* p, float (&f)[8]) {
                using E = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
                if (c.whole) unpack<E, 8>(load_written<E, 8>(p), f);
                else
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = i < left ? to_float(p[i]) : 0.0f;
            };
            some(c.x + at, v);
            if (c.momentum) {
                float m[8];
                some(c.momentum + at, m);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float g = c.rest * v[i];
                    m[i] = fmaf(c.beta, m[i], g);
                    v[i] = c.nesterov ? fmaf(c.beta, m[i], g) : m[i];
                }
                if (c.whole) {
                    store<M, 8>(c.new_momentum + at, pack<M, 8>(m));
                    store<float, 8>(c.update + at, pack<float, 8>(v));
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i < left) c.new_momentum[at + i] = from_float<M>(m[i]), c.update[at + i] = v[i];
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fma(double(v[i]), double(v[i]), sum);
        }
    for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
    if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = sum;
    __syncthreads();
    if (threadIdx.x) return;
    for (int i = 1; i < 8; ++i) sum += shared[i];
    c.sums[blockIdx.y * c.blocks + blockIdx.x] = sum;
}

// Divides by norm + eps and splits into parts.
template <class V>
__global__ void __launch_bounds__(256)
    k_normalise(const V* x, const double* sums, __half* out, int64_t rows, int64_t pitch, int64_t plane, int32_t columns,
                int32_t lanes, int32_t blocks, float scale, double eps, bool whole) {
    __shared__ double shared[8];
    next_launch_may_begin();
    after_previous_launch();
    double sum = 0.0;
    for (int i = threadIdx.x; i < blocks; i += 256) sum += sums[blockIdx.y * blocks + i];
    for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
    if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = sum;
    __syncthreads();
    sum = 0.0;
    for (int i = 0; i < 8; ++i) sum += shared[i];
    const float by = float(scale / (sqrt(sum) + eps));
    const int lane = threadIdx.x % lanes, high = 256 / lanes, wide = lanes * 8;
    for (int64_t row = blockIdx.x * int64_t(high) + threadIdx.x / lanes; row < rows; row += int64_t(gridDim.x) * high)
        for (int column = lane * 8; column < columns; column += wide) {  // the padding behind is never read
            const V* p = x + (blockIdx.y * rows + row) * columns + column;
            float v[8], h[8];
            if (whole) unpack<V, 8>(load_written<V, 8>(p), v);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = column + i < columns ? to_float(p[i]) : 0.0f;
            __half* to = out + blockIdx.y * 2 * plane + row * pitch + column;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= by;
            const auto high_part = pack<__half, 8>(v);
            unpack<__half, 8>(high_part, h);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] -= h[i];
            store<__half, 8>(to, high_part);
            store<__half, 8>(to + plane, pack<__half, 8>(v));
        }
}

}  // namespace cpde::ops
