// Linear layers too small, or of too few points, for the tensor cores' long way from
// loads to epilogue: products on the FP32 units, from arrays of any type and layout, in
// one launch.
#pragma once
#include "kernels_linear.cuh"

namespace cpde::ops {

// --- few points ------------------------------------------------------------
//
// z = x W' for POINTS rows of x: the weights pass through the GPU once, which is all that
// bounds it. A warp takes OUTPUTS rows of W, each lane eight neighbouring inputs at a time,
// and holds a sum for each pair of a point and an output; x comes from L1. One point of
// 4096 x 4096 bf16: 9.5 us a call (3.5 TB/s), launch and host's way included.

template <int POINTS> constexpr int FEW_OUTPUTS = POINTS >= 4 ? 2 : 1;
constexpr int FEW_THREADS = 256;

// TURNED: x and W change places, for layers of at most 8 outputs (a field's head): then x is
// what passes through once.
template <class T, int POINTS, bool TURNED>
__global__ void __launch_bounds__(FEW_THREADS) k_few_points(const Source<T> x, const Source<T> w, LinearEpilogue<T> epilogue, GemmShape s) {
    constexpr int R = FEW_OUTPUTS<POINTS>;
    next_launch_may_begin();
    after_previous_launch();
    const int lane = threadIdx.x % 32;
    const int64_t output = (blockIdx.x * int64_t(FEW_THREADS / 32) + threadIdx.x / 32) * R;
    const int64_t points = x.rows, outputs = w.rows;
    if (output >= outputs) return;
    float sum[R][POINTS] = {};
    auto add = [&](const Vector<T, 8> (&a)[R], const Vector<T, 8>& b, int p) {
        float y[8];
        unpack<T, 8>(b, y);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float v[8];
            unpack<T, 8>(a[r], v);
            float eight = v[0] * y[0];  // by itself: the long sum has an eighth of the roundings then
#pragma unroll
            for (int j = 1; j < 8; ++j) eight = fmaf(v[j], y[j], eight);
            sum[r][p] += eight;
        }
    };
    int k = lane * 8;
    if (x.width == 8 && w.width == 8 && outputs % R == 0) {
        // DEEP rounds' weights are under way at a time.
        constexpr int DEEP = POINTS == 1 ? 8 : 4;
        for (; k + 256 * (DEEP - 1) + 8 <= x.columns; k += 256 * DEEP) {
            Vector<T, 8> a[DEEP][R];
#pragma unroll
            for (int i = 0; i < DEEP; ++i)
#pragma unroll
                for (int r = 0; r < R; ++r) a[i][r] = load_written<T, 8>(w.p + (output + r) * w.stride + k + 256 * i);
#pragma unroll
            for (int i = 0; i < DEEP; ++i)
#pragma unroll
                for (int p = 0; p < POINTS; ++p)
                    add(a[i], load_written<T, 8>(x.p + min(int64_t(p), points - 1) * x.stride + k + 256 * i), p);
        }
    }
    for (; k < x.columns; k += 256) {
        Vector<T, 8> a[R];
#pragma unroll
        for (int r = 0; r < R; ++r) a[r] = gemm::gather(w, output + r, k);
#pragma unroll
        for (int p = 0; p < POINTS; ++p) add(a, gemm::gather(x, p, k), p);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int p = 0; p < POINTS; ++p)
#pragma unroll
            for (int o = 16; o; o /= 2) sum[r][p] += __shfl_xor_sync(~0u, sum[r][p], o);
    // One lane ends one result.
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int p = 0; p < POINTS; ++p)
            if (lane == r * POINTS + p && p < points && output + r < outputs) {
                float v[1] = {sum[r][p]};
                if constexpr (TURNED) epilogue.template some<1>(v, output + r, p, s);
                else epilogue.template some<1>(v, p, int(output + r), s);
            }
}

// --- small products ----------------------------------------------------------
//
// A block computes 32 x 32 results, its eight warps an eighth of each slab of the
// contraction each, so that also a small result keeps a block's warps busy: a lane holds
// 4 x 8 of the warp's sums. The warps' sums are added in order. Two products go in one
// launch: a layer's two gradients, whose dz is computed from dy and z as it is read.
// 257 points of 48 x 128 FP32 take 5.8 us a call, the host's way; with parts and tensor
// cores 12.6. Gradients of 300 points of 100 x 77: 12.7, before 29.6.

template <class T>
struct SmallOperand {
    const T* p;
    const T* z;             // p times the activation's slope at z, or null
    int64_t row, k;         // strides
    int64_t z_row, z_k;
    int32_t activation;
};
template <class T>
struct SmallProduct {
    SmallOperand<T> a, b;
    LinearEpilogue<T> epilogue;
    void* sums;             // sums of A's rows, of T or FP32, or null
    bool sums_wide;
    int32_t m, n, tiles_n;
    int64_t k;
    int32_t tiles;
};

constexpr int SMALL_TILE = 32, SMALL_SLAB = 64, SMALL_PITCH = SMALL_TILE + 4, SMALL_WARPS = 8;

template <class T>
struct SmallChunk {
    T v[8], z[8];
    // The lanes run along whichever way is contiguous.
    __device__ __forceinline__ static int row_of(int i, bool along_k) {
        const int q = threadIdx.x + 256 * i;
        return along_k ? q / SMALL_SLAB : q % SMALL_TILE;
    }
    __device__ __forceinline__ static int k_of(int i, bool along_k) {
        const int q = threadIdx.x + 256 * i;
        return along_k ? q % SMALL_SLAB : q / SMALL_TILE;
    }
    __device__ __forceinline__ void load(const SmallOperand<T>& o, int64_t row0, int64_t rows, int64_t k0, int64_t k, bool along_k) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t r = row0 + row_of(i, along_k), c = k0 + k_of(i, along_k);
            const bool there = r < rows && c < k;
            v[i] = there ? o.p[r * o.row + c * o.k] : from_float<T>(0.0f);
            z[i] = there && o.z ? o.z[r * o.z_row + c * o.z_k] : from_float<T>(0.0f);
        }
    }
    // The slopes here, behind the loads: a branch between those would make them wait for each other.
    __device__ __forceinline__ void store(float* to, const SmallOperand<T>& o, bool along_k) const {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = to_float(v[i]);
        if (o.z) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] *= layer_slope<sizeof(T) == 4>(to_float(z[i]), o.activation);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) to[k_of(i, along_k) * SMALL_PITCH + row_of(i, along_k)] = f[i];
    }
};

template <class T>
__global__ void __launch_bounds__(32 * SMALL_WARPS) k_small_products(const SmallProduct<T> first, const SmallProduct<T> second) {
    __shared__ float shared[SMALL_WARPS * SMALL_TILE * SMALL_TILE];
    static_assert(2 * SMALL_SLAB * SMALL_PITCH <= SMALL_WARPS * SMALL_TILE * SMALL_TILE);
    next_launch_may_begin();
    after_previous_launch();
    const bool other = int(blockIdx.x) >= first.tiles;
    const SmallProduct<T>& c = other ? second : first;
    const int tile = int(blockIdx.x) - (other ? first.tiles : 0);
    const int64_t row0 = int64_t(tile / c.tiles_n) * SMALL_TILE, column0 = int64_t(tile % c.tiles_n) * SMALL_TILE;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int r0 = lane / 4 * 4, c0 = lane % 4 * 8;
    const bool a_along = c.a.k == 1, b_along = c.b.k == 1;
    float *as = shared, *bs = shared + SMALL_SLAB * SMALL_PITCH;
    float sum[4][8] = {}, row_sum = 0.0f;
    const bool row_sums = c.sums && column0 == 0;
    SmallChunk<T> a, b;
    a.load(c.a, row0, c.m, 0, c.k, a_along);
    b.load(c.b, column0, c.n, 0, c.k, b_along);
    for (int64_t k0 = 0; k0 < c.k; k0 += SMALL_SLAB) {
        __syncthreads();
        a.store(as, c.a, a_along);
        b.store(bs, c.b, b_along);
        __syncthreads();
        if (k0 + SMALL_SLAB < c.k) {
            a.load(c.a, row0, c.m, k0 + SMALL_SLAB, c.k, a_along);
            b.load(c.b, column0, c.n, k0 + SMALL_SLAB, c.k, b_along);
        }
#pragma unroll
        for (int i = 0; i < SMALL_SLAB / SMALL_WARPS; ++i) {
            const int k = i * SMALL_WARPS + warp;
            const float4 x = *reinterpret_cast<const float4*>(as + k * SMALL_PITCH + r0);
            const float4 y = *reinterpret_cast<const float4*>(bs + k * SMALL_PITCH + c0);
            const float4 z = *reinterpret_cast<const float4*>(bs + k * SMALL_PITCH + c0 + 4);
            const float av[4] = {x.x, x.y, x.z, x.w}, bv[8] = {y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[r][j] = fmaf(av[r], bv[j], sum[r][j]);
            if (row_sums) row_sum += as[k * SMALL_PITCH + lane];
        }
    }
    __syncthreads();
    if (row_sums) {
        shared[warp * SMALL_TILE + lane] = row_sum;
        __syncthreads();
        if (warp == 0 && row0 + lane < c.m) {
            for (int i = 1; i < SMALL_WARPS; ++i) row_sum += shared[i * SMALL_TILE + lane];
            if (c.sums_wide) static_cast<float*>(c.sums)[row0 + lane] = row_sum;
            else static_cast<T*>(c.sums)[row0 + lane] = from_float<T>(row_sum);
        }
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < 8; j += 4)
            *reinterpret_cast<float4*>(shared + (warp * SMALL_TILE + r0 + r) * SMALL_TILE + c0 + j) =
                make_float4(sum[r][j], sum[r][j + 1], sum[r][j + 2], sum[r][j + 3]);
    __syncthreads();
    const int row = threadIdx.x / 8, column = threadIdx.x % 8 * 4;
    float v[4] = {};
#pragma unroll
    for (int i = 0; i < SMALL_WARPS; ++i) {
        const float4 d = *reinterpret_cast<const float4*>(shared + (i * SMALL_TILE + row) * SMALL_TILE + column);
        v[0] += d.x, v[1] += d.y, v[2] += d.z, v[3] += d.w;
    }
    GemmShape s = {};
    s.m = c.m, s.n = c.n;
    if (row0 + row >= c.m || column0 + column >= c.n) return;
    if (c.epilogue.fours) {
        c.epilogue.template some<4>(v, row0 + row, int(column0) + column, s);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (column0 + column + j < c.n) {
                float one[1] = {v[j]};
                c.epilogue.template some<1>(one, row0 + row, int(column0) + column + j, s);
            }
    }
}

}  // namespace cpde::ops
