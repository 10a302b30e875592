// Orthogonalised matrices whose smaller side is at most 128 and larger at most 256, an
// optimiser step's with its momentum and weights: the whole of it in one launch, a CTA a
// matrix. The formulas and parts are those of kernels_orthogonal.cuh, two of everything; X (transposed
// where it is tall) and A stay in shared memory, in the layout that the MMAs read, and
// each product's epilogue writes over what the product has read: Q over A, the next X
// over X. Bound by the chain of 15 products of 128 x 128 and their epilogues, each of
// which has to wait for the one before: 4 x 128 x 128 FP32 in 39 us (of the 67,000 clocks
// 21,000 are MMAs, 26,000 epilogues, 9,000 loads and results; 88 us in 17 launches).
#pragma once
#include "kernels_orthogonal.cuh"

namespace cpde::ops {

constexpr int SMALL_SIDE = 128, SMALL_LENGTH = 256, SMALL_STEPS = 64, SMALL_THREADS = 512;
constexpr int SMALL_BLOCK = SMALL_SIDE * 128;  // bytes of 64 columns

// A step's factors: of D for A; of A and D for Q; of X and D for the next X.
struct SmallStep {
    float gram, poly_in, poly_d, x_in, x_d;
};

template <class T, class M>
struct SmallCall {
    const T* x;             // or the gradient
    const M* momentum;      // an optimiser step's, or null
    M* new_momentum;
    const T* weight;        // or null
    T* out;
    int32_t rows, columns;  // of the given matrix
    int32_t steps;
    float beta, rest, keep, rate, scale;  // scale: 2^s of the first X
    double eps;
    bool nesterov, whole;   // whole: rows of eights, at 16 bytes, in every array
    SmallStep step[SMALL_STEPS];
};

// One product into tensor memory, in two sums that the epilogue adds: the first and the
// second half of the contraction, SMALL_LENGTH columns apart. In each the small products
// of parts come first: sums are cut toward zero at their size, and what that does to the
// steps is seen in the result (of one matrix 1.2e-6 of its norm with one sum, 0.8e-6 with two;
// with two the updates of four layers of 128 x 128 come out at 1.7e-6, FP32 products at 2.9e-6).
template <bool B_ROWS>
__device__ __forceinline__ void small_product(uint32_t d, uint32_t a, uint32_t a_part, uint32_t b, uint32_t b_part, int n, int k) {
    const uint32_t instruction = 1u << 4 | uint32_t(B_ROWS) << 16 | uint32_t(n >> 3) << 17 | uint32_t(SMALL_SIDE >> 4) << 24;
    // MN-major blocks of 64 columns are SMALL_BLOCK apart.
    const uint64_t b_base = B_ROWS ? (gemm::descriptor<true>(0) & ~(uint64_t(0x3FFFu) << 16)) | uint64_t(SMALL_BLOCK >> 4) << 16
                                   : gemm::descriptor<false>(0);
    const int middle = (k / 16 + 1) / 2 * 16;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const uint32_t from_a = a + (i == 0 ? a_part : 0), from_b = b + (i == 1 ? b_part : 0);
        const uint64_t da = gemm::descriptor<false>(from_a), db = b_base | uint64_t((from_b >> 4) & 0x3FFFu);
#pragma unroll
        for (int at = 0; at < SMALL_LENGTH; at += 16) {
            if (at >= k) break;
            const uint32_t to_a = at / 64 * SMALL_BLOCK + at % 64 * 2, to_b = B_ROWS ? at * 128 : to_a;
            gemm::mma<1>(at < middle ? d : d + SMALL_LENGTH, da + (to_a >> 4), db + (to_b >> 4), instruction,
                         i > 0 || (at != 0 && at != middle));
        }
    }
}

// 32 columns of a warp's lanes: thread i gets lane i's.
__device__ __forceinline__ void tmem_piece(uint32_t at, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
    tc::tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
    tc::tmem_landed(v);
}

// Eight neighbouring columns of a row, in the swizzle.
__device__ __forceinline__ uint32_t small_at(int row, int column) {
    return column / 64 * SMALL_BLOCK + row * 128 + ((column % 64 / 8) ^ (row & 7)) * 16;
}
__device__ __forceinline__ void small_get(const uint8_t* base, uint32_t part, uint32_t at, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        Vector<__half, 8> h;
        h.word[0] = *reinterpret_cast<const uint4*>(base + p * part + at);
        float f[8];
        unpack<__half, 8>(h, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += f[i];
    }
}
__device__ __forceinline__ void small_put(uint8_t* base, uint32_t part, uint32_t at, float (&v)[8]) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const auto h = pack<__half, 8>(v);
        *reinterpret_cast<uint4*>(base + p * part + at) = h.word[0];
        float f[8];
        unpack<__half, 8>(h, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] -= f[i];
    }
}

template <class T, class M>
__global__ void __launch_bounds__(SMALL_THREADS, 1) k_orthogonal_small(const __grid_constant__ SmallCall<T, M> c, int* error) {
    extern __shared__ uint8_t raw_shared[];
    __shared__ double sums[SMALL_THREADS / 32];
    __shared__ uint64_t done;
    __shared__ uint32_t slot;
    __shared__ int abort_flag;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const bool tall = c.rows > c.columns;
    const int side = tall ? c.columns : c.rows, length = tall ? c.rows : c.columns;
    const int side16 = (side + 15) / 16 * 16, length16 = (length + 15) / 16 * 16;
    const int x_blocks = (length + 63) / 64, a_blocks = (side + 63) / 64;
    uint8_t* x_shared = raw_shared + (1024 - (tc::smem_u32(raw_shared) & 1023)) % 1024;
    const uint32_t x_part = x_blocks * SMALL_BLOCK, a_part = a_blocks * SMALL_BLOCK;
    uint8_t* a_shared = x_shared + 2 * x_part;
    volatile int* abort = &abort_flag;
    if (threadIdx.x == 0) {
        tc::mbar_init(&done, 1);
        tc::fence_barrier_init();
        *abort = 0;
    }
    __syncwarp();
    if (warp == 0) gemm::tmem_take<1>(&slot, 512);
    tc::tc_fence_before();
    // A block of the launch behind that took its tensor memory first would wait for this
    // one's end, and this one for the columns: nothing says that it may begin before they
    // are here.
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = slot;
    next_launch_may_begin();
    after_previous_launch();

    // COUNT values from `at` on, an optimiser step's updates and its new momentum.
    const int64_t base = int64_t(blockIdx.x) * c.rows * c.columns;
    auto values = [&](int64_t at, bool whole, auto& v, auto& m) {
        constexpr int COUNT = sizeof(v) / 4;
        load_some<T, COUNT>(c.x + base + at, v, COUNT, whole);
        if (!c.momentum) return;
        load_some<M, COUNT>(c.momentum + base + at, m, COUNT, whole);
#pragma unroll
        for (int j = 0; j < COUNT; ++j) {
            const float part = c.rest * v[j];
            m[j] = fmaf(c.beta, m[j], part);
            v[j] = c.nesterov ? fmaf(c.beta, m[j], part) : m[j];
        }
    };
    double sum = 0.0;
    const int all = c.rows * c.columns, eights = c.whole ? all / 8 : 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < eights; i += SMALL_THREADS) {
        float v[8], m[8];
        values(i * 8, true, v, m);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fma(double(v[j]), double(v[j]), sum);
    }
#pragma unroll 8
    for (int i = eights * 8 + threadIdx.x; i < all; i += SMALL_THREADS) {
        float v[1], m[1];
        values(i, false, v, m);
        sum = fma(double(v[0]), double(v[0]), sum);
    }
    // The rows and columns behind the matrix are zeros.
    for (uint32_t i = threadIdx.x * 16; i < 2 * x_part; i += SMALL_THREADS * 16)
        *reinterpret_cast<uint4*>(x_shared + i) = make_uint4(0, 0, 0, 0);
    for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    sum = 0.0;
    for (int i = 0; i < SMALL_THREADS / 32; ++i) sum += sums[i];
    const float by = float(c.scale / (sqrt(sum) + c.eps));
    const int chunks = (length + 7) / 8;
#pragma unroll 2
    for (int i = threadIdx.x; i < side * chunks; i += SMALL_THREADS) {
        // Neighbouring threads read neighbouring elements.
        const int row = tall ? i % side : i / chunks, column = (tall ? i / side : i % chunks) * 8;
        float v[8], m[8];
        if (c.whole && !tall) {
            const int64_t at = row * c.columns + column;
            values(at, true, v, m);
            if (c.momentum) store<M, 8>(c.new_momentum + base + at, pack<M, 8>(m));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = 0.0f;
                if (column + j >= length) continue;
                const int64_t at = tall ? (column + j) * c.columns + row : row * c.columns + column + j;
                float one[1], its[1];
                values(at, false, one, its);
                v[j] = one[0];
                if (c.momentum) c.new_momentum[base + at] = from_float<M>(its[0]);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= by;
        small_put(x_shared, x_part, small_at(row, column), v);
    }

    uint32_t parity = 0;
    // Waits until every thread has written its part, has a product computed and waits for that.
    auto run = [&](auto issue) {
        tc::fence_proxy_async();
        tc::tc_fence_before();
        __syncthreads();
        if (warp == 0) {
            tc::tc_fence_after();
            if (gemm::elected()) {
                issue();
                tc::mma_commit(&done);
            }
            __syncwarp();
        }
        const bool ok = gemm::wait_for(&done, parity, abort);
        parity ^= 1;
        tc::tc_fence_after();
        return __syncthreads_and(ok) != 0;
    };
    const int row = warp % 4 * 32 + lane, group = warp / 4;
    const uint32_t lanes = tmem + (uint32_t(warp % 4 * 32) << 16);
    const uint32_t x0 = tc::smem_u32(x_shared), a0 = tc::smem_u32(a_shared);
    // The product's pieces of 32 columns, in turn to the four warps of a row: f(column, eight of them).
    auto pieces = [&](int n, int k, auto f) {
        for (int column = group * 32; column < n; column += SMALL_THREADS / 4) {
            float v[32];
            __syncwarp();  // behind the branches of the piece before: the warp loads as one
            tmem_piece(lanes + column, v);
            if (k > 16) {  // the second half's sums
                float u[32];
                tmem_piece(lanes + SMALL_LENGTH + column, u);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] += u[i];
            }
#pragma unroll
            for (int i = 0; i < 32; i += 8)
                if (column + i < n) f(column + i, *reinterpret_cast<float(*)[8]>(v + i));
        }
    };
    bool ok = true;
    for (int k = 0; ok && k < c.steps; ++k) {
        const SmallStep s = c.step[k];
        if (!(ok = run([&] { small_product<false>(tmem, x0, x_part, x0, x_part, side16, length16); }))) break;
        pieces(side16, length16, [&](int column, float(&d)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] *= s.gram;
            small_put(a_shared, a_part, small_at(row, column), d);
        });
        if (!(ok = run([&] { small_product<false>(tmem, a0, a_part, a0, a_part, side16, side16); }))) break;
        pieces(side16, side16, [&](int column, float(&d)[8]) {
            const uint32_t at = small_at(row, column);
            float v[8];
            small_get(a_shared, a_part, at, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = fmaf(s.poly_in, v[i], s.poly_d * d[i]);
            small_put(a_shared, a_part, at, v);
        });
        if (!(ok = run([&] { small_product<true>(tmem, a0, a_part, x0, x_part, length16, side16); }))) break;
        const bool last = k + 1 == c.steps;
        pieces(length16, side16, [&](int column, float(&d)[8]) {
            const uint32_t at = small_at(row, column);
            float v[8];
            small_get(x_shared, x_part, at, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = fmaf(s.x_in, v[i], s.x_d * d[i]);
            if (!last) {
                small_put(x_shared, x_part, at, v);
            } else if (row < side && column < length) {
                float w[8];
                auto ended = [&](int i) { return c.weight ? fmaf(-c.rate, v[i], c.keep * w[i]) : v[i]; };
                if (c.whole && !tall) {
                    const int64_t to = base + row * c.columns + column;
                    if (c.weight) load_some<T, 8>(c.weight + to, w, 8, true);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = ended(i);
                    store<T, 8>(c.out + to, pack<T, 8>(v));
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (column + i >= length) continue;
                        const int64_t to = base + (tall ? (column + i) * c.columns + row : row * c.columns + column + i);
                        if (c.weight) w[i] = to_float(c.weight[to]);
                        c.out[to] = from_float<T>(ended(i));
                    }
                }
            }
        });
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc::tc_fence_after();
        gemm::tmem_release<1>(tmem, 512);
    }
    if (threadIdx.x == 0 && *abort) gemm::report(error);
}

}  // namespace cpde::ops
