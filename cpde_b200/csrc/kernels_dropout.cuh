// Dropout from a counter-based generator: the mask is a function of (seed,
// offset, element index) and is computed again wherever it is needed.
#pragma once
#include "device_vector.cuh"

namespace cpde::ops {

// Philox4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", SC 2011): ten rounds of two 32x32-bit
// products over a 128-bit counter under a 64-bit key.
__device__ __forceinline__ uint4 philox(uint64_t index, uint64_t offset, uint64_t seed) {
    uint32_t c0 = uint32_t(index), c1 = uint32_t(index >> 32), c2 = uint32_t(offset), c3 = uint32_t(offset >> 32);
    uint32_t k0 = uint32_t(seed), k1 = uint32_t(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t a = uint64_t(c0) * 0xD2511F53u, b = uint64_t(c2) * 0xCD9E8D57u;
        c0 = uint32_t(b >> 32) ^ c1 ^ k0;
        c1 = uint32_t(b);
        c2 = uint32_t(a >> 32) ^ c3 ^ k1;
        c3 = uint32_t(a);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// Which elements stay. Element i takes 16 of the 128 bits of counter i / 8
// (word (i % 8) / 2, low half first) and stays when they are >= threshold =
// round(65536 rate). 16 bits an element halve the integer work of 32: at 32 the
// generator, not memory, would bound the 16-bit types. The rate is thereby a
// multiple of 1/65536, and `factor` is the exact inverse of that rate's keep
// probability, so expectations are kept.
struct DropoutRule {
    uint64_t seed, offset;
    uint32_t threshold;  // 0: nothing is dropped
    float factor;
};

// Elements V * j .. V * j + V - 1 of the eight that `bits` decides (V <= 8).
template <int V>
__device__ __forceinline__ void drop(float (&f)[V], const uint4& bits, uint32_t first, const DropoutRule& rule) {
    const uint32_t word[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
    for (int i = 0; i < V; ++i) {
        uint32_t w;
        if constexpr (V == 8) {
            w = word[i / 2];
        } else {
            const uint32_t at = (first + i) >> 1;
            w = at == 0 ? word[0] : at == 1 ? word[1] : at == 2 ? word[2] : word[3];
        }
        const uint32_t half = V == 1 ? ((first & 1) ? w >> 16 : w & 0xffffu) : (i & 1) ? w >> 16 : w & 0xffffu;
        f[i] = half >= rule.threshold ? f[i] * rule.factor : 0.0f;  // a dropped NaN or infinity is a zero
    }
}

// V elements from logical index `index`, a multiple of V (V divides 8).
template <int V>
__device__ __forceinline__ void drop_at(float (&f)[V], uint64_t index, const DropoutRule& rule) {
    drop<V>(f, philox(index >> 3, rule.offset, rule.seed), uint32_t(index & 7), rule);
}

struct DropoutShape {
    int64_t rows, columns, x_stride, residual_stride;
};

// y = residual + drop(x). One thread has the eight elements of a counter.
// VECTORS: 2 rows are contiguous and aligned, 1 rows of a multiple of eight
// columns at aligned strides, 0 anything.
template <class T, bool RESIDUAL, int VECTORS>
__global__ void __launch_bounds__(256) k_dropout(const T* __restrict__ x, const T* __restrict__ residual,
                                                  T* __restrict__ y, DropoutShape shape, int64_t count,
                                                  DropoutRule rule) {
    const int64_t group = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    const int64_t first = group * 8;
    if (first >= count) return;
    const bool random = rule.threshold != 0;
    uint4 bits = make_uint4(0, 0, 0, 0);
    if (VECTORS && first + 8 <= count) {
        int64_t at = first, rat = first;
        if (VECTORS == 1) {
            const int64_t row = first / shape.columns, column = first - row * shape.columns;
            at = row * shape.x_stride + column;
            rat = row * shape.residual_stride + column;
        }
        const auto vx = load<T, 8>(x + at);
        float f[8];
        unpack<T, 8>(vx, f);
        if (random) {
            bits = philox(uint64_t(group), rule.offset, rule.seed);
            drop<8>(f, bits, 0, rule);
        }
        if (RESIDUAL) {
            float r[8];
            unpack<T, 8>(load<T, 8>(residual + rat), r);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] += r[i];
        }
        store<T, 8>(y + first, pack<T, 8>(f));
        return;
    }
    if (random) bits = philox(uint64_t(group), rule.offset, rule.seed);
    for (int i = 0; i < 8 && first + i < count; ++i) {
        int64_t at = first + i, rat = at;
        if (VECTORS != 2) {
            const int64_t row = at / shape.columns, column = at - row * shape.columns;
            at = row * shape.x_stride + column;
            rat = row * shape.residual_stride + column;
        }
        float f[1] = {to_float(x[at])};
        if (random) drop<1>(f, bits, uint32_t(i), rule);
        if (RESIDUAL) f[0] += to_float(residual[rat]);
        y[first + i] = from_float<T>(f[0]);
    }
}

}  // namespace cpde::ops
