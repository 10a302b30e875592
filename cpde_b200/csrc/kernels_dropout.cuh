// Dropout from a counter-based generator: the mask is a function of (seed,
// offset, element index) and is computed again wherever it is needed.
#pragma once
#include "device_vector.cuh"

namespace cpde::ops {

// Which elements stay. Element i takes 16 of the 128 bits of counter i / 8
// (word (i % 8) / 2, low half first) and stays when they are >= threshold =
// round(65536 rate). 16 bits an element halve the integer work of 32: at 32 the
// generator, not memory, would bound the 16-bit types. The rate is thereby a
// multiple of 1/65536, and `factor` is the exact inverse of that rate's keep
// probability, so expectations are kept.
struct DropoutRule {
    uint64_t offset;
    uint32_t key[20];    // the rounds' keys, from the seed: constants of the launch
    uint32_t threshold;  // 0: nothing is dropped
    float factor;
};

// Philox4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", SC 2011): ten rounds of two 32x32-bit
// products over a 128-bit counter under a 64-bit key.
inline DropoutRule keyed_rule(uint32_t threshold, float factor, uint64_t seed, uint64_t offset) {
    DropoutRule rule = {offset, {}, threshold, factor};
    uint32_t k0 = uint32_t(seed), k1 = uint32_t(seed >> 32);
    for (int round = 0; round < 10; ++round) {
        rule.key[2 * round] = k0;
        rule.key[2 * round + 1] = k1;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return rule;
}
__device__ __forceinline__ uint4 philox(uint64_t index, const DropoutRule& rule) {
    uint32_t c0 = uint32_t(index), c1 = uint32_t(index >> 32);
    uint32_t c2 = uint32_t(rule.offset), c3 = uint32_t(rule.offset >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t a = uint64_t(c0) * 0xD2511F53u, b = uint64_t(c2) * 0xCD9E8D57u;
        c0 = uint32_t(b >> 32) ^ c1 ^ rule.key[2 * round];
        c1 = uint32_t(b);
        c2 = uint32_t(a >> 32) ^ c3 ^ rule.key[2 * round + 1];
        c3 = uint32_t(a);
    }
    return make_uint4(c0, c1, c2, c3);
}

// Zeros in the places of V elements that are dropped (a NaN or an infinity
// there too); the others are left for the caller to scale. `index`, a multiple
// of V, is the first one's; `bits` are its counter's.
template <int V>
__device__ __forceinline__ void drop(Pairs<V>& f, const uint4& bits, uint32_t index, const DropoutRule& rule) {
    static_assert(V == 8 || V == 4 || V == 1);
    if constexpr (V == 1) {
        const uint32_t at = index & 7;
        const uint32_t word = at < 4 ? (at < 2 ? bits.x : bits.y) : (at < 6 ? bits.z : bits.w);
        const uint32_t half = at & 1 ? word >> 16 : word & 0xffffu;
        if (half < rule.threshold) f.p[0].x = 0.0f;
    } else {
        const bool back = V == 4 && (index & 4);
        const uint32_t word[4] = {back ? bits.z : bits.x, back ? bits.w : bits.y, bits.z, bits.w};
        // A half is below the threshold where it, in the upper half of a word, is no more
        // than the largest word below threshold << 16. (One instruction compares both
        // halves and has two predicates as results; but with f16 values behind it the
        // compiler lost one of the two, depending on how it placed registers, and dropped
        // elements' neighbours became NaN.)
        const uint32_t last = (rule.threshold << 16) - 1;
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            if (word[i] << 16 <= last) f.p[i].x = 0.0f;
            if (word[i] <= last) f.p[i].y = 0.0f;
        }
    }
}
template <int V>
__device__ __forceinline__ void drop_at(Pairs<V>& f, uint64_t index, const DropoutRule& rule) {
    drop<V>(f, philox(index >> 3, rule), uint32_t(index), rule);
}
template <int V>
__device__ __forceinline__ void scale(Pairs<V>& f, float by) {
#pragma unroll
    for (int i = 0; i < Pairs<V>::N; ++i) f.p[i] = __fmul2_rn(f.p[i], both(by));
}

struct DropoutShape {
    int64_t rows, columns, x_stride, residual_stride;
};

// y = residual + drop(x). One thread has the eight elements of a counter. Bound by
// memory: 67M bf16 with a residual (403 MB) take 61 to 63 us, 6.4 to 6.6 TB/s;
// with the keys in registers 74.
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
        Vector<T, 8> vr;
        if (RESIDUAL) vr = load<T, 8>(residual + rat);
        if (random) bits = philox(uint64_t(group), rule);
        Pairs<8> f = unpack_pairs<T, 8>(vx);
        if (random) drop<8>(f, bits, 0, rule);
        // Rounded before the residual is added, so that the sum does not depend
        // on whether a compiler joins the two operations.
#pragma unroll
        for (int j = 0; j < 8; ++j) f.set(j, __fmul_rn(f.get(j), rule.factor));
        if (RESIDUAL) {
            const Pairs<8> r = unpack_pairs<T, 8>(vr);
#pragma unroll
            for (int i = 0; i < 4; ++i) f.p[i] = __fadd2_rn(f.p[i], r.p[i]);
        }
        store<T, 8>(y + first, pack_pairs<T, 8>(f));
        return;
    }
    if (random) bits = philox(uint64_t(group), rule);
    for (int i = 0; i < 8 && first + i < count; ++i) {
        int64_t at = first + i, rat = at;
        if (VECTORS != 2) {
            const int64_t row = at / shape.columns, column = at - row * shape.columns;
            at = row * shape.x_stride + column;
            rat = row * shape.residual_stride + column;
        }
        Pairs<1> f = {{make_float2(to_float(x[at]), 0.0f)}};
        if (random) drop<1>(f, bits, uint32_t(i), rule);
        const float kept = __fmul_rn(f.p[0].x, rule.factor);
        y[first + i] = from_float<T>(RESIDUAL ? __fadd_rn(kept, to_float(residual[rat])) : kept);
    }
}

}  // namespace cpde::ops
