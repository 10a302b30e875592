// Element types and short vectors of the device-tensor operators: a thread
// moves V neighbouring elements with as few and as wide accesses as their bytes
// allow and computes on them in FP32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace cpde::ops {

// Bytes of V elements as one or more machine words.
template <int BYTES> struct Words { using type = uint4; static constexpr int count = BYTES / 16; };
template <> struct Words<8> { using type = uint2; static constexpr int count = 1; };
template <> struct Words<4> { using type = uint32_t; static constexpr int count = 1; };
template <> struct Words<2> { using type = uint16_t; static constexpr int count = 1; };

template <class T, int V>
struct Vector {
    using W = Words<int(sizeof(T)) * V>;
    using Word = typename W::type;
    Word word[W::count];
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Inputs that the kernel never writes.
template <class T, int V>
__device__ __forceinline__ Vector<T, V> load(const T* p) {
    Vector<T, V> v;
    const auto* w = reinterpret_cast<const typename Vector<T, V>::Word*>(p);
#pragma unroll
    for (int i = 0; i < Vector<T, V>::W::count; ++i) v.word[i] = __ldg(w + i);
    return v;
}

template <class T, int V>
__device__ __forceinline__ void store(T* p, const Vector<T, V>& v) {
    auto* w = reinterpret_cast<typename Vector<T, V>::Word*>(p);
#pragma unroll
    for (int i = 0; i < Vector<T, V>::W::count; ++i) w[i] = v.word[i];
}

template <class T, int V>
__device__ __forceinline__ void unpack(const Vector<T, V>& v, float (&f)[V]) {
    T e[V];
    memcpy(e, &v, sizeof(e));
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_float(e[i]);
}

template <class T, int V>
__device__ __forceinline__ Vector<T, V> pack(const float (&f)[V]) {
    T e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_float<T>(f[i]);
    Vector<T, V> v;
    memcpy(&v, e, sizeof(v));
    return v;
}

template <class T, int V>
__device__ __forceinline__ Vector<T, V> zeros() {
    Vector<T, V> v;
    memset(&v, 0, sizeof(v));
    return v;
}

// Quotient of 31-bit integers by a divisor that is fixed for the launch
// (multiply-high with a precomputed reciprocal; exact for n < 2^31).
struct Divisor {
    uint32_t divisor, multiplier, shift;
    explicit Divisor(uint32_t d) : divisor(d), shift(0) {
        while ((uint64_t(1) << shift) < d) ++shift;
        multiplier = uint32_t((uint64_t(1) << 32) * ((uint64_t(1) << shift) - d) / d + 1);
    }
    __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
        return (__umulhi(n, multiplier) + n) >> shift;
    }
};

}  // namespace cpde::ops
