// Element types and short vectors of the device-tensor operators: a thread
// moves V neighbouring elements with as few and as wide accesses as their bytes
// allow and computes on them in FP32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <cstring>
#include <type_traits>

namespace cpde::ops {

// A kernel that is launched as dependent (launch_dependent in operators.cu) may
// begin before the launch ahead of it has ended: it waits here before it touches
// what that one wrote, or anything that an earlier launch may still use.
__device__ __forceinline__ void after_previous_launch() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets the launch behind begin once every block has said so.
__device__ __forceinline__ void next_launch_may_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

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

// Inputs that nothing writes while the kernel runs: the read-only path, and loads
// that a compiler may move freely.
template <class T, int V>
__device__ __forceinline__ Vector<T, V> load(const T* p) {
    Vector<T, V> v;
    const auto* w = reinterpret_cast<const typename Vector<T, V>::Word*>(p);
#pragma unroll
    for (int i = 0; i < Vector<T, V>::W::count; ++i) v.word[i] = __ldg(w + i);
    return v;
}

// What the launch ahead writes while this kernel may already be there: ordinary
// loads, which stay behind after_previous_launch(). For the same reason a pointer to
// such data is never __restrict__.
template <class T, int V>
__device__ __forceinline__ Vector<T, V> load_written(const T* p) {
    Vector<T, V> v;
    const auto* w = reinterpret_cast<const typename Vector<T, V>::Word*>(p);
#pragma unroll
    for (int i = 0; i < Vector<T, V>::W::count; ++i) v.word[i] = w[i];
    return v;
}

template <class T, int V>
__device__ __forceinline__ void store(T* p, const Vector<T, V>& v) {
    auto* w = reinterpret_cast<typename Vector<T, V>::Word*>(p);
#pragma unroll
    for (int i = 0; i < Vector<T, V>::W::count; ++i) w[i] = v.word[i];
}

// For what this kernel will not read again.
template <class T, int V>
__device__ __forceinline__ void store_streaming(T* p, const Vector<T, V>& v) {
    auto* w = reinterpret_cast<typename Vector<T, V>::Word*>(p);
#pragma unroll
    for (int i = 0; i < Vector<T, V>::W::count; ++i) __stcs(w + i, v.word[i]);
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

// V values as pairs for the packed FP32 instructions (two operations an issue
// slot); V = 1 leaves the second of its pair at zero.
template <int V>
struct Pairs {
    static constexpr int N = (V + 1) / 2;
    float2 p[N];
    __device__ __forceinline__ float get(int j) const { return j % 2 ? p[j / 2].y : p[j / 2].x; }
    __device__ __forceinline__ void set(int j, float v) { (j % 2 ? p[j / 2].y : p[j / 2].x) = v; }
    __device__ __forceinline__ void fill(float v) {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = make_float2(v, v);
    }
};
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

template <class T, int V>
__device__ __forceinline__ Pairs<V> unpack_pairs(const Vector<T, V>& v) {
    Pairs<V> f;
    if constexpr (V == 1) {
        float e[1];
        unpack<T, 1>(v, e);
        f.p[0] = make_float2(e[0], 0.0f);
    } else if constexpr (sizeof(T) == 4) {
        memcpy(&f, &v, sizeof(f));
    } else {
        uint32_t w[V / 2];
        memcpy(w, &v, sizeof(w));
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                f.p[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
            } else {
                __half2 h;
                memcpy(&h, &w[i], 4);
                f.p[i] = __half22float2(h);
            }
        }
    }
    return f;
}

template <class T, int V>
__device__ __forceinline__ Vector<T, V> pack_pairs(const Pairs<V>& f) {
    if constexpr (V == 1) {
        const float e[1] = {f.p[0].x};
        return pack<T, 1>(e);
    } else {
        Vector<T, V> v;
        if constexpr (sizeof(T) == 4) {
            memcpy(&v, &f, sizeof(v));
        } else {
            uint32_t w[V / 2];
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                    const __nv_bfloat162 h = __float22bfloat162_rn(f.p[i]);
                    memcpy(&w[i], &h, 4);
                } else {
                    const __half2 h = __float22half2_rn(f.p[i]);
                    memcpy(&w[i], &h, 4);
                }
            }
            memcpy(&v, w, sizeof(v));
        }
        return v;
    }
}

// `v`, or zero where rounding has made it negative. A NaN stays one: fmaxf would make
// it a zero too.
__device__ __forceinline__ float not_negative(float v) { return v < 0.0f ? 0.0f : v; }
__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }
// A value to take deviations from: one that is not finite would make a NaN of every
// mean, also where the definition gives an infinity.
__device__ __forceinline__ float finite_or_zero(float v) { return finite(v) ? v : 0.0f; }

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
