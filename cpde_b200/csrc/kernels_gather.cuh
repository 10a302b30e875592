// Products of FP32 arrays as in kernels_gemm.cuh, without parts in memory: warps of loads
// read A, split it and write the parts into shared memory themselves, in the layout that
// TMA would give, and B's parts stay there. For layers of at most 128 inputs and outputs
// at many points, which are bound by how often x goes through memory: 65,536 points of
// 128 x 128 with tanh take 40 us (two passes at the copy rate 10), 51 with parts.
// What is left is the way of a tile from load to epilogue at 3.5 tiles a CTA (the
// conversion is six operations an element, the tensor core is busy for a sixth of the time).
#pragma once
#include "kernels_gemm.cuh"

namespace cpde::ops {

template <class T>
struct Source {
    const T* p;
    int64_t stride, rows;
    int32_t columns;
    int32_t width;  // elements that are read at a time: 8, 4, 2 or 1, by the rows' alignment
};

// T's parts: FP32 as three BF16, what each leaves going to the next (24 bits, all
// exponents); the 16-bit types as they are.
template <class T> struct Parts { using type = T; static constexpr int count = 1; };
template <> struct Parts<float> { using type = __nv_bfloat16; static constexpr int count = 3; };

// The part of v, and in v the rest. A value that rounds to infinity is cut to the
// largest finite one, and an infinity's rest is nothing.
__device__ __forceinline__ float next_part(float& v) {
    float h = __bfloat162float(__float2bfloat16_rn(v));
    if (!finite(h) && finite(v)) h = copysignf(__uint_as_float(0x7f7f0000u), v);
    v = finite(h) ? v - h : 0.0f;
    return h;
}

// Eight values' parts. Pairs go through the packed conversion, about six operations an
// element; values that may round to infinity, and those that are not finite, one by one.
template <class T>
__device__ __forceinline__ void split_eight(float (&v)[8], uint4 (&part)[Parts<T>::count]) {
    using O = typename Parts<T>::type;
    if constexpr (Parts<T>::count == 1) {
        part[0] = pack<O, 8>(v).word[0];
    } else {
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
        uint32_t w[Parts<T>::count][4];
        if (most < 0x7f7f0000u) {
#pragma unroll
            for (int p = 0; p < Parts<T>::count; ++p)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __nv_bfloat162 h = __float22bfloat162_rn(make_float2(v[2 * j], v[2 * j + 1]));
                    memcpy(&w[p][j], &h, 4);
                    if (p + 1 < Parts<T>::count) {
                        v[2 * j] -= __uint_as_float(w[p][j] << 16);
                        v[2 * j + 1] -= __uint_as_float(w[p][j] & 0xffff0000u);
                    }
                }
        } else {
#pragma unroll
            for (int p = 0; p < Parts<T>::count; ++p)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float low = next_part(v[2 * j]), high = next_part(v[2 * j + 1]);
                    w[p][j] = __float_as_uint(low) >> 16 | (__float_as_uint(high) & 0xffff0000u);
                }
        }
#pragma unroll
        for (int p = 0; p < Parts<T>::count; ++p) memcpy(&part[p], w[p], 16);
    }
}

constexpr int GATHER_WARPS = 8, GATHER_CHUNKS = 1024 / (32 * GATHER_WARPS);

namespace gemm {

template <class T>
__device__ __forceinline__ Vector<T, 8> gather(const Source<T>& s, int64_t row, int column) {
    if (row >= s.rows || column >= s.columns) return zeros<T, 8>();
    const T* p = s.p + row * s.stride + column;
    if (column + 8 <= s.columns) {
        Vector<T, 8> v;
        if (s.width == 8) {
            if constexpr (sizeof(T) == 4) {
                const Wide w = load_wide(p);
                memcpy(&v, &w, sizeof(v));
                return v;
            } else {
                return load_written<T, 8>(p);
            }
        }
        if (s.width == 4) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const auto part = load_written<T, 4>(p + 4 * i);
                memcpy(reinterpret_cast<T*>(&v) + 4 * i, &part, sizeof(part));
            }
            return v;
        }
        if (s.width == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const auto part = load_written<T, 2>(p + 2 * i);
                memcpy(reinterpret_cast<T*>(&v) + 2 * i, &part, sizeof(part));
            }
            return v;
        }
    }
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = column + i < s.columns ? p[i] : from_float<T>(0.0f);
    Vector<T, 8> v;
    memcpy(&v, e, sizeof(v));
    return v;
}

// An operand's 128 x 64 of a slab as 1024 chunks of eight, shared by the threads. Neighbouring
// threads read neighbouring chunks of a row and write different banks.
template <class T, bool ROWS>
struct Chunks {
    Vector<T, 8> raw[GATHER_CHUNKS];
    __device__ __forceinline__ void load(const Source<T>& s, int64_t at, int64_t k, int thread) {
#pragma unroll
        for (int i = 0; i < GATHER_CHUNKS; ++i) {
            const int q = thread + 32 * GATHER_WARPS * i;
            if constexpr (ROWS) raw[i] = gather(s, k + q % 512 / 8, int(at) + q / 512 * 64 + q % 8 * 8);
            else raw[i] = gather(s, at + q / 8, int(k) + q % 8 * 8);
        }
    }
    // To part p's place at to[p].
    __device__ __forceinline__ void store(uint8_t* const (&to)[Parts<T>::count], int thread) const {
#pragma unroll
        for (int i = 0; i < GATHER_CHUNKS; ++i) {
            const int q = thread + 32 * GATHER_WARPS * i, row = ROWS ? q % 512 / 8 : q / 8;
            const int at = (ROWS ? q / 512 * 8192 : 0) + row * 128 + ((q ^ row) & 7) * 16;
            float v[8];
            uint4 part[Parts<T>::count];
            unpack<T, 8>(raw[i], v);
            split_eight<T>(v, part);
#pragma unroll
            for (int p = 0; p < Parts<T>::count; ++p) *reinterpret_cast<uint4*>(to[p] + at) = part[p];
        }
    }
};

// The work's slabs one after the other.
template <class C>
struct Walk {
    const GemmShape& s;
    int at, items, stride, slab;
    Work w;
    __device__ Walk(const GemmShape& shape, int first, int step, int count) : s(shape), at(first), items(count), stride(step) {
        if (there()) w = work_at<C>(s, at), slab = w.from;
    }
    __device__ bool there() const { return at < items; }
    __device__ void next() {
        if (++slab < w.to) return;
        at += stride;
        if (there()) w = work_at<C>(s, at), slab = w.from;
    }
};

}  // namespace gemm

template <class C>
constexpr int GATHER_THREADS = 32 * (GATHER_WARPS + 1 + C::WARPS);

template <class C, class T, class E>
__global__ void __launch_bounds__(GATHER_THREADS<C>, 1)
    k_gather(const Source<T> a, const Source<T> b, const GemmShape s, const E epilogue, int* error) {
    using namespace gemm;
    static_assert(C::CTAS == 1 && C::BN == 128 && C::P == Parts<T>::count && C::P > 1 && C::RESIDENT && !C::A_ROWS);
    extern __shared__ uint8_t raw_shared[];
    const Shared<C> sh(raw_shared);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int first = blockIdx.x, stride = gridDim.x;
    const int items = s.tiles * s.splits;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; ++i) tc::mbar_init(sh.full + i, GATHER_WARPS), tc::mbar_init(sh.empty + i, 1);
        for (int i = 0; i < 2; ++i) tc::mbar_init(sh.ready + i, 1), tc::mbar_init(sh.taken + i, C::WARPS);
        tc::mbar_init(sh.held, GATHER_WARPS);
        *sh.abort = 0;
        tc::fence_barrier_init();
    }
    if (warp == GATHER_WARPS) tmem_take<1>(sh.slot, C::TMEM);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *sh.slot;
    next_launch_may_begin();
    after_previous_launch();

    if (warp < GATHER_WARPS) {
        Chunks<T, false> ra;
        Chunks<T, C::B_ROWS> rb;
        Walk<C> walk(s, first, stride, items);
        // The rows of the tile after the next are brought into L2: what is under way into the
        // registers covers the latency of L2, not that of memory. (Tiles follow each other down A.)
        auto ahead = [&](int64_t row) {
            row += threadIdx.x;
            const uint32_t bytes = uint32_t(a.columns * sizeof(T)) / 16 * 16;
            if (a.width < 8 || threadIdx.x >= GEMM_ROWS || row >= a.rows || !bytes) return;
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a.p + row * a.stride), "r"(bytes) : "memory");
        };
        // A slab into registers, one ahead; false behind the last.
        auto load = [&] {
            if (!walk.there()) return false;
            if (walk.slab == walk.w.from) ahead(int64_t(walk.w.tile_m + 2 * stride) * C::BM);
            ra.load(a, int64_t(walk.w.tile_m) * C::BM, int64_t(walk.slab) * GEMM_SLAB, threadIdx.x);
            walk.next();
            return true;
        };
        bool there = load();
        for (int slab = 0; slab < s.slabs; ++slab) {
            uint8_t* to[C::P];
#pragma unroll
            for (int p = 0; p < C::P; ++p) to[p] = sh.stages + C::STAGES * C::STAGE + (slab * C::P + p) * C::B_BYTES;
            rb.load(b, 0, int64_t(slab) * GEMM_SLAB, threadIdx.x);
            rb.store(to, threadIdx.x);
        }
        // What this thread has written is there for the MMAs.
        tc::fence_proxy_async();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(sh.held);
        int st = 0;
        uint32_t parity = 1;
        while (there) {
            // The slab's stages, the last part's first.
            uint8_t* to[C::P];
            uint64_t* bar[C::P];
            bool ok = true;
#pragma unroll
            for (int p = C::P - 1; p >= 0; --p) {
                ok = ok && (lane || wait_for(sh.empty + st, parity, sh.abort));
                to[p] = sh.stages + st * C::STAGE, bar[p] = sh.full + st;
                if (++st == C::STAGES) st = 0, parity ^= 1;
            }
            if (!__all_sync(~0u, ok)) break;
            ra.store(to, threadIdx.x);
            there = load();
            tc::fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
#pragma unroll
                for (int p = 0; p < C::P; ++p) tc::mbar_arrive(bar[p]);
            }
        }
        // No commit may be under way to the stages' barriers when the CTA ends.
        if (threadIdx.x == 0)
            for (int i = 0; i < C::STAGES && wait_for(sh.empty + st, parity, sh.abort); ++i)
                if (++st == C::STAGES) st = 0, parity ^= 1;
    } else if (warp == GATHER_WARPS) {
        if (elected()) issue<C>(sh, s, tmem, first, stride, items);
    } else {
        finish<C>(sh, s, epilogue, tmem, warp - GATHER_WARPS - 1, warp % 4, 0, first, stride, items);
    }
    tc::tc_fence_before();
    __syncwarp();
    __syncthreads();
    if (warp == GATHER_WARPS) {
        tc::tc_fence_after();
        tmem_release<1>(tmem, C::TMEM);
    }
    if (threadIdx.x == 0 && *sh.abort) gemm::report(error);
}

}  // namespace cpde::ops
