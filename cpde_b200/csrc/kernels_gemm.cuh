// Matrix products of 16-bit operands on the tensor cores, D = A B' with FP32
// accumulators in tensor memory; what becomes of D is an epilogue's.
//
// An operand is an array of rows of 64-element slabs that TMA brings into shared
// memory in the 128-byte swizzle. The contraction runs along a row (K-major) or
// over the rows (MN-major): the bytes in shared memory are the same, only the
// descriptors differ, so that no operand is ever transposed.
//
// An operand of P > 1 parts is the sum of P arrays of 16-bit numbers, each part
// the rest that the parts before leave: two FP16 parts hold 22 bits, three BF16
// parts the 24 of FP32 with its exponents. Of the products of parts those are
// taken that are not below the last part's own rounding: 3 for two parts, 6 for
// three, the small ones first. The tensor core rounds its sums toward zero, which
// adds up over a long contraction: 262,144 terms of one sign fall short by 1.5e-3, 6e-9 a
// term. The accumulator is therefore taken out after a unit of slabs, and units are added
// in registers, rounded to nearest. With P > 1 a unit is a slab or two, which over 65,536
// terms leaves the error of an FP32 sum. With one part it is 2048 terms: that sum is then
// within 1.2e-5 however long it is, for 1% to 2% of the time. (1024 terms: 5e-6 and 4%;
// 4096: 2.4e-5 and the time of 2048. Short contractions keep the kernel without units: the
// other one takes 6% more there, for the registers.)
//
// A tile of 128 x BN of one CTA, or 256 x BN of a cluster of two whose CTAs hold
// half of each operand (cta_group::2), by three roles that are up to two accumulators
// ahead of each other: a thread that issues the loads, one that issues the MMAs, and
// warps that take the accumulators out. CTAs go through the tiles in strides. The tile of
// 256 x 256 has the tensor core's rate: a slab takes 518 clocks where its MMAs take 512.
// 32,768 points of 2048 x 2048 bf16: 185 us (1.49 PFLOP/s; the library's product takes
// 183), with bias and SiLU 188, with a residual and the sums kept 223. 8192 x 8192 x 8192:
// 710 us (678), bound by what L2 brings (47 bytes a clock an SM). Six products of FP32's
// parts: 2048 x 2048 x 2048 in 88 us (195 TFLOP/s, 1.2 PFLOP/s of BF16).
// Every wait is bounded: a role that gives up raises the CTA's abort flag, the
// loads in flight are waited for, tensor memory is released and `error` is set.
#pragma once
#include "device_vector.cuh"
#include "tc.cuh"

namespace cpde::ops {

constexpr int GEMM_ROWS = 128;   // rows of a CTA's tile: the lanes of tensor memory
constexpr int GEMM_SLAB = 64;    // elements of a slab: 128 bytes, one swizzled row
constexpr int GEMM_LONG = 32;    // slabs of one part that an accumulator sums at most
constexpr int GEMM_PIECE = 16;   // columns that an epilogue warp handles at a time
constexpr int GEMM_STRIDE = 17;  // floats between rows of 16 columns in shared memory: no bank conflicts
constexpr long long GEMM_WAIT = 2000000000LL;  // clocks, about a second

struct GemmShape {
    int m, n;                        // rows and columns of the result
    int slabs, splits, split_slabs;  // slabs of the contraction, and how they are split
    int array_slabs;                 // of which an array of A has so many: a contraction of one part goes on in the next
    int tiles_m, tiles_n, tiles, batches;
    int a_planes, b_planes;          // arrays of an operand a batch (of which P are read)
    uint32_t stage_bytes;            // what a stage's loads bring, of all CTAs of the cluster
    uint32_t instruction;            // the MMA's descriptor
    bool lower;                      // only tiles that reach the diagonal or below
};

// What a CTA holds. A_ROWS and B_ROWS: the contraction runs over the rows of the operand's array.
// RESIDENT: the whole of B stays in shared memory, HELD parts of slabs at most.
template <int CTAS_, int BN_, int P_, bool A_ROWS_, bool B_ROWS_, bool RESIDENT_ = false, bool LONG_ = false>
struct GemmTile {
    static constexpr int CTAS = CTAS_, BN = BN_, P = P_;
    static constexpr bool A_ROWS = A_ROWS_, B_ROWS = B_ROWS_, RESIDENT = RESIDENT_, LONG = LONG_;
    static constexpr int BM = GEMM_ROWS * CTAS;
    static constexpr int B_PART = BN / CTAS;  // columns of the tile whose operand this CTA loads
    static constexpr int A_BYTES = GEMM_ROWS * 128, B_BYTES = B_PART * 128;
    static constexpr int HELD = RESIDENT ? 6 : 0;
    static constexpr int STAGE = A_BYTES + (RESIDENT ? 0 : B_BYTES);  // one part of a slab of both operands
    // Of the epilogue. Its loads, conversions and stores are long chains, of which a
    // scheduler needs two warps' at least: four warps took twice the time.
    static constexpr int WARPS = 8;
    // Slabs that are summed in the accumulator before it is taken out. The way from the
    // last MMA to the epilogue and back takes 1.4 us a slab with two CTAs of 256 columns:
    // less than the six products of three parts (1.7), more than the three of two (0.83).
    // A resident B's few slabs are one unit, whose large products come last, and so is a
    // contraction of one part, unless it is LONG.
    static constexpr bool WHOLE = (P == 1 && !LONG) || RESIDENT;
    static constexpr int UNIT = WHOLE ? 1 << 30 : P == 1 ? GEMM_LONG : P == 2 ? 2 : 1;
    static constexpr int COLUMNS = BN / (WARPS / 4);  // of an epilogue warp
    static constexpr int THREADS = 64 + 32 * WARPS;
    static constexpr int PIECES = WARPS * 32 * GEMM_STRIDE * 4;
    static constexpr int ROOM = (227 * 1024 - 1024 - 256 - PIECES - HELD * B_BYTES) / STAGE;
    static constexpr int STAGES = ROOM > 12 ? 12 : ROOM;
    static constexpr int SHARED = 1024 + STAGES * STAGE + HELD * B_BYTES + PIECES + 256;
    static constexpr uint32_t TMEM = BN * 2 <= 32 ? 32 : BN * 2 <= 64 ? 64 : BN * 2 <= 128 ? 128 : BN * 2 <= 256 ? 256 : 512;
    static_assert(STAGES > P && BN * 2 <= 512 && BN % 32 == 0 && COLUMNS % GEMM_PIECE == 0);
    static_assert(!B_ROWS || B_PART % 64 == 0, "boxes of rows are 64 columns wide");
};

namespace gemm {

// As tc::mbar_wait_or_abort, without a clock where there is nothing to wait for.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort) {
    return tc::mbar_try_wait(bar, parity) || tc::mbar_wait_or_abort(bar, parity, GEMM_WAIT, abort);
}

// Says on the host's word that a wait ran out.
__device__ __forceinline__ void report(int* error) {
    *const_cast<volatile int*>(error) = 3;
    __threadfence_system();
}

// One thread of the warp. The loads and MMAs take their operands from registers of the
// whole warp: a thread that the compiler knows to be the only one issues them directly.
__device__ __forceinline__ bool elected() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of `p` in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t at_rank(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(tc::smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ void arrive_at(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// A box into this CTA's memory; its bytes count at `bar`, for two CTAs that of the first.
template <int CTAS>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    if constexpr (CTAS == 2)
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], "
                     "[%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y),
                     "r"(z)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], "
                     "[%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y),
                     "r"(z)
                     : "memory");
}

template <int CTAS>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, bool accumulate) {
    if constexpr (CTAS == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                     "r"(instruction), "r"(uint32_t(accumulate))
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                     "r"(instruction), "r"(uint32_t(accumulate))
                     : "memory");
}
// Arrives at `bar`, in every CTA of the cluster, when this thread's MMAs have ended.
template <int CTAS>
__device__ __forceinline__ void commit(uint64_t* bar) {
    if constexpr (CTAS == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                         tc::smem_u32(bar)),
                     "h"(uint16_t(3))
                     : "memory");
    else
        tc::mma_commit(bar);
}
template <int CTAS>
__device__ __forceinline__ void tmem_take(uint32_t* slot, uint32_t columns) {
    if constexpr (CTAS == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(slot)), "r"(columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        tc::tmem_alloc(slot, columns);
        tc::tmem_relinquish();
    }
}
template <int CTAS>
__device__ __forceinline__ void tmem_release(uint32_t base, uint32_t columns) {
    if constexpr (CTAS == 2)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
    else
        tc::tmem_dealloc(base, columns);
}

// Descriptors of a tile in shared memory, 128-byte swizzle, 8-row groups 1024 bytes
// apart. K-major: the groups follow each other along M or N. MN-major: they follow
// each other along K, and blocks of 64 along M or N are 64 rows apart.
template <bool ROWS>
__device__ __forceinline__ uint64_t descriptor(uint32_t at) {
    return uint64_t((at >> 4) & 0x3FFFu) | uint64_t(ROWS ? 8192u >> 4 : 1u) << 16 | uint64_t(1024u >> 4) << 32 |
           uint64_t(1u) << 46 | uint64_t(2u) << 61;
}
// Bytes from one MMA's 16 elements of the contraction to the next one's.
template <bool ROWS> constexpr uint32_t STEP = ROWS ? 16 * 128 : 32;

struct Work {
    int tile_m, tile_n, split, batch, from, to;  // and its slabs
};
// Work items in an order that keeps the operands of neighbours in L2: bands of 8
// tiles high, batch after batch and split after split.
template <class C>
__device__ __forceinline__ Work work_at(const GemmShape& s, int at) {
    Work w;
    const int each = s.tiles * s.splits;
    w.batch = at / each;
    const int rest = at % each, tile = rest % s.tiles;
    w.split = rest / s.tiles;
    if (s.lower) {
        constexpr int RATIO = C::BM / C::BN;  // tiles of a band up to the diagonal, a band
        int left = tile, m = 0, wide;
        while (left >= (wide = min(s.tiles_n, RATIO * (m + 1)))) left -= wide, ++m;
        w.tile_m = m, w.tile_n = left;
    } else {
        const int band = tile / (8 * s.tiles_n), high = min(8, s.tiles_m - 8 * band), in = tile - band * 8 * s.tiles_n;
        w.tile_m = 8 * band + in % high, w.tile_n = in / high;
    }
    w.from = w.split * s.split_slabs;
    w.to = min(s.slabs, w.from + s.split_slabs);
    return w;
}

template <class C>
struct Shared {
    uint8_t* stages;
    float* pieces;
    uint64_t *full, *empty, *ready, *taken, *held;  // of the stages; of the two accumulators; of a resident B
    volatile int* abort;
    uint32_t* slot;
    __device__ explicit Shared(uint8_t* raw) {
        stages = raw + (1024 - (tc::smem_u32(raw) & 1023)) % 1024;
        uint8_t* behind = stages + C::STAGES * C::STAGE + C::HELD * C::B_BYTES;
        pieces = reinterpret_cast<float*>(behind);
        full = reinterpret_cast<uint64_t*>(behind + C::PIECES);
        empty = full + 12, ready = empty + 12, taken = ready + 2;
        held = taken + 2;
        slot = reinterpret_cast<uint32_t*>(held + 1);
        abort = reinterpret_cast<volatile int*>(slot + 1);
    }
};

}  // namespace gemm

// Products of parts: all but those below the last part's own rounding.
template <int P> constexpr int PRODUCTS = P * (P + 1) / 2;

// Up to V elements of a row that has `left` of them from here on.
template <class T, int V>
__device__ __forceinline__ void load_some(const T* p, float (&f)[V], int64_t left, bool whole) {
    if (whole) {
        unpack<T, V>(load_written<T, V>(p), f);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = i < left ? to_float(p[i]) : 0.0f;
    }
}
// 32 bytes that one thread moves, 32-byte aligned: whole sectors, also where every
// thread of a warp is in a row of its own.
struct Wide {
    uint32_t w[8];
};
__device__ __forceinline__ Wide load_wide(const void* p) {
    Wide v;
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
                 : "l"(p));
    return v;
}
__device__ __forceinline__ void store_wide(void* p, const Wide& v) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v.w[0]), "r"(v.w[1]), "r"(v.w[2]),
                 "r"(v.w[3]), "r"(v.w[4]), "r"(v.w[5]), "r"(v.w[6]), "r"(v.w[7])
                 : "memory");
}

// 16 elements of T as one or two of them.
template <class T>
struct Sixteen {
    static constexpr int COUNT = sizeof(T) / 2;
    Wide part[COUNT];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) part[i] = load_wide(reinterpret_cast<const char*>(p) + 32 * i);
    }
    __device__ __forceinline__ void get(float (&f)[16]) const {
        Vector<T, 16> v;
        memcpy(&v, part, sizeof(v));
        unpack<T, 16>(v, f);
    }
    __device__ __forceinline__ static void store(T* p, const float (&f)[16]) {
        const Vector<T, 16> v = pack<T, 16>(f);
        Wide w[COUNT];
        memcpy(w, &v, sizeof(v));
#pragma unroll
        for (int i = 0; i < COUNT; ++i) store_wide(reinterpret_cast<char*>(p) + 32 * i, w[i]);
    }
};

namespace gemm {

// The MMAs of this cluster's work, by the one thread that calls this.
template <class C>
__device__ __forceinline__ void issue(const Shared<C>& sh, const GemmShape& s, uint32_t tmem, int first, int stride, int items) {
    const uint32_t stages = tc::smem_u32(sh.stages), held = stages + C::STAGES * C::STAGE;
    if (C::RESIDENT && !wait_for(sh.held, 0, sh.abort)) return;
    int st = 0;
    uint32_t parity = 0, unit = 0;
    int waiting = 0;  // the first part's stage of a resident unit's slab before
    bool ok = true;
    for (int at = first; ok && at < items; at += stride) {
        const Work w = work_at<C>(s, at);
        for (int slab = w.from; ok && slab < w.to; ++slab) {
            const int in = (slab - w.from) % C::UNIT;
            const bool begins = in == 0, ends = in == C::UNIT - 1 || slab + 1 == w.to;
            const uint32_t d = tmem + (unit & 1) * C::BN;
            if (begins) ok = wait_for(sh.taken + (unit & 1), ((unit >> 1) & 1) ^ 1, sh.abort);
            // The slab's stages, by part.
            int stage[C::P];
            uint32_t round[C::P];
#pragma unroll
            for (int p = C::P - 1; p >= 0; --p) {
                stage[p] = st, round[p] = parity;
                if (++st == C::STAGES) st = 0, parity ^= 1;
            }
            auto there = [&](int p) { ok = ok && wait_for(sh.full + stage[p], round[p], sh.abort); };
            auto multiply_at = [&](int a_stage, uint32_t b_at, bool accumulate) {
                const uint64_t a = descriptor<C::A_ROWS>(stages + a_stage * C::STAGE), b = descriptor<C::B_ROWS>(b_at);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mma<C::CTAS>(d, a + k * (STEP<C::A_ROWS> >> 4), b + k * (STEP<C::B_ROWS> >> 4), s.instruction,
                                 accumulate || k > 0);
            };
            auto multiply = [&](int pa, int pb, bool accumulate) {
                multiply_at(stage[pa], C::RESIDENT ? held + (slab * C::P + pb) * C::B_BYTES : stages + stage[pb] * C::STAGE + C::A_BYTES,
                            accumulate);
            };
            there(0);
            if constexpr (C::P > 1) there(C::P - 1);
            if (!ok) break;
            tc::tc_fence_after();
            if constexpr (C::P == 3) {
                multiply(2, 0, !begins);
                multiply(0, 2, true);
                commit<C::CTAS>(sh.empty + stage[2]);
                there(1);
                if (!ok) break;
                tc::tc_fence_after();
                multiply(1, 1, true);
                multiply(1, 0, true);
                multiply(0, 1, true);
                commit<C::CTAS>(sh.empty + stage[1]);
            } else if constexpr (C::P == 2) {
                multiply(1, 0, !begins);
                multiply(0, 1, true);
                commit<C::CTAS>(sh.empty + stage[1]);
            }
            if constexpr (C::RESIDENT && C::P > 1) {
                // Sums are cut toward zero at their size: the large products of a unit, of
                // two slabs at most, follow when all of the small ones are in.
                if (!ends) {
                    waiting = stage[0];
                    continue;
                }
                if (!begins) {
                    multiply_at(waiting, held + (slab - 1) * C::P * C::B_BYTES, true);
                    commit<C::CTAS>(sh.empty + waiting);
                }
            }
            multiply(0, 0, C::P > 1 || !begins);
            commit<C::CTAS>(sh.empty + stage[0]);
            if (ends) commit<C::CTAS>(sh.ready + (unit & 1)), ++unit;
        }
    }
}

// The accumulators' way out, by epilogue warp e whose lanes are those of `quarter`. The
// loop over a tile's pieces is not unrolled: its code would run out of the instruction
// cache. (Unrolled, a piece of 32 columns without an activation took 1200 clocks.)
template <class C, class E>
__device__ __forceinline__ void finish(const Shared<C>& sh, const GemmShape& s, const E& epilogue, uint32_t tmem, int e, int quarter,
                                       uint32_t rank, int first, int stride, int items) {
    const int lane = threadIdx.x % 32, c0 = e / 4 * C::COLUMNS;
    float* piece = sh.pieces + e * 32 * GEMM_STRIDE;
    uint32_t unit = 0;
    // Waits for an accumulator, one lane for all; false where a role gave up.
    auto wait = [&] {
        const bool ok = lane || wait_for(sh.ready + (unit & 1), (unit >> 1) & 1, sh.abort);
        const bool all = __all_sync(~0u, ok);
        tc::tc_fence_after();
        return all;
    };
    auto taken = [&] {
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
            if constexpr (C::CTAS == 2) arrive_at(at_rank(sh.taken + (unit & 1), 0));
            else tc::mbar_arrive(sh.taken + (unit & 1));
        }
        ++unit;
    };
    bool ok = true;
    for (int at = first; ok && at < items; at += stride) {
        const Work w = work_at<C>(s, at);
        const int row = w.tile_m * C::BM + rank * GEMM_ROWS + quarter * 32, column0 = w.tile_n * C::BN + c0;
        const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16) + c0;
        const bool mine = row + lane < s.m;
        // What a piece needs beside D is read ahead of it.
        typename E::Fetched ahead;
        auto fetch = [&](int column) {
            if (epilogue.whole && mine && column < s.n) epilogue.fetch(ahead, row + lane, column, w.batch, s);
        };
        fetch(column0);
        if constexpr (C::WHOLE) {
            if (!(ok = wait())) break;
        } else {
            // The units are added in registers, and their sum goes back to where the last was.
            float sum[C::COLUMNS / 16][16] = {};
            for (int slab = w.from; ok && slab < w.to; slab += C::UNIT) {
                if (!(ok = wait())) break;
#pragma unroll
                for (int c = 0; c < C::COLUMNS / 16; ++c) {
                    float v[16];
                    tc::tmem_read<16>(lanes + (unit & 1) * C::BN + 16 * c, v);
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum[c][i] += v[i];
                }
                if (slab + C::UNIT < w.to) taken();
            }
            if (!ok) break;
#pragma unroll
            for (int c = 0; c < C::COLUMNS / 16; ++c) {
                tc::tmem_st8(lanes + (unit & 1) * C::BN + 16 * c, *reinterpret_cast<const float(*)[8]>(sum[c]));
                tc::tmem_st8(lanes + (unit & 1) * C::BN + 16 * c + 8, *reinterpret_cast<const float(*)[8]>(sum[c] + 8));
            }
            tc::tmem_wait_st();
        }
        const uint32_t from = lanes + (unit & 1) * C::BN;
#pragma unroll 1
        for (int c = 0; c < C::COLUMNS; c += GEMM_PIECE) {
            const int column = column0 + c, left = s.n - column;
            float v[16];
            __syncwarp();  // behind the branches of the piece before: the warp loads as one
            tc::tmem_read<16>(from + c, v);
            const typename E::Fetched now = ahead;
            if (c + GEMM_PIECE == C::COLUMNS) taken();
            else fetch(column + GEMM_PIECE);
            if (row >= s.m || left <= 0) continue;
            if (epilogue.whole) {
                if (mine) epilogue.whole_row(v, now, row + lane, column, w.batch, w.split, C::BM, C::BN, s);
                continue;
            }
            // A thread ends its row's elements, then neighbouring threads write neighbouring ones.
            float z[16];
            if (mine) epilogue.odd(v, z, row + lane, column, left, w.batch, s);
            auto out = [&](const float (&f)[16], auto which) {
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 16; ++i) piece[lane * GEMM_STRIDE + i] = f[i];
                __syncwarp();
                if (lane % 16 >= left) return;
#pragma unroll 4
                for (int r = lane / 16; r < 32; r += 2)
                    if (row + r < s.m)
                        epilogue.template write<which>(piece[r * GEMM_STRIDE + lane % 16], row + r, column + lane % 16, w.batch, s);
            };
            if (epilogue.writes_z()) out(z, std::integral_constant<int, 0>{});
            out(v, std::integral_constant<int, 1>{});
        }
    }
}

}  // namespace gemm

// The epilogue E gets a tile in pieces of 32 rows and 16 columns, a thread the row of its
// lane. Where its arrays have rows of whole 32 bytes (`whole`), `fetch` reads what belongs
// to a thread's 16 elements ahead of `whole_row`, which ends them. Otherwise the results (`odd`)
// go through shared memory, so that neighbouring threads write neighbouring elements.
template <class C, class E>
__global__ void __launch_bounds__(C::THREADS, 1)
    k_gemm(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, const GemmShape s, const E epilogue,
           int* error) {
    using namespace gemm;
    extern __shared__ uint8_t raw_shared[];
    const Shared<C> sh(raw_shared);
    const int warp = threadIdx.x / 32;
    const uint32_t rank = C::CTAS == 2 ? cluster_rank() : 0;
    const int first = blockIdx.x / C::CTAS, stride = gridDim.x / C::CTAS;
    const int items = s.tiles * s.splits * s.batches;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; ++i) tc::mbar_init(sh.full + i, 1), tc::mbar_init(sh.empty + i, 1);
        for (int i = 0; i < 2; ++i) tc::mbar_init(sh.ready + i, 1), tc::mbar_init(sh.taken + i, C::CTAS * C::WARPS);
        *sh.abort = 0;
        tc::fence_barrier_init();
    }
    if (threadIdx.x == 32 * 2) {
        for (const CUtensorMap* map : {&a_map, &b_map})
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
    }
    if (warp == 1) tmem_take<C::CTAS>(sh.slot, C::TMEM);
    tc::tc_fence_before();
    __syncwarp();  // the cluster's barrier is for whole warps
    if constexpr (C::CTAS == 2) cluster_sync();
    else __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *sh.slot;
    next_launch_may_begin();
    after_previous_launch();

    if (warp == 0) {
        if (elected()) {
            int st = 0;
            uint32_t parity = 1, loaded = 0;
            // The barriers that the bytes count at, and the boxes' places.
            const uint32_t bars = C::CTAS == 2 ? at_rank(sh.full, 0) : tc::smem_u32(sh.full);
            const uint32_t stages = tc::smem_u32(sh.stages);
            for (int at = first; at < items && !*sh.abort; at += stride) {
                const Work w = work_at<C>(s, at);
                const int m0 = w.tile_m * C::BM + rank * GEMM_ROWS, n0 = w.tile_n * C::BN + rank * C::B_PART;
                const int za = w.batch * s.a_planes, zb = w.batch * s.b_planes;
                bool ok = true;
                for (int slab = w.from; ok && slab < w.to; ++slab) {
                    const bool next = C::P == 1 && slab >= s.array_slabs;
                    const int k0 = (next ? slab - s.array_slabs : slab) * GEMM_SLAB, at_a = za + next;
#pragma unroll
                    for (int i = 0; i < C::P; ++i, ++loaded) {  // the last part first: it is the first to be done with
                        const int p = C::P - 1 - i;
                        if (!(ok = wait_for(sh.empty + st, parity, sh.abort))) break;
                        if (rank == 0) tc::mbar_expect_tx(sh.full + st, s.stage_bytes);
                        const uint32_t bar = bars + 8 * st;
                        const uint32_t a = stages + st * C::STAGE, b = a + C::A_BYTES;
                        if constexpr (C::A_ROWS) {
                            load_box<C::CTAS>(a, &a_map, bar, m0, k0, at_a + p);
                            load_box<C::CTAS>(a + 8192, &a_map, bar, m0 + 64, k0, at_a + p);
                        } else {
                            load_box<C::CTAS>(a, &a_map, bar, k0, m0, at_a + p);
                        }
                        if constexpr (C::B_ROWS) {
#pragma unroll
                            for (int j = 0; j < C::B_PART; j += 64) load_box<C::CTAS>(b + j * 128, &b_map, bar, n0 + j, k0, zb + p);
                        } else {
                            load_box<C::CTAS>(b, &b_map, bar, k0, n0, zb + p);
                        }
                        if (++st == C::STAGES) st = 0, parity ^= 1;
                    }
                }
            }
            // No load may be in flight when the CTA ends, also where a role gave up, nor a
            // commit under way to the other CTA's barriers.
            for (uint32_t k = loaded - min(loaded, uint32_t(C::STAGES)); k < loaded; ++k) {
                const uint32_t round = (k / C::STAGES) & 1;
                if (rank == 0 && !tc::mbar_wait(sh.full + k % C::STAGES, round, GEMM_WAIT)) *sh.abort = 1;
                if (!*sh.abort) wait_for(sh.empty + k % C::STAGES, round, sh.abort);
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && elected()) issue<C>(sh, s, tmem, first, stride, items);
    } else {
        finish<C>(sh, s, epilogue, tmem, warp - 2, warp % 4, rank, first, stride, items);
    }
    tc::tc_fence_before();
    __syncwarp();
    if constexpr (C::CTAS == 2) cluster_sync();
    else __syncthreads();
    if (warp == 1) {
        tc::tc_fence_after();
        tmem_release<C::CTAS>(tmem, C::TMEM);
    }
    if (threadIdx.x == 0 && *sh.abort) gemm::report(error);
}

}  // namespace cpde::ops
