// Launches of kernels_gemm.cuh: tensor maps, tiles and splits; what the launches of layers
// and of orthogonalised matrices have in common.
#pragma once
#include <algorithm>
#include <atomic>

#include "common.hpp"
#include "expression.hpp"
#include "kernels_gemm.cuh"

namespace cpde::ops {

constexpr int GEMM_SMS = 148;

enum Type : int32_t { F32 = 0, BF16 = 1, F16 = 2 };
template <class T> struct Tag { using type = T; };

// Parts of a workspace, 256-byte aligned.
struct Room {
    char* base;
    size_t bytes = 0;
    template <class T> T* take(size_t count) {
        T* p = base ? reinterpret_cast<T*>(base + bytes) : nullptr;
        bytes += (count * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

inline bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Threads of a row, eight columns each: a power of two.
inline int row_lanes(int64_t columns) {
    int lanes = 1;
    while (lanes < 32 && lanes * 8 < columns) lanes *= 2;
    return lanes;
}

// A launch that may begin before the one ahead in the stream has ended: every kernel
// behind it says after_previous_launch() before it touches memory. CLUSTER CTAs each.
template <class... P, class... A>
void launch_early(void (*kernel)(P...), dim3 grid, unsigned threads, size_t shared, int cluster, cudaStream_t stream,
                  A&&... arguments) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attributes[2] = {};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = cluster;
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = cluster > 1 ? 2 : 1;
    CPDE_CUDA(cudaLaunchKernelEx(&config, kernel, P(arguments)...));
}

// A 16-bit operand: `planes` arrays (parts, batches) of rows of `pitch` elements.
struct Operand {
    const void* base;
    int64_t pitch, rows, columns, planes, plane;  // `plane` elements from one array to the next
    int each;                                     // arrays a batch
};

// Boxes of 64 columns and `box` rows; what lies outside the array is read as zeros.
inline CUtensorMap operand_map(const Operand& o, int box, bool bf16) {
    CUtensorMap map;
    // The stride of a single row or array is never used, but has to be a valid one.
    const int64_t pitch = o.rows > 1 ? o.pitch : (o.columns + 7) / 8 * 8, plane = o.planes > 1 ? o.plane : 8;
    cuuint64_t dims[3] = {cuuint64_t(o.columns), cuuint64_t(o.rows), cuuint64_t(o.planes)};
    cuuint64_t strides[2] = {cuuint64_t(pitch) * 2, cuuint64_t(plane) * 2};
    cuuint32_t boxes[3] = {GEMM_SLAB, cuuint32_t(box), 1};
    cuuint32_t element_strides[3] = {1, 1, 1};
    driver_check(driver_api().encode_tiled(&map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                                           const_cast<void*>(o.base), dims, strides, boxes, element_strides,
                                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE),
                 "cuTensorMapEncodeTiled");
    return map;
}

// Which tile a product takes, into how many parts its contraction is split, and the
// clocks that it is estimated to take.
struct GemmPlan {
    int ctas, bn, splits, split_slabs;
    double clocks;
};

// The tiles (GemmTile), and the clocks that an MMA of theirs was measured to take in a
// long contraction: only the largest has the rate of the tensor core, the others are
// bound by what an MMA reads of shared memory.
struct GemmChoice {
    int ctas, bn, clocks;
};
constexpr GemmChoice GEMM_CHOICES[4] = {{2, 256, 130}, {2, 128, 100}, {1, 128, 75}, {1, 64, 70}};

inline int64_t lower_tiles(int64_t tiles_m, int64_t tiles_n, int64_t ratio) {
    int64_t sum = 0;
    for (int64_t m = 0; m < tiles_m; ++m) sum += std::min(tiles_n, ratio * (m + 1));
    return sum;
}

// Clocks around a tile, those of 32 columns in the epilogue, those of a launch, and of
// joining a split contraction besides its partial sums' way through memory.
constexpr double TILE_CLOCKS = 700, PIECE_CLOCKS = 900, LAUNCH_CLOCKS = 3000, JOIN_CLOCKS = 5000;

// Takes the tile into `best` if it is estimated to be faster, with its best split. A
// tile's epilogue runs beside the next one's products.
inline void consider(GemmPlan& best, int ctas, int bn, double slab, int64_t m, int64_t n, int64_t k, int64_t batches, bool lower,
                     bool may_split) {
    const int64_t slabs = (k + GEMM_SLAB - 1) / GEMM_SLAB;
    const int64_t bm = 128 * ctas, tm = (m + bm - 1) / bm, tn = (n + bn - 1) / bn;
    const int64_t tiles = (lower ? lower_tiles(tm, tn, bm / bn) : tm * tn) * batches, slots = GEMM_SMS / ctas;
    const int64_t fill = std::max<int64_t>(1, slots / std::max<int64_t>(tiles, 1));
    const int64_t most = may_split ? std::min(slabs / 2, 4 * fill) : 1;
    const double epilogue = PIECE_CLOCKS * bn / 64;
    for (int64_t want : {int64_t(1), int64_t(2), int64_t(3), int64_t(4), int64_t(6), int64_t(8), fill, 2 * fill}) {
        if (want > 1 && want > most) continue;
        const int64_t each = (slabs + want - 1) / want, splits = (slabs + each - 1) / each;
        double time = double((tiles * splits + slots - 1) / slots) * (std::max(each * slab, epilogue) + TILE_CLOCKS) + epilogue;
        if (splits > 1) time += JOIN_CLOCKS + double(splits) * m * n * 8 / 4000;
        if (!best.ctas || time < best.clocks) best = {ctas, bn, int(splits), int(each), time};
    }
}

// The choice of the shortest estimate: waves of tiles, a slab at the rate of the MMAs, of
// what L2 brings (64 bytes a clock an SM), or of the accumulators' way out and back, which
// is long between two CTAs (GemmTile::UNIT).
template <int P>
GemmPlan gemm_plan(int64_t m, int64_t n, int64_t k, int64_t batches, bool lower, bool may_split) {
    GemmPlan best = {};
    for (const GemmChoice& c : GEMM_CHOICES) {
        const double bytes = P * (128 + c.bn / c.ctas) * 128.0, way = P == 1 || c.ctas == 1 ? 0 : P == 2 ? 1300 : 2600;
        consider(best, c.ctas, c.bn, std::max({PRODUCTS<P> * 4.0 * c.clocks, bytes / 64, way}), m, n, k, batches, lower, may_split);
    }
    return best;
}

inline GemmShape gemm_shape(int64_t m, int64_t n, int64_t k, int64_t batches, int bm, int bn, bool lower, const GemmPlan& plan) {
    GemmShape s = {};
    s.m = int(m), s.n = int(n);
    s.slabs = int((k + GEMM_SLAB - 1) / GEMM_SLAB);
    s.splits = plan.splits, s.split_slabs = plan.split_slabs;
    s.tiles_m = int((m + bm - 1) / bm), s.tiles_n = int((n + bn - 1) / bn);
    s.tiles = int(lower ? lower_tiles(s.tiles_m, s.tiles_n, bm / bn) : int64_t(s.tiles_m) * s.tiles_n);
    s.batches = int(batches);
    s.lower = lower;
    return s;
}
inline uint32_t mma_instruction(int m, int n, bool a_rows, bool b_rows, bool bf16) {
    const uint32_t kind = bf16 ? 1 : 0;
    return 1u << 4 | kind << 7 | kind << 10 | uint32_t(a_rows) << 15 | uint32_t(b_rows) << 16 | uint32_t(n >> 3) << 17 |
           uint32_t(m >> 4) << 24;
}
// Raises the kernel's limit of shared memory, once a device.
template <class K>
void allow_shared(K kernel, int bytes, std::atomic<uint64_t>& ready) {
    int device = 0;
    CPDE_CUDA(cudaGetDevice(&device));
    if (ready.load() >> (device & 63) & 1) return;
    CPDE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    ready.fetch_or(uint64_t(1) << (device & 63));
}

template <class C, class E>
void launch_gemm(const Operand& a, const Operand& b, int64_t m, int64_t n, int64_t k, int64_t batches, bool bf16, bool lower,
                 const GemmPlan& plan, const E& epilogue, int* error, cudaStream_t stream) {
    GemmShape s = gemm_shape(m, n, k, batches, C::BM, C::BN, lower, plan);
    s.a_planes = a.each, s.b_planes = b.each;
    s.array_slabs = int(((C::A_ROWS ? a.rows : a.columns) + GEMM_SLAB - 1) / GEMM_SLAB);
    // A single tile of few rows loads no more of them than there are; what the other
    // lanes compute from old bytes is never read.
    const bool few = !C::A_ROWS && C::CTAS == 1 && m < GEMM_ROWS;
    const int a_box = C::A_ROWS ? 64 : few ? int((m + 7) / 8 * 8) : GEMM_ROWS;
    const int b_box = C::B_ROWS ? 64 : C::B_PART;
    s.stage_bytes = uint32_t(C::CTAS * ((few ? a_box * 128 : C::A_BYTES) + C::B_BYTES));
    s.instruction = mma_instruction(C::BM, C::BN, C::A_ROWS, C::B_ROWS, bf16);
    static std::atomic<uint64_t> ready{0};
    allow_shared(k_gemm<C, E>, C::SHARED, ready);
    const int64_t items = int64_t(s.tiles) * s.splits * s.batches;
    require(items < (int64_t(1) << 31), "too many tiles for one product");
    const int clusters = int(std::min<int64_t>(items, GEMM_SMS / C::CTAS));
    launch_early(k_gemm<C, E>, dim3(clusters * C::CTAS), C::THREADS, C::SHARED, C::CTAS, stream, operand_map(a, a_box, bf16),
                 operand_map(b, b_box, bf16), s, epilogue, error);
}

// The tile of the plan as a type, that of a contraction of one part by its length.
template <int P, bool A_ROWS, bool B_ROWS, class F>
void with_tile(const GemmPlan& plan, F&& f) {
    auto with = [&](auto is_long) {
        constexpr bool LONG = decltype(is_long)::value;
        if (plan.bn == 256) return f(GemmTile<2, 256, P, A_ROWS, B_ROWS, false, LONG>{});
        if (plan.bn == 128 && plan.ctas == 2) return f(GemmTile<2, 128, P, A_ROWS, B_ROWS, false, LONG>{});
        if (plan.bn == 128) return f(GemmTile<1, 128, P, A_ROWS, B_ROWS, false, LONG>{});
        f(GemmTile<1, 64, P, A_ROWS, B_ROWS, false, LONG>{});
    };
    if constexpr (P == 1)
        if (plan.split_slabs > GEMM_LONG) return with(std::true_type{});
    with(std::false_type{});
}

}  // namespace cpde::ops
