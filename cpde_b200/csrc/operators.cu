// Launches of the device-tensor operators (operators.hpp).
#include "operators.hpp"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <map>
#include <mutex>
#include <tuple>

#include "common.hpp"
#include "kernels_dropout.cuh"
#include "kernels_embedding.cuh"
#include "kernels_norm.cuh"
#include "kernels_norm_slab.cuh"

namespace cpde::ops {
namespace {

constexpr int SMS = 148;

enum Type : int32_t { F32 = 0, BF16 = 1, F16 = 2 };
size_t bytes_of(int32_t type) { return type == F32 ? 4 : 2; }

template <class T> struct Tag { using type = T; };

// Calls f with the C++ type of a type code.
template <class F>
void with_type(int32_t type, F&& f) {
    if (type == F32) f(Tag<float>{});
    else if (type == BF16) f(Tag<__nv_bfloat16>{});
    else f(Tag<__half>{});
}

// Equal types, or the one on the WIDE_IN side FP32 and the other of 16 bits.
template <bool WIDE_IN, class F>
void with_types(int32_t in, int32_t out, F&& f) {
    with_type(WIDE_IN ? out : in, [&](auto narrow) {
        using N = typename decltype(narrow)::type;
        if (in == out) f(Tag<N>{}, Tag<N>{});
        else if constexpr (WIDE_IN) f(Tag<float>{}, Tag<N>{});
        else f(Tag<N>{}, Tag<float>{});
    });
}

uint32_t power_of_two_from(int64_t n) {
    uint32_t p = 1;
    while (p < n) p *= 2;
    return p;
}

// The most elements, a power of two up to `most`, that divide a row of
// `channels` and whose accesses are aligned at every given address and stride.
struct Alignment {
    uint64_t odd = 0;  // bits that an access's alignment must not have
    Alignment& at(const void* p, size_t element) { odd |= reinterpret_cast<uintptr_t>(p) / element; return *this; }
    Alignment& stride(int64_t elements) { odd |= uint64_t(elements); return *this; }
    int vector(int most) const {
        int v = most;
        while (v > 1 && odd % v) v /= 2;
        return v;
    }
};

template <int... VS, class F>
void with_vector(int v, F&& f) {
    ((v == VS ? f(std::integral_constant<int, VS>{}) : void()), ...);
}

// A launch that may begin before the launch ahead of it in the stream has ended:
// for kernels that say after_previous_launch() first, behind one of this file's
// kernels. It hides a launch's start, about a microsecond.
template <class... P, class... A>
void launch_dependent(void (*kernel)(P...), dim3 grid, unsigned threads, size_t shared, cudaStream_t stream, A... arguments) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    CPDE_CUDA(cudaLaunchKernelEx(&config, kernel, P(arguments)...));
}

template <class K>
void dynamic_shared(K kernel, size_t bytes) {
    CPDE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
}

size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }

// --- embedding -------------------------------------------------------------

// Above this many tokens a sort takes the whole GPU, three launches a pass, and
// below it one cluster in one launch.
constexpr int64_t CLUSTER_TOKENS = 65536;

struct SortPlan {
    int passes, digit_bits;
    uint32_t cluster;   // CTAs of the one-launch sort
    uint32_t tiles;     // CTAs of a launch of the other (0: it is not taken)
    uint32_t per_warp;  // its pairs of a warp
};
SortPlan sort_plan(int64_t tokens, int64_t rows) {
    int bits = 1;
    while ((int64_t(1) << bits) < rows + 1) ++bits;
    SortPlan p;
    const bool large = tokens > CLUSTER_TOKENS;
    const int most = large ? 9 : 10;  // bits of a digit, from the shared memory of its warps' counts
    p.passes = (bits + most - 1) / most;
    p.digit_bits = (bits + p.passes - 1) / p.passes;
    p.cluster = std::min<uint32_t>(16, power_of_two_from((tokens + 2047) / 2048));
    // Tiles of at most 512 pairs a warp: 128 KB, beside 64 KB of counts.
    const int64_t warps = SMS * SORT_WARPS, waves = std::max<int64_t>(1, (tokens + warps * 512 - 1) / (warps * 512));
    p.tiles = large ? uint32_t(SMS * waves) : 0;
    p.per_warp = large ? uint32_t((tokens + warps * waves - 1) / (warps * waves)) : 0;
    return p;
}

SumShape sum_shape(int64_t tokens, int64_t rows, int64_t channels, int v) {
    SumShape s = {};
    s.tokens = uint32_t(tokens);
    s.rows = uint32_t(rows);
    s.channels = channels;
    s.vectors = uint32_t(channels / v);
    s.lanes = power_of_two_from(std::min<int64_t>(s.vectors, 32));
    s.tiles = (s.vectors + s.lanes - 1) / s.lanes;
    s.chunk = 64;
    while (s.chunk > 8 && (tokens / s.chunk) * s.tiles * s.lanes / 32 < SMS * 12) s.chunk /= 2;
    s.chunks = uint32_t((tokens + s.chunk - 1) / s.chunk);
    s.sum_blocks = uint32_t((uint64_t(s.chunks) * s.tiles * s.lanes + 255) / 256);
    return s;
}

// The parts of the workspace.
struct GradientWorkspace {
    uint2* pairs[2];
    uint32_t* counts;
    float* partial;
    size_t bytes;
    GradientWorkspace(void* base, int64_t tokens, int64_t rows, int64_t channels) : bytes(0) {
        auto take = [&](size_t n) {
            char* p = static_cast<char*>(base) + bytes;
            bytes += padded(n);
            return p;
        };
        const SortPlan plan = sort_plan(tokens, rows);
        for (auto& p : pairs) p = reinterpret_cast<uint2*>(take(size_t(tokens) * sizeof(uint2)));
        counts = reinterpret_cast<uint32_t*>(take((size_t(plan.tiles + 1) << plan.digit_bits) * 4));
        size_t partials = 0;
        for (int v : {8, 4, 2, 1})
            if (channels % v == 0)
                partials = std::max(partials, size_t(sum_shape(tokens, rows, channels, v).chunks) * 2 * channels);
        partial = reinterpret_cast<float*>(take(partials * sizeof(float)));
    }
};

// What the sort's launches clear while they leave memory idle: in the one launch
// as much as it takes to sort (16 us for 32768 tokens), in each of the others a
// few microseconds' worth.
constexpr int64_t CLEARED_BY_CLUSTER = 72 << 20, CLEARED_BY_LAUNCH = 12 << 20;

// Sorts the tokens into pairs[sorted_buffer(passes)] and clears the first
// clearing.whole words of the output.
template <class Id>
void sort_tokens(const EmbeddingCall& c, const Id* ids, const SortPlan& plan, const GradientWorkspace& w,
                 const Clearing& clearing, int device, cudaStream_t stream) {
    static std::atomic<uint64_t> ready{0};  // devices on which the kernels' limits are raised
    if (!(ready.load() >> (device & 63) & 1)) {
        dynamic_shared(k_sort_tokens<Id>, (size_t(SORT_WARPS) + 1) * 4096);
        dynamic_shared(k_place_tokens<Id>, SORT_WARPS * (512 * sizeof(uint2) + 512 * 4));
        CPDE_CUDA(cudaFuncSetAttribute(k_sort_tokens<Id>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        ready.fetch_or(uint64_t(1) << (device & 63));
    }
    if (plan.tiles) {
        SortPass s = {uint32_t(c.tokens), plan.per_warp, 1u << plan.digit_bits, 0, 0, 0};
        for (int pass = 0; pass < plan.passes; ++pass) {
            const SortInput<Id> in = {ids, c.rows, pass ? w.pairs[(pass + 1) & 1] : nullptr};
            s.shift = pass * plan.digit_bits;
            s.from = clearing.whole * (2 * pass) / (2 * plan.passes);
            s.to = clearing.whole * (2 * pass + 1) / (2 * plan.passes);
            if (pass == 0) {
                k_count_digits<Id><<<plan.tiles, SORT_THREADS, s.bins * 4, stream>>>(in, s, w.counts, clearing);
                CPDE_LAUNCHED();
            } else {
                launch_dependent(k_count_digits<Id>, plan.tiles, SORT_THREADS, s.bins * 4, stream, in, s, w.counts, clearing);
            }
            launch_dependent(k_scan_counts, (s.bins + 7) / 8, 256, 0, stream, w.counts, plan.tiles, s.bins);
            s.from = s.to;
            s.to = clearing.whole * (2 * pass + 2) / (2 * plan.passes);
            const size_t shared = SORT_WARPS * (plan.per_warp * sizeof(uint2) + s.bins * 4);
            launch_dependent(k_place_tokens<Id>, plan.tiles, SORT_THREADS, shared, stream, in, s, w.counts,
                             w.pairs[pass & 1], clearing);
        }
        return;
    }
    // At most seven clusters of 16 beside the sort's: a GPC holds one of them.
    const int64_t fillers = std::min<int64_t>(112, (clearing.whole + 4 * SORT_THREADS - 1) / (4 * SORT_THREADS));
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(unsigned(plan.cluster + (fillers + plan.cluster - 1) / plan.cluster * plan.cluster));
    config.blockDim = dim3(SORT_THREADS);
    config.dynamicSmemBytes = (size_t(SORT_WARPS) + 1) * (size_t(4) << plan.digit_bits);
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = plan.cluster;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    CPDE_CUDA(cudaLaunchKernelEx(&config, k_sort_tokens<Id>, ids, uint32_t(c.tokens), c.rows, plan.passes,
                                 plan.digit_bits, w.pairs[0], w.pairs[1], clearing));
}

bool small_gradient(int64_t tokens, int64_t rows, int64_t channels) {
    return tokens <= SMALL_TOKENS && rows * channels <= SMALL_TABLE;
}

}  // namespace

void embedding(const EmbeddingCall& c, cudaStream_t stream) {
    if (!c.tokens) return;
    with_types<true>(c.in_type, c.out_type, [&](auto in, auto out) {
        using TI = typename decltype(in)::type;
        using TO = typename decltype(out)::type;
        const int v = Alignment().at(c.in, sizeof(TI)).at(c.out, sizeof(TO)).stride(c.in_stride).stride(c.channels)
                          .vector(16 / sizeof(TO));
        with_vector<8, 4, 2, 1>(v, [&](auto width) {
            constexpr int V = decltype(width)::value;
            if constexpr (V * sizeof(TO) <= 16) {
                const int64_t vectors = c.channels / V;
                // Slabs of tokens whose vectors a 31-bit index counts.
                const int64_t slab = std::max<int64_t>(1, ((int64_t(1) << 30) - 1) / vectors);
                for (int64_t t = 0; t < c.tokens; t += slab) {
                    const uint32_t count = uint32_t(std::min(slab, c.tokens - t) * vectors);
                    TO* to = static_cast<TO*>(c.out) + t * c.channels;
                    auto launch = [&](auto* ids, auto lookups) {
                        constexpr int LOOKUPS = decltype(lookups)::value, THREADS = lookup_threads(LOOKUPS);
                        const uint32_t blocks = (count + THREADS * LOOKUPS - 1) / (THREADS * LOOKUPS);
                        k_embedding<TI, TO, std::remove_const_t<std::remove_pointer_t<decltype(ids)>>, V, LOOKUPS>
                            <<<blocks, THREADS, 0, stream>>>(static_cast<const TI*>(c.in), c.in_stride, c.rows, ids + t, to,
                                                             c.channels, Divisor(uint32_t(vectors)), count, c.scale);
                    };
                    auto launch_ids = [&](auto lookups) {
                        if (c.id_type) launch(static_cast<const int64_t*>(c.ids), lookups);
                        else launch(static_cast<const int32_t*>(c.ids), lookups);
                    };
                    if (vectors < 4) launch_ids(std::integral_constant<int, 2>{});
                    else launch_ids(std::integral_constant<int, 4>{});
                    CPDE_LAUNCHED();
                }
            }
        });
    });
}

size_t embedding_gradient_workspace(int64_t tokens, int64_t rows, int64_t channels) {
    return GradientWorkspace(nullptr, tokens, rows, channels).bytes;
}

void embedding_gradient(const EmbeddingCall& c, int device, cudaStream_t stream) {
    const size_t out_bytes = size_t(c.rows) * c.channels * bytes_of(c.out_type);
    if (!c.tokens) {
        CPDE_CUDA(cudaMemsetAsync(c.out, 0, out_bytes, stream));
        return;
    }
    // Calls f with the types and the vector width.
    auto typed = [&](auto&& f) {
        with_types<false>(c.in_type, c.out_type, [&](auto in, auto out) {
            using TI = typename decltype(in)::type;
            using TO = typename decltype(out)::type;
            const int v = Alignment().at(c.in, sizeof(TI)).at(c.out, sizeof(TO)).stride(c.in_stride).stride(c.channels)
                              .vector(16 / sizeof(TI));
            with_vector<8, 4, 2, 1>(v, [&](auto width) {
                if constexpr (decltype(width)::value * sizeof(TI) <= 16) f(in, out, width);
            });
        });
    };
    if (small_gradient(c.tokens, c.rows, c.channels)) {
        typed([&](auto in, auto out, auto width) {
            using TI = typename decltype(in)::type;
            using TO = typename decltype(out)::type;
            constexpr int V = decltype(width)::value;
            const uint32_t vectors = uint32_t(c.channels / V), lanes = power_of_two_from(std::min<uint32_t>(vectors, 8));
            const uint32_t blocks = (vectors + lanes - 1) / lanes, size = std::max(32u, power_of_two_from(c.tokens));
            auto launch = [&](auto* ids) {
                k_small_gradient<TI, TO, std::remove_const_t<std::remove_pointer_t<decltype(ids)>>, V>
                    <<<dim3(blocks, lanes), size, 0, stream>>>(static_cast<const TI*>(c.in), c.in_stride, ids, uint32_t(c.tokens), size,
                                                 c.rows, c.channels, vectors, lanes, static_cast<TO*>(c.out), c.scale);
            };
            if (c.id_type) launch(static_cast<const int64_t*>(c.ids));
            else launch(static_cast<const int32_t*>(c.ids));
            CPDE_LAUNCHED();
        });
        return;
    }
    const GradientWorkspace w(c.workspace, c.tokens, c.rows, c.channels);
    const SortPlan plan = sort_plan(c.tokens, c.rows);
    Clearing clearing = {static_cast<uint4*>(c.out), 0};
    const size_t row_bytes = size_t(c.channels) * bytes_of(c.out_type);
    uint32_t clear_from = uint32_t(c.rows);
    if ((reinterpret_cast<uintptr_t>(c.out) | out_bytes) % 16) {
        CPDE_CUDA(cudaMemsetAsync(c.out, 0, out_bytes, stream));
    } else {
        const int64_t idle = plan.tiles ? CLEARED_BY_LAUNCH * 2 * plan.passes : CLEARED_BY_CLUSTER;
        clearing.whole = int64_t(out_bytes / 16);
        if (row_bytes % 16 == 0 && int64_t(out_bytes) > 2 * idle) {
            clear_from = uint32_t(idle / row_bytes);
            clearing.whole = int64_t(clear_from * row_bytes / 16);
        }
    }
    if (c.id_type) sort_tokens(c, static_cast<const int64_t*>(c.ids), plan, w, clearing, device, stream);
    else sort_tokens(c, static_cast<const int32_t*>(c.ids), plan, w, clearing, device, stream);
    const uint2* pairs = w.pairs[sorted_buffer(plan.passes)];
    typed([&](auto in, auto out, auto width) {
        using TI = typename decltype(in)::type;
        using TO = typename decltype(out)::type;
        constexpr int V = decltype(width)::value;
        SumShape s = sum_shape(c.tokens, c.rows, c.channels, V);
        s.grad_stride = c.in_stride;
        s.clear_from = clear_from;
        const unsigned clear_blocks = clear_from < s.rows ? SMS * 4 : 0;
        launch_dependent(k_sum_tokens<TI, TO, V>, s.sum_blocks + clear_blocks, 256, 0, stream, pairs,
                         static_cast<const TI*>(c.in), static_cast<TO*>(c.out), w.partial, s, clearing, c.scale);
        if (c.tokens >= 2 * int64_t(s.chunk)) {  // else no run covers a chunk behind its first
            launch_dependent(k_join_chunks<TO, V>, dim3((s.chunks + JOIN_CHUNKS - 1) / JOIN_CHUNKS, s.tiles), JOIN_WARPS * 32,
                             0, stream, pairs, static_cast<TO*>(c.out), w.partial, s, c.scale);
        }
    });
}

// --- dropout ---------------------------------------------------------------

namespace {

DropoutRule dropout_rule(double rate, uint64_t seed, uint64_t offset) {
    const uint32_t threshold = uint32_t(std::lround(rate * 65536));
    return keyed_rule(threshold, threshold < 65536 ? float(65536.0 / (65536.0 - threshold)) : 0.0f, seed, offset);
}

}  // namespace

void dropout(const DropoutCall& c, cudaStream_t stream) {
    if (!c.rows || !c.columns) return;
    DropoutShape s = {c.rows, c.columns, c.x_stride, c.residual ? c.residual_stride : c.columns};
    const int64_t count = c.rows * c.columns;
    const bool contiguous = c.rows == 1 || (s.x_stride == c.columns && s.residual_stride == c.columns);
    with_type(c.type, [&](auto tag) {
        using T = typename decltype(tag)::type;
        Alignment a;
        a.at(c.x, sizeof(T)).at(c.residual, sizeof(T)).at(c.y, sizeof(T));
        if (!contiguous) a.stride(s.x_stride).stride(s.residual_stride).stride(c.columns);
        const int mode = a.vector(8) == 8 ? (contiguous ? 2 : 1) : 0;
        const unsigned blocks = unsigned((count + 2047) / 2048);
        const DropoutRule rule = dropout_rule(c.rate, c.seed, c.offset);
        with_vector<0, 1, 2>(mode, [&](auto m) {
            constexpr int MODE = decltype(m)::value;
            const T *x = static_cast<const T*>(c.x), *r = static_cast<const T*>(c.residual);
            if (r) k_dropout<T, true, MODE><<<blocks, 256, 0, stream>>>(x, r, static_cast<T*>(c.y), s, count, rule);
            else k_dropout<T, false, MODE><<<blocks, 256, 0, stream>>>(x, r, static_cast<T*>(c.y), s, count, rule);
            CPDE_LAUNCHED();
        });
    });
}

// --- group norm --------------------------------------------------------------

namespace {

NormShape norm_shape(int64_t instances, int64_t points, int64_t channels, int64_t groups, int v) {
    NormShape s = {};
    s.instances = int32_t(instances);
    s.points = int32_t(points);
    s.channels = int32_t(channels);
    s.groups = int32_t(groups);
    s.width = int32_t(channels / groups);
    s.vectors = s.channels / v;
    s.tiles = (s.vectors + 63) / 64;
    s.tile = (s.vectors + s.tiles - 1) / s.tiles;
    s.tiles = (s.vectors + s.tile - 1) / s.tile;
    s.pieces = std::min(s.groups, (s.tile * v - 1) / s.width + 2);
    const int64_t ys = NORM_THREADS / s.tile, blocks = instances * s.tiles;
    s.splits = int32_t(std::max<int64_t>(1, std::min(std::max<int64_t>(1, SMS * NORM_BLOCKS / blocks), (points + ys * 4 - 1) / (ys * 4))));
    s.splits = int32_t(std::max<int64_t>(s.splits, (points + ys * 512 - 1) / (ys * 512)));
    return s;
}

// The workspace of two passes: the groups' pieces, and the gradient's sums by channel.
size_t piece_bytes(const NormShape& s, size_t piece) {
    return padded(size_t(s.instances) * s.splits * s.tiles * s.pieces * piece);
}
size_t channel_sum_bytes(const NormShape& s, int64_t parts) {
    return padded(size_t(s.instances) * parts * s.channels * sizeof(float2));
}

// Strides, lengths and dropout of a call.
void add_call(NormShape& s, const NormCall& c) {
    s.x_point = c.x_point;
    s.x_instance = c.x_instance;
    s.grad_point = c.grad_point;
    s.grad_instance = c.grad_instance;
    s.activation = c.activation;
    s.eps = float(c.eps);
    s.lengths = c.lengths;
    s.rule = dropout_rule(c.rate, c.seed, c.offset);
}

// How a cluster holds one instance's points in a tile of whole groups.
struct SlabPlan {
    int32_t cluster = 0;  // CTAs; 0: it does not hold them
    int32_t tile, tiles;  // vectors of a tile, tiles
    int32_t slots;        // vectors of a thread, and array
    size_t shared;
};
constexpr size_t SLAB_SIX = 36 << 10, SLAB_THREE = 72 << 10, SLAB_TWO = 108 << 10, SLAB_ONE = 220 << 10;  // shared memory of a CTA
constexpr int64_t MOST_ITEMS = int64_t(1) << 30;  // items of a launch are counted in 31 bits

// Vectors of at most 16 bytes (a copy's most) whose channels are of one group.
int slab_vector(int fit, size_t element, int64_t width) {
    int v = std::min<int>(fit, int(16 / element));
    while (v > 1 && width % v) v /= 2;
    return v;
}

SlabPlan slab_plan(const NormShape& s, int v, size_t element, size_t parameter, int arrays) {
    SlabPlan p;
    const size_t vector_bytes = v * element;
    const int64_t group = s.width / v, groups = s.groups;
    int64_t tile_groups = std::max<int64_t>(1, int64_t(SLAB_TILE_BYTES / vector_bytes) / group);  // whole lines
    tile_groups = std::min(tile_groups, groups);
    p.tile = int32_t(tile_groups * group);
    if (p.tile > SLAB_THREADS) return p;
    p.tiles = int32_t((groups + tile_groups - 1) / tile_groups);
    if (int64_t(s.instances) * p.tiles > MOST_ITEMS) return p;
    const int64_t ys = SLAB_THREADS / p.tile;
    auto plan = [&](int32_t cluster) {
        const int64_t points = (int64_t(s.points) + cluster - 1) / cluster;
        const int64_t slots = (points + ys - 1) / ys;
        p.slots = int32_t(std::min<int64_t>(slots, 1 << 16));
        const int64_t width = int64_t(p.tile) * v, rows = slab_rows_are_warps(p.tile) ? SLAB_WARPS : ys;
        const size_t parameters = tile_parameter_bytes(width, parameter);
        p.shared = size_t(p.slots) * SLAB_THREADS * vector_bytes * arrays +
                   2 * SlabExchange::bytes(int32_t(tile_groups), cluster) + parameters +
                   (arrays == 1 ? SLAB_THREADS : size_t((rows + 1) * width)) * sizeof(float2);
        return p.shared;
    };
    int32_t cluster = 0;
    for (size_t limit : {arrays == 1 ? SLAB_SIX : SLAB_THREE, SLAB_THREE, SLAB_TWO, SLAB_ONE}) {
        for (int32_t c = 1; c <= SLAB_CLUSTER && !cluster; c *= 2)
            if (plan(c) <= limit) cluster = c;
        if (cluster) break;
    }
    if (!cluster) return p;
    // Few instances: smaller shares, for more of the GPU.
    while (cluster < SLAB_CLUSTER && int64_t(s.instances) * p.tiles * cluster < 2 * SMS && (plan(cluster), p.slots >= 4))
        cluster *= 2;
    plan(cluster);
    p.cluster = cluster;
    return p;
}

// Launches a slab kernel over the items of a call, with as many clusters as the
// GPU holds at once; `counter` (four bytes) deals out the items behind those.
template <auto kernel, class... A>
void launch_slab(const SlabPlan& plan, const NormShape& norm, int v, const NormCall& c, size_t parameter,
                 uint32_t* counter, int device, cudaStream_t stream, A... arguments) {
    static std::mutex mutex;
    // Clusters that a device holds at once, by its number, their size and their memory in
    // KB: a property of the kernel, looked up once; at most 5 x 220 a device.
    static std::map<std::tuple<int, int32_t, int32_t>, int32_t> resident;
    cudaLaunchConfig_t config = {};
    config.blockDim = dim3(SLAB_THREADS);
    config.dynamicSmemBytes = plan.shared;
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = plan.cluster;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    int32_t clusters;
    {
        std::lock_guard<std::mutex> lock(mutex);
        const int32_t kilobytes = int32_t((plan.shared + 1023) / 1024);
        int32_t& known = resident[{device, plan.cluster, kilobytes}];
        if (!known) {
            dynamic_shared(kernel, SLAB_ONE);
            CPDE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
            config.gridDim = dim3(plan.cluster);
            config.dynamicSmemBytes = size_t(kilobytes) * 1024;
            int most = 0;
            CPDE_CUDA(cudaOccupancyMaxActiveClusters(&most, kernel, &config));
            config.dynamicSmemBytes = plan.shared;
            known = std::max(1, most);
        }
        clusters = known;
    }
    const int32_t ys = SLAB_THREADS / plan.tile, group_vectors = norm.width / v;
    auto by = [](int32_t d) { return Divisor(uint32_t(d)); };
    SlabShape s = {norm, plan.cluster, plan.slots, 0, norm.instances * plan.tiles, nullptr, ys, group_vectors,
                   plan.tile * v, plan.tile / group_vectors, by(plan.cluster), by(plan.tiles), by(plan.tile), by(ys),
                   by(group_vectors), false};
    s.clusters = std::min(clusters, s.items);
    s.norm.tile = plan.tile;
    s.norm.tiles = plan.tiles;
    add_call(s.norm, c);
    s.wide_parameters = Alignment().at(c.weight, parameter).at(c.bias, parameter).vector(v) == v;
    if (s.clusters < s.items) {
        s.counter = counter;
        CPDE_CUDA(cudaMemsetAsync(counter, 0, sizeof(*counter), stream));
    }
    config.gridDim = dim3(unsigned(s.clusters * plan.cluster));
    CPDE_CUDA(cudaLaunchKernelEx(&config, kernel, arguments..., s));
}

// The widest vectors that the call's addresses and strides allow. The forward
// takes eight channels of any type (160 us against 169 for a million points of 64
// f32 channels in two passes), the gradient one access of 16 bytes an array (234
// us; with eight channels 232, within what the sums' registers allow).
template <class T>
int norm_vector(const NormCall& c) {
    Alignment a;
    a.at(c.x, sizeof(T)).at(c.out, sizeof(T)).stride(c.x_point).stride(c.channels);
    if (c.instances > 1) a.stride(c.x_instance);
    if (c.grad) {
        a.at(c.grad, sizeof(T)).stride(c.grad_point);
        if (c.instances > 1) a.stride(c.grad_instance);
    }
    return a.vector(c.grad ? int(16 / sizeof(T)) : 8);
}

// Calls f with the types of the array and of the parameters.
template <class F>
void with_norm_types(const NormCall& c, F&& f) {
    with_type(c.type, [&](auto tag) {
        if (c.parameter_type == F32) f(tag, Tag<float>{});
        else f(tag, tag);
    });
}

// Calls f with the vector width, one of 8, 4 and 1, and whether a vector's
// channels are of one group. The gradient's eight channels of several groups
// would want more registers than a thread has: it takes four.
template <bool GRADIENT, class F>
void with_norm_vector(int v, int64_t width, F&& f) {
    if (GRADIENT && v == 8 && width % 8) v = 4;
    with_vector<8, 4, 1>(v == 2 ? 1 : v, [&](auto w) {
        constexpr int V = decltype(w)::value;
        if (width % V == 0) f(w, std::true_type{});
        else if constexpr (V > 1 && !(GRADIENT && V == 8)) f(w, std::false_type{});
    });
}

}  // namespace

size_t group_norm_workspace(int64_t instances, int64_t points, int64_t channels, int64_t groups, bool gradient) {
    size_t bytes = padded(4);
    for (int v : {8, 4, 1}) {
        if (channels % v) continue;
        const NormShape s = norm_shape(instances, points, channels, groups, v);
        bytes = std::max(bytes, gradient ? piece_bytes(s, sizeof(float2)) + channel_sum_bytes(s, s.splits)
                                         : piece_bytes(s, sizeof(Moments)));
        if (!gradient || v == 1 || s.width % v) continue;
        // Every plan that a call of these sizes can take.
        const size_t types[][2] = {{4, 4}, {2, 4}, {2, 2}};  // bytes of an element and of a parameter
        for (auto [element, parameter] : types) {
            if (v * element > 16) continue;
            const SlabPlan plan = slab_plan(s, v, element, parameter, 2);
            if (plan.cluster) bytes = std::max(bytes, padded(4) + channel_sum_bytes(s, plan.cluster));
        }
    }
    return bytes;
}

void group_norm(const NormCall& c, int device, cudaStream_t stream) {
    if (!c.instances) return;
    if (!c.points) {
        CPDE_CUDA(cudaMemsetAsync(c.mean, 0, size_t(c.instances * c.groups) * 4, stream));
        CPDE_CUDA(cudaMemsetAsync(c.rstd, 0, size_t(c.instances * c.groups) * 4, stream));
        return;
    }
    with_norm_types(c, [&](auto type, auto parameter_type) {
        using T = typename decltype(type)::type;
        using P = typename decltype(parameter_type)::type;
        const T* x = static_cast<const T*>(c.x);
        const P *weight = static_cast<const P*>(c.weight), *bias = static_cast<const P*>(c.bias);
        T* y = static_cast<T*>(c.out);
        const int fit = norm_vector<T>(c);
        bool done = false;
        with_vector<8, 4>(slab_vector(fit, sizeof(T), c.channels / c.groups), [&](auto width) {
            constexpr int V = decltype(width)::value;
            if constexpr (V * sizeof(T) <= 16) {
                const NormShape s = norm_shape(c.instances, c.points, c.channels, c.groups, V);
                const SlabPlan plan = slab_plan(s, V, sizeof(T), sizeof(P), 1);
                if (!plan.cluster) return;
                launch_slab<k_norm_slab<T, P, V>>(plan, s, V, c, sizeof(P), static_cast<uint32_t*>(c.workspace), device,
                                                  stream, x, weight, bias, y, c.mean, c.rstd);
                done = true;
            }
        });
        if (done) return;
        with_norm_vector<false>(fit, c.channels / c.groups, [&](auto width, auto one) {
            constexpr int V = decltype(width)::value;
            NormShape s = norm_shape(c.instances, c.points, c.channels, c.groups, V);
            add_call(s, c);
            auto* pieces = static_cast<Moments*>(c.workspace);
            const size_t shared = size_t(NORM_THREADS / s.tile) * s.tile * V * 8;
            k_norm_moments<T, V><<<dim3(unsigned(s.instances) * s.splits, s.tiles), NORM_THREADS, shared, stream>>>(
                x, s, pieces);
            CPDE_LAUNCHED();
            launch_dependent(k_norm_apply<T, P, V, decltype(one)::value>, dim3(unsigned(s.instances) * s.splits, s.tiles),
                             NORM_THREADS, size_t(s.pieces) * 8, stream, x, weight, bias, y, c.mean, c.rstd, pieces, s);
        });
    });
}

void group_norm_gradient(const NormCall& c, int device, cudaStream_t stream) {
    if (!c.instances || !c.points) {
        const size_t bytes = size_t(c.channels) * bytes_of(c.parameter_type);
        if (c.dweight) CPDE_CUDA(cudaMemsetAsync(c.dweight, 0, bytes, stream));
        if (c.dbias) CPDE_CUDA(cudaMemsetAsync(c.dbias, 0, bytes, stream));
        return;
    }
    with_norm_types(c, [&](auto type, auto parameter_type) {
        using T = typename decltype(type)::type;
        using P = typename decltype(parameter_type)::type;
        const T *grad = static_cast<const T*>(c.grad), *x = static_cast<const T*>(c.x);
        const P *weight = static_cast<const P*>(c.weight), *bias = static_cast<const P*>(c.bias);
        T* dx = static_cast<T*>(c.out);
        P *dweight = static_cast<P*>(c.dweight), *dbias = static_cast<P*>(c.dbias);
        const unsigned parameter_blocks = dweight || dbias ? unsigned(c.channels + 31) / 32 : 0;
        const int fit = norm_vector<T>(c);
        bool done = false;
        with_vector<8, 4>(slab_vector(fit, sizeof(T), c.channels / c.groups), [&](auto width) {
            constexpr int V = decltype(width)::value;
            if constexpr (V * sizeof(T) <= 16) {
                const NormShape s = norm_shape(c.instances, c.points, c.channels, c.groups, V);
                const SlabPlan plan = slab_plan(s, V, sizeof(T), sizeof(P), 2);
                if (!plan.cluster) return;
                auto* counter = static_cast<uint32_t*>(c.workspace);
                auto* channel_sums = reinterpret_cast<float2*>(static_cast<char*>(c.workspace) + padded(4));
                launch_slab<k_norm_slab_gradient<T, P, V>>(plan, s, V, c, sizeof(P), counter, device, stream, grad, x,
                                                           c.mean, c.rstd, weight, bias, dx, channel_sums);
                if (parameter_blocks) {
                    launch_dependent(k_norm_parameters<P>, parameter_blocks, 1024, 0, stream, dweight, dbias, channel_sums,
                                     s.instances * plan.cluster, s.channels);
                }
                done = true;
            }
        });
        if (done) return;
        with_norm_vector<true>(fit, c.channels / c.groups, [&](auto width, auto one) {
            constexpr int V = decltype(width)::value;
            constexpr bool ONE = decltype(one)::value;
            NormShape s = norm_shape(c.instances, c.points, c.channels, c.groups, V);
            add_call(s, c);
            auto* pieces = static_cast<float2*>(c.workspace);
            auto* channel_sums = reinterpret_cast<float2*>(
                static_cast<char*>(c.workspace) + piece_bytes(s, sizeof(float2)));
            const size_t shared = size_t(NORM_THREADS / s.tile) * s.tile * V * 8;
            k_norm_sums<T, P, V, ONE><<<dim3(unsigned(s.instances) * s.splits, s.tiles), NORM_THREADS, shared, stream>>>(
                grad, x, c.mean, c.rstd, weight, bias, s, channel_sums, pieces);
            CPDE_LAUNCHED();
            launch_dependent(k_norm_input_gradient<T, P, V, ONE>,
                             dim3(unsigned(s.instances) * s.splits + parameter_blocks, s.tiles), NORM_THREADS,
                             size_t(s.pieces) * 8, stream, grad, x, c.mean, c.rstd, weight, bias, dx, dweight, dbias,
                             channel_sums, pieces, s);
        });
    });
}

}  // namespace cpde::ops
