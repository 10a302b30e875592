// Embedding lookup with scaling, and its gradient by sorted tokens.
#pragma once
#include <cooperative_groups.h>

#include "device_vector.cuh"

namespace cpde::ops {

// out[t,:] = scale * table[ids[t],:]; an id outside [0, rows) is absent and
// gives a zero row. A thread has LOOKUPS vectors of V channels, a block's
// vectors apart, so that its loads of ids and then of rows are in flight
// together. Bound by memory: 32768 rows of 2048 bf16 (181 MB) take 32.9 us, 5.5
// TB/s, with four lookups a thread; with two 35.1, with eight 36.9. Rows of fewer
// than four vectors wait for an id and then a row, and more threads hide that
// better: 1M rows of 8 f32 (40 MB) take 12.3 us with two lookups, 14.3 with four.
constexpr int lookup_threads(int lookups) { return 256 / lookups; }
template <class TI, class TO, class Id, int V, int LOOKUPS>
__global__ void __launch_bounds__(lookup_threads(LOOKUPS)) k_embedding(const TI* __restrict__ table, int64_t table_stride, int64_t rows,
                                                    const Id* __restrict__ ids, TO* __restrict__ out,
                                                    int64_t channels, Divisor vectors, uint32_t count, float scale) {
    constexpr int THREADS = lookup_threads(LOOKUPS);
    const uint32_t base = blockIdx.x * (THREADS * LOOKUPS) + threadIdx.x;
    int64_t source[LOOKUPS];
#pragma unroll
    for (int u = 0; u < LOOKUPS; ++u) {
        const uint32_t i = base + u * THREADS;
        source[u] = -1;
        if (i < count) {
            const uint32_t t = vectors.quotient(i), k = i - t * vectors.divisor;
            const int64_t id = int64_t(ids[t]);
            if (id >= 0 && id < rows) source[u] = id * table_stride + int64_t(k) * V;
        }
    }
    Vector<TI, V> v[LOOKUPS];
#pragma unroll
    for (int u = 0; u < LOOKUPS; ++u) v[u] = source[u] >= 0 ? load<TI, V>(table + source[u]) : zeros<TI, V>();
#pragma unroll
    for (int u = 0; u < LOOKUPS; ++u) {
        const uint32_t i = base + u * THREADS;
        if (i >= count) continue;
        float f[V];
        unpack<TI, V>(v[u], f);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = source[u] >= 0 ? f[j] * scale : 0.0f;
        store_streaming<TO, V>(out + int64_t(i) * V, pack<TO, V>(f));  // the table stays in L2
    }
}

// --- gradient: tokens sorted by row --------------------------------------

constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;

// Row of a token; absent ids sort behind every row, as row `rows`.
template <class Id>
__device__ __forceinline__ uint32_t row_of(Id id, int64_t rows) {
    return uint32_t(int64_t(id) >= 0 && int64_t(id) < rows ? int64_t(id) : rows);
}

// (row, token) pairs. The passes of a sort alternate between two buffers, pass p
// writing buffer p % 2; the first reads the ids themselves.
__host__ __device__ inline int sorted_buffer(int passes) { return (passes - 1) & 1; }
template <class Id>
struct SortInput {
    const Id* ids;
    int64_t rows;
    const uint2* pairs;  // null in the first pass
    __device__ __forceinline__ uint2 at(uint32_t i) const {
        return pairs ? pairs[i] : make_uint2(row_of(ids[i], rows), i);
    }
};

// The table's gradient is cleared where no token adds to it. Of a large one the
// sort's launches clear the first words whole while memory idles, and the sums'
// launch those of the rows behind that the sorted tokens do not hold.
struct Clearing {
    uint4* words;   // the table's gradient
    int64_t whole;  // words that the sort clears
};
__device__ __forceinline__ void clear_words(uint4* words, int64_t from, int64_t to, int64_t first, int64_t step) {
    for (int64_t i = from + first; i < to; i += step) words[i] = make_uint4(0, 0, 0, 0);
}

// A pass is stable because each warp has a contiguous range of the pairs: a
// pair's place is (smaller digits anywhere) + (its digit in the CTAs before) +
// (in the warps before) + (before it in its warp, from the lanes with the same
// digit). No order depends on timing. SORT_BATCH loads of a lane are in flight at
// once.
constexpr int SORT_BATCH = 8;

template <class Id>
__device__ __forceinline__ void count_digits(const SortInput<Id>& in, uint32_t lo, uint32_t hi, uint32_t step,
                                             int shift, uint32_t mask, uint32_t* histogram) {
    for (uint32_t at = lo; at < hi; at += SORT_BATCH * step) {
        uint32_t r[SORT_BATCH];
#pragma unroll
        for (int u = 0; u < SORT_BATCH; ++u) r[u] = at + u * step < hi ? in.at(at + u * step).x : 0;
#pragma unroll
        for (int u = 0; u < SORT_BATCH; ++u)
            if (at + u * step < hi) atomicAdd(&histogram[(r[u] >> shift) & mask], 1u);
    }
}

// The lanes of a warp whose digits of `bits` bits are equal to the caller's, by a
// vote a bit: a warp's match instruction took 280 cycles here, nine votes 40.
__device__ __forceinline__ uint32_t equal_lanes(uint32_t lanes, uint32_t digit, uint32_t mask) {
    uint32_t equal = lanes;
    for (uint32_t bit = 1; bit <= mask; bit *= 2) {
        const uint32_t set = __ballot_sync(lanes, digit & bit);
        equal &= digit & bit ? set : ~set;
    }
    return equal;
}

// `place`: this warp's next place in `out` for each digit.
template <class Id>
__device__ __forceinline__ void place_pairs(const SortInput<Id>& in, uint32_t lo, uint32_t hi, int shift,
                                            uint32_t mask, uint32_t* place, uint2* out) {
    const uint32_t lane = threadIdx.x % 32;
    for (uint32_t at = lo; at < hi; at += SORT_BATCH * 32) {
        uint2 pair[SORT_BATCH];
#pragma unroll
        for (int u = 0; u < SORT_BATCH; ++u) {
            const uint32_t i = at + u * 32 + lane;
            pair[u] = i < hi ? in.at(i) : make_uint2(0, 0);
        }
#pragma unroll
        for (int u = 0; u < SORT_BATCH; ++u) {
            const bool active = at + u * 32 + lane < hi;
            const uint32_t lanes = __ballot_sync(~0u, active);
            if (active) {
                const uint32_t digit = (pair[u].x >> shift) & mask;
                const uint32_t peers = equal_lanes(lanes, digit, mask);
                const uint32_t mine = __popc(peers & ((1u << lane) - 1));
                const uint32_t to = place[digit] + mine;
                __syncwarp(lanes);
                if (mine == 0) place[digit] += __popc(peers);
                out[to] = pair[u];
            }
            __syncwarp();
        }
    }
}

// Exclusive prefix of the warps' counts by digit in shared memory, which become
// places within the digit; returns the CTA's count of digit threadIdx.x.
__device__ __forceinline__ uint32_t prefix_warps(uint32_t* histogram, uint32_t bins) {
    uint32_t sum = 0;
    if (threadIdx.x < bins) {
        uint32_t n[SORT_WARPS];
#pragma unroll
        for (int w = 0; w < SORT_WARPS; ++w) n[w] = histogram[w * bins + threadIdx.x];
#pragma unroll
        for (int w = 0; w < SORT_WARPS; ++w) {
            histogram[w * bins + threadIdx.x] = sum;
            sum += n[w];
        }
    }
    return sum;
}

// Adds the places' base to a digit's warps.
__device__ __forceinline__ void add_to_warps(uint32_t* histogram, uint32_t bins, uint32_t base) {
    if (threadIdx.x >= bins) return;
    uint32_t n[SORT_WARPS];
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) n[w] = histogram[w * bins + threadIdx.x];
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) histogram[w * bins + threadIdx.x] = n[w] + base;
}

// Exclusive prefix over the block's threads.
__device__ __forceinline__ uint32_t prefix_block(uint32_t value, uint32_t* warp_sums) {
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint32_t scan = value;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint32_t n = __shfl_up_sync(~0u, scan, d);
        if (lane >= uint32_t(d)) scan += n;
    }
    if (lane == 31) warp_sums[warp] = scan;
    __syncthreads();
    if (warp == 0) {
        uint32_t s = warp_sums[lane];
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const uint32_t n = __shfl_up_sync(~0u, s, d);
            if (lane >= uint32_t(d)) s += n;
        }
        warp_sums[lane] = s;
    }
    __syncthreads();
    return scan - value + (warp ? warp_sums[warp - 1] : 0);
}

// Few tokens: all passes in one launch, by the first cluster of the grid, whose
// CTAs exchange their counts through distributed shared memory; the other
// clusters clear the table's gradient meanwhile. Bound by its chain of barriers
// and trips: 16 us for 4000 tokens of 17 bits, 19 for 32768, 26 with 72 MB cleared
// beside; a launch a step would take nine launches.
template <class Id>
__global__ void __launch_bounds__(SORT_THREADS) k_sort_tokens(const Id* __restrict__ ids, uint32_t tokens,
                                                               int64_t rows, int passes, int digit_bits,
                                                               uint2* pairs0, uint2* pairs1, Clearing clearing) {
    namespace cg = cooperative_groups;
    next_launch_may_begin();
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t size = cluster.num_blocks();
    if (blockIdx.x >= size) {
        clear_words(clearing.words, 0, clearing.whole, int64_t(blockIdx.x - size) * SORT_THREADS + threadIdx.x,
                    int64_t(gridDim.x - size) * SORT_THREADS);
        return;
    }
    extern __shared__ uint32_t sort_shared[];
    const uint32_t bins = 1u << digit_bits;
    uint32_t* histogram = sort_shared;                 // [warp][bin]
    uint32_t* totals = histogram + SORT_WARPS * bins;  // [bin]: this CTA's
    __shared__ uint32_t warp_sums[SORT_WARPS];
    const uint32_t rank = cluster.block_rank();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, bin = threadIdx.x;
    const uint32_t per_warp = (tokens + size * SORT_WARPS - 1) / (size * SORT_WARPS);
    const uint64_t start = uint64_t(rank * SORT_WARPS + warp) * per_warp;
    const uint32_t lo = uint32_t(start < tokens ? start : tokens);
    const uint32_t hi = uint32_t(start + per_warp < tokens ? start + per_warp : tokens);
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * digit_bits;
        const SortInput<Id> in = {ids, rows, pass == 0 ? nullptr : pass & 1 ? pairs0 : pairs1};
        for (uint32_t i = threadIdx.x; i < SORT_WARPS * bins; i += SORT_THREADS) histogram[i] = 0;
        __syncthreads();
        count_digits(in, lo + lane, hi, 32, shift, bins - 1, histogram + warp * bins);
        __syncthreads();
        const uint32_t mine = prefix_warps(histogram, bins);
        if (bin < bins) totals[bin] = mine;
        cluster.sync();
        uint32_t before = 0, all = 0;
        if (bin < bins) {
#pragma unroll 8
            for (uint32_t c = 0; c < size; ++c) {
                const uint32_t n = cluster.map_shared_rank(totals, c)[bin];
                before += c < rank ? n : 0;
                all += n;
            }
        }
        const uint32_t base = prefix_block(all, warp_sums) + before;
        add_to_warps(histogram, bins, base);
        __syncthreads();
        place_pairs(in, lo, hi, shift, bins - 1, histogram + warp * bins, pass & 1 ? pairs1 : pairs0);
        // Orders this pass's pairs in global memory, and its reads of the other
        // CTAs' totals, before the next pass's.
        __threadfence();
        cluster.sync();
    }
}

// Many tokens: a pass is three launches over the whole GPU (one cluster took 217
// us for 1M tokens in two passes, these take 45). The first counts the digits of
// each tile (a CTA's range of pairs): 4.8 us for 1M tokens.
struct SortPass {
    uint32_t tokens, per_warp, bins;
    int shift;
    int64_t from, to;  // the words of the table's gradient that this launch clears
};
template <class Id>
__global__ void __launch_bounds__(SORT_THREADS) k_count_digits(SortInput<Id> in, SortPass s,
                                                                uint32_t* counts, Clearing clearing) {
    extern __shared__ uint32_t sort_shared[];
    after_previous_launch();
    next_launch_may_begin();
    clear_words(clearing.words, s.from, s.to, int64_t(blockIdx.x) * SORT_THREADS + threadIdx.x,
                int64_t(gridDim.x) * SORT_THREADS);
    if (threadIdx.x < s.bins) sort_shared[threadIdx.x] = 0;
    __syncthreads();
    const uint64_t per_tile = uint64_t(s.per_warp) * SORT_WARPS, start = blockIdx.x * per_tile;
    const uint32_t lo = uint32_t(start < s.tokens ? start : s.tokens);
    const uint32_t hi = uint32_t(start + per_tile < s.tokens ? start + per_tile : s.tokens);
    count_digits(in, lo + threadIdx.x, hi, SORT_THREADS, s.shift, s.bins - 1, sort_shared);
    __syncthreads();
    if (threadIdx.x < s.bins) counts[blockIdx.x * s.bins + threadIdx.x] = sort_shared[threadIdx.x];
}

// The second replaces the tiles' counts of each digit by their exclusive prefix
// over the tiles and writes the digits' totals behind them: a warp a digit. (Were
// each CTA of the third to sum them itself, all of them would read 45 MB from L2
// where 148 tiles have 512 digits, 9 us.)
__global__ void __launch_bounds__(256) k_scan_counts(uint32_t* counts, uint32_t tiles, uint32_t bins) {
    const uint32_t bin = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
    after_previous_launch();
    next_launch_may_begin();
    if (bin >= bins) return;
    uint32_t sum = 0;
    for (uint32_t base = 0; base < tiles; base += 32 * 8) {
        uint32_t n[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const uint32_t tile = base + u * 32 + lane;
            n[u] = tile < tiles ? counts[tile * bins + bin] : 0;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            uint32_t scan = n[u];
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const uint32_t v = __shfl_up_sync(~0u, scan, d);
                if (lane >= uint32_t(d)) scan += v;
            }
            const uint32_t tile = base + u * 32 + lane;
            if (tile < tiles) counts[tile * bins + bin] = sum + scan - n[u];
            sum += __shfl_sync(~0u, scan, 31);
        }
    }
    if (lane == 0) counts[tiles * bins + bin] = sum;
}

// The third sorts its tile by the digit in shared memory and writes it out from
// there, so that pairs of a digit leave side by side: 13 us for 1M pairs, half of
// it the votes and trips to shared memory that keep the order; written straight to
// their places, as two words, they took 27.
template <class Id>
__global__ void __launch_bounds__(SORT_THREADS) k_place_tokens(SortInput<Id> in, SortPass s,
                                                                const uint32_t* counts, uint2* out, Clearing clearing) {
    extern __shared__ uint32_t sort_shared[];
    __shared__ uint32_t warp_sums[SORT_WARPS], shift_of[SORT_THREADS];
    uint2* staged = reinterpret_cast<uint2*>(sort_shared);  // the tile
    const uint32_t per_tile = s.per_warp * SORT_WARPS;
    uint32_t* histogram = sort_shared + 2 * per_tile;  // [warp][bin]
    after_previous_launch();
    next_launch_may_begin();
    clear_words(clearing.words, s.from, s.to, int64_t(blockIdx.x) * SORT_THREADS + threadIdx.x,
                int64_t(gridDim.x) * SORT_THREADS);
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, bin = threadIdx.x;
    for (uint32_t i = threadIdx.x; i < SORT_WARPS * s.bins; i += SORT_THREADS) histogram[i] = 0;
    const uint32_t prefix = bin < s.bins ? counts[blockIdx.x * s.bins + bin] : 0;
    const uint32_t total = bin < s.bins ? counts[gridDim.x * s.bins + bin] : 0;
    __syncthreads();
    const uint64_t tile = uint64_t(blockIdx.x) * per_tile, start = tile + uint64_t(warp) * s.per_warp;
    const uint32_t lo = uint32_t(start < s.tokens ? start : s.tokens);
    const uint32_t hi = uint32_t(start + s.per_warp < s.tokens ? start + s.per_warp : s.tokens);
    count_digits(in, lo + lane, hi, 32, s.shift, s.bins - 1, histogram + warp * s.bins);
    const uint32_t base = prefix_block(total, warp_sums) + prefix;  // where the tile's pairs of the digit go
    __syncthreads();
    const uint32_t mine = prefix_warps(histogram, s.bins);
    const uint32_t local = prefix_block(mine, warp_sums);  // and where they are staged
    if (bin < s.bins) shift_of[bin] = base - local;
    add_to_warps(histogram, s.bins, local);
    __syncthreads();
    place_pairs(in, lo, hi, s.shift, s.bins - 1, histogram + warp * s.bins, staged);
    __syncthreads();
    const uint32_t count = tile < s.tokens ? uint32_t(s.tokens - tile < per_tile ? s.tokens - tile : per_tile) : 0;
    for (uint32_t i = threadIdx.x; i < count; i += SORT_THREADS) {
        const uint2 pair = staged[i];
        out[i + shift_of[(pair.x >> s.shift) & (s.bins - 1)]] = pair;
    }
}

constexpr uint32_t NO_ROW = 0xffffffffu;

// Segmented sums over the sorted tokens. A group of `lanes` lanes looks after
// `chunk` consecutive sorted tokens and `lanes` vectors of V channels: it adds the
// gradients of each run of equal rows that begins in the chunk, in FP32 and in
// token order, on into the next chunk where the run ends there. A run that covers
// a whole chunk behind the one in which it begins is long: each chunk writes
// what it has of it to partial[chunk][0] (or [1] where it begins), and
// k_join_chunks adds those: through partial sums for every run that crosses a
// border, sums and joins of 1M x 8 f32 took 31 us and not 22. Bound by memory where
// rows are wide: 32768 x 2048 bf16 into 128000 rows (634 MB with the rows cleared
// beside) in 100 us, 6.3 TB/s.
constexpr int SUM_BATCH = 8;
struct SumShape {
    uint32_t tokens, rows, chunk, chunks, vectors, lanes, tiles;
    uint32_t sum_blocks, clear_from;  // blocks that sum; the first row that the others clear
    int64_t channels, grad_stride;
};

template <class TI, class TO, int V>
__global__ void __launch_bounds__(256) k_sum_tokens(const uint2* pairs, const TI* __restrict__ grad, TO* out,
                                                     float* partial, SumShape s, Clearing clearing, float scale) {
    after_previous_launch();
    next_launch_may_begin();
    if (blockIdx.x >= s.sum_blocks) {
        // Rows without a token: a lane looks for a row among the sorted tokens, then
        // the warp clears those that are not there.
        const uint32_t lane = threadIdx.x % 32, warps = (gridDim.x - s.sum_blocks) * 8;
        const int64_t row_words = s.channels * sizeof(TO) / 16;
        for (uint32_t base = s.clear_from + ((blockIdx.x - s.sum_blocks) * 8 + threadIdx.x / 32) * 32; base < s.rows;
             base += warps * 32) {
            uint32_t lo = 0, hi = s.tokens;  // the first token whose row is not below
            while (lo < hi) {
                const uint32_t middle = lo + (hi - lo) / 2;
                if (pairs[middle].x < base + lane) lo = middle + 1;
                else hi = middle;
            }
            const bool absent = base + lane < s.rows && (lo == s.tokens || pairs[lo].x != base + lane);
            for (uint32_t which = __ballot_sync(~0u, absent); which; which &= which - 1) {
                uint4* to = clearing.words + int64_t(base + __ffs(which) - 1) * row_words;
                for (int64_t i = lane; i < row_words; i += 32) to[i] = make_uint4(0, 0, 0, 0);
            }
        }
        return;
    }
    const uint64_t group = (uint64_t(blockIdx.x) * 256 + threadIdx.x) / s.lanes;
    const uint32_t chunk = uint32_t(group / s.tiles), tile = uint32_t(group - uint64_t(chunk) * s.tiles);
    const uint32_t vector = tile * s.lanes + threadIdx.x % s.lanes;
    if (chunk >= s.chunks || vector >= s.vectors) return;
    const int64_t column = int64_t(vector) * V;
    const uint32_t lo = chunk * s.chunk, end = min(lo + s.chunk, s.tokens);
    auto row_at = [&](uint32_t i) { return pairs[i].x; };
    uint32_t current = row_at(lo);
    if (current >= s.rows) return;
    const uint32_t last = row_at(end - 1);
    const bool continued = lo && row_at(lo - 1) == current;  // began in a chunk before
    // Whether the run that ends the chunk, if it begins here, is long; and the one
    // that begins the chunk, if it began before: it covers this chunk, or it
    // covers the one before and began before that.
    const bool tail_long = end + s.chunk <= s.tokens && row_at(end + s.chunk - 1) == last;
    const bool head_long = continued && ((last == current && end - lo == s.chunk) ||
                                         (lo > s.chunk && row_at(lo - s.chunk - 1) == current));
    uint32_t stop = end;  // of what this group adds
    if (!tail_long && end < s.tokens && last < s.rows && row_at(end) == last && !(continued && last == current))
        stop = min(end + s.chunk, s.tokens);
    int state = continued ? (head_long ? 1 : 2) : 0;  // of the run at hand: 1 to partial[0], 2 another's, 0 own
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.0f;
    auto to_partial = [&](int which) {
        store<float, V>(partial + (int64_t(chunk) * 2 + which) * s.channels + column, pack<float, V>(sum));
    };
    auto flush = [&] {
        if (state == 1) {
            to_partial(0);
        } else if (state == 0) {
            float f[V];
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = sum[j] * scale;
            store<TO, V>(out + int64_t(current) * s.channels + column, pack<TO, V>(f));
        }
    };
    bool done = false;
    for (uint32_t at = lo; at < stop && !done; at += SUM_BATCH) {
        // `at` is a multiple of SUM_BATCH, and the buffers are padded to it.
        uint32_t r[SUM_BATCH], from[SUM_BATCH];
        Vector<TI, V> v[SUM_BATCH];
#pragma unroll
        for (int u = 0; u < SUM_BATCH; u += 2) {
            const uint4 a = *reinterpret_cast<const uint4*>(pairs + at + u);
            r[u] = a.x, from[u] = a.y, r[u + 1] = a.z, from[u + 1] = a.w;
        }
#pragma unroll
        for (int u = 0; u < SUM_BATCH; ++u) {
            // Behind the chunk only its last run goes on.
            if (at + u >= stop || (at + u >= end && r[u] != last)) r[u] = NO_ROW;
            const bool wanted = r[u] < s.rows && !(state == 2 && r[u] == current);
            v[u] = wanted ? load<TI, V>(grad + int64_t(from[u]) * s.grad_stride + column) : zeros<TI, V>();
        }
#pragma unroll
        for (int u = 0; u < SUM_BATCH; ++u) {
            if (r[u] != current && !done) {
                if (r[u] == NO_ROW) {
                    done = true;
                } else {
                    flush();
                    current = r[u];
                    state = 0;
#pragma unroll
                    for (int j = 0; j < V; ++j) sum[j] = 0.0f;
                    done = current >= s.rows;
                }
            }
            float f[V];
            unpack<TI, V>(v[u], f);
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += done ? 0.0f : f[j];
        }
    }
    if (current >= s.rows) return;
    if (state == 0 && tail_long && current == last)
        to_partial(1);
    else
        flush();
}

// Long runs: the block of the chunk in which such a run begins adds its partial
// sums in a tile of `lanes` times V columns. A warp takes a run, its lanes
// sharing the chunks where the columns leave lanes over; runs of over JOIN_LONG
// chunks are shared by the block's warps. All orders are fixed by the sizes and
// the ids.
constexpr int JOIN_WARPS = 8, JOIN_CHUNKS = 32;
constexpr uint32_t JOIN_LONG = 8;

template <int V>
__device__ __forceinline__ void add_chunks(const float* partial, int64_t channels, int64_t column,
                                           uint32_t first, uint32_t last, uint32_t step, float (&sum)[V]) {
#pragma unroll 8
    for (uint32_t c = first; c <= last; c += step) {
        float f[V];
        unpack<float, V>(load_written<float, V>(partial + int64_t(c) * 2 * channels + column), f);
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] += f[j];
    }
}

template <class TO, int V>
__global__ void __launch_bounds__(JOIN_WARPS * 32) k_join_chunks(const uint2* pairs, TO* out, const float* partial,
                                                                  SumShape s, float scale) {
    __shared__ uint32_t starts[JOIN_CHUNKS], rows[JOIN_CHUNKS], lasts[JOIN_CHUNKS], found;
    __shared__ float sums[JOIN_WARPS][32 * V];
    after_previous_launch();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    auto row_at = [&](uint32_t i) { return pairs[i].x; };
    if (warp == 0) {  // a lane a chunk
        const uint32_t chunk = blockIdx.x * JOIN_CHUNKS + lane, lo = chunk * s.chunk, end = lo + s.chunk;
        uint32_t r = NO_ROW, last = chunk + 1;
        if (chunk + 1 < s.chunks && end + s.chunk <= s.tokens) {
            r = row_at(end - 1);
            if (r >= s.rows || row_at(end + s.chunk - 1) != r || (lo && row_at(lo) == r && row_at(lo - 1) == r)) r = NO_ROW;
        }
        if (r != NO_ROW) {
            // The last chunk that begins with row r: by doubled steps, then by halving.
            uint32_t step = 1;
            while (last + step < s.chunks && row_at((last + step) * s.chunk) == r) {
                last += step;
                step *= 2;
            }
            uint32_t beyond = min(last + step, s.chunks);
            while (beyond - last > 1) {
                const uint32_t middle = last + (beyond - last) / 2;
                if (row_at(middle * s.chunk) == r) last = middle;
                else beyond = middle;
            }
        }
        const uint32_t which = __ballot_sync(~0u, r != NO_ROW);
        if (r != NO_ROW) {
            const uint32_t at = __popc(which & ((1u << lane) - 1));
            starts[at] = chunk;
            rows[at] = r;
            lasts[at] = last;
        }
        if (lane == 0) found = __popc(which);
    }
    __syncthreads();
    if (!found) return;
    const uint32_t x = lane % s.lanes, y = lane / s.lanes, ys = 32 / s.lanes;
    const uint32_t vector = blockIdx.y * s.lanes + x;
    const int64_t column = int64_t(vector) * V;
    const bool inside = vector < s.vectors;
    float sum[V];
    auto start = [&](bool begins, uint32_t from) {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] = 0.0f;
        if (begins && inside && y == 0)
            unpack<float, V>(load_written<float, V>(partial + (int64_t(from) * 2 + 1) * s.channels + column), sum);
    };
    auto write = [&](uint32_t r) {
        for (uint32_t d = 16; d >= s.lanes; d /= 2) {
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += __shfl_down_sync(~0u, sum[j], d);
        }
        if (y == 0 && inside) {
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] *= scale;
            store<TO, V>(out + int64_t(r) * s.channels + column, pack<TO, V>(sum));
        }
    };
    for (uint32_t i = warp; i < found; i += JOIN_WARPS) {
        if (lasts[i] - starts[i] > JOIN_LONG) continue;
        start(true, starts[i]);
        if (inside) add_chunks<V>(partial, s.channels, column, starts[i] + 1 + y, lasts[i], ys, sum);
        write(rows[i]);
    }
    for (uint32_t i = 0; i < found; ++i) {
        if (lasts[i] - starts[i] <= JOIN_LONG) continue;
        start(warp == 0, starts[i]);
        if (inside)
            add_chunks<V>(partial, s.channels, column, starts[i] + 1 + warp * ys + y, lasts[i], JOIN_WARPS * ys, sum);
#pragma unroll
        for (int j = 0; j < V; ++j) sums[warp][lane * V + j] = sum[j];
        __syncthreads();
        if (warp == 0) {
            for (int k = 1; k < JOIN_WARPS; ++k) {
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] += sums[k][lane * V + j];
            }
            write(rows[i]);
        }
        __syncthreads();
    }
}

// Few tokens and a small table: one launch. Each block sorts all tokens in shared
// memory (a bitonic network over keys (row, token), a thread a key; keys differ,
// so that the order is the ids'), and clears and sums its own columns of the rows
// r with r % gridDim.y = blockIdx.y, a group of lanes a run: most groups then wait
// for one run's gradients instead of several in turn.
constexpr int SMALL_TOKENS = 1024, SMALL_BITS = 10;
constexpr int64_t SMALL_TABLE = 1 << 18;  // elements; a row fits in the key's other 22 bits
template <class TI, class TO, class Id, int V>
__global__ void __launch_bounds__(SMALL_TOKENS) k_small_gradient(const TI* __restrict__ grad, int64_t grad_stride,
                                                                  const Id* __restrict__ ids, uint32_t tokens,
                                                                  uint32_t size, int64_t rows, int64_t channels,
                                                                  uint32_t vectors, uint32_t lanes,
                                                                  TO* __restrict__ out, float scale) {
    __shared__ uint32_t keys[2][SMALL_TOKENS];
    const uint32_t vector = blockIdx.x * lanes + threadIdx.x % lanes;
    const uint32_t group = threadIdx.x / lanes, groups = blockDim.x / lanes;
    const bool inside = vector < vectors;
    const int64_t column = int64_t(vector) * V;
    const uint32_t t = threadIdx.x;
    uint32_t key = t < tokens ? row_of(ids[t], rows) << SMALL_BITS | t : ~0u;
    if (inside)
        for (int64_t r = blockIdx.y + group * gridDim.y; r < rows; r += groups * gridDim.y)
            store<TO, V>(out + r * channels + column, zeros<TO, V>());
    int buffer = 0;
    for (uint32_t k = 2; k <= size; k *= 2)
        for (uint32_t j = k / 2; j; j /= 2) {
            uint32_t other;
            if (j < 32) {
                other = __shfl_xor_sync(~0u, key, j);
            } else {  // between warps; the two buffers alternate, so that one barrier a step does
                keys[buffer][t] = key;
                __syncthreads();
                other = keys[buffer][t ^ j];
                buffer ^= 1;
            }
            key = ((t & j) == 0) == ((t & k) == 0) ? min(key, other) : max(key, other);
        }
    uint32_t* sorted = keys[buffer];
    sorted[t] = key;
    __syncthreads();
    if (!inside) return;
    for (uint32_t i = group; i < tokens; i += groups) {
        const uint32_t row = sorted[i] >> SMALL_BITS;
        if (row >= rows || row % gridDim.y != blockIdx.y || (i && sorted[i - 1] >> SMALL_BITS == row)) continue;
        float sum[V];
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] = 0.0f;
        for (uint32_t at = i; at < tokens && sorted[at] >> SMALL_BITS == row; at += SUM_BATCH) {
            Vector<TI, V> v[SUM_BATCH];
#pragma unroll
            for (int u = 0; u < SUM_BATCH; ++u) {
                const bool mine = at + u < tokens && sorted[at + u] >> SMALL_BITS == row;
                v[u] = mine ? load<TI, V>(grad + int64_t(sorted[at + u] % SMALL_TOKENS) * grad_stride + column) : zeros<TI, V>();
            }
#pragma unroll
            for (int u = 0; u < SUM_BATCH; ++u) {
                float f[V];
                unpack<TI, V>(v[u], f);
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] += f[j];
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] *= scale;
        store<TO, V>(out + int64_t(row) * channels + column, pack<TO, V>(sum));
    }
}

}  // namespace cpde::ops
