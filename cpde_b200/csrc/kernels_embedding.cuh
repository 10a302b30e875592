// Embedding lookup with scaling, and its gradient by sorted tokens.
#pragma once
#include <cooperative_groups.h>

#include "device_vector.cuh"

namespace cpde::ops {

// out[t,:] = scale * table[ids[t],:]; an id outside [0, rows) is absent and
// gives a zero row. A thread has LOOKUPS vectors of V channels, a block's
// vectors apart, so that its loads of ids and then of rows are in flight
// together.
constexpr int LOOKUPS = 4;
template <class TI, class TO, class Id, int V>
__global__ void __launch_bounds__(256) k_embedding(const TI* __restrict__ table, int64_t table_stride, int64_t rows,
                                                    const Id* __restrict__ ids, TO* __restrict__ out,
                                                    int64_t channels, Divisor vectors, uint32_t count, float scale) {
    const uint32_t base = blockIdx.x * (256 * LOOKUPS) + threadIdx.x;
    int64_t source[LOOKUPS];
#pragma unroll
    for (int u = 0; u < LOOKUPS; ++u) {
        const uint32_t i = base + u * 256;
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
        const uint32_t i = base + u * 256;
        if (i >= count) continue;
        float f[V];
        unpack<TI, V>(v[u], f);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = source[u] >= 0 ? f[j] * scale : 0.0f;
        store<TO, V>(out + int64_t(i) * V, pack<TO, V>(f));
    }
}

// --- gradient: tokens sorted by row --------------------------------------

constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;

// Two buffers of (row, token) pairs that the passes of the sort alternate
// between, pass p writing buffer p % 2.
struct SortBuffers {
    uint32_t* row[2];
    uint32_t* token[2];
};
__host__ __device__ inline int sorted_buffer(int passes) { return (passes - 1) & 1; }

// Row of a token; absent ids sort behind every row, as row `rows`.
template <class Id>
__device__ __forceinline__ uint32_t row_of(Id id, int64_t rows) {
    return uint32_t(int64_t(id) >= 0 && int64_t(id) < rows ? int64_t(id) : rows);
}

// What a pass of the sort reads: the ids themselves at first, then the pairs
// that the pass before wrote.
template <class Id>
struct SortInput {
    const Id* ids;
    int64_t rows;
    const uint32_t *row, *token;  // null in the first pass
    __device__ __forceinline__ uint32_t row_at(uint32_t i) const { return row ? row[i] : row_of(ids[i], rows); }
    __device__ __forceinline__ uint32_t token_at(uint32_t i) const { return row ? token[i] : i; }
};

// A pass is stable because each warp has a contiguous range of the pairs: a
// pair's place is (smaller digits anywhere) + (its digit in the CTAs before) +
// (in the warps before) + (before it in its warp, from a match over the lanes).
// No order depends on timing. SORT_BATCH loads of a lane are in flight at once.
constexpr int SORT_BATCH = 8;

template <class Id>
__device__ __forceinline__ void count_digits(const SortInput<Id>& in, uint32_t lo, uint32_t hi, uint32_t step,
                                             int shift, uint32_t mask, uint32_t* histogram) {
    for (uint32_t at = lo; at < hi; at += SORT_BATCH * step) {
        uint32_t r[SORT_BATCH];
#pragma unroll
        for (int u = 0; u < SORT_BATCH; ++u) r[u] = at + u * step < hi ? in.row_at(at + u * step) : 0;
#pragma unroll
        for (int u = 0; u < SORT_BATCH; ++u)
            if (at + u * step < hi) atomicAdd(&histogram[(r[u] >> shift) & mask], 1u);
    }
}

// `place`: this warp's next place for each digit.
template <class Id>
__device__ __forceinline__ void place_pairs(const SortInput<Id>& in, uint32_t lo, uint32_t hi, int shift,
                                            uint32_t mask, uint32_t* place, uint32_t* __restrict__ row_out,
                                            uint32_t* __restrict__ token_out) {
    const uint32_t lane = threadIdx.x % 32;
    for (uint32_t at = lo; at < hi; at += SORT_BATCH * 32) {
        uint32_t r[SORT_BATCH], token[SORT_BATCH];
#pragma unroll
        for (int u = 0; u < SORT_BATCH; ++u) {
            const uint32_t i = at + u * 32 + lane;
            r[u] = i < hi ? in.row_at(i) : 0;
            token[u] = i < hi ? in.token_at(i) : 0;
        }
#pragma unroll
        for (int u = 0; u < SORT_BATCH; ++u) {
            const bool active = at + u * 32 + lane < hi;
            const uint32_t lanes = __ballot_sync(~0u, active);
            if (active) {
                const uint32_t digit = (r[u] >> shift) & mask;
                const uint32_t peers = __match_any_sync(lanes, digit);
                const uint32_t mine = __popc(peers & ((1u << lane) - 1));
                const uint32_t to = place[digit] + mine;
                __syncwarp(lanes);
                if (mine == 0) place[digit] += __popc(peers);
                row_out[to] = r[u];
                token_out[to] = token[u];
            }
            __syncwarp();
        }
    }
}

// Exclusive prefix of the warps' counts by digit in shared memory, which become
// places within the CTA; returns the CTA's count of digit threadIdx.x.
__device__ __forceinline__ uint32_t prefix_warps(uint32_t* histogram, uint32_t bins) {
    uint32_t sum = 0;
    if (threadIdx.x < bins)
        for (int w = 0; w < SORT_WARPS; ++w) {
            const uint32_t n = histogram[w * bins + threadIdx.x];
            histogram[w * bins + threadIdx.x] = sum;
            sum += n;
        }
    return sum;
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

__device__ __forceinline__ void clear_words(uint4* words, int64_t from, int64_t to, int64_t first, int64_t step) {
    for (int64_t i = from + first; i < to; i += step) words[i] = make_uint4(0, 0, 0, 0);
}

// Few tokens: all passes in one launch, by the first cluster of the grid, whose
// CTAs exchange their counts through distributed shared memory; the other
// clusters clear `fill` meanwhile.
template <class Id>
__global__ void __launch_bounds__(SORT_THREADS) k_sort_tokens(const Id* __restrict__ ids, uint32_t tokens,
                                                               int64_t rows, int passes, int digit_bits,
                                                               SortBuffers buffers, uint4* __restrict__ fill,
                                                               int64_t fill_words) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t size = cluster.num_blocks();
    if (blockIdx.x >= size) {
        clear_words(fill, 0, fill_words, int64_t(blockIdx.x - size) * SORT_THREADS + threadIdx.x,
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
        const int shift = pass * digit_bits, from = (pass + 1) & 1, to = pass & 1;
        const SortInput<Id> in = {ids, rows, pass ? buffers.row[from] : nullptr, buffers.token[from]};
        for (uint32_t i = threadIdx.x; i < SORT_WARPS * bins; i += SORT_THREADS) histogram[i] = 0;
        __syncthreads();
        count_digits(in, lo + lane, hi, 32, shift, bins - 1, histogram + warp * bins);
        __syncthreads();
        const uint32_t mine = prefix_warps(histogram, bins);
        if (bin < bins) totals[bin] = mine;
        cluster.sync();
        uint32_t before = 0, all = 0;
        if (bin < bins)
            for (uint32_t c = 0; c < size; ++c) {
                const uint32_t n = cluster.map_shared_rank(totals, c)[bin];
                before += c < rank ? n : 0;
                all += n;
            }
        const uint32_t base = prefix_block(all, warp_sums) + before;
        if (bin < bins)
            for (int w = 0; w < SORT_WARPS; ++w) histogram[w * bins + bin] += base;
        __syncthreads();
        place_pairs(in, lo, hi, shift, bins - 1, histogram + warp * bins, buffers.row[to], buffers.token[to]);
        // Orders this pass's pairs in global memory, and its reads of the other
        // CTAs' totals, before the next pass's.
        __threadfence();
        cluster.sync();
    }
}

// Many tokens: a pass is two launches over the whole GPU. The first counts the
// digits of each tile (a CTA's range of pairs).
struct SortPass {
    uint32_t tokens, per_warp, bins;
    int shift;
    int64_t fill_from, fill_to;  // the words of the output that this launch clears
};
template <class Id>
__global__ void __launch_bounds__(SORT_THREADS) k_count_digits(SortInput<Id> in, SortPass s,
                                                                uint32_t* __restrict__ counts,
                                                                uint4* __restrict__ fill) {
    extern __shared__ uint32_t sort_shared[];
    clear_words(fill, s.fill_from, s.fill_to, int64_t(blockIdx.x) * SORT_THREADS + threadIdx.x,
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

// The second sums the tiles' counts (each CTA all of them: they stay in L2) and
// places the pairs.
template <class Id>
__global__ void __launch_bounds__(SORT_THREADS) k_place_tokens(SortInput<Id> in, SortPass s,
                                                                const uint32_t* __restrict__ counts,
                                                                uint32_t* __restrict__ row_out,
                                                                uint32_t* __restrict__ token_out,
                                                                uint4* __restrict__ fill) {
    extern __shared__ uint32_t sort_shared[];
    __shared__ uint32_t warp_sums[SORT_WARPS], sums[2][SORT_THREADS];
    uint32_t* histogram = sort_shared;  // [warp][bin]
    clear_words(fill, s.fill_from, s.fill_to, int64_t(blockIdx.x) * SORT_THREADS + threadIdx.x,
                int64_t(gridDim.x) * SORT_THREADS);
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, bin = threadIdx.x & (s.bins - 1);
    for (uint32_t i = threadIdx.x; i < SORT_WARPS * s.bins; i += SORT_THREADS) histogram[i] = 0;
    __syncthreads();
    const uint64_t start = (uint64_t(blockIdx.x) * SORT_WARPS + warp) * s.per_warp;
    const uint32_t lo = uint32_t(start < s.tokens ? start : s.tokens);
    const uint32_t hi = uint32_t(start + s.per_warp < s.tokens ? start + s.per_warp : s.tokens);
    count_digits(in, lo + lane, hi, 32, s.shift, s.bins - 1, histogram + warp * s.bins);
    // Threads with equal bin share the tiles.
    const uint32_t share = threadIdx.x / s.bins, shares = SORT_THREADS / s.bins;
    uint32_t before = 0, all = 0;
#pragma unroll 16
    for (uint32_t tile = share; tile < gridDim.x; tile += shares) {
        const uint32_t n = counts[tile * s.bins + bin];
        before += tile < blockIdx.x ? n : 0;
        all += n;
    }
    sums[0][threadIdx.x] = before;
    sums[1][threadIdx.x] = all;
    __syncthreads();
    prefix_warps(histogram, s.bins);
    before = all = 0;
    if (threadIdx.x < s.bins)
        for (uint32_t i = threadIdx.x; i < SORT_THREADS; i += s.bins) {
            before += sums[0][i];
            all += sums[1][i];
        }
    const uint32_t base = prefix_block(all, warp_sums) + before;
    if (threadIdx.x < s.bins)
        for (int w = 0; w < SORT_WARPS; ++w) histogram[w * s.bins + threadIdx.x] += base;
    __syncthreads();
    place_pairs(in, lo, hi, s.shift, s.bins - 1, histogram + warp * s.bins, row_out, token_out);
}

constexpr uint32_t NO_ROW = 0xffffffffu;

// Segmented sums over the sorted tokens. A group of `lanes` lanes has `chunk`
// consecutive sorted tokens and `lanes` vectors of V channels, and adds the
// gradients of a run of equal rows in FP32, in token order. A run inside the
// chunk is written to the table's gradient; what a run that crosses a chunk's
// border has in this chunk goes to partial[chunk][0] (runs that began before)
// or partial[chunk][1] (runs that begin here and go on).
constexpr int SUM_BATCH = 8;
struct SumShape {
    uint32_t tokens, rows, chunk, chunks, vectors, lanes, tiles;
    int64_t channels, grad_stride;
};
template <class TI, class TO, int V>
__global__ void __launch_bounds__(256) k_sum_tokens(const uint32_t* __restrict__ row, const uint32_t* __restrict__ token,
                                                     const TI* __restrict__ grad, TO* __restrict__ out,
                                                     float* __restrict__ partial, SumShape s, float scale) {
    const uint64_t group = (uint64_t(blockIdx.x) * 256 + threadIdx.x) / s.lanes;
    const uint32_t chunk = uint32_t(group / s.tiles), tile = uint32_t(group - uint64_t(chunk) * s.tiles);
    const uint32_t vector = tile * s.lanes + threadIdx.x % s.lanes;
    if (chunk >= s.chunks || vector >= s.vectors) return;
    const int64_t column = int64_t(vector) * V;
    const uint32_t lo = chunk * s.chunk, hi = min(lo + s.chunk, s.tokens);
    const uint32_t before = lo ? row[lo - 1] : NO_ROW, after = hi < s.tokens ? row[hi] : NO_ROW;
    uint32_t current = row[lo];
    bool continued = current == before;
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.0f;
    auto to_partial = [&](int which) {
        store<float, V>(partial + (int64_t(chunk) * 2 + which) * s.channels + column, pack<float, V>(sum));
    };
    auto flush = [&] {
        if (continued) {
            to_partial(0);
        } else {
            float f[V];
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = sum[j] * scale;
            store<TO, V>(out + int64_t(current) * s.channels + column, pack<TO, V>(f));
        }
    };
    for (uint32_t at = lo; at < hi && current < s.rows; at += SUM_BATCH) {
        // `at` is a multiple of SUM_BATCH, and the buffers are padded to it.
        uint32_t r[SUM_BATCH], from[SUM_BATCH];
        Vector<TI, V> v[SUM_BATCH];
#pragma unroll
        for (int u = 0; u < SUM_BATCH; u += 4) {
            const uint4 a = *reinterpret_cast<const uint4*>(row + at + u);
            const uint4 b = *reinterpret_cast<const uint4*>(token + at + u);
            r[u] = a.x, r[u + 1] = a.y, r[u + 2] = a.z, r[u + 3] = a.w;
            from[u] = b.x, from[u + 1] = b.y, from[u + 2] = b.z, from[u + 3] = b.w;
        }
#pragma unroll
        for (int u = 0; u < SUM_BATCH; ++u) {
            if (at + u >= hi) r[u] = NO_ROW;
            v[u] = r[u] < s.rows ? load<TI, V>(grad + int64_t(from[u]) * s.grad_stride + column) : zeros<TI, V>();
        }
#pragma unroll
        for (int u = 0; u < SUM_BATCH; ++u) {
            if (r[u] == NO_ROW) break;
            if (r[u] != current) {
                flush();
                current = r[u];
                continued = false;
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] = 0.0f;
                if (current >= s.rows) break;
            }
            float f[V];
            unpack<TI, V>(v[u], f);
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += f[j];
        }
    }
    if (current >= s.rows) return;
    if (current == after && !continued)
        to_partial(1);
    else
        flush();
}

// Rows whose runs cross chunk borders. A warp looks after one chunk: where such
// a run begins in it, it adds the run's partial sums in a tile of `lanes` times
// V columns, its lanes sharing the chunks where the columns leave lanes over.
// Runs of over JOIN_LONG chunks are shared by the block's warps. All orders are
// fixed by the sizes and the ids.
constexpr int JOIN_WARPS = 8;
constexpr uint32_t JOIN_LONG = 64;
struct Run {
    uint32_t row, last;  // the last chunk that begins with `row`
};

template <int V>
__device__ __forceinline__ void add_chunks(const float* __restrict__ partial, int64_t channels, int64_t column,
                                           uint32_t first, uint32_t last, uint32_t step, float (&sum)[V]) {
#pragma unroll 4
    for (uint32_t c = first; c <= last; c += step) {
        float f[V];
        unpack<float, V>(load<float, V>(partial + int64_t(c) * 2 * channels + column), f);
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] += f[j];
    }
}

template <class TO, int V>
__global__ void __launch_bounds__(JOIN_WARPS * 32) k_join_chunks(const uint32_t* __restrict__ row,
                                                                  TO* __restrict__ out,
                                                                  const float* __restrict__ partial, SumShape s,
                                                                  float scale) {
    __shared__ Run runs[JOIN_WARPS];
    __shared__ float sums[JOIN_WARPS][32 * V];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t chunk = blockIdx.x * JOIN_WARPS + warp;
    Run run = {NO_ROW, 0};
    if (chunk + 1 < s.chunks) {
        const uint32_t lo = chunk * s.chunk, hi = lo + s.chunk, r = row[hi - 1];
        if (r < s.rows && row[hi] == r && !(lo && row[lo] == r && row[lo - 1] == r)) {
            uint32_t first = chunk + 1, last = chunk + 1;  // gallop, then halve
            for (uint32_t step = 1; last + step < s.chunks && row[(last + step) * s.chunk] == r; step *= 2) last += step;
            first = last;
            uint32_t end = s.chunks - 1 - last < last - chunk + 1 ? s.chunks - 1 : last + (last - chunk + 1);
            while (first < end) {
                const uint32_t middle = first + (end - first + 1) / 2;
                if (row[middle * s.chunk] == r) first = middle;
                else end = middle - 1;
            }
            run = {r, first};
        }
    }
    const uint32_t x = lane % s.lanes, y = lane / s.lanes, ys = 32 / s.lanes;
    const uint32_t vector = blockIdx.y * s.lanes + x;
    const int64_t column = int64_t(vector) * V;
    const bool inside = vector < s.vectors;
    const bool is_long = run.row != NO_ROW && run.last - chunk > JOIN_LONG;
    float sum[V];
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
    auto start = [&](uint32_t from) {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] = 0.0f;
        if (inside && y == 0)
            unpack<float, V>(load<float, V>(partial + (int64_t(from) * 2 + 1) * s.channels + column), sum);
    };
    if (run.row != NO_ROW && !is_long) {
        start(chunk);
        if (inside) add_chunks<V>(partial, s.channels, column, chunk + 1 + y, run.last, ys, sum);
        write(run.row);
    }
    if (lane == 0) runs[warp] = is_long ? run : Run{NO_ROW, 0};
    __syncthreads();
    for (uint32_t w = 0; w < JOIN_WARPS; ++w) {
        const Run r = runs[w];
        if (r.row == NO_ROW) continue;
        const uint32_t from = blockIdx.x * JOIN_WARPS + w;
        if (warp == 0) {
            start(from);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] = 0.0f;
        }
        if (inside) add_chunks<V>(partial, s.channels, column, from + 1 + warp * ys + y, r.last, JOIN_WARPS * ys, sum);
#pragma unroll
        for (int j = 0; j < V; ++j) sums[warp][lane * V + j] = sum[j];
        __syncthreads();
        if (warp == 0) {
            for (int k = 1; k < JOIN_WARPS; ++k) {
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] += sums[k][lane * V + j];
            }
            write(r.row);
        }
        __syncthreads();
    }
}

}  // namespace cpde::ops
