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
// between; the last pass ends in buffer 1 - passes % 2 ... see sorted_buffer().
struct SortBuffers {
    uint32_t* row[2];
    uint32_t* token[2];
};
__host__ __device__ inline int sorted_buffer(int passes) { return (passes - 1) & 1; }

// Stable radix sort of the tokens by row, least significant digit first, by the
// first cluster of the grid; the other clusters clear `fill` meanwhile. Each
// warp keeps a contiguous range of the pairs, so a pair's place in its digit is
// (digits below) + (same digit in CTAs before) + (in warps before) + (in its
// warp before, from a match over the lanes): no order depends on timing.
// Absent ids sort behind every row, as row `rows`.
template <class Id>
__global__ void __launch_bounds__(SORT_THREADS) k_sort_tokens(const Id* __restrict__ ids, uint32_t tokens,
                                                               int64_t rows, int passes, int digit_bits,
                                                               SortBuffers buffers, uint4* __restrict__ fill,
                                                               int64_t fill_words) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t size = cluster.num_blocks();
    if (blockIdx.x >= size) {
        const int64_t step = int64_t(gridDim.x - size) * SORT_THREADS;
        for (int64_t i = int64_t(blockIdx.x - size) * SORT_THREADS + threadIdx.x; i < fill_words; i += step)
            fill[i] = make_uint4(0, 0, 0, 0);
        return;
    }
    extern __shared__ uint32_t sort_shared[];
    const uint32_t bins = 1u << digit_bits;
    uint32_t* histogram = sort_shared;                   // [warp][bin]
    uint32_t* totals = histogram + SORT_WARPS * bins;    // [bin]: this CTA's
    __shared__ uint32_t warp_sums[SORT_WARPS];
    const uint32_t rank = cluster.block_rank();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t per_warp = (tokens + size * SORT_WARPS - 1) / (size * SORT_WARPS);
    const uint64_t start = uint64_t(rank * SORT_WARPS + warp) * per_warp;
    const uint32_t lo = uint32_t(start < tokens ? start : tokens);
    const uint32_t hi = uint32_t(start + per_warp < tokens ? start + per_warp : tokens);
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * digit_bits;
        const uint32_t* row_in = buffers.row[(pass + 1) & 1];
        const uint32_t* token_in = buffers.token[(pass + 1) & 1];
        uint32_t* row_out = buffers.row[pass & 1];
        uint32_t* token_out = buffers.token[pass & 1];
        auto row_at = [&](uint32_t i) {
            if (pass) return row_in[i];
            const int64_t id = int64_t(ids[i]);
            return uint32_t(id >= 0 && id < rows ? id : rows);
        };
        for (uint32_t i = threadIdx.x; i < SORT_WARPS * bins; i += SORT_THREADS) histogram[i] = 0;
        __syncthreads();
        for (uint32_t i = lo + lane; i < hi; i += 32)
            atomicAdd(&histogram[warp * bins + ((row_at(i) >> shift) & (bins - 1))], 1u);
        __syncthreads();
        const uint32_t bin = threadIdx.x;
        if (bin < bins) {
            uint32_t sum = 0;
            for (int w = 0; w < SORT_WARPS; ++w) {
                const uint32_t n = histogram[w * bins + bin];
                histogram[w * bins + bin] = sum;
                sum += n;
            }
            totals[bin] = sum;
        }
        cluster.sync();
        uint32_t before = 0, all = 0;
        if (bin < bins) {
            for (uint32_t c = 0; c < size; ++c) {
                const uint32_t n = cluster.map_shared_rank(totals, c)[bin];
                before += c < rank ? n : 0;
                all += n;
            }
        }
        uint32_t scan = all;
        for (int d = 1; d < 32; d *= 2) {
            const uint32_t n = __shfl_up_sync(~0u, scan, d);
            if (lane >= uint32_t(d)) scan += n;
        }
        if (lane == 31) warp_sums[warp] = scan;
        __syncthreads();
        if (warp == 0) {
            uint32_t s = warp_sums[lane];
            for (int d = 1; d < 32; d *= 2) {
                const uint32_t n = __shfl_up_sync(~0u, s, d);
                if (lane >= uint32_t(d)) s += n;
            }
            warp_sums[lane] = s;
        }
        __syncthreads();
        if (bin < bins) {
            const uint32_t base = scan - all + (warp ? warp_sums[warp - 1] : 0) + before;
            for (int w = 0; w < SORT_WARPS; ++w) histogram[w * bins + bin] += base;
        }
        __syncthreads();
        for (uint32_t at = lo; at < hi; at += 32) {
            const uint32_t i = at + lane;
            const bool active = i < hi;
            const uint32_t lanes = __ballot_sync(~0u, active);
            if (active) {
                const uint32_t r = row_at(i), token = pass ? token_in[i] : i;
                const uint32_t digit = (r >> shift) & (bins - 1);
                const uint32_t peers = __match_any_sync(lanes, digit);
                const uint32_t mine = __popc(peers & ((1u << lane) - 1));
                const uint32_t place = histogram[warp * bins + digit] + mine;
                __syncwarp(lanes);
                if (mine == 0) histogram[warp * bins + digit] += __popc(peers);
                row_out[place] = r;
                token_out[place] = token;
            }
            __syncwarp();
        }
        // Orders this pass's pairs in global memory, and its reads of the other
        // CTAs' totals, before the next pass's.
        __threadfence();
        cluster.sync();
    }
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
        float* p = partial + (int64_t(chunk) * 2 + which) * s.channels + column;
#pragma unroll
        for (int j = 0; j < V; ++j) p[j] = sum[j];
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
        uint32_t r[SUM_BATCH];
        Vector<TI, V> v[SUM_BATCH];
#pragma unroll
        for (int u = 0; u < SUM_BATCH; ++u) r[u] = at + u < hi ? row[at + u] : NO_ROW;
#pragma unroll
        for (int u = 0; u < SUM_BATCH; ++u)
            v[u] = r[u] < s.rows ? load<TI, V>(grad + int64_t(token[at + u]) * s.grad_stride + column)
                                 : zeros<TI, V>();
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

// Rows whose runs cross chunk borders: the block of the chunk in which such a
// run begins adds its partial sums. Thread (y, x) of the block adds those of
// every blockDim.y-th chunk for a column, and the block joins them in a fixed
// tree.
template <class TO>
__global__ void __launch_bounds__(256) k_join_chunks(const uint32_t* __restrict__ row, TO* __restrict__ out,
                                                      const float* __restrict__ partial, SumShape s, float scale) {
    __shared__ float shared[256];
    const uint32_t chunk = blockIdx.x, lo = chunk * s.chunk, hi = lo + s.chunk;
    if (hi >= s.tokens) return;
    const uint32_t r = row[hi - 1];
    if (r >= s.rows || row[hi] != r) return;
    if (lo && row[lo] == r && row[lo - 1] == r) return;  // the run began in an earlier chunk
    // The last chunk whose first token has row r.
    uint32_t first = chunk + 1, last = s.chunks - 1;
    while (first < last) {
        const uint32_t middle = (first + last + 1) / 2;
        if (row[middle * s.chunk] == r)
            first = middle;
        else
            last = middle - 1;
    }
    for (int64_t base = 0; base < s.channels; base += blockDim.x) {
        const int64_t column = base + threadIdx.x;
        float sum = 0.0f;
        if (column < s.channels) {
            if (threadIdx.y == 0) sum = partial[(int64_t(chunk) * 2 + 1) * s.channels + column];
            for (uint32_t c = chunk + 1 + threadIdx.y; c <= last; c += blockDim.y)
                sum += partial[int64_t(c) * 2 * s.channels + column];
        }
        shared[threadIdx.y * blockDim.x + threadIdx.x] = sum;
        __syncthreads();
        for (uint32_t half = blockDim.y / 2; half; half /= 2) {
            if (threadIdx.y < half)
                shared[threadIdx.y * blockDim.x + threadIdx.x] +=
                    shared[(threadIdx.y + half) * blockDim.x + threadIdx.x];
            __syncthreads();
        }
        if (threadIdx.y == 0 && column < s.channels)
            out[int64_t(r) * s.channels + column] = from_float<TO>(shared[threadIdx.x] * scale);
        __syncthreads();
    }
}

}  // namespace cpde::ops
