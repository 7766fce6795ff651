// Which tokens a row has seen (a bit per token) and how often it generated each (a 32-bit count).
//
// The ids come as the encoder leaves them: padded rows with their lengths, or flat ids with offsets.  Bits are set and
// counts are raised by atomics on whole numbers, so that the order in which they happen does not show.  An id outside
// the vocabulary is no token, a history row outside the history takes nothing.
#pragma once
#include "common.cuh"

namespace dnatok {

constexpr int HISTORY_THREADS = 256;

struct HistoryArgs {
    uint32_t* seen;               // [history_rows, words]
    int32_t* counts;              // [history_rows, width], or NULL: nothing is counted
    int64_t history_rows, width;
    int64_t n_rows, columns;      // columns: ids per padded row
    int64_t id_stride;            // ids from one padded row to the next
    const int64_t* offsets;       // [n_rows + 1] for flat ids, else NULL
    int64_t total;                // flat ids
    const int32_t* lengths;       // [n_rows] ids of each padded row, or NULL: all columns
    int32_t pad_left;
    const void* rows;             // history row of each row, or NULL: the same
    int32_t rows_bits;
};

// Row `row`'s ids lie at [lo, hi) of the ids; its history row, or -1.
__device__ __forceinline__ int64_t history_row(const HistoryArgs& a, int64_t row, int64_t* lo, int64_t* hi) {
    if (a.offsets) {
        int64_t b = a.offsets[row], e = a.offsets[row + 1];
        if (b < 0) b = 0;
        if (e > a.total) e = a.total;
        *lo = b;
        *hi = e;
    } else {
        int64_t n = a.lengths ? (int64_t)a.lengths[row] : a.columns;
        n = n < 0 ? 0 : n > a.columns ? a.columns : n;
        *lo = row * a.id_stride + (a.pad_left ? a.columns - n : 0);
        *hi = *lo + n;
    }
    int64_t h = row;
    if (a.rows) h = a.rows_bits == 64 ? static_cast<const int64_t*>(a.rows)[row] : static_cast<const int32_t*>(a.rows)[row];
    return h >= 0 && h < a.history_rows ? h : -1;
}

// A warp takes a row; its lanes take the row's ids in turn.
template <typename IdT>
__global__ void __launch_bounds__(HISTORY_THREADS)
history_add_kernel(HistoryArgs a, const IdT* __restrict__ ids) {
    const int lane = threadIdx.x & 31;
    const int64_t words = (a.width + 31) / 32;
    const int64_t warps = (int64_t)gridDim.x * (HISTORY_THREADS / 32);
    for (int64_t row = (int64_t)blockIdx.x * (HISTORY_THREADS / 32) + (threadIdx.x >> 5); row < a.n_rows; row += warps) {
        int64_t lo, hi;
        const int64_t h = history_row(a, row, &lo, &hi);
        if (h < 0) continue;
        for (int64_t i = lo + lane; i < hi; i += 32) {
            const int64_t id = (int64_t)ids[i];
            if (id < 0 || id >= a.width) continue;
            atomicOr(a.seen + h * words + (id >> 5), 1u << (id & 31));
            if (a.counts) atomicAdd(a.counts + h * a.width + id, 1);
        }
    }
}

}  // namespace dnatok
