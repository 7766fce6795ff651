// Which tokens a row has seen (a bit per token) and how often it generated each (a 32-bit count).
//
// The ids come as the encoder leaves them: padded rows with their lengths, or flat ids with offsets.  Bits are set and
// counts are raised by atomics on whole numbers, so that the order in which they happen does not show.  An id outside
// the vocabulary is no token, a history row outside the history takes nothing.
//
// What bounds it: launch latency for prompts and single tokens (256 padded rows of up to 1,000 ids: 3.7 us with the clearing of
// a new history, calls following one another in a graph), instructions and atomics in shared memory for long rows (8 rows,
// 6.2 M ids together: 8.6 us counted and 8.9 marked, 2.9 TB/s; about 24 warp instructions for 32 ids, clearing and joining the
// tables among them).
//
// Rows are divided by their mean length, which is what the host knows: one row much longer than the others is entered by few
// threads (10,000 rows of 200 ids and one of 1,000,000: 1,220 us, for 24 MB of ids).
#pragma once
#include <type_traits>
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

// Rows shorter than the vocabulary: 2^log_group threads of one of `splits` parts of a row take its ids in turn and enter them
// where they belong.  Four ids a thread are under way at a time.
template <typename IdT>
__global__ void __launch_bounds__(HISTORY_THREADS)
history_add_kernel(HistoryArgs a, const IdT* __restrict__ ids, int log_group, int splits) {
    const int64_t words = (a.width + 31) / 32;
    const int64_t unit = ((int64_t)blockIdx.x * HISTORY_THREADS + threadIdx.x) >> log_group;
    const int64_t row = splits == 1 ? unit : unit / splits;
    if (row >= a.n_rows) return;
    int64_t lo, hi;
    const int64_t h = history_row(a, row, &lo, &hi);
    if (h < 0) return;
    uint32_t* seen = a.seen + h * words;
    int32_t* counts = a.counts ? a.counts + h * a.width : nullptr;
    const int64_t step = (int64_t)splits << log_group;
    for (int64_t i = lo + ((unit - row * splits) << log_group) + (threadIdx.x & ((1 << log_group) - 1)); i < hi; i += 4 * step) {
        int64_t id[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) id[k] = i + k * step < hi ? (int64_t)ids[i + k * step] : -1;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (id[k] < 0 || id[k] >= a.width) continue;
            atomicOr(seen + (id[k] >> 5), 1u << (id[k] & 31));
            if (counts) atomicAdd(counts + id[k], 1);
        }
    }
}

constexpr int HISTORY_LONG_THREADS = 512;

// The part of a row that one of `splits` blocks takes.
__device__ __forceinline__ void history_part(int64_t& lo, int64_t& hi, int split, int splits) {
    const int64_t each = (hi - lo + splits - 1) / splits;
    const int64_t end = hi;
    lo += each * split;
    hi = lo + each < end ? lo + each : end;
}

// f(id) for every id of [lo, hi) that is a token, by the block's threads; eight loads a thread are under way at a time.  (In
// steps of 2^30 ids, so that the places inside one fit 32 bits.)
template <typename IdT, typename F>
__device__ __forceinline__ void history_each(const IdT* __restrict__ ids, int64_t lo, int64_t hi, int width, F f) {
    using Unsigned = typename std::conditional<sizeof(IdT) == 8, uint64_t, uint32_t>::type;     // below 0: beyond every width
    constexpr int64_t STEP = 1 << 30;
    constexpr int EACH = 8;
    for (; lo < hi; lo += STEP) {
        const Unsigned* p = reinterpret_cast<const Unsigned*>(ids) + lo;
        const int n = (int)(hi - lo < STEP ? hi - lo : STEP);
        int i = threadIdx.x;
        for (; i + (EACH - 1) * HISTORY_LONG_THREADS < n; i += EACH * HISTORY_LONG_THREADS) {
            Unsigned id[EACH];
#pragma unroll
            for (int k = 0; k < EACH; ++k) id[k] = p[i + k * HISTORY_LONG_THREADS];
#pragma unroll
            for (int k = 0; k < EACH; ++k) if (id[k] < (Unsigned)width) f((int)id[k]);
        }
        for (; i < n; i += HISTORY_LONG_THREADS) {
            const Unsigned id = p[i];
            if (id < (Unsigned)width) f((int)id);
        }
    }
}

// Long rows, counted: a block counts its part of a row in shared memory and then adds what it found.  A long row of few
// different tokens (bases) would queue up at a handful of counters: there are 2^log_copies of each, one for every 32 / copies
// lanes of a warp, in banks of their own.
template <typename IdT>
__global__ void __launch_bounds__(HISTORY_LONG_THREADS)
history_count_kernel(HistoryArgs a, const IdT* __restrict__ ids, int splits, int log_copies) {
    extern __shared__ int32_t found[];            // [width][copies]
    const int64_t row = blockIdx.x / splits;
    int64_t lo, hi;
    const int64_t h = history_row(a, row, &lo, &hi);
    if (h < 0) return;
    history_part(lo, hi, (int)(blockIdx.x % splits), splits);
    if (lo >= hi) return;
    const int width = (int)a.width, copies = 1 << log_copies;
    for (int v = threadIdx.x; v < width << log_copies; v += HISTORY_LONG_THREADS) found[v] = 0;
    __syncthreads();
    const int copy = threadIdx.x & (copies - 1);
    history_each(ids, lo, hi, width, [&](int id) { atomicAdd(found + ((id << log_copies) | copy), 1); });
    __syncthreads();
    const int words = (width + 31) / 32;
    for (int v = threadIdx.x; v < words * 32; v += HISTORY_LONG_THREADS) {
        int32_t n = 0;
        if (v < width)
            for (int k = 0; k < copies; ++k) n += found[(v << log_copies) | ((v + k) & (copies - 1))];   // (lanes start at banks of their own)
        const uint32_t word = __ballot_sync(0xffffffffu, n > 0);
        if (n > 0) atomicAdd(a.counts + h * a.width + v, n);
        if (word && (threadIdx.x & 31) == 0) atomicOr(a.seen + h * words + (v >> 5), word);
    }
}

// Long rows, only marked: the same with a bit per token; a bit that is there already is not set again.
template <typename IdT>
__global__ void __launch_bounds__(HISTORY_LONG_THREADS)
history_mark_kernel(HistoryArgs a, const IdT* __restrict__ ids, int splits) {
    extern __shared__ uint32_t marked[];          // [words]
    const int64_t row = blockIdx.x / splits;
    int64_t lo, hi;
    const int64_t h = history_row(a, row, &lo, &hi);
    if (h < 0) return;
    history_part(lo, hi, (int)(blockIdx.x % splits), splits);
    if (lo >= hi) return;
    const int width = (int)a.width, words = (width + 31) / 32;
    for (int w = threadIdx.x; w < words; w += HISTORY_LONG_THREADS) marked[w] = 0;
    __syncthreads();
    history_each(ids, lo, hi, width, [&](int id) {
        const uint32_t bit = 1u << (id & 31);
        if (!(*reinterpret_cast<volatile uint32_t*>(marked + (id >> 5)) & bit)) atomicOr(marked + (id >> 5), bit);
    });
    __syncthreads();
    for (int w = threadIdx.x; w < words; w += HISTORY_LONG_THREADS)
        if (marked[w]) atomicOr(a.seen + h * words + w, marked[w]);
}

}  // namespace dnatok
