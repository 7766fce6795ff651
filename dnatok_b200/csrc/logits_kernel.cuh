// Penalties for repeated tokens, a bias and a mask on logits, and the gradient of that.
//
//   x1 = seen ? (x > 0 ? x / r : x * r) : x          r, f, p: repetition, frequency, presence of the row
//   x2 = c > 0 ? x1 - f c - p : x1                   c: how often the row generated the token
//   y  = allowed ? x2 + bias : -inf
//   dx = allowed ? dy (seen ? (x > 0 ? 1 / r : r) : 1) : 0,   dbias = allowed ? dy : 0, over the rows for a shared bias
//
// All of it is computed in 32 bits, with a rounding an operation (x / r is x * (1 / r): two of them); y and dx are then rounded
// once, to the type of the output.  seen and allowed hold a bit per token (bit v % 32 of word v / 32), so that a count is only
// read where a token was seen, and a logit in the backward pass too.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>
#include "common.cuh"

namespace dnatok {

constexpr int LOGITS_THREADS = 256;

struct LogitsArgs {
    int32_t n_rows, width;
    int64_t stride;
    const uint32_t* seen;         // [history_rows, words] or NULL
    const int32_t* counts;        // [history_rows, width] or NULL: no row generated anything
    int32_t history_rows;
    const void* rows;             // history row of each logits row, or NULL: the same
    int32_t rows_bits;            // 32 or 64
    float repetition, frequency, presence;
    const float *d_repetition, *d_frequency, *d_presence;   // one value a row; NULL: the number above
    const float* bias;            // [width] (bias_stride 0), [n_rows, width] or NULL
    int64_t bias_stride;
    const uint32_t* allowed;      // [words] (allowed_stride 0), [n_rows, words] or NULL: all are
    int64_t allowed_stride;
};

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The history row of a row, -1 for none.
__device__ __forceinline__ int32_t history_of(const LogitsArgs& a, int32_t row) {
    if (!a.rows) return row;
    const int64_t h = a.rows_bits == 64 ? __ldg(static_cast<const int64_t*>(a.rows) + row) : __ldg(static_cast<const int32_t*>(a.rows) + row);
    return h >= 0 && h < a.history_rows ? (int32_t)h : -1;
}
__device__ __forceinline__ float of_row(const float* each, float all, int32_t row) { return each ? __ldg(each + row) : all; }

__device__ __forceinline__ bool bit_at(const uint32_t* words, int v) { return __ldg(words + (v >> 5)) >> (v & 31) & 1; }

// Small calls, a thread a logit: nothing is shared, but few instructions stand between the loads (73 rows of 4,106 bf16
// logits with everything: 3.3 us, the kernel below 3.6, calls following one another in a graph; the rule and where the two
// meet stand at the launch).
template <typename T, typename O>
__global__ void __launch_bounds__(LOGITS_THREADS)
process_each_kernel(LogitsArgs a, const T* logits, O* out, int64_t out_stride) {
    const uint32_t i = blockIdx.x * LOGITS_THREADS + threadIdx.x;
    if (i >= (uint32_t)a.n_rows * (uint32_t)a.width) return;
    const int row = (int)(i / (uint32_t)a.width), v = (int)(i - (uint32_t)row * (uint32_t)a.width);
    float y = as_float(logits[row * a.stride + v]);
    const bool ok = !a.allowed || bit_at(a.allowed + row * a.allowed_stride, v);
    const int32_t h = a.seen ? history_of(a, row) : -1;
    if (h >= 0 && bit_at(a.seen + (int64_t)h * ((a.width + 31) >> 5), v)) {
        const int32_t c = a.counts ? __ldg(a.counts + ((int64_t)h * a.width + v)) : 0;
        const float r = of_row(a.d_repetition, a.repetition, row);
        y *= y > 0.f ? __frcp_rn(r) : r;
        if (c > 0) y = y - of_row(a.d_frequency, a.frequency, row) * (float)c - of_row(a.d_presence, a.presence, row);
    }
    if (a.bias) y += __ldg(a.bias + row * a.bias_stride + v);
    out[row * out_stride + v] = from_float<O>(ok ? y : -INFINITY);
}

// A warp takes a tile of one or two parts (PARTS) of 256 columns of a row, 8 columns a lane in each: two where that leaves
// warps for the whole GPU, since a row's own words and numbers are then fetched for twice as many columns.  Which columns of
// a part a lane has (MAP):
//   CONTIGUOUS  8 neighbouring ones, for 16-bit arrays that begin and go on at multiples of 16 bytes: one access each
//   HALVES      4 and 4 at a distance of 128, where a 32-bit array is among them: its two accesses fill whole sectors
//   APART       32 apart, at any alignment (a vocabulary of 4,106 tokens in 16 bits, a view that begins anywhere)
//
// All columns get bias, mask and repetition penalty on this way.  Where counts matter too, the hits (seen and allowed) are
// mended afterwards: they are few among many, as a rule, and fetching and subtracting counts for 8 columns a lane took more
// instructions than all the rest together.  The warp lists the hits' columns in shared memory and takes 32 at a time.  (The
// repetition penalty alone, 333 x 32,000 fp16: 12.4 us among all columns, 14.4 by the list.)
//
// What bounds it: instructions and memory about alike.  2,048 x 32,000 bf16 to float, a quarter allowed, 5 % seen: 94 us, issue
// slots 73 % busy, 444 MB = 4.7 TB/s (the counts of scattered tokens cost 64 bytes each from DRAM); 4,096 x 32,000 bf16 with
// nine tenths allowed: 176 us, 5.3 TB/s; 333 x 32,000 fp16 with the repetition penalty alone 12.4 us, 3.5 TB/s (one
// row of 512 takes 4).
constexpr int LOGITS_PART = 256;
constexpr int LOGITS_WARPS = LOGITS_THREADS / 32;
enum { APART, CONTIGUOUS, HALVES };
enum { NO_HISTORY, SEEN_ONLY, COUNTED };           // what the penalties need

template <int MAP> __device__ __forceinline__ int tile_column(int lane, int j) {
    return MAP == CONTIGUOUS ? lane * 8 + j : MAP == HALVES ? (j >> 2) * 128 + lane * 4 + (j & 3) : j * 32 + lane;
}

// Bit j: column j of this lane lies in the row, of which `left` columns are left from the part on.  (Widths of the maps with
// neighbouring columns are multiples of what a lane moves at a time: those columns lie in the row together or not at all.)
template <int MAP> __device__ __forceinline__ uint32_t tile_all(int left, int lane) {
    if (MAP == CONTIGUOUS) return lane * 8 < left ? 0xff : 0;
    if (MAP == HALVES) return (lane * 4 < left ? 0xf : 0) | (128 + lane * 4 < left ? 0xf0 : 0);
    uint32_t b = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) b |= (uint32_t)(j * 32 + lane < left) << j;
    return b;
}

// A set's words of this tile, lane l holding word l % (8 PARTS); and bit j: the set holds column j of this lane in part u.
template <int PARTS> __device__ __forceinline__ uint32_t tile_word(const uint32_t* words, int left, int lane) {
    const int w = lane & (8 * PARTS - 1);
    return w * 32 < left ? __ldg(words + w) : 0;
}
template <int MAP> __device__ __forceinline__ uint32_t tile_bits(uint32_t word, int u, int lane) {
    constexpr uint32_t FULL = 0xffffffffu;
    if (MAP == CONTIGUOUS) return __shfl_sync(FULL, word, u * 8 + (lane >> 2)) >> (lane & 3) * 8 & 0xff;
    if (MAP == HALVES) {
        const int shift = (lane & 7) * 4;
        return (__shfl_sync(FULL, word, u * 8 + (lane >> 3)) >> shift & 0xf) | (__shfl_sync(FULL, word, u * 8 + 4 + (lane >> 3)) >> shift & 0xf) << 4;
    }
    uint32_t b = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) b |= (__shfl_sync(FULL, word, u * 8 + j) >> lane & 1) << j;
    return b;
}

template <typename T> struct alignas(16) Raw8 { T v[8]; };        // 8 values as they lie in memory

// The values of this lane's columns, from `p` on, where `want` has a bit.
template <int MAP, typename T>
__device__ __forceinline__ void load_tile(const T* p, uint32_t want, int lane, Raw8<T>& raw) {
    constexpr int EACH = MAP == APART ? 1 : MAP == HALVES ? 4 : 8;     // neighbouring columns
#pragma unroll
    for (int k = 0; k < 8 / EACH; ++k) {
        if (!(want >> k * EACH & ((1u << EACH) - 1))) continue;
        const T* q = p + tile_column<MAP>(lane, k * EACH);
        T* to = raw.v + k * EACH;
        if constexpr (EACH == 1) {
            *to = *q;
        } else if constexpr (EACH * sizeof(T) == 8) {
            *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(q);
        } else {
#pragma unroll
            for (int i = 0; i < (int)(EACH * sizeof(T) / 16); ++i)
                reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(q)[i];
        }
    }
}

// The values rounded, two an instruction where the type has one, and -inf where `may` has no bit.
__device__ __forceinline__ void round_all(const float (&y)[8], uint32_t may, Raw8<float>& raw) {
#pragma unroll
    for (int j = 0; j < 8; ++j) raw.v[j] = may >> j & 1 ? y[j] : -INFINITY;
}
__device__ __forceinline__ uint32_t round_two(float x, float y, __half) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t round_two(float x, float y, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T> __device__ __forceinline__ void round_all(const float (&y)[8], uint32_t may, Raw8<T>& raw) {
    constexpr uint32_t NONE = std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;     // -inf twice
    uint32_t* words = reinterpret_cast<uint32_t*>(&raw);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        // bit j of four into the top bit of byte j; a byte's top bit then fills the 16 bits of a value
        const uint32_t tops = (may >> 4 * i & 0xf) * 0x10204080u;
        uint32_t m0, m1;
        asm("prmt.b32 %0, %1, 0, 0x9988;" : "=r"(m0) : "r"(tops));
        asm("prmt.b32 %0, %1, 0, 0xbbaa;" : "=r"(m1) : "r"(tops));
        words[2 * i] = (round_two(y[4 * i], y[4 * i + 1], T()) & m0) | (NONE & ~m0);
        words[2 * i + 1] = (round_two(y[4 * i + 2], y[4 * i + 3], T()) & m1) | (NONE & ~m1);
    }
}

template <int MAP, typename T>
__device__ __forceinline__ void store_tile(T* p, uint32_t all, int lane, const float (&y)[8], uint32_t may = 0xff) {
    constexpr int EACH = MAP == APART ? 1 : MAP == HALVES ? 4 : 8;
    Raw8<T> raw;
    round_all(y, may, raw);
#pragma unroll
    for (int k = 0; k < 8 / EACH; ++k) {
        if (!(all >> k * EACH & 1)) continue;
        T* q = p + tile_column<MAP>(lane, k * EACH);
        const T* from = raw.v + k * EACH;
        if constexpr (EACH == 1) {
            *q = *from;
        } else if constexpr (EACH * sizeof(T) == 8) {
            *reinterpret_cast<uint2*>(q) = *reinterpret_cast<const uint2*>(from);
        } else {
#pragma unroll
            for (int i = 0; i < (int)(EACH * sizeof(T) / 16); ++i)
                reinterpret_cast<uint4*>(q)[i] = reinterpret_cast<const uint4*>(from)[i];
        }
    }
}

// x / r of a seen token is x * (1 / r): two roundings in 32 bits instead of one, and no division a token.
struct Penalty { float up, down; };
__device__ __forceinline__ Penalty penalty_of(float r) { return {__frcp_rn(r), r}; }
__device__ __forceinline__ float penalise(const Penalty& q, float x, float by) { return by * (x > 0.f ? q.up : q.down); }

// The hits of the tile that this lane lists, from the tile's words: bit j stands for column hit_column(lane) + j.
template <int PARTS> __device__ __forceinline__ int hit_shift(int lane) { return lane / (8 * PARTS) * (8 * PARTS); }
template <int PARTS> __device__ __forceinline__ int hit_column(int lane) { return (lane & (8 * PARTS - 1)) * 32 + hit_shift<PARTS>(lane); }

// The words of the tile's hits: what row h of the history has seen among `ok`.
template <int PARTS>
__device__ __forceinline__ uint32_t hit_word(const LogitsArgs& a, int32_t h, uint32_t ok, int base, int left, int lane) {
    return h < 0 ? 0 : tile_word<PARTS>(a.seen + ((int64_t)h * ((a.width + 31) >> 5) + (base >> 5)), left, lane) & ok;
}

// The hits that this lane lists.  (Bits behind the last column are no tokens.)
template <int PARTS> __device__ __forceinline__ uint32_t lane_hits(uint32_t word, int left, int lane) {
    constexpr int BITS = 8 * PARTS;
    const int behind = left - hit_column<PARTS>(lane);
    return word >> hit_shift<PARTS>(lane) & ((1u << (behind >= BITS ? BITS : behind > 0 ? behind : 0)) - 1);
}

// by[j] times the penalty of x[j] where `hit` has a bit.
__device__ __forceinline__ void penalise_hits(const Penalty& q, uint32_t hit, const float (&x)[8], float (&by)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float z = penalise(q, x[j], by[j]);
        by[j] = hit >> j & 1 ? z : by[j];
    }
}

// The columns of a warp's hits, in their order, into `list`; how many there are.
template <int PARTS>
__device__ __forceinline__ int list_hits(uint32_t hits, uint16_t* list, int lane) {
    const int mine = __popc(hits);
    int upto = mine;                                          // hits of the lanes up to this one
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int before = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += before;
    }
    uint16_t* to = list + (upto - mine);
    for (; hits; hits &= hits - 1) *to++ = (uint16_t)(hit_column<PARTS>(lane) + __ffs(hits) - 1);
    __syncwarp();
    return __shfl_sync(0xffffffffu, upto, 31);
}

// A tile's values as they were before this warp wrote over them, by column.
template <int MAP, typename T>
__device__ __forceinline__ void keep_tile(T* kept, const Raw8<T>& raw, int lane) {
    constexpr int EACH = MAP == APART ? 1 : MAP == HALVES ? 4 : 8;
#pragma unroll
    for (int k = 0; k < 8 / EACH; ++k) {
        T* q = kept + tile_column<MAP>(lane, k * EACH);
        const T* from = raw.v + k * EACH;
        if constexpr (EACH == 1) {
            *q = *from;
        } else if constexpr (EACH * sizeof(T) == 8) {
            *reinterpret_cast<uint2*>(q) = *reinterpret_cast<const uint2*>(from);
        } else {
#pragma unroll
            for (int i = 0; i < (int)(EACH * sizeof(T) / 16); ++i) reinterpret_cast<uint4*>(q)[i] = reinterpret_cast<const uint4*>(from)[i];
        }
    }
}

template <typename T, typename O, int MAP, int MODE, int PARTS>
__global__ void __launch_bounds__(LOGITS_THREADS, 6)
process_logits_kernel(LogitsArgs a, const T* logits, O* out, int64_t out_stride) {
    constexpr bool LIST = MODE == COUNTED;
    __shared__ Raw8<T> kept[LIST ? LOGITS_WARPS : 1][LOGITS_PART * PARTS / 8];
    __shared__ uint16_t listed[LIST ? LOGITS_WARPS : 1][LOGITS_PART * PARTS];
    const int lane = threadIdx.x & 31;
    const int base = blockIdx.x * LOGITS_PART * PARTS, left = a.width - base;
#pragma unroll 1
    for (int row = blockIdx.y * LOGITS_WARPS + (threadIdx.x >> 5); row < a.n_rows; row += gridDim.y * LOGITS_WARPS) {
        const T* x_row = logits + (row * a.stride + base);
        Raw8<T> x[PARTS];
#pragma unroll
        for (int u = 0; u < PARTS; ++u) {
            x[u] = {};
            load_tile<MAP>(x_row + u * LOGITS_PART, tile_all<MAP>(left - u * LOGITS_PART, lane), lane, x[u]);
        }
        const uint32_t ok = a.allowed ? tile_word<PARTS>(a.allowed + (row * a.allowed_stride + (base >> 5)), left, lane) : 0xffffffffu;
        uint32_t seen = 0;
        const int32_t* counts = nullptr;
        if (MODE != NO_HISTORY) {
            const int32_t h = history_of(a, row);
            seen = hit_word<PARTS>(a, h, ok, base, left, lane);
            if (LIST && h >= 0) counts = a.counts + ((int64_t)h * a.width + base);
        }
        T* before = kept[LIST ? threadIdx.x >> 5 : 0][0].v;
        uint16_t* list = listed[LIST ? threadIdx.x >> 5 : 0];
        bool mend = false;
        int n_hits = 0, c = 0;                                // c: of this lane's first hit, ahead of time
        if (LIST) {
            const uint32_t hits = lane_hits<PARTS>(seen, left, lane);
            mend = __any_sync(0xffffffffu, hits);
            if (mend) {
                n_hits = list_hits<PARTS>(hits, list, lane);
                if (lane < n_hits) c = __ldg(counts + list[lane]);
            }
        }
        const float* bias = a.bias ? a.bias + (row * a.bias_stride + base) : nullptr;
        O* y_row = out + (row * out_stride + base);
#pragma unroll
        for (int u = 0; u < PARTS; ++u) {
            const uint32_t all = tile_all<MAP>(left - u * LOGITS_PART, lane);
            if (mend) keep_tile<MAP>(before + u * LOGITS_PART, x[u], lane);
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = as_float(x[u].v[j]);
            if (MODE == SEEN_ONLY) {
                const uint32_t hit = tile_bits<MAP>(seen, u, lane);
                if (hit) penalise_hits(penalty_of(of_row(a.d_repetition, a.repetition, row)), hit, y, y);
            }
            if (bias) {
                Raw8<float> b;
                load_tile<MAP>(bias + u * LOGITS_PART, all, lane, b);
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] += b.v[j];
            }
            store_tile<MAP>(y_row + u * LOGITS_PART, all, lane, y, a.allowed ? tile_bits<MAP>(ok, u, lane) : 0xff);
        }
        if (!mend) continue;
        __syncwarp();                                         // the values kept, and the order of the stores
        const Penalty pen = penalty_of(of_row(a.d_repetition, a.repetition, row));
        const float f = of_row(a.d_frequency, a.frequency, row), p = of_row(a.d_presence, a.presence, row);
        for (int i = lane; i < n_hits; i += 32) {
            const int v = list[i], now = c;
            if (i + 32 < n_hits) c = __ldg(counts + list[i + 32]);
            const float x1 = as_float(before[v]);
            float y = penalise(pen, x1, x1);
            if (now > 0) y = y - f * (float)now - p;
            if (bias) y += __ldg(bias + v);
            y_row[v] = from_float<O>(y);
        }
        __syncwarp();
    }
}

// The gradients of the logits at a row's hits, over those of its other allowed tokens.  x: the logit of this lane's first hit,
// fetched ahead of time.  (By the list, because only there are logits read: among all columns, as the repetition penalty of
// the forward pass, 2,048 x 32,000 took 119 us instead of 83 when that was tried; 74 now, bf16, nine tenths allowed, 5 % seen.)
template <typename T, typename G>
__device__ __forceinline__ void mend_gradient(const LogitsArgs& a, int row, int n_hits, const uint16_t* list, T x, const T* x_row, const G* g_row, T* d_row, int lane) {
    __syncwarp();                                             // the order of the stores
    const Penalty pen = penalty_of(of_row(a.d_repetition, a.repetition, row));
    for (int i = lane; i < n_hits; i += 32) {
        const int v = list[i];
        const T now = x;
        if (i + 32 < n_hits) x = x_row[list[i + 32]];
        d_row[v] = from_float<T>(penalise(pen, as_float(now), as_float(g_row[v])));
    }
    __syncwarp();
}

// The gradients of the logits and of a bias of every row.
template <typename T, typename G, int MAP, bool SEEN, int PARTS>
__global__ void __launch_bounds__(LOGITS_THREADS, 6)
logits_gradient_kernel(LogitsArgs a, const T* logits, const G* grad, int64_t grad_stride, T* dlogits, int64_t dlogits_stride, float* dbias) {
    __shared__ uint16_t listed[SEEN ? LOGITS_WARPS : 1][LOGITS_PART * PARTS];
    const int lane = threadIdx.x & 31;
    const int base = blockIdx.x * LOGITS_PART * PARTS, left = a.width - base;
#pragma unroll 1
    for (int row = blockIdx.y * LOGITS_WARPS + (threadIdx.x >> 5); row < a.n_rows; row += gridDim.y * LOGITS_WARPS) {
        const G* g_row = grad + (row * grad_stride + base);
        Raw8<G> raw[PARTS];
#pragma unroll
        for (int u = 0; u < PARTS; ++u) {
            raw[u] = {};
            load_tile<MAP>(g_row + u * LOGITS_PART, tile_all<MAP>(left - u * LOGITS_PART, lane), lane, raw[u]);
        }
        const uint32_t ok = a.allowed ? tile_word<PARTS>(a.allowed + (row * a.allowed_stride + (base >> 5)), left, lane) : 0xffffffffu;
        const uint32_t hits = SEEN ? lane_hits<PARTS>(hit_word<PARTS>(a, history_of(a, row), ok, base, left, lane), left, lane) : 0;
        const T* x_row = logits + (row * a.stride + base);
        int n_hits = 0;
        T x = {};
        if (SEEN && __any_sync(0xffffffffu, hits)) {
            n_hits = list_hits<PARTS>(hits, listed[threadIdx.x >> 5], lane);
            if (lane < n_hits) x = x_row[listed[threadIdx.x >> 5][lane]];
        }
        T* d_row = dlogits ? dlogits + (row * dlogits_stride + base) : nullptr;
#pragma unroll
        for (int u = 0; u < PARTS; ++u) {
            const uint32_t all = tile_all<MAP>(left - u * LOGITS_PART, lane), may = tile_bits<MAP>(ok, u, lane);
            float g[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = may >> j & 1 ? as_float(raw[u].v[j]) : 0.f;
            if (dbias) store_tile<MAP>(dbias + ((int64_t)row * a.width + base + u * LOGITS_PART), all, lane, g);
            if (d_row) store_tile<MAP>(d_row + u * LOGITS_PART, all, lane, g);
        }
        if (SEEN && n_hits) mend_gradient(a, row, n_hits, listed[threadIdx.x >> 5], x, x_row, g_row, d_row, lane);
    }
}

// The same with the gradient of a bias that all rows share: a block keeps one tile of columns for rows_per_block rows, each
// warp adds up every eighth of them in registers, the warps' sums are joined in shared memory, those of several blocks by
// bias_gradient_kernel.  The incoming gradient is read once for both, and the order of the additions depends on the sizes
// alone.  4,096 x 32,000 bf16: 165 us, 780 MB = 4.7 TB/s; 209 us before the logits of the hits were fetched ahead of the row's
// own stores and the blocks made whole rounds.
template <typename T, typename G, int MAP, bool SEEN, int PARTS>
__global__ void __launch_bounds__(LOGITS_THREADS, sizeof(G) == 2 ? 4 : 3)
logits_bias_gradient_kernel(LogitsArgs a, const T* logits, const G* grad, int64_t grad_stride, T* dlogits, int64_t dlogits_stride,
                            float* sums, int rows_per_block) {
    constexpr int R = 2;                                      // rows under way at a time
    __shared__ float part[LOGITS_WARPS][LOGITS_PART * PARTS];
    __shared__ uint16_t listed[SEEN ? LOGITS_WARPS : 1][R][LOGITS_PART * PARTS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int base = blockIdx.x * LOGITS_PART * PARTS, left = a.width - base;
    const int first = blockIdx.y * rows_per_block, last = a.n_rows - first < rows_per_block ? a.n_rows : first + rows_per_block;
    float acc[PARTS][8] = {};
#pragma unroll 1
    for (int row = first + warp; row < last; row += LOGITS_WARPS * R) {
        Raw8<G> raw[R][PARTS];
        uint32_t ok[R], hits[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int i = row + k * LOGITS_WARPS;
            ok[k] = hits[k] = 0;
#pragma unroll
            for (int u = 0; u < PARTS; ++u) raw[k][u] = {};
            if (i < last) {
#pragma unroll
                for (int u = 0; u < PARTS; ++u)
                    load_tile<MAP>(grad + (i * grad_stride + base + u * LOGITS_PART), tile_all<MAP>(left - u * LOGITS_PART, lane), lane, raw[k][u]);
                ok[k] = a.allowed ? tile_word<PARTS>(a.allowed + (i * a.allowed_stride + (base >> 5)), left, lane) : 0xffffffffu;
                if (SEEN) hits[k] = lane_hits<PARTS>(hit_word<PARTS>(a, history_of(a, i), ok[k], base, left, lane), left, lane);
            }
        }
        int n_hits[R] = {};
        T x[R] = {};
        if (SEEN) {
#pragma unroll
            for (int k = 0; k < R; ++k) {
                if (!__any_sync(0xffffffffu, hits[k])) continue;
                n_hits[k] = list_hits<PARTS>(hits[k], listed[warp][k], lane);
                if (lane < n_hits[k]) x[k] = logits[(row + k * LOGITS_WARPS) * a.stride + base + listed[warp][k][lane]];
            }
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int i = row + k * LOGITS_WARPS;
            if (i >= last) break;
            T* d_row = dlogits ? dlogits + (i * dlogits_stride + base) : nullptr;
#pragma unroll
            for (int u = 0; u < PARTS; ++u) {
                const uint32_t may = tile_bits<MAP>(ok[k], u, lane);
                float g[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    g[j] = may >> j & 1 ? as_float(raw[k][u].v[j]) : 0.f;
                    acc[u][j] += g[j];
                }
                if (d_row) store_tile<MAP>(d_row + u * LOGITS_PART, tile_all<MAP>(left - u * LOGITS_PART, lane), lane, g);
            }
            if (SEEN && n_hits[k])
                mend_gradient(a, i, n_hits[k], listed[warp][k], x[k], logits + (i * a.stride + base), grad + (i * grad_stride + base), d_row, lane);
        }
    }
#pragma unroll
    for (int u = 0; u < PARTS; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j) part[warp][u * LOGITS_PART + tile_column<MAP>(lane, j)] = acc[u][j];
    __syncthreads();
    for (int v = threadIdx.x; v < LOGITS_PART * PARTS && v < left; v += LOGITS_THREADS) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < LOGITS_WARPS; ++w) sum += part[w][v];
        sums[(int64_t)blockIdx.y * a.width + base + v] = sum;
    }
}

// The sums of several blocks of rows joined, in their order.
__global__ void __launch_bounds__(LOGITS_THREADS)
bias_gradient_kernel(const float* __restrict__ sums, int blocks, int64_t width, float* __restrict__ dbias) {
    const int64_t v = (int64_t)blockIdx.x * LOGITS_THREADS + threadIdx.x;
    if (v >= width) return;
    float sum = 0.f;
#pragma unroll 8
    for (int k = 0; k < blocks; ++k) sum += sums[(int64_t)k * width + v];
    dbias[v] = sum;
}

}  // namespace dnatok
