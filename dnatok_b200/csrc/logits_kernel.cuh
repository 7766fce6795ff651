// Penalties for repeated tokens, a bias and a mask on logits, and the gradient of that.
//
//   x1 = seen ? (x > 0 ? x / r : x * r) : x          r, f, p: repetition, frequency, presence of the row
//   x2 = c > 0 ? x1 - f c - p : x1                   c: how often the row generated the token
//   y  = allowed ? x2 + bias : -inf
//   dx = allowed ? dy (seen ? (x > 0 ? 1 / r : r) : 1) : 0,   dbias = allowed ? dy : 0, over the rows for a shared bias
//
// All of it is computed in 32 bits; y and dx are rounded once, to the type of the output.  seen and allowed hold a bit
// per token (bit v % 32 of word v / 32), so that a count is only read where there is one.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace dnatok {

constexpr int LOGITS_THREADS = 256;

struct LogitsArgs {
    int64_t n_rows, width, stride;
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
__device__ __forceinline__ int32_t history_of(const LogitsArgs& a, int64_t row) {
    if (!a.rows) return (int32_t)row;
    const int64_t h = a.rows_bits == 64 ? __ldg(static_cast<const int64_t*>(a.rows) + row) : __ldg(static_cast<const int32_t*>(a.rows) + row);
    return h >= 0 && h < a.history_rows ? (int32_t)h : -1;
}
__device__ __forceinline__ float of_row(const float* each, float all, int64_t row) { return each ? __ldg(each + row) : all; }

// A block keeps one tile of 512 columns and goes through rows of it, a warp a row, 8 columns a lane in each of the tile's
// two parts: what belongs to the columns is worked out once, neighbouring blocks read neighbouring columns of the same
// rows, and a row's own words and numbers are fetched for 16 columns a lane.
// Which columns of a part a lane has (MAP):
//   CONTIGUOUS  8 neighbouring ones, for 16-bit arrays that begin and go on at multiples of 16 bytes: one access each
//   HALVES      4 and 4 at a distance of 128, where a 32-bit array is among them: its two accesses fill whole sectors
//   APART       32 apart, at any alignment (a vocabulary of 4,106 tokens in 16 bits, a view that begins anywhere)
constexpr int LOGITS_PART = 256, LOGITS_PARTS = 2, LOGITS_TILE = LOGITS_PART * LOGITS_PARTS;
constexpr int LOGITS_WARPS = LOGITS_THREADS / 32;
constexpr int LOGITS_BLOCKS = 4;                   // an SM: 64 registers a thread
enum { APART, CONTIGUOUS, HALVES };

template <int MAP> __device__ __forceinline__ int tile_column(int lane, int j) {
    return MAP == CONTIGUOUS ? lane * 8 + j : MAP == HALVES ? (j >> 2) * 128 + lane * 4 + (j & 3) : j * 32 + lane;
}

// Columns of the row from this block's tile on, at most a tile's.
__device__ __forceinline__ int tile_left(int64_t width, int64_t base) { return width - base < LOGITS_TILE ? (int)(width - base) : LOGITS_TILE; }

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

// A set's words of this tile, lane l holding word l % 16; and bit j: the set holds column j of this lane in part u.
__device__ __forceinline__ uint32_t tile_word(const uint32_t* words, int left, int lane) {
    return (lane & 15) * 32 < left ? __ldg(words + (lane & 15)) : 0;
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

template <int MAP, typename T>
__device__ __forceinline__ void store_tile(T* p, uint32_t all, int lane, const float (&y)[8]) {
    constexpr int EACH = MAP == APART ? 1 : MAP == HALVES ? 4 : 8;
    Raw8<T> raw;
#pragma unroll
    for (int j = 0; j < 8; ++j) raw.v[j] = from_float<T>(y[j]);
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

// *p where `want` is not 0, else 0: one predicated load, not a branch.
__device__ __forceinline__ int32_t load_where(const int32_t* p, uint32_t want) {
    int32_t v = 0;
    asm("{\n.reg .pred q;\nsetp.ne.u32 q, %2, 0;\n@q ld.global.nc.s32 %0, [%1];\n}" : "+r"(v) : "l"(p), "r"(want));
    return v;
}

template <typename T, typename O, int MAP>
__global__ void __launch_bounds__(LOGITS_THREADS, LOGITS_BLOCKS)
process_logits_kernel(LogitsArgs a, const T* logits, O* out, int64_t out_stride) {
    const int lane = threadIdx.x & 31;
    const int64_t base = (int64_t)blockIdx.x * LOGITS_TILE;
    const int left = tile_left(a.width, base);
    const int words = ((int)a.width + 31) >> 5;
#pragma unroll 1
    for (int64_t row = (int64_t)blockIdx.y * LOGITS_WARPS + (threadIdx.x >> 5); row < a.n_rows; row += (int64_t)gridDim.y * LOGITS_WARPS) {
        const T* x_row = logits + row * a.stride + base;
        Raw8<T> x[LOGITS_PARTS];
#pragma unroll
        for (int u = 0; u < LOGITS_PARTS; ++u) {
            x[u] = {};
            load_tile<MAP>(x_row + u * LOGITS_PART, tile_all<MAP>(left - u * LOGITS_PART, lane), lane, x[u]);
        }
        const uint32_t ok_word = a.allowed ? tile_word(a.allowed + row * a.allowed_stride + (base >> 5), left, lane) : 0xffffffffu;
        const int32_t h = a.seen ? history_of(a, row) : -1;
        const uint32_t hit_word = h >= 0 ? tile_word(a.seen + ((int64_t)h * words + (base >> 5)), left, lane) & ok_word : 0;
        const bool any_hit = __any_sync(0xffffffffu, hit_word);
        const float* b_row = a.bias ? a.bias + row * a.bias_stride + base : nullptr;
        O* y_row = out + row * out_stride + base;
#pragma unroll
        for (int u = 0; u < LOGITS_PARTS; ++u) {
            const uint32_t all = tile_all<MAP>(left - u * LOGITS_PART, lane);
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = as_float(x[u].v[j]);
            if (any_hit) {
                const uint32_t hit = tile_bits<MAP>(hit_word, u, lane) & all;
                const Penalty pen = penalty_of(of_row(a.d_repetition, a.repetition, row));
                if (hit) {
                    int32_t c[8] = {};
                    if (a.counts) {
                        const int32_t* counts = a.counts + ((int64_t)h * (int32_t)a.width + base) + u * LOGITS_PART;
#pragma unroll
                        for (int j = 0; j < 8; ++j) c[j] = load_where(counts + tile_column<MAP>(lane, j), hit >> j & 1);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float z = y[j] * (y[j] > 0.f ? pen.up : pen.down);
                        y[j] = hit >> j & 1 ? z : y[j];
                    }
                    if (c[0] | c[1] | c[2] | c[3] | c[4] | c[5] | c[6] | c[7]) {
                        const float f = of_row(a.d_frequency, a.frequency, row), p = of_row(a.d_presence, a.presence, row);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float z = y[j] - f * (float)c[j] - p;
                            y[j] = c[j] > 0 ? z : y[j];
                        }
                    }
                }
            }
            if (b_row) {
                Raw8<float> bias;
                load_tile<MAP>(b_row + u * LOGITS_PART, all, lane, bias);
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] += bias.v[j];
            }
            if (a.allowed) {
                const uint32_t ok = tile_bits<MAP>(ok_word, u, lane);
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = ok >> j & 1 ? y[j] : -INFINITY;
            }
            store_tile<MAP>(y_row + u * LOGITS_PART, all, lane, y);
        }
    }
}

// A row's logits are read only where its mask allows, its counts only where its history has a bit: a warp fetches those
// words a row ahead, and the number of the history row two ahead, so that a row costs one trip to memory and not three.
struct Ahead {
    const uint32_t* allowed;      // this tile's words of the mask of the next row
    const uint32_t* seen;         // this tile's words of history row 0; NULL: no history
    int32_t h;                    // history row of the next row
    uint32_t ok, hit;             // words fetched

    // The words of `row`, whose history row is h; then the history row of the one after, if there is one.
    __device__ __forceinline__ void fetch(const LogitsArgs& a, int64_t row, bool more, int left, int lane) {
        ok = 0xffffffffu;
        hit = 0;
        if (allowed) {
            ok = tile_word(allowed, left, lane);
            allowed += a.allowed_stride * LOGITS_WARPS;
        }
        if (seen) {
            if (h >= 0) hit = tile_word(seen + (int64_t)h * (((int32_t)a.width + 31) >> 5), left, lane);
            if (more) h = history_of(a, row + LOGITS_WARPS);
        }
    }
};

// The gradients of the logits and, SHARED, of a bias that all rows share: each warp adds up its rows of the block's columns
// in registers, the warps' sums are joined in shared memory, those of several blocks by bias_gradient_kernel.  The incoming
// gradient is read once for both, and the order of the additions depends on the sizes alone.
template <typename T, typename G, int MAP, bool SHARED>
__global__ void __launch_bounds__(LOGITS_THREADS, LOGITS_BLOCKS)
logits_gradient_kernel(LogitsArgs a, const T* logits, const G* grad, int64_t grad_stride, T* dlogits, int64_t dlogits_stride,
                       float* dbias, int rows_per_block) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t base = (int64_t)blockIdx.x * LOGITS_TILE;
    const int left = tile_left(a.width, base);
    uint32_t all[LOGITS_PARTS];
#pragma unroll
    for (int u = 0; u < LOGITS_PARTS; ++u) all[u] = tile_all<MAP>(left - u * LOGITS_PART, lane);
    float acc[LOGITS_PARTS][8] = {};
    int64_t row = (int64_t)blockIdx.y * rows_per_block + warp;
    int rows = (int)((a.n_rows - row < rows_per_block - warp ? a.n_rows - row : rows_per_block - warp) + LOGITS_WARPS - 1) / LOGITS_WARPS;
    const T* x_row = logits + row * a.stride + base;
    const G* g_row = grad + row * grad_stride + base;
    T* d_row = dlogits ? dlogits + row * dlogits_stride + base : nullptr;
    Ahead next;
    next.allowed = a.allowed ? a.allowed + row * a.allowed_stride + (base >> 5) : nullptr;
    next.seen = a.seen && dlogits ? a.seen + (base >> 5) : nullptr;
    next.h = -1;
    if (rows > 0) {
        if (next.seen) next.h = history_of(a, row);
        next.fetch(a, row, rows > 1, left, lane);
    }
#pragma unroll 1
    for (; rows > 0; --rows) {
        uint32_t ok[LOGITS_PARTS], hit[LOGITS_PARTS];
        Raw8<T> x[LOGITS_PARTS];
        Raw8<G> raw[LOGITS_PARTS];
#pragma unroll
        for (int u = 0; u < LOGITS_PARTS; ++u) {
            ok[u] = tile_bits<MAP>(next.ok, u, lane) & all[u];
            hit[u] = tile_bits<MAP>(next.hit, u, lane) & ok[u];
            raw[u] = {};
            load_tile<MAP>(g_row + u * LOGITS_PART, ok[u], lane, raw[u]);
        }
#pragma unroll
        for (int u = 0; u < LOGITS_PARTS; ++u) {
            x[u] = {};
            load_tile<MAP>(x_row + u * LOGITS_PART, hit[u], lane, x[u]);
        }
        const int64_t here = row;
        row += LOGITS_WARPS;
        if (rows > 1) next.fetch(a, row, rows > 2, left, lane);
#pragma unroll
        for (int u = 0; u < LOGITS_PARTS; ++u) {
            float g[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                g[j] = ok[u] >> j & 1 ? as_float(raw[u].v[j]) : 0.f;
                if (SHARED) acc[u][j] += g[j];
            }
            if (!SHARED && dbias) store_tile<MAP>(dbias + here * a.width + base + u * LOGITS_PART, all[u], lane, g);
            if (!d_row) continue;
            if (hit[u]) {
                const Penalty pen = penalty_of(of_row(a.d_repetition, a.repetition, here));
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float z = g[j] * (as_float(x[u].v[j]) > 0.f ? pen.up : pen.down);
                    g[j] = hit[u] >> j & 1 ? z : g[j];
                }
            }
            store_tile<MAP>(d_row + u * LOGITS_PART, all[u], lane, g);
        }
        x_row += a.stride * LOGITS_WARPS;
        g_row += grad_stride * LOGITS_WARPS;
        if (d_row) d_row += dlogits_stride * LOGITS_WARPS;
    }
    if (SHARED) {
        __shared__ float part[LOGITS_WARPS][LOGITS_TILE];
#pragma unroll
        for (int u = 0; u < LOGITS_PARTS; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j) part[warp][u * LOGITS_PART + tile_column<MAP>(lane, j)] = acc[u][j];
        __syncthreads();
        for (int v = threadIdx.x; v < left; v += LOGITS_THREADS) {
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < LOGITS_WARPS; ++w) sum += part[w][v];
            dbias[(int64_t)blockIdx.y * a.width + base + v] = sum;
        }
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
