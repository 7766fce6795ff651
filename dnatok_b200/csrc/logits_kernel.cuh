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
    int64_t history_rows;
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

// What one row brings along.  A history row outside the history gives a row without one.
struct LogitsRow {
    const uint32_t* seen;
    const int32_t* counts;
    const uint32_t* allowed;
    const float* bias;
    float r, f, p;
};

__device__ __forceinline__ LogitsRow logits_row(const LogitsArgs& a, int64_t row) {
    LogitsRow o;
    const int64_t words = (a.width + 31) / 32;
    int64_t h = row;
    if (a.rows) h = a.rows_bits == 64 ? static_cast<const int64_t*>(a.rows)[row] : static_cast<const int32_t*>(a.rows)[row];
    const bool known = a.seen && h >= 0 && h < a.history_rows;
    o.seen = known ? a.seen + h * words : nullptr;
    o.counts = known && a.counts ? a.counts + h * a.width : nullptr;
    o.allowed = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
    o.bias = a.bias ? a.bias + row * a.bias_stride : nullptr;
    o.r = a.d_repetition ? a.d_repetition[row] : a.repetition;
    o.f = a.d_frequency ? a.d_frequency[row] : a.frequency;
    o.p = a.d_presence ? a.d_presence[row] : a.presence;
    return o;
}

__device__ __forceinline__ bool bit_at(const uint32_t* words, int64_t v) { return (words[v >> 5] >> (v & 31)) & 1; }

template <typename T, typename O>
__global__ void __launch_bounds__(LOGITS_THREADS)
process_logits_kernel(LogitsArgs a, const T* __restrict__ logits, O* __restrict__ out, int64_t out_stride) {
    const int64_t n = a.n_rows * a.width;
    for (int64_t i = (int64_t)blockIdx.x * LOGITS_THREADS + threadIdx.x; i < n; i += (int64_t)gridDim.x * LOGITS_THREADS) {
        const int64_t row = i / a.width, v = i - row * a.width;
        const LogitsRow q = logits_row(a, row);
        float y = -INFINITY;
        if (!q.allowed || bit_at(q.allowed, v)) {
            y = as_float(logits[row * a.stride + v]);
            if (q.seen && bit_at(q.seen, v)) {
                y = y > 0.f ? y / q.r : y * q.r;
                const int32_t c = q.counts ? q.counts[v] : 0;
                if (c > 0) y = y - q.f * (float)c - q.p;
            }
            if (q.bias) y += q.bias[v];
        }
        out[row * out_stride + v] = from_float<O>(y);
    }
}

template <typename T, typename G>
__global__ void __launch_bounds__(LOGITS_THREADS)
logits_gradient_kernel(LogitsArgs a, const T* __restrict__ logits, const G* __restrict__ grad, int64_t grad_stride,
                       T* __restrict__ dlogits, int64_t dlogits_stride, float* __restrict__ dbias_rows) {
    const int64_t n = a.n_rows * a.width;
    for (int64_t i = (int64_t)blockIdx.x * LOGITS_THREADS + threadIdx.x; i < n; i += (int64_t)gridDim.x * LOGITS_THREADS) {
        const int64_t row = i / a.width, v = i - row * a.width;
        const LogitsRow q = logits_row(a, row);
        float g = 0.f, d = 0.f;
        if (!q.allowed || bit_at(q.allowed, v)) {
            d = g = as_float(grad[row * grad_stride + v]);
            if (q.seen && bit_at(q.seen, v)) d = as_float(logits[row * a.stride + v]) > 0.f ? g / q.r : g * q.r;
        }
        if (dlogits) dlogits[row * dlogits_stride + v] = from_float<T>(d);
        if (dbias_rows) dbias_rows[row * a.width + v] = g;
    }
}

// Shared bias: a thread adds up its column, in the order of the rows.
template <typename G>
__global__ void __launch_bounds__(LOGITS_THREADS)
bias_gradient_kernel(LogitsArgs a, const G* __restrict__ grad, int64_t grad_stride, float* __restrict__ dbias) {
    const int64_t v = (int64_t)blockIdx.x * LOGITS_THREADS + threadIdx.x;
    if (v >= a.width) return;
    float sum = 0.f;
    for (int64_t row = 0; row < a.n_rows; ++row)
        if (!a.allowed || bit_at(a.allowed + row * a.allowed_stride, v)) sum += as_float(grad[row * grad_stride + v]);
    dbias[v] = sum;
}

}  // namespace dnatok
