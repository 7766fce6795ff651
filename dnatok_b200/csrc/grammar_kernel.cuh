// Grammar masks: which tokens a finite automaton over bytes lets follow.
//
// Tokens are several bytes long, so the automaton is walked along every token's bytes from the row's state; a token is
// allowed if the walk ends in a live state.  Rows carry a state: 0 and above, GRAMMAR_DEAD (a token that was not allowed
// was taken: nothing may follow) or GRAMMAR_FINISHED (after the end token: only the end token may follow).
#pragma once
#include "common.cuh"

namespace dnatok {

constexpr int GRAMMAR_THREADS = 256;
constexpr int32_t GRAMMAR_DEAD = -1, GRAMMAR_FINISHED = -2;

struct GrammarTables {
    const int32_t* next;          // [n_states * n_classes], -1: no way on
    const uint8_t* accepting;     // [n_states]
    const uint8_t* codes;         // classes of the tokens' bytes, token after token
    const int32_t* token_at;      // [width + 1] first code of each token; a token without codes is never allowed
    int32_t n_states, n_classes;
    int64_t width;
    int64_t end_id;               // -1: none
};

__device__ __forceinline__ int32_t grammar_walk(const GrammarTables& t, int32_t state, int64_t token) {
    const int32_t lo = t.token_at[token], hi = t.token_at[token + 1];
    if (state < 0 || state >= t.n_states || lo == hi) return GRAMMAR_DEAD;
    for (int32_t i = lo; i < hi && state >= 0; ++i) state = t.next[(int64_t)state * t.n_classes + t.codes[i]];
    return state < 0 ? GRAMMAR_DEAD : state;
}

__device__ __forceinline__ bool grammar_may_end(const GrammarTables& t, int32_t state) {
    return state == GRAMMAR_FINISHED || (state >= 0 && state < t.n_states && t.accepting[state]);
}

// The state after a token; a token outside the vocabulary leaves the row as it was.
__device__ __forceinline__ int32_t grammar_after(const GrammarTables& t, int32_t state, int64_t token) {
    if (token < 0 || token >= t.width) return state;
    if (token == t.end_id) return grammar_may_end(t, state) ? GRAMMAR_FINISHED : GRAMMAR_DEAD;
    return grammar_walk(t, state, token);
}

__global__ void __launch_bounds__(GRAMMAR_THREADS)
grammar_advance_kernel(GrammarTables t, const int32_t* states, const void* __restrict__ tokens, int token_bits, int64_t n_rows,
                       int32_t* out) {
    const int64_t row = (int64_t)blockIdx.x * GRAMMAR_THREADS + threadIdx.x;
    if (row >= n_rows) return;
    const int64_t token = token_bits == 64 ? static_cast<const int64_t*>(tokens)[row] : static_cast<const int32_t*>(tokens)[row];
    out[row] = grammar_after(t, states[row], token);
}

// A warp takes one word of a row: 32 tokens.
__global__ void __launch_bounds__(GRAMMAR_THREADS)
grammar_allowed_kernel(GrammarTables t, const int32_t* __restrict__ states, int64_t n_rows, uint32_t* __restrict__ allowed) {
    const int64_t words = (t.width + 31) / 32;
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * (GRAMMAR_THREADS / 32);
    for (int64_t w = (int64_t)blockIdx.x * (GRAMMAR_THREADS / 32) + (threadIdx.x >> 5); w < n_rows * words; w += warps) {
        const int64_t row = w / words, token = (w - row * words) * 32 + lane;
        const int32_t state = states[row];
        bool ok = false;
        if (token < t.width) ok = token == t.end_id ? grammar_may_end(t, state) : grammar_walk(t, state, token) >= 0;
        const uint32_t word = __ballot_sync(0xffffffffu, ok);
        if (lane == 0) allowed[w] = word;
    }
}

}  // namespace dnatok
