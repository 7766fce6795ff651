// Grammar masks: which tokens a finite automaton over bytes lets follow.
//
// Tokens are several bytes long, so the automaton is walked along every token's bytes from the row's state; a token is
// allowed if the walk ends in a live state.  Rows carry a state: 0 and above, GRAMMAR_DEAD (a token that was not allowed
// was taken: nothing may follow) or GRAMMAR_FINISHED (after the end token: only the end token may follow).
//
// The tokens are kept sorted by their text, those longer than the average after the others, in groups of 32 that share a
// prefix, and 32 groups share the beginning of their prefixes.  A row walks those beginnings first, a lane each, then the
// prefixes of the groups behind the ones that live, a lane a group, and then, a warp a group, only the rest of the tokens
// whose prefix lives: automata that allow little leave most tokens after a few steps for 1,024 of them, and one that allows
// nearly all walks the shared bases once.  (The order trades the length of the prefixes,
// which is what a row that allows little lives by, against the steps behind them, those of a group's longest token: with
// 32,000 random tokens 3.3 bases and 4.8 steps this way, 3.7 and 6.4 in one order of all texts.  Groups cut at the nodes of
// the texts' trie share 4.7 bases and halve a typical row of a pattern, 22 -> 10 us for 1,024 of them, but there are 1.6
// times as many: rows that allow nearly all, which the others wait for, go from 95 to 165 us.)
//
// What bounds it: instructions, about 85 a group and warp with its share of everything (1,024 rows of a 2,000-position
// pattern over 32,000 tokens: 10.2 M, 29 us, of which the last third is a few rows that allow most tokens), and for few rows
// the latency of the dependent loads (one row 5 to 6 us).  The bytes are nothing: 4 MB of masks.
#pragma once
#include <cooperative_groups.h>
#include <type_traits>
#include "common.cuh"

namespace dnatok {

constexpr int GRAMMAR_THREADS = 256;
constexpr int32_t GRAMMAR_DEAD = -1, GRAMMAR_FINISHED = -2;

// A text of up to 14 classes below 16 in 64 bits: class i in bits 4 i, its length in the top 4 (15: longer).
constexpr int GRAMMAR_PACKED = 14;
// What 32 groups share, and a group behind that, has up to 8 classes; a token's rest has up to 16, or its group is walked
// code by code (GRAMMAR_SLOW).  All are filled up with the class that leaves every state as it is.
constexpr int GRAMMAR_SHARED = 8, GRAMMAR_REST = 16, GRAMMAR_SLOW = 255, GRAMMAR_RUN = 256;

struct GrammarTables {
    const int32_t* next;          // [n_states << log_pitch], -1: no way on
    const uint8_t* accepting;     // [n_states]
    const uint8_t* codes;         // classes of the tokens' bytes, token after token
    const int32_t* token_at;      // [width + 1] first code of each token; a token without codes is never allowed
    const uint64_t* text;         // [width] packed texts, 0: none; NULL: more than 15 classes
    // Masks: `step16` or `step32` [(n_states + 1) << log_pitch] holds (following state << log_pitch); state n_states is the
    // dead one, and the last class leads from every state to itself: a walk needs no test.
    const uint16_t* step16;
    const uint32_t* step32;
    const uint32_t* super;        // [n_super] what 32 groups share
    const uint2* prefix;          // [n_super * 32] x: what a group shares behind that; y: steps that its tokens take then, 0: no group, and
                                  // GRAMMAR_RUN if their ids follow one another
    const uint2* rest;            // [n_super * 1024] x: the first 8 classes that each token has behind the prefix; y: its id, -1: none
    const uint32_t* more;         // [n_super * 1024] the 8 classes behind those, read for groups that have any
    int32_t n_states, log_pitch, n_groups, n_super, super_steps, prefix_steps, n_runs;
    int64_t width;
    int64_t end_id;               // -1: none
};

template <typename S> __device__ __forceinline__ const S* grammar_steps(const GrammarTables& t);
template <> __device__ __forceinline__ const uint32_t* grammar_steps<uint32_t>(const GrammarTables& t) { return t.step32; }
template <> __device__ __forceinline__ const uint16_t* grammar_steps<uint16_t>(const GrammarTables& t) { return t.step16; }

// The state after a token's codes, for any number of classes.
__device__ __forceinline__ int32_t grammar_walk_codes(const GrammarTables& t, int32_t state, int64_t token) {
    const int32_t lo = t.token_at[token], hi = t.token_at[token + 1];
    if (lo == hi) return GRAMMAR_DEAD;
    for (int32_t i = lo; i < hi && state >= 0; ++i) state = __ldg(t.next + (((int64_t)state << t.log_pitch) | __ldg(t.codes + i)));
    return state < 0 ? GRAMMAR_DEAD : state;
}

__device__ __forceinline__ bool grammar_may_end(const GrammarTables& t, int32_t state) {
    return state == GRAMMAR_FINISHED || (state >= 0 && state < t.n_states && t.accepting[state]);
}

// The state after a token; a token outside the vocabulary leaves the row as it was.
__device__ __forceinline__ int32_t grammar_after(const GrammarTables& t, int32_t state, int64_t token) {
    if (token < 0 || token >= t.width) return state;
    if (token == t.end_id) return grammar_may_end(t, state) ? GRAMMAR_FINISHED : GRAMMAR_DEAD;
    if (state < 0 || state >= t.n_states) return GRAMMAR_DEAD;
    const uint64_t text = t.text ? t.text[token] : 15ull << 60;
    int n = (int)(text >> 60);
    if (n > GRAMMAR_PACKED) return grammar_walk_codes(t, state, token);
    if (n == 0) return GRAMMAR_DEAD;
    uint64_t left = text;
    for (; n > 0 && state >= 0; --n, left >>= 4) state = __ldg(t.next + (((int64_t)state << t.log_pitch) | (left & 15)));
    return state < 0 ? GRAMMAR_DEAD : state;
}

__device__ __forceinline__ int64_t grammar_token(const void* tokens, int token_bits, int64_t row) {
    return token_bits == 64 ? static_cast<const int64_t*>(tokens)[row] : static_cast<const int32_t*>(tokens)[row];
}

__global__ void __launch_bounds__(GRAMMAR_THREADS)
grammar_advance_kernel(GrammarTables t, const int32_t* states, const void* tokens, int token_bits, int64_t n_rows,
                       int32_t* out) {                        // (out may be the states, or the tokens)
    const int64_t row = (int64_t)blockIdx.x * GRAMMAR_THREADS + threadIdx.x;
    if (row < n_rows) out[row] = grammar_after(t, states[row], grammar_token(tokens, token_bits, row));
}

// Any number of classes and tokens: a warp takes one word of a row, a lane a token.
__global__ void __launch_bounds__(GRAMMAR_THREADS)
grammar_any_kernel(GrammarTables t, const int32_t* __restrict__ states, int64_t n_rows, uint32_t* __restrict__ allowed) {
    const int64_t words = (t.width + 31) / 32;
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * (GRAMMAR_THREADS / 32);
    for (int64_t w = (int64_t)blockIdx.x * (GRAMMAR_THREADS / 32) + (threadIdx.x >> 5); w < n_rows * words; w += warps) {
        const int64_t row = w / words, token = (w - row * words) * 32 + lane;
        const int32_t state = states[row];
        bool ok = false;
        if (token < t.width) {
            if (token == t.end_id) ok = grammar_may_end(t, state);
            else if (state >= 0 && state < t.n_states) ok = grammar_walk_codes(t, state, token) >= 0;
        }
        const uint32_t word = __ballot_sync(0xffffffffu, ok);
        if (lane == 0) allowed[w] = word;
    }
}

// A cluster of `parts` blocks takes a row.  Its warps share the sets of 32 groups that live (`split` warps a set: each takes
// every split-th of the groups); the tokens that live set their bits in the block's shared memory, and each block joins and
// writes its share of the words.  All counts are powers of two.  With `tokens` the row's state is advanced first (by every
// thread for itself: a warp that does it for the others keeps them waiting, 31 -> 39 us) and written by the cluster's first.
// NEAR: the table is small and copied to shared memory, so that a walk's steps do not each wait for the L2 the first time.
// RUNS: many groups' ids follow one another, as those of k-mers do; their bits are set as one word, since 32 lanes would
// queue up at it (1,024 rows of 4,106 tokens: 18 us, 22 without).
constexpr int GRAMMAR_NEAR_BYTES = 16 * 1024;
constexpr int GRAMMAR_MOST = 512;                             // threads a block; 40 registers: 3 blocks an SM

template <typename S, bool NEAR, bool CLUSTER, bool RUNS>
__global__ void __launch_bounds__(GRAMMAR_MOST, 3)
grammar_allowed_kernel(GrammarTables t, const int32_t* __restrict__ states, const void* __restrict__ tokens, int token_bits,
                       int32_t* __restrict__ states_out, uint32_t* __restrict__ allowed, int parts, int split) {
    extern __shared__ uint4 shared[];
    constexpr uint32_t FULL = 0xffffffffu;
    constexpr int TOGETHER = 4;                               // groups a warp walks at a time: their loads overlap
    const int words = (int)((t.width + 31) / 32);
    const S* table = grammar_steps<S>(t);
    S* near = reinterpret_cast<S*>(shared);
    uint32_t* set = reinterpret_cast<uint32_t*>(shared);      // [words], behind the table
    if (NEAR) {
        const int pieces = (int)((((size_t)(t.n_states + 1) << t.log_pitch) * sizeof(S) + 15) / 16);
        const uint4* from = reinterpret_cast<const uint4*>(table);
        for (int i = threadIdx.x; i < pieces; i += blockDim.x) shared[i] = __ldg(from + i);
        set += pieces * 4;
    }
    auto step = [&](uint32_t s, uint32_t code) -> uint32_t { return NEAR ? near[s | code] : __ldg(table + (s | code)); };
    const int64_t row = blockIdx.x / parts;
    const int part = (int)(blockIdx.x % parts);
    for (int w = threadIdx.x; w < words; w += blockDim.x) set[w] = 0;
    const uint32_t dead = (uint32_t)t.n_states << t.log_pitch;
    int32_t state = states[row];
    __syncthreads();
    if (tokens) {
        const int64_t token = grammar_token(tokens, token_bits, row);
        const uint64_t text = token >= 0 && token < t.width && token != t.end_id && state >= 0 && state < t.n_states ? __ldg(t.text + token) : 0;
        const int n = (int)(text >> 60);
        if (n > 0 && n <= GRAMMAR_PACKED) {                   // (everything else: grammar_after)
            uint32_t s = (uint32_t)state << t.log_pitch;
            uint64_t left = text;
            for (int i = 0; i < n; ++i, left >>= 4) s = step(s, (uint32_t)left & 15);
            state = s == dead ? GRAMMAR_DEAD : (int32_t)(s >> t.log_pitch);
        } else {
            state = grammar_after(t, state, token);
        }
        if (part == 0 && threadIdx.x == 0) states_out[row] = state;
    }
    if (state >= 0 && state < t.n_states) {
        const int lane = threadIdx.x & 31, all_warps = (int)(blockDim.x >> 5) * parts, me = part * (int)(blockDim.x >> 5) + (int)(threadIdx.x >> 5);
        int ranks = 0;                                        // sets that lived so far
        for (int s0 = 0; s0 < t.n_super; s0 += 32) {
            uint32_t of_set = dead;                           // state behind what this lane's set shares
            if (s0 + lane < t.n_super) {
                uint32_t text = __ldg(t.super + s0 + lane);
                of_set = (uint32_t)state << t.log_pitch;
                for (int n = 0; n < t.super_steps && of_set != dead; ++n, text >>= 4) of_set = step(of_set, text & 15);
            }
            __syncwarp();
            const uint32_t live = __ballot_sync(FULL, of_set != dead);
            const int share = (me - (ranks + __popc(live & ((1u << lane) - 1))) * split) & (all_warps - 1);   // which of a set's shares is this warp's
            uint32_t sets = __ballot_sync(FULL, of_set != dead && share < split);
            ranks += __popc(live);
            while (sets) {
                const int k0 = __ffs(sets) - 1;
                sets &= sets - 1;
                const int g0 = (s0 + k0) * 32;
                const uint2 group = __ldg(t.prefix + g0 + lane);
                const int steps_mine = (int)(group.y & 255), run_mine = (int)(group.y & GRAMMAR_RUN);
                uint32_t mine = __shfl_sync(FULL, of_set, k0);    // state behind the prefix of this lane's group
                if ((lane & (split - 1)) != __shfl_sync(FULL, share, k0) || steps_mine == 0) mine = dead;
                uint32_t prefix = group.x;
                for (int n = 0; n < t.prefix_steps && mine != dead; ++n, prefix >>= 4) mine = step(mine, prefix & 15);
                __syncwarp();
                uint32_t alive = __ballot_sync(FULL, mine != dead && steps_mine != GRAMMAR_SLOW);
                uint32_t slow = __ballot_sync(FULL, mine != dead && steps_mine == GRAMMAR_SLOW);
                auto walk = [&](auto together) {                  // the next groups of `alive`, that many at a time
                    constexpr int N = decltype(together)::value;
                    uint2 text[N];
                    int at[N];
                    uint32_t s[N];
                    int run[N], steps = 0;
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const int k = __ffs(alive) - 1;
                        alive &= alive - 1;
                        at[i] = (g0 + k) * 32 + lane;
                        text[i] = __ldg(t.rest + at[i]);
                        s[i] = __shfl_sync(FULL, mine, k);
                        steps = max(steps, __shfl_sync(FULL, steps_mine, k));
                        run[i] = RUNS ? __shfl_sync(FULL, run_mine, k) : 0;
                    }
                    for (int n = 0; n < steps; ++n) {
                        if (n == 8) {
#pragma unroll
                            for (int i = 0; i < N; ++i) text[i].x = __ldg(t.more + at[i]);
                        }
#pragma unroll
                        for (int i = 0; i < N; ++i) {
                            s[i] = step(s[i], text[i].x & 15);
                            text[i].x >>= 4;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const bool ok = s[i] != dead && (int)text[i].y >= 0;
                        if (RUNS && run[i]) {
                            const uint32_t word = __ballot_sync(FULL, ok);
                            const uint32_t at = __shfl_sync(FULL, text[i].y, 0);
                            if (lane < 2 && word) {
                                const uint32_t bits = lane == 0 ? word << (at & 31) : (at & 31) ? word >> (32 - (at & 31)) : 0;
                                if (bits) atomicOr(set + (at >> 5) + lane, bits);
                            }
                        } else if (ok) {
                            atomicOr(set + (text[i].y >> 5), 1u << (text[i].y & 31));
                        }
                    }
                };
                while (__popc(alive) >= TOGETHER) walk(std::integral_constant<int, TOGETHER>());
                while (__popc(alive) >= 2) walk(std::integral_constant<int, 2>());
                if (alive) walk(std::integral_constant<int, 1>());
                while (slow) {                                    // groups with a longer token: from the row's state, code by code
                    const int k = __ffs(slow) - 1;
                    slow &= slow - 1;
                    const int32_t id = (int32_t)__ldg(&t.rest[(g0 + k) * 32 + lane].y);
                    if (id >= 0 && grammar_walk_codes(t, state, id) >= 0) atomicOr(set + (id >> 5), 1u << (id & 31));
                }
            }
        }
    }
    if (threadIdx.x == 0 && part == 0 && t.end_id >= 0 && grammar_may_end(t, state)) atomicOr(set + (t.end_id >> 5), 1u << (t.end_id & 31));
    uint32_t* out = allowed + row * words;
    if (CLUSTER) {
        cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
        cluster.sync();
        const int each = (words + parts - 1) / parts;
        const int end = (part + 1) * each < words ? (part + 1) * each : words;
        for (int w = part * each + threadIdx.x; w < end; w += blockDim.x) {
            uint32_t word = 0;
            for (int p = 0; p < parts; ++p) word |= cluster.map_shared_rank(set, p)[w];
            out[w] = word;
        }
        cluster.sync();                                       // nobody leaves while its words are read
    } else {
        __syncthreads();
        for (int w = threadIdx.x; w < words; w += blockDim.x) out[w] = set[w];
    }
}

}  // namespace dnatok
