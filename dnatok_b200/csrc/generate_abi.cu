// C ABI of the operators between a model's logits and the choice of its next token (see include/dnatok_b200.h).
#include "../../include/dnatok_b200.h"

#include <climits>
#include <map>
#include <mutex>
#include <new>
#include <vector>

#include "abi_shared.h"
#include "grammar_kernel.cuh"
#include "history_kernel.cuh"
#include "logits_kernel.cuh"

using namespace dnatok;

namespace {

#define CUDA_TRY(expr)                                                                              \
    do {                                                                                            \
        cudaError_t e_ = (expr);                                                                    \
        if (e_ != cudaSuccess) return abi_fail(DNATOK_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(e_)); \
    } while (0)

#define LAUNCH_CHECK(name)                                                                          \
    do {                                                                                            \
        abi_count_launch();                                                                         \
        cudaError_t e_ = cudaGetLastError();                                                        \
        if (e_ != cudaSuccess) return abi_fail(DNATOK_ERR_CUDA, "launch of %s: %s", name, cudaGetErrorString(e_)); \
    } while (0)

bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
size_t size_of(int dtype) { return dtype == DNATOK_F32 ? 4 : 2; }
bool known(int dtype) { return dtype == DNATOK_F32 || dtype == DNATOK_F16 || dtype == DNATOK_BF16; }

// Blocks for `n` threads' worth of work in blocks of `threads`, at most what a grid-stride loop needs to fill the GPU.
unsigned blocks_for(int64_t n, int threads, int64_t most = 148 * 16) {
    const int64_t b = (n + threads - 1) / threads;
    return (unsigned)(b < 1 ? 1 : b > most ? most : b);
}

int check_rows(const void* rows, int bits, int64_t n_rows, int64_t history_rows) {
    if (rows) {
        if (bits != 32 && bits != 64) return abi_fail(DNATOK_ERR_INVALID, "rows_bits must be 32 or 64");
        if (!aligned(rows, (size_t)bits / 8)) return abi_fail(DNATOK_ERR_INVALID, "misaligned row numbers");
    } else if (history_rows != n_rows) {
        return abi_fail(DNATOK_ERR_INVALID, "the history has %lld rows, the call %lld", (long long)history_rows, (long long)n_rows);
    }
    return 0;
}

int check_logits(const dnatok_logits* in) {
    if (!in) return abi_fail(DNATOK_ERR_INVALID, "NULL argument");
    if (!known(in->dtype)) return abi_fail(DNATOK_ERR_INVALID, "unknown type of logits");
    if (in->n_rows < 0 || in->width < 1 || in->width > INT32_MAX) return abi_fail(DNATOK_ERR_INVALID, "bad number of rows or columns");
    if (in->stride < 0) return abi_fail(DNATOK_ERR_INVALID, "stride < 0");
    if (in->n_rows && !in->logits) return abi_fail(DNATOK_ERR_INVALID, "logits is NULL");
    if (!aligned(in->logits, size_of(in->dtype))) return abi_fail(DNATOK_ERR_INVALID, "misaligned logits");
    if (in->counts && !in->seen) return abi_fail(DNATOK_ERR_INVALID, "counts without seen");
    if (in->seen) {
        if (in->history_rows < 0) return abi_fail(DNATOK_ERR_INVALID, "history_rows < 0");
        if (int rc = check_rows(in->rows, in->rows_bits, in->n_rows, in->history_rows)) return rc;
    }
    const int64_t words = (in->width + 31) / 32;
    if (in->bias && in->bias_stride != 0 && in->bias_stride < in->width) return abi_fail(DNATOK_ERR_INVALID, "bias_stride smaller than a row");
    if (in->allowed && in->allowed_stride != 0 && in->allowed_stride < words) return abi_fail(DNATOK_ERR_INVALID, "allowed_stride smaller than a row");
    const void* words32[] = {in->seen, in->counts, in->d_repetition, in->d_frequency, in->d_presence, in->bias, in->allowed};
    for (const void* p : words32) if (!aligned(p, 4)) return abi_fail(DNATOK_ERR_INVALID, "misaligned 32-bit array");
    if (!in->d_repetition && !(in->repetition > 0.f)) return abi_fail(DNATOK_ERR_INVALID, "repetition must be positive");
    return 0;
}

LogitsArgs logits_args(const dnatok_logits* in) {
    LogitsArgs a;
    a.n_rows = in->n_rows; a.width = in->width; a.stride = in->stride;
    a.seen = in->seen; a.counts = in->counts; a.history_rows = in->history_rows;
    a.rows = in->rows; a.rows_bits = in->rows_bits;
    a.repetition = in->repetition; a.frequency = in->frequency; a.presence = in->presence;
    a.d_repetition = in->d_repetition; a.d_frequency = in->d_frequency; a.d_presence = in->d_presence;
    a.bias = in->bias; a.bias_stride = in->bias_stride;
    a.allowed = in->allowed; a.allowed_stride = in->allowed_stride;
    return a;
}

int check_output(const char* what, const void* p, size_t size, int64_t stride, const dnatok_logits* in) {
    if (in->n_rows && !p) return abi_fail(DNATOK_ERR_INVALID, "%s is NULL", what);
    if (!aligned(p, size)) return abi_fail(DNATOK_ERR_INVALID, "misaligned %s", what);
    if (in->n_rows > 1 && stride < in->width) return abi_fail(DNATOK_ERR_INVALID, "rows of %s overlap", what);
    return 0;
}

// Calls f with a null pointer of the element type.
template <typename F>
void with_type(int dtype, F f) {
    if (dtype == DNATOK_F32) f((float*)nullptr);
    else if (dtype == DNATOK_F16) f((__half*)nullptr);
    else f((__nv_bfloat16*)nullptr);
}

}  // namespace

extern "C" {

int dnatok_process_logits(const dnatok_logits* in, void* d_out, int32_t out_dtype, int64_t out_stride, dnatok_stream stream) {
    if (int rc = check_logits(in)) return rc;
    if (out_dtype != in->dtype && out_dtype != DNATOK_F32) return abi_fail(DNATOK_ERR_INVALID, "the output has the logits' type or is float");
    if (int rc = check_output("output", d_out, size_of(out_dtype), out_stride, in)) return rc;
    if (d_out == in->logits && in->n_rows && (out_dtype != in->dtype || (in->n_rows > 1 && out_stride != in->stride)))
        return abi_fail(DNATOK_ERR_INVALID, "in place the output has the logits' type and stride");
    if (in->n_rows == 0) return DNATOK_OK;
    cudaStream_t st = (cudaStream_t)stream;
    const LogitsArgs a = logits_args(in);
    const unsigned grid = blocks_for(a.n_rows * a.width, LOGITS_THREADS);
    with_type(in->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (out_dtype == in->dtype) process_logits_kernel<T, T><<<grid, LOGITS_THREADS, 0, st>>>(a, (const T*)in->logits, (T*)d_out, out_stride);
        else process_logits_kernel<T, float><<<grid, LOGITS_THREADS, 0, st>>>(a, (const T*)in->logits, (float*)d_out, out_stride);
    });
    LAUNCH_CHECK("process_logits_kernel");
    return DNATOK_OK;
}

size_t dnatok_logits_scratch_bytes(int64_t n_rows, int64_t width) {
    (void)n_rows; (void)width;
    return 0;
}

int dnatok_process_logits_backward(const dnatok_logits* in, const void* d_grad, int32_t grad_dtype, int64_t grad_stride,
                                   void* d_dlogits, int64_t dlogits_stride, float* d_dbias, void* d_scratch,
                                   size_t scratch_bytes, dnatok_stream stream) {
    if (int rc = check_logits(in)) return rc;
    if (grad_dtype != in->dtype && grad_dtype != DNATOK_F32) return abi_fail(DNATOK_ERR_INVALID, "the gradient has the logits' type or is float");
    if (grad_stride < 0) return abi_fail(DNATOK_ERR_INVALID, "grad_stride < 0");
    if (in->n_rows && !d_grad) return abi_fail(DNATOK_ERR_INVALID, "gradient is NULL");
    if (!aligned(d_grad, size_of(grad_dtype)) || !aligned(d_dbias, 4)) return abi_fail(DNATOK_ERR_INVALID, "misaligned gradient");
    if (d_dlogits) if (int rc = check_output("logits' gradient", d_dlogits, size_of(in->dtype), dlogits_stride, in)) return rc;
    if (d_dlogits && d_dlogits == d_grad && in->n_rows && (grad_dtype != in->dtype || (in->n_rows > 1 && grad_stride != dlogits_stride)))
        return abi_fail(DNATOK_ERR_INVALID, "in place both gradients have one type and stride");
    (void)d_scratch; (void)scratch_bytes;
    cudaStream_t st = (cudaStream_t)stream;
    const bool shared = in->bias_stride == 0;
    if (in->n_rows == 0) {
        if (d_dbias && shared) CUDA_TRY(cudaMemsetAsync(d_dbias, 0, (size_t)in->width * 4, st));
        return DNATOK_OK;
    }
    const LogitsArgs a = logits_args(in);
    auto run = [&](auto* t, auto* g) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        using G = std::remove_pointer_t<decltype(g)>;
        if (d_dbias && shared) {       // before the logits' gradient, which may overwrite the gradient
            bias_gradient_kernel<G><<<(unsigned)((a.width + LOGITS_THREADS - 1) / LOGITS_THREADS), LOGITS_THREADS, 0, st>>>(
                a, (const G*)d_grad, grad_stride, d_dbias);
            LAUNCH_CHECK("bias_gradient_kernel");
        }
        if (d_dlogits || (d_dbias && !shared)) {
            logits_gradient_kernel<T, G><<<blocks_for(a.n_rows * a.width, LOGITS_THREADS), LOGITS_THREADS, 0, st>>>(
                a, (const T*)in->logits, (const G*)d_grad, grad_stride, (T*)d_dlogits, dlogits_stride, shared ? nullptr : d_dbias);
            LAUNCH_CHECK("logits_gradient_kernel");
        }
        return DNATOK_OK;
    };
    int rc = DNATOK_OK;
    with_type(in->dtype, [&](auto* t) { rc = grad_dtype == in->dtype ? run(t, t) : run(t, (float*)nullptr); });
    return rc;
}

// ------------------------------------------------------------------ history

int dnatok_history_add(const dnatok_history* h, int32_t generated, dnatok_stream stream) {
    if (!h) return abi_fail(DNATOK_ERR_INVALID, "NULL argument");
    if (h->n_rows < 0 || h->history_rows < 0 || h->width < 1 || h->width > INT32_MAX) return abi_fail(DNATOK_ERR_INVALID, "bad sizes of the history");
    if (h->id_bits != 32 && h->id_bits != 64) return abi_fail(DNATOK_ERR_INVALID, "id_bits must be 32 or 64");
    if (int rc = check_rows(h->rows, h->rows_bits, h->n_rows, h->history_rows)) return rc;
    if (h->offsets && h->lengths) return abi_fail(DNATOK_ERR_INVALID, "flat ids have offsets, padded ones lengths");
    if (h->offsets ? h->total < 0 : (h->columns < 0 || h->id_stride < 0)) return abi_fail(DNATOK_ERR_INVALID, "bad sizes of the ids");
    if (h->n_rows == 0 || (h->offsets ? h->total : h->columns) == 0 || h->history_rows == 0) return DNATOK_OK;
    if (!h->seen || !h->ids) return abi_fail(DNATOK_ERR_INVALID, "NULL argument");
    if (!aligned(h->ids, (size_t)h->id_bits / 8) || !aligned(h->seen, 4) || !aligned(h->counts, 4) || !aligned(h->lengths, 4) || !aligned(h->offsets, 8))
        return abi_fail(DNATOK_ERR_INVALID, "misaligned array");
    HistoryArgs a;
    a.seen = h->seen; a.counts = generated ? h->counts : nullptr; a.history_rows = h->history_rows; a.width = h->width;
    a.n_rows = h->n_rows; a.columns = h->columns; a.id_stride = h->id_stride;
    a.offsets = h->offsets; a.total = h->total; a.lengths = h->lengths; a.pad_left = h->pad_left;
    a.rows = h->rows; a.rows_bits = h->rows_bits;
    cudaStream_t st = (cudaStream_t)stream;
    const unsigned grid = blocks_for(a.n_rows * 32, HISTORY_THREADS);
    if (h->id_bits == 64) history_add_kernel<int64_t><<<grid, HISTORY_THREADS, 0, st>>>(a, (const int64_t*)h->ids);
    else history_add_kernel<int32_t><<<grid, HISTORY_THREADS, 0, st>>>(a, (const int32_t*)h->ids);
    LAUNCH_CHECK("history_add_kernel");
    return DNATOK_OK;
}

}  // extern "C"

// ------------------------------------------------------------------ grammars

struct dnatok_grammar {
    std::vector<int32_t> next;
    std::vector<uint8_t> accepting, codes;
    std::vector<int32_t> token_at;
    int32_t n_states = 0, n_classes = 0;
    int64_t width = 0, end_id = -1;
    struct Device { void* memory = nullptr; GrammarTables tables{}; };
    std::mutex mu;
    std::map<int, Device> dev;
};

namespace {

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// The tables on the current device, uploaded on first use: one allocation, filled on a stream of its own.
int grammar_tables(dnatok_grammar* g, cudaStream_t stream, GrammarTables* out) {
    int dev = 0;
    CUDA_TRY(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(g->mu);
    auto it = g->dev.find(dev);
    if (it == g->dev.end()) {
        cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
        CUDA_TRY(cudaStreamIsCapturing(stream, &capturing));
        if (capturing != cudaStreamCaptureStatusNone)
            return abi_fail(DNATOK_ERR_INVALID, "a grammar's first use on a device must be outside of stream capture");
        const size_t sizes[4] = {g->next.size() * 4, g->accepting.size(), g->codes.size(), g->token_at.size() * 4};
        const void* from[4] = {g->next.data(), g->accepting.data(), g->codes.data(), g->token_at.data()};
        size_t at[5] = {0};
        for (int i = 0; i < 4; ++i) at[i + 1] = at[i] + up256(sizes[i] + 1);
        struct Undo {
            void* memory = nullptr;
            cudaStream_t copies = nullptr;
            ~Undo() { if (copies) cudaStreamDestroy(copies); if (memory) cudaFree(memory); }
        } undo;
        CUDA_TRY(cudaMalloc(&undo.memory, at[4]));
        CUDA_TRY(cudaStreamCreateWithFlags(&undo.copies, cudaStreamNonBlocking));
        char* base = (char*)undo.memory;
        for (int i = 0; i < 4; ++i)
            if (sizes[i]) CUDA_TRY(cudaMemcpyAsync(base + at[i], from[i], sizes[i], cudaMemcpyHostToDevice, undo.copies));
        CUDA_TRY(cudaStreamSynchronize(undo.copies));
        dnatok_grammar::Device d;
        GrammarTables& t = d.tables;
        t.next = (const int32_t*)(base + at[0]);
        t.accepting = (const uint8_t*)(base + at[1]);
        t.codes = (const uint8_t*)(base + at[2]);
        t.token_at = (const int32_t*)(base + at[3]);
        t.n_states = g->n_states; t.n_classes = g->n_classes; t.width = g->width; t.end_id = g->end_id;
        d.memory = undo.memory;
        it = g->dev.emplace(dev, d).first;
        undo.memory = nullptr;
    }
    *out = it->second.tables;
    return 0;
}

int check_states(const dnatok_grammar* g, const void* states, int64_t n_rows) {
    if (!g || n_rows < 0 || (n_rows && !states)) return abi_fail(DNATOK_ERR_INVALID, "bad argument");
    if (!aligned(states, 4)) return abi_fail(DNATOK_ERR_INVALID, "misaligned states");
    return 0;
}

int launch_allowed(const GrammarTables& t, const int32_t* states, int64_t n_rows, uint32_t* allowed, cudaStream_t st) {
    grammar_allowed_kernel<<<blocks_for(n_rows * ((t.width + 31) / 32) * 32, GRAMMAR_THREADS), GRAMMAR_THREADS, 0, st>>>(t, states, n_rows, allowed);
    LAUNCH_CHECK("grammar_allowed_kernel");
    return DNATOK_OK;
}

}  // namespace

extern "C" {

int dnatok_create_grammar(const int32_t* next, int32_t n_states, int32_t n_classes, const uint8_t* accepting,
                          const uint8_t byte_class[256], const uint8_t* token_bytes, const int64_t* token_offsets,
                          int64_t width, int64_t end_id, dnatok_grammar** out) {
    if (!next || !accepting || !byte_class || !token_offsets || !out) return abi_fail(DNATOK_ERR_INVALID, "NULL argument");
    if (n_states < 1 || n_classes < 1 || n_classes > 256) return abi_fail(DNATOK_ERR_INVALID, "bad number of states or classes");
    if (width < 1 || width > INT32_MAX) return abi_fail(DNATOK_ERR_INVALID, "bad number of tokens");
    if (end_id < -1 || end_id >= width) return abi_fail(DNATOK_ERR_INVALID, "end_id outside the vocabulary");
    for (int i = 0; i < 256; ++i) if (byte_class[i] >= n_classes) return abi_fail(DNATOK_ERR_INVALID, "class of byte %d outside the automaton", i);
    for (int64_t i = 0; i < (int64_t)n_states * n_classes; ++i)
        if (next[i] < -1 || next[i] >= n_states) return abi_fail(DNATOK_ERR_INVALID, "state %lld leads to state %d", (long long)(i / n_classes), next[i]);
    if (token_offsets[0] != 0) return abi_fail(DNATOK_ERR_INVALID, "token_offsets must start at 0");
    for (int64_t v = 0; v < width; ++v)
        if (token_offsets[v + 1] < token_offsets[v]) return abi_fail(DNATOK_ERR_INVALID, "token_offsets decrease at token %lld", (long long)v);
    const int64_t total = token_offsets[width];
    if (total > INT32_MAX) return abi_fail(DNATOK_ERR_UNSUPPORTED, "more than 2^31 - 1 bytes of tokens");
    if (total && !token_bytes) return abi_fail(DNATOK_ERR_INVALID, "NULL argument");
    try {
        auto* g = new dnatok_grammar();
        struct Undo { dnatok_grammar* g; ~Undo() { delete g; } } undo{g};
        g->n_states = n_states; g->n_classes = n_classes; g->width = width; g->end_id = end_id;
        g->next.assign(next, next + (int64_t)n_states * n_classes);
        g->accepting.resize((size_t)n_states);
        for (int32_t i = 0; i < n_states; ++i) g->accepting[(size_t)i] = accepting[i] != 0;
        g->codes.resize((size_t)total);
        for (int64_t i = 0; i < total; ++i) g->codes[(size_t)i] = byte_class[token_bytes[i]];
        g->token_at.resize((size_t)width + 1);
        for (int64_t v = 0; v <= width; ++v) g->token_at[(size_t)v] = (int32_t)token_offsets[v];
        undo.g = nullptr;
        *out = g;
    } catch (const std::bad_alloc&) {
        return abi_fail(DNATOK_ERR_INVALID, "out of memory");
    }
    return DNATOK_OK;
}

void dnatok_destroy_grammar(dnatok_grammar* g) {
    if (!g) return;
    int cur = 0;
    if (!g->dev.empty()) cudaGetDevice(&cur);
    // may run while some stream is captured: a free is no part of the capture and must not end it
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    if (!g->dev.empty()) cudaThreadExchangeStreamCaptureMode(&mode);
    for (auto& kv : g->dev) if (cudaSetDevice(kv.first) == cudaSuccess) cudaFree(kv.second.memory);
    if (!g->dev.empty()) {
        cudaThreadExchangeStreamCaptureMode(&mode);
        cudaSetDevice(cur);
    }
    delete g;
}

int dnatok_grammar_allowed(dnatok_grammar* g, const int32_t* d_states, int64_t n_rows, uint32_t* d_allowed, dnatok_stream stream) {
    if (int rc = check_states(g, d_states, n_rows)) return rc;
    if (n_rows && !d_allowed) return abi_fail(DNATOK_ERR_INVALID, "mask is NULL");
    if (!aligned(d_allowed, 4)) return abi_fail(DNATOK_ERR_INVALID, "misaligned mask");
    if (n_rows == 0) return DNATOK_OK;
    GrammarTables t;
    if (int rc = grammar_tables(g, (cudaStream_t)stream, &t)) return rc;
    return launch_allowed(t, d_states, n_rows, d_allowed, (cudaStream_t)stream);
}

int dnatok_grammar_step(dnatok_grammar* g, const int32_t* d_states, const void* d_tokens, int32_t token_bits, int64_t n_rows,
                        int32_t* d_states_out, uint32_t* d_allowed, dnatok_stream stream) {
    if (int rc = check_states(g, d_states, n_rows)) return rc;
    if (token_bits != 32 && token_bits != 64) return abi_fail(DNATOK_ERR_INVALID, "token_bits must be 32 or 64");
    if (n_rows && (!d_tokens || !d_states_out)) return abi_fail(DNATOK_ERR_INVALID, "NULL argument");
    if (!aligned(d_tokens, (size_t)token_bits / 8) || !aligned(d_states_out, 4) || !aligned(d_allowed, 4))
        return abi_fail(DNATOK_ERR_INVALID, "misaligned array");
    if (d_allowed && d_states_out == d_states && n_rows) return abi_fail(DNATOK_ERR_INVALID, "with a mask the new states need an array of their own");
    if (n_rows == 0) return DNATOK_OK;
    GrammarTables t;
    cudaStream_t st = (cudaStream_t)stream;
    if (int rc = grammar_tables(g, st, &t)) return rc;
    grammar_advance_kernel<<<(unsigned)((n_rows + GRAMMAR_THREADS - 1) / GRAMMAR_THREADS), GRAMMAR_THREADS, 0, st>>>(t, d_states, d_tokens, token_bits, n_rows, d_states_out);
    LAUNCH_CHECK("grammar_advance_kernel");
    return d_allowed ? launch_allowed(t, d_states_out, n_rows, d_allowed, st) : DNATOK_OK;
}

}  // extern "C"
