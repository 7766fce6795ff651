// C ABI of the operators between a model's logits and the choice of its next token (see include/dnatok_b200.h).
#include "../../include/dnatok_b200.h"

#include <algorithm>
#include <climits>
#include <cstring>
#include <map>
#include <mutex>
#include <new>
#include <type_traits>
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
constexpr int SMS = 148;
unsigned blocks_for(int64_t n, int threads, int64_t most = SMS * 16) {
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

constexpr int64_t LOGITS_MOST = INT32_MAX - 1024 * 1024;        // rows or columns: what is added to them stays in 32 bits

int check_logits(const dnatok_logits* in) {
    if (!in) return abi_fail(DNATOK_ERR_INVALID, "NULL argument");
    if (!known(in->dtype)) return abi_fail(DNATOK_ERR_INVALID, "unknown type of logits");
    if (in->n_rows < 0 || in->n_rows > LOGITS_MOST || in->width < 1 || in->width > LOGITS_MOST)
        return abi_fail(DNATOK_ERR_INVALID, "bad number of rows or columns");
    if (in->stride < 0) return abi_fail(DNATOK_ERR_INVALID, "stride < 0");
    if (in->n_rows && !in->logits) return abi_fail(DNATOK_ERR_INVALID, "logits is NULL");
    if (!aligned(in->logits, size_of(in->dtype))) return abi_fail(DNATOK_ERR_INVALID, "misaligned logits");
    if (in->counts && !in->seen) return abi_fail(DNATOK_ERR_INVALID, "counts without seen");
    if (in->seen) {
        if (in->history_rows < 0 || in->history_rows > INT32_MAX) return abi_fail(DNATOK_ERR_INVALID, "bad number of history rows");
        if (int rc = check_rows(in->rows, in->rows_bits, in->n_rows, in->history_rows)) return rc;
    }
    const int64_t words = (in->width + 31) / 32;
    if (in->bias && in->bias_stride != 0 && in->bias_stride < in->width) return abi_fail(DNATOK_ERR_INVALID, "bias_stride smaller than a row");
    if (in->allowed && in->allowed_stride != 0 && in->allowed_stride < words) return abi_fail(DNATOK_ERR_INVALID, "allowed_stride smaller than a row");
    const void* words32[] = {in->seen, in->counts, in->d_repetition, in->d_frequency, in->d_presence, in->bias, in->allowed};
    for (const void* p : words32) if (!aligned(p, 4)) return abi_fail(DNATOK_ERR_INVALID, "misaligned 32-bit array");
    if (!in->d_repetition && !(in->repetition >= 0x1p-126f && in->repetition <= 0x1p126f))      // (so that 1 / r is a normal number too)
        return abi_fail(DNATOK_ERR_INVALID, "repetition must be positive and finite (2^-126 to 2^126)");
    return 0;
}

LogitsArgs logits_args(const dnatok_logits* in) {
    LogitsArgs a;
    a.n_rows = (int32_t)in->n_rows; a.width = (int32_t)in->width; a.stride = in->stride;
    a.seen = in->seen; a.counts = in->counts; a.history_rows = (int32_t)in->history_rows;
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

// Rows of an array, all in bytes.  (128 bits: no stride is too long.)
using Wide = __int128;
struct Rows {
    const void* p;
    Wide n, stride, row;
};

// Whether two arrays have a byte in common.  Rows may lie between those of the other array, as the columns of a view of one
// wider array do.
bool overlap(Rows a, Rows b) {
    if (!a.p || !b.p || a.n < 1 || b.n < 1 || a.row < 1 || b.row < 1) return false;
    if (a.stride == 0) a.n = 1;
    if (b.stride == 0) b.n = 1;
    const Wide a0 = (Wide)(uintptr_t)a.p, b0 = (Wide)(uintptr_t)b.p;
    const Wide a1 = a0 + (a.n - 1) * a.stride + a.row, b1 = b0 + (b.n - 1) * b.stride + b.row;
    if (a1 <= b0 || b1 <= a0) return false;
    if (a.n > 1 && b.n > 1 && a.stride == b.stride) {
        // row j of b is b0 - a0 + (j - i) stride behind row i of a: the first such distance that does not end before a's row
        const Wide d = b0 - a0, from = -b.row - d, s = a.stride;
        Wide m = (from >= 0 ? from / s : -((-from + s - 1) / s)) + 1;
        if (m < 1 - a.n) m = 1 - a.n;
        return m <= b.n - 1 && d + m * s < a.row;
    }
    for (Wide i = 0, j = 0; i < a.n && j < b.n;) {             // both in order: the row that ends first is passed
        const Wide x = a0 + i * a.stride, y = b0 + j * b.stride;
        if (x + a.row <= y) i += a.n == 1 ? 1 : (y - x - a.row) / a.stride + 1;
        else if (y + b.row <= x) j += b.n == 1 ? 1 : (x - y - b.row) / b.stride + 1;
        else return true;
    }
    return false;
}

// An output may not overlap what other threads still read.  The logits themselves are the caller's to look at.
int check_apart(const char* what, const Rows& out, const dnatok_logits* in) {
    const Wide n = in->n_rows, width = in->width, words = (width + 31) / 32;
    const struct { const char* name; Rows rows; } read[] = {
        {"bias", {in->bias, n, (Wide)in->bias_stride * 4, width * 4}},
        {"mask", {in->allowed, n, (Wide)in->allowed_stride * 4, words * 4}},
        {"history's words", {in->seen, in->history_rows, words * 4, words * 4}},
        {"history's counts", {in->counts, in->history_rows, width * 4, width * 4}},
        {"row numbers", {in->seen ? in->rows : nullptr, n, in->rows_bits / 8, in->rows_bits / 8}},
        {"repetition penalties", {in->d_repetition, n, 4, 4}},
        {"frequency penalties", {in->d_frequency, n, 4, 4}},
        {"presence penalties", {in->d_presence, n, 4, 4}},
    };
    for (const auto& r : read)
        if (overlap(out, r.rows)) return abi_fail(DNATOK_ERR_INVALID, "%s and %s overlap", what, r.name);
    return 0;
}

// Whether rows of elements of `size` bytes can be moved 16 bytes at a time.  An array that is not there can.
bool vector_rows(const void* p, int64_t stride, size_t size, int64_t n_rows) {
    return !p || (aligned(p, 16) && (n_rows <= 1 || stride * (int64_t)size % 16 == 0));
}

int64_t rows_per_block(int64_t n_rows, int64_t groups) {
    const int64_t per_warp = (n_rows + groups * LOGITS_WARPS - 1) / (groups * LOGITS_WARPS);
    return per_warp * LOGITS_WARPS;
}

int64_t tiles_of(int64_t width, int parts) { return (width + LOGITS_PART * parts - 1) / (LOGITS_PART * parts); }

// Parts a tile (see logits_kernel.cuh): one as long as that gives at most 4 warps to each of the GPU's schedulers.
int logits_parts(int64_t n_rows, int64_t width) { return n_rows * tiles_of(width, 1) <= (int64_t)SMS * 16 ? 1 : 2; }

// A warp for every tile of columns and row.
dim3 logits_grid(int64_t n_rows, int64_t width, int parts) {
    const int64_t groups = (n_rows + LOGITS_WARPS - 1) / LOGITS_WARPS;
    return dim3((unsigned)tiles_of(width, parts), (unsigned)(groups < 65535 ? groups : 65535));
}

// With a shared bias' gradient a block goes through several groups of rows, as many as leave at most 12 blocks an SM (three
// whole rounds of 4, four of 3): their partial sums are few beside what they read.  Up to 32 rows one block does them all,
// four a warp, which saves the launch that joins: about 3 us of the host.  On the GPU alone, calls following one another in a
// graph, it gains up to 16 rows and loses behind (float, one block and two launches: 16 x 32,000 4.6 and 5.3 us, 9 x 4,096 4.2
// and 4.6, 32 x 4,096 7.4 and 4.9, 32 x 32,000 10.6 and 6.9).
dim3 bias_grid(int64_t n_rows, int64_t width, int parts) {
    const int64_t tiles = tiles_of(width, parts);
    int64_t groups = (int64_t)SMS * 12 / tiles;
    const int64_t most = (n_rows + LOGITS_WARPS - 1) / LOGITS_WARPS;
    if (groups > most) groups = most;
    if (groups < 1 || n_rows <= 32) groups = 1;
    const int64_t rows = rows_per_block(n_rows, groups);
    return dim3((unsigned)tiles, (unsigned)((n_rows + rows - 1) / rows));
}

// Which columns a lane takes, whether there is a history, and the parts of a tile (see logits_kernel.cuh).
template <size_t S, size_t U, typename F>
void with_variant(bool vector, int64_t width, bool seen, int parts, F f) {
    constexpr int MAP = (S > 2 || U > 2) ? HALVES : CONTIGUOUS;
    auto tiled = [&](auto m, auto s) { if (parts == 1) f(m, s, std::integral_constant<int, 1>()); else f(m, s, std::integral_constant<int, 2>()); };
    auto known = [&](auto m) { if (seen) tiled(m, std::true_type()); else tiled(m, std::false_type()); };
    if (!vector || width % (MAP == HALVES ? 4 : 8)) known(std::integral_constant<int, APART>());
    else known(std::integral_constant<int, MAP>());
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
    const Wide size = size_of(in->dtype), out_size = size_of(out_dtype);
    const Rows out = {d_out, in->n_rows, out_stride * out_size, in->width * out_size};
    if (d_out != in->logits && overlap(out, {in->logits, in->n_rows, in->stride * size, in->width * size}))
        return abi_fail(DNATOK_ERR_INVALID, "output and logits overlap (the output may be the logits themselves)");
    if (int rc = check_apart("output", out, in)) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    const LogitsArgs a = logits_args(in);
    const bool vector = vector_rows(in->logits, in->stride, size_of(in->dtype), in->n_rows) &&
                        vector_rows(d_out, out_stride, size_of(out_dtype), in->n_rows) &&
                        vector_rows(in->bias, in->bias_stride, 4, in->n_rows);
    const int parts = logits_parts(a.n_rows, a.width);
    const dim3 grid = logits_grid(a.n_rows, a.width, parts);
    const int64_t logits = (int64_t)a.n_rows * a.width;
    // A thread each, all of them on the GPU at once.  With everything, bf16, a thread a logit and by tiles: 585 x 512 3.2 and 3.2 us,
    // 1,171 x 512 4.8 and 3.4; 73 x 4,106 3.3 and 3.6, 146 x 4,106 5.0 and 5.8, 292 x 4,106 8.0 and 6.8; 9 x 32,000 3.3 and 3.1 to
    // 3.8, 18 x 32,000 4.9 and 3.4.  (Rows of few tokens leave most of a tile empty: 120,000 x 10 7.8 and 97.)
    const bool few = logits <= (int64_t)SMS * 2048;
    with_type(in->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        auto typed = [&](auto* o) {
            using O = std::remove_pointer_t<decltype(o)>;
            if (few) {
                process_each_kernel<T, O><<<(unsigned)((logits + LOGITS_THREADS - 1) / LOGITS_THREADS), LOGITS_THREADS, 0, st>>>(
                    a, (const T*)in->logits, (O*)d_out, out_stride);
                return;
            }
            with_variant<sizeof(T), sizeof(O)>(vector, a.width, a.seen != nullptr, parts, [&](auto m, auto seen, auto n) {
                constexpr int MAP = decltype(m)::value, PARTS = decltype(n)::value;
                if constexpr (!decltype(seen)::value)
                    process_logits_kernel<T, O, MAP, NO_HISTORY, PARTS><<<grid, LOGITS_THREADS, 0, st>>>(a, (const T*)in->logits, (O*)d_out, out_stride);
                else if (a.counts)
                    process_logits_kernel<T, O, MAP, COUNTED, PARTS><<<grid, LOGITS_THREADS, 0, st>>>(a, (const T*)in->logits, (O*)d_out, out_stride);
                else
                    process_logits_kernel<T, O, MAP, SEEN_ONLY, PARTS><<<grid, LOGITS_THREADS, 0, st>>>(a, (const T*)in->logits, (O*)d_out, out_stride);
            });
        };
        if (out_dtype == in->dtype) typed(t); else typed((float*)nullptr);
    });
    LAUNCH_CHECK("process_logits_kernel");
    return DNATOK_OK;
}

size_t dnatok_logits_scratch_bytes(int64_t n_rows, int64_t width) {
    if (n_rows < 1 || width < 1) return 0;
    const unsigned blocks = bias_grid(n_rows, width, logits_parts(n_rows, width)).y;
    return blocks > 1 ? (size_t)blocks * (size_t)width * 4 : 0;
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
    if (d_dlogits && d_dlogits == in->logits && in->n_rows) return abi_fail(DNATOK_ERR_INVALID, "the logits are still read: their gradient needs an array of its own");
    if (d_dlogits && d_dlogits == d_grad && in->n_rows && (grad_dtype != in->dtype || (in->n_rows > 1 && grad_stride != dlogits_stride)))
        return abi_fail(DNATOK_ERR_INVALID, "in place both gradients have one type and stride");
    cudaStream_t st = (cudaStream_t)stream;
    const bool shared = in->bias_stride == 0;
    if (in->n_rows == 0) {
        if (d_dbias && shared) CUDA_TRY(cudaMemsetAsync(d_dbias, 0, (size_t)in->width * 4, st));
        return DNATOK_OK;
    }
    if (!d_dlogits && !d_dbias) return DNATOK_OK;
    const LogitsArgs a = logits_args(in);
    const bool vector = vector_rows(in->logits, in->stride, size_of(in->dtype), in->n_rows) &&
                        vector_rows(d_grad, grad_stride, size_of(grad_dtype), in->n_rows) &&
                        vector_rows(d_dlogits, dlogits_stride, size_of(in->dtype), in->n_rows) &&
                        (shared || vector_rows(d_dbias, in->width, 4, in->n_rows));
    const bool add = d_dbias && shared;
    const int parts = logits_parts(a.n_rows, a.width);
    const dim3 grid = add ? bias_grid(a.n_rows, a.width, parts) : logits_grid(a.n_rows, a.width, parts);
    const bool join = add && grid.y > 1;
    if (join && (!d_scratch || scratch_bytes < dnatok_logits_scratch_bytes(a.n_rows, a.width) || !aligned(d_scratch, 256)))
        return abi_fail(DNATOK_ERR_SCRATCH, "the gradient of a shared bias needs %zu bytes of 256-byte aligned scratch",
                        dnatok_logits_scratch_bytes(a.n_rows, a.width));
    dnatok_logits read = *in;                                 // what the kernels read of it
    read.bias = read.d_frequency = read.d_presence = nullptr;
    read.counts = nullptr;
    if (!in->seen || !d_dlogits) {
        read.logits = read.rows = nullptr;
        read.seen = nullptr;
        read.d_repetition = nullptr;
    }
    const Wide size = size_of(in->dtype), width = in->width;
    const Rows grad = {d_grad, in->n_rows, grad_stride * (Wide)size_of(grad_dtype), width * size_of(grad_dtype)};
    const Rows logits = {read.logits, in->n_rows, in->stride * size, width * size};
    const Rows outs[] = {{d_dlogits, in->n_rows, dlogits_stride * size, width * size},
                         {d_dbias, shared ? 1 : in->n_rows, width * 4, width * 4},
                         {join ? d_scratch : nullptr, 1, 0, join ? (Wide)dnatok_logits_scratch_bytes(a.n_rows, a.width) : 0}};
    const char* names[] = {"logits' gradient", "bias' gradient", "scratch"};
    for (int i = 0; i < 3; ++i) {
        if (overlap(outs[i], logits)) return abi_fail(DNATOK_ERR_INVALID, "%s and logits overlap", names[i]);
        if (!(i == 0 && d_dlogits == d_grad) && overlap(outs[i], grad))
            return abi_fail(DNATOK_ERR_INVALID, "%s and gradient overlap (that of the logits may be the gradient itself)", names[i]);
        for (int k = 0; k < i; ++k)
            if (overlap(outs[i], outs[k])) return abi_fail(DNATOK_ERR_INVALID, "%s and %s overlap", names[i], names[k]);
        if (int rc = check_apart(names[i], outs[i], &read)) return rc;
    }
    float* sums = join ? (float*)d_scratch : d_dbias;
    with_type(in->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        auto typed = [&](auto* g) {
            using G = std::remove_pointer_t<decltype(g)>;
            with_variant<sizeof(T), sizeof(G)>(vector, a.width, a.seen && d_dlogits, parts, [&](auto m, auto seen, auto n) {
                constexpr int MAP = decltype(m)::value, PARTS = decltype(n)::value;
                constexpr bool SEEN = decltype(seen)::value;
                if (add)
                    logits_bias_gradient_kernel<T, G, MAP, SEEN, PARTS><<<grid, LOGITS_THREADS, 0, st>>>(
                        a, (const T*)in->logits, (const G*)d_grad, grad_stride, (T*)d_dlogits, dlogits_stride, sums,
                        (int)rows_per_block(a.n_rows, grid.y));
                else
                    logits_gradient_kernel<T, G, MAP, SEEN, PARTS><<<grid, LOGITS_THREADS, 0, st>>>(
                        a, (const T*)in->logits, (const G*)d_grad, grad_stride, (T*)d_dlogits, dlogits_stride, d_dbias);
            });
        };
        if (grad_dtype == in->dtype) typed(t); else typed((float*)nullptr);
    });
    LAUNCH_CHECK("logits_gradient_kernel");
    if (join) {
        bias_gradient_kernel<<<(unsigned)((a.width + LOGITS_THREADS - 1) / LOGITS_THREADS), LOGITS_THREADS, 0, st>>>(sums, (int)grid.y, a.width, d_dbias);
        LAUNCH_CHECK("bias_gradient_kernel");
    }
    return DNATOK_OK;
}

}  // extern "C"

// ------------------------------------------------------------------ history

namespace {

template <typename IdT>
int launch_history(const HistoryArgs& a, const IdT* ids, cudaStream_t st) {
    const int64_t mean = a.offsets ? a.total / a.n_rows : a.columns;     // ids a row, as far as the host knows
    // A row with at least as many ids as there are tokens is counted in shared memory first (8 rows of up to 1,048,576 ids of
    // bytes: 8.1 us; entered one by one they queue up at ten counters a row: 10,800 us).  A row that is only marked needs 32
    // times less to clear and to join.
    const int64_t words = (a.width + 31) / 32, table = a.counts ? a.width : words;
    if (mean >= 1024 && mean >= (a.counts ? table : 4 * table) && table * 4 <= 192 * 1024 && a.n_rows <= (1 << 20)) {
        // up to 8 counters a token (these rows: 8.1 us, 8.2 with 32, which take longer to clear and to join, 7.6 with one: ten
        // tokens in use do not make the lanes of a warp wait for one another as long as one or two would)
        int log_copies = 0;
        while (a.counts && log_copies < 3 && (table << (log_copies + 1)) * 4 <= 48 * 1024) ++log_copies;
        int64_t resident = 220 * 1024 / ((table << log_copies) * 4 + 1024);       // blocks an SM, all of them at once
        if (resident > 3) resident = 3;
        int64_t splits = (int64_t)SMS * resident / a.n_rows;
        const int64_t least = table > 1024 ? table : 1024;                // ids a block
        if (splits > mean / least) splits = mean / least;
        if (splits < 1) splits = 1;
        while (log_copies > 0 && (table << log_copies) > mean / splits) --log_copies;
        const size_t shared = (size_t)(table << log_copies) * 4;
        const unsigned grid = (unsigned)(a.n_rows * splits);
        if (a.counts) {
            if (shared > 48 * 1024) CUDA_TRY(cudaFuncSetAttribute(history_count_kernel<IdT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 192 * 1024));
            history_count_kernel<IdT><<<grid, HISTORY_LONG_THREADS, shared, st>>>(a, ids, (int)splits, log_copies);
            LAUNCH_CHECK("history_count_kernel");
        } else {
            if (shared > 48 * 1024) CUDA_TRY(cudaFuncSetAttribute(history_mark_kernel<IdT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 192 * 1024));
            history_mark_kernel<IdT><<<grid, HISTORY_LONG_THREADS, shared, st>>>(a, ids, (int)splits);
            LAUNCH_CHECK("history_mark_kernel");
        }
        return DNATOK_OK;
    }
    int log_group = 0;                                                    // threads a row: about one for four ids
    while (1 << log_group < HISTORY_THREADS && 4ll << log_group < mean) ++log_group;
    int64_t splits = (mean + (8ll << log_group) - 1) / (8ll << log_group);
    const int64_t most = ((int64_t)SMS * 2048 >> log_group) / a.n_rows;
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    const int64_t blocks = ((a.n_rows * splits << log_group) + HISTORY_THREADS - 1) / HISTORY_THREADS;
    if (blocks > INT32_MAX) return abi_fail(DNATOK_ERR_UNSUPPORTED, "too many rows for one call");
    history_add_kernel<IdT><<<(unsigned)blocks, HISTORY_THREADS, 0, st>>>(a, ids, log_group, (int)splits);
    LAUNCH_CHECK("history_add_kernel");
    return DNATOK_OK;
}

}  // namespace

extern "C" {

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
    return h->id_bits == 64 ? launch_history(a, (const int64_t*)h->ids, st) : launch_history(a, (const int32_t*)h->ids, st);
}

}  // extern "C"

// ------------------------------------------------------------------ grammars

struct dnatok_grammar {
    std::vector<int32_t> next;
    std::vector<uint16_t> step16;
    std::vector<uint32_t> step32;
    std::vector<uint8_t> accepting, codes;
    std::vector<int32_t> token_at;
    std::vector<uint64_t> text;
    std::vector<uint32_t> super;
    std::vector<uint2> prefix;
    std::vector<uint2> rest;
    std::vector<uint32_t> more;
    int32_t n_states = 0, log_pitch = 0, n_groups = 0, super_steps = 0, prefix_steps = 0, n_runs = 0;
    int64_t width = 0, end_id = -1;
    struct Device { void* memory = nullptr; GrammarTables tables{}; };
    std::mutex mu;
    std::map<int, Device> dev;
};

namespace {

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// While it lives, calls of this thread that a capture does not allow leave the captures of other streams alone: allocations,
// frees and waits that are no part of them.
struct OutsideCaptures {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    bool on = cudaThreadExchangeStreamCaptureMode(&mode) == cudaSuccess;
    ~OutsideCaptures() { if (on) cudaThreadExchangeStreamCaptureMode(&mode); }
};

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
        OutsideCaptures outside;
        constexpr int N = 11;
        const size_t sizes[N] = {g->next.size() * 4, g->step16.size() * 2, g->accepting.size(), g->codes.size(), g->token_at.size() * 4,
                                 g->text.size() * 8, g->prefix.size() * 8, g->rest.size() * 8, g->step32.size() * 4, g->super.size() * 4, g->more.size() * 4};
        const void* from[N] = {g->next.data(), g->step16.data(), g->accepting.data(), g->codes.data(), g->token_at.data(),
                               g->text.data(), g->prefix.data(), g->rest.data(), g->step32.data(), g->super.data(), g->more.data()};
        size_t at[N + 1] = {0};
        for (int i = 0; i < N; ++i) at[i + 1] = at[i] + up256(sizes[i] + 1);
        struct Undo {
            void* memory = nullptr;
            cudaStream_t copies = nullptr;
            ~Undo() { if (copies) cudaStreamDestroy(copies); if (memory) cudaFree(memory); }
        } undo;
        CUDA_TRY(cudaMalloc(&undo.memory, at[N]));
        CUDA_TRY(cudaStreamCreateWithFlags(&undo.copies, cudaStreamNonBlocking));
        char* base = (char*)undo.memory;
        for (int i = 0; i < N; ++i)
            if (sizes[i]) CUDA_TRY(cudaMemcpyAsync(base + at[i], from[i], sizes[i], cudaMemcpyHostToDevice, undo.copies));
        CUDA_TRY(cudaStreamSynchronize(undo.copies));
        dnatok_grammar::Device d;
        GrammarTables& t = d.tables;
        t.next = (const int32_t*)(base + at[0]);
        t.step16 = g->step16.empty() ? nullptr : (const uint16_t*)(base + at[1]);
        t.step32 = (const uint32_t*)(base + at[8]);
        t.accepting = (const uint8_t*)(base + at[2]);
        t.codes = (const uint8_t*)(base + at[3]);
        t.token_at = (const int32_t*)(base + at[4]);
        t.text = g->text.empty() ? nullptr : (const uint64_t*)(base + at[5]);
        t.prefix = (const uint2*)(base + at[6]);
        t.super = (const uint32_t*)(base + at[9]);
        t.rest = (const uint2*)(base + at[7]);
        t.more = (const uint32_t*)(base + at[10]);
        t.n_states = g->n_states; t.log_pitch = g->log_pitch; t.n_groups = g->n_groups;
        t.n_super = (int32_t)g->super.size();
        t.n_runs = g->n_runs;
        t.super_steps = g->super_steps; t.prefix_steps = g->prefix_steps;
        t.width = g->width; t.end_id = g->end_id;
        d.memory = undo.memory;
        try {
            it = g->dev.emplace(dev, d).first;
        } catch (const std::bad_alloc&) {
            return abi_fail(DNATOK_ERR_INVALID, "out of memory");
        }
        undo.memory = nullptr;
    }
    *out = it->second.tables;
    return 0;
}

Rows row_array(const void* p, int64_t n_rows, Wide row) { return {p, n_rows, row, row}; }
Wide mask_bytes(const dnatok_grammar* g) { return (Wide)((g->width + 31) / 32) * 4; }

int check_states(const dnatok_grammar* g, const void* states, int64_t n_rows) {
    if (!g || n_rows < 0 || (n_rows && !states)) return abi_fail(DNATOK_ERR_INVALID, "bad argument");
    if (!aligned(states, 4)) return abi_fail(DNATOK_ERR_INVALID, "misaligned states");
    return 0;
}

// With tokens: the states are advanced first.
int launch_allowed(const GrammarTables& t, const int32_t* states, const void* tokens, int token_bits, int32_t* states_out, int64_t n_rows,
                   uint32_t* allowed, cudaStream_t st) {
    const int64_t words = (t.width + 31) / 32;
    // The groups need a row's words in shared memory, 32 KB beside a small table; vocabularies beyond 262,144 tokens and automata with more than
    // 15 classes go token by token.  (By groups and token by token, motifs to avoid: 64 x 4,106 5.3 and 3.5 us, 1 x 32,000 6.1 and
    // 3.4, but 1,024 x 4,106 17.6 and 27.5, 64 x 32,000 11.7 and 21.7, 1,024 x 32,000 72 and 312.)
    if (!t.text || words > 8192 || n_rows > INT32_MAX / 8) {
        if (tokens) {
            grammar_advance_kernel<<<(unsigned)((n_rows + GRAMMAR_THREADS - 1) / GRAMMAR_THREADS), GRAMMAR_THREADS, 0, st>>>(
                t, states, tokens, token_bits, n_rows, states_out);
            LAUNCH_CHECK("grammar_advance_kernel");
            states = states_out;
        }
        grammar_any_kernel<<<blocks_for(n_rows * words * 32, GRAMMAR_THREADS), GRAMMAR_THREADS, 0, st>>>(t, states, n_rows, allowed);
        LAUNCH_CHECK("grammar_any_kernel");
        return DNATOK_OK;
    }
    // Few rows: up to 8 blocks a row, as long as all are on the GPU at once (3 an SM) and each has 128 groups.  A warp for
    // every 4 groups, up to 16: rows differ, and one that may go on with anything holds up the others (1,024 rows of a pattern
    // over 32,000 tokens: 29 us, 35 with 8 warps, 47 in clusters of 2 blocks; 148 rows that all may: 20 us in 296 blocks, 25 in
    // 592, which are two rounds).
    const int64_t room = (int64_t)SMS * 3;
    int parts = 1;
    while (parts < 8 && n_rows * parts * 2 <= room && t.n_groups > parts * 128) parts *= 2;
    int warps = 1;
    while (warps < GRAMMAR_MOST / 32 && warps * 4 * parts < t.n_groups) warps *= 2;
    int split = 1;                                            // warps a set of 32 groups
    while (split < 32 && split < warps * parts && t.n_super * split < warps * parts) split *= 2;
    const size_t table = (((size_t)(t.n_states + 1) << t.log_pitch) * (t.step16 ? 2 : 4) + 15) / 16 * 16;
    const bool near = table <= GRAMMAR_NEAR_BYTES;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n_rows * parts));
    cfg.blockDim = dim3((unsigned)warps * 32);
    cfg.dynamicSmemBytes = (near ? table : 0) + (size_t)words * 4;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)parts; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    cudaError_t e = cudaSuccess;
    auto run = [&](auto s, auto n, auto c, auto r) {
        e = cudaLaunchKernelEx(&cfg, grammar_allowed_kernel<decltype(s), decltype(n)::value, decltype(c)::value, decltype(r)::value>, t,
                               states, tokens, token_bits, states_out, allowed, parts, split);
    };
    auto marked = [&](auto s, auto n, auto c) { if (t.n_runs * 2 > t.n_groups) run(s, n, c, std::true_type()); else run(s, n, c, std::false_type()); };
    auto placed = [&](auto s, auto n) { if (parts > 1) marked(s, n, std::true_type()); else marked(s, n, std::false_type()); };
    if (!t.step16) placed(uint32_t(), std::false_type());              // (such a table is never small)
    else if (near) placed(uint16_t(), std::true_type());
    else placed(uint16_t(), std::false_type());
    if (e != cudaSuccess) return abi_fail(DNATOK_ERR_CUDA, "launch of grammar_allowed_kernel: %s", cudaGetErrorString(e));
    LAUNCH_CHECK("grammar_allowed_kernel");
    return DNATOK_OK;
}

// The tokens in the order of their groups (see grammar_kernel.cuh): what a group shares, what each has behind it, who it is.
void sort_tokens(dnatok_grammar* g) {
    auto code = [&](int32_t v, int64_t i) { return g->codes[(size_t)(g->token_at[(size_t)v] + i)]; };
    auto length = [&](int32_t v) { return (int64_t)g->token_at[(size_t)v + 1] - g->token_at[(size_t)v]; };
    auto classes = [&](int32_t v, int64_t from, int64_t to, int64_t filled) {
        uint64_t p = 0;
        for (int64_t i = 0; i < filled; ++i)
            p |= (uint64_t)(from + i < to ? code(v, from + i) : (1 << g->log_pitch) - 1) << (4 * i);
        return p;
    };
    std::vector<int32_t> order;
    g->text.assign((size_t)g->width, 0);
    for (int32_t v = 0; v < g->width; ++v) {
        const int64_t n = length(v);
        g->text[(size_t)v] = n > GRAMMAR_PACKED ? 15ull << 60 : (uint64_t)n << 60 | classes(v, 0, n, n);
        if (length(v) && v != g->end_id) order.push_back(v);
    }
    const int64_t mean = order.empty() ? 0 : ((int64_t)g->codes.size() + (int64_t)order.size() - 1) / (int64_t)order.size();
    std::vector<uint64_t> key((size_t)g->width);              // the first 16 classes, ends first
    for (int32_t v : order)
        for (int64_t i = 0; i < 16; ++i) key[(size_t)v] = key[(size_t)v] << 4 | (uint64_t)(i < length(v) ? code(v, i) + 1 : 0);
    std::sort(order.begin(), order.end(), [&](int32_t x, int32_t y) {
        if ((length(x) > mean) != (length(y) > mean)) return length(y) > mean;
        if (key[(size_t)x] != key[(size_t)y]) return key[(size_t)x] < key[(size_t)y];
        const int64_t n = std::min(length(x), length(y));
        const int c = memcmp(&g->codes[(size_t)g->token_at[(size_t)x]], &g->codes[(size_t)g->token_at[(size_t)y]], (size_t)n);
        return c ? c < 0 : length(x) != length(y) ? length(x) < length(y) : x < y;
    });
    // what order[from .. to) have in common from class `done` on, at most `most` classes
    auto common = [&](size_t from, size_t to, int64_t done, int64_t most) {
        int64_t n = std::min(most, length(order[from]) - done);
        for (size_t i = from; i < to; ++i)
            for (int64_t j = 0; j < n; ++j)
                if (done + j >= length(order[i]) || code(order[i], done + j) != code(order[from], done + j)) n = j;
        return n;
    };
    const size_t sets = (order.size() + 1023) / 1024;
    g->n_groups = (int32_t)((order.size() + 31) / 32);
    g->prefix.assign(sets * 32, make_uint2(0, 0));
    g->rest.assign(sets * 1024, make_uint2(0, ~0u));
    g->more.assign(sets * 1024, 0);
    for (size_t s = 0; s < sets; ++s) {
        const size_t end = std::min(order.size(), (s + 1) * 1024);
        const int64_t m = common(s * 1024, end, 0, GRAMMAR_SHARED);
        g->super.push_back((uint32_t)classes(order[s * 1024], 0, m, GRAMMAR_SHARED));
        g->super_steps = std::max(g->super_steps, (int32_t)m);
        for (size_t k = s * 32; k * 32 < end; ++k) {
            const size_t last = std::min(end, k * 32 + 32);
            const int64_t n = common(k * 32, last, m, GRAMMAR_SHARED);
            int64_t steps = 1;                                // (0 says that there is no group)
            bool run = true;
            for (size_t i = k * 32; i < last; ++i) {
                const int32_t v = order[i];
                steps = std::max(steps, length(v) - m - n);
                const uint64_t rest = classes(v, m + n, length(v), GRAMMAR_REST);
                g->rest[i] = make_uint2((uint32_t)rest, (uint32_t)v);
                g->more[i] = (uint32_t)(rest >> 32);
                run = run && v == order[k * 32] + (int32_t)(i - k * 32);
            }
            g->prefix[k] = make_uint2((uint32_t)classes(order[k * 32], m, m + n, GRAMMAR_SHARED), (uint32_t)(steps > GRAMMAR_REST ? GRAMMAR_SLOW : steps) | (run ? GRAMMAR_RUN : 0));
            g->prefix_steps = std::max(g->prefix_steps, (int32_t)n);
            g->n_runs += run;
        }
    }
}

// The automaton for masks (see GrammarTables).
void make_steps(dnatok_grammar* g) {
    const int64_t columns = 1ll << g->log_pitch;
    g->step32.resize((size_t)((g->n_states + 1) * columns));
    for (int64_t s = 0; s <= g->n_states; ++s)
        for (int64_t c = 0; c < columns; ++c) {
            const int32_t to = s == g->n_states ? -1 : c == columns - 1 ? (int32_t)s : g->next[(size_t)(s * columns + c)];
            g->step32[(size_t)(s * columns + c)] = (uint32_t)(to < 0 ? g->n_states : to) << g->log_pitch;
        }
    if ((g->n_states + 1ll) * columns <= 1 << 16) {
        g->step16.assign(g->step32.begin(), g->step32.end());
        g->step32.clear();
    }
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
        g->n_states = n_states; g->width = width; g->end_id = end_id;
        while (1 << g->log_pitch < n_classes + 1) ++g->log_pitch;
        g->next.assign((size_t)n_states << g->log_pitch, -1);
        for (int64_t s = 0; s < n_states; ++s)
            for (int32_t c = 0; c < n_classes; ++c) g->next[(size_t)((s << g->log_pitch) + c)] = next[s * n_classes + c];
        g->accepting.resize((size_t)n_states);
        for (int32_t i = 0; i < n_states; ++i) g->accepting[(size_t)i] = accepting[i] != 0;
        g->codes.resize((size_t)total);
        for (int64_t i = 0; i < total; ++i) g->codes[(size_t)i] = byte_class[token_bytes[i]];
        g->token_at.resize((size_t)width + 1);
        for (int64_t v = 0; v <= width; ++v) g->token_at[(size_t)v] = (int32_t)token_offsets[v];
        if (n_classes <= 15 && n_states < 1 << 27) {
            sort_tokens(g);
            make_steps(g);
        }
        undo.g = nullptr;
        *out = g;
    } catch (const std::bad_alloc&) {
        return abi_fail(DNATOK_ERR_INVALID, "out of memory");
    }
    return DNATOK_OK;
}

void dnatok_destroy_grammar(dnatok_grammar* g) {
    if (!g) return;
    if (!g->dev.empty()) {
        OutsideCaptures outside;                              // may run while some stream is captured
        int cur = 0;
        cudaGetDevice(&cur);
        for (auto& kv : g->dev) if (cudaSetDevice(kv.first) == cudaSuccess) cudaFree(kv.second.memory);
        cudaSetDevice(cur);
    }
    delete g;
}

int dnatok_grammar_allowed(dnatok_grammar* g, const int32_t* d_states, int64_t n_rows, uint32_t* d_allowed, dnatok_stream stream) {
    if (int rc = check_states(g, d_states, n_rows)) return rc;
    if (n_rows && !d_allowed) return abi_fail(DNATOK_ERR_INVALID, "mask is NULL");
    if (!aligned(d_allowed, 4)) return abi_fail(DNATOK_ERR_INVALID, "misaligned mask");
    if (n_rows == 0) return DNATOK_OK;
    if (overlap(row_array(d_allowed, n_rows, mask_bytes(g)), row_array(d_states, n_rows, 4))) return abi_fail(DNATOK_ERR_INVALID, "mask and states overlap");
    GrammarTables t;
    if (int rc = grammar_tables(g, (cudaStream_t)stream, &t)) return rc;
    return launch_allowed(t, d_states, nullptr, 0, nullptr, n_rows, d_allowed, (cudaStream_t)stream);
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
    // With a mask every block of a row reads its state and token while the first writes the new state.  Without one a thread has
    // a row, and may write where it read.
    const Rows states = row_array(d_states, n_rows, 4), tokens = row_array(d_tokens, n_rows, token_bits / 8), out = row_array(d_states_out, n_rows, 4);
    if (d_states_out != d_states && overlap(out, states)) return abi_fail(DNATOK_ERR_INVALID, "new states and states overlap");
    if ((d_allowed || token_bits != 32 || d_states_out != d_tokens) && overlap(out, tokens))
        return abi_fail(DNATOK_ERR_INVALID, "new states and tokens overlap");
    const Rows mask = row_array(d_allowed, n_rows, mask_bytes(g));
    if (overlap(mask, states) || overlap(mask, tokens) || overlap(mask, out)) return abi_fail(DNATOK_ERR_INVALID, "mask and states or tokens overlap");
    GrammarTables t;
    cudaStream_t st = (cudaStream_t)stream;
    if (int rc = grammar_tables(g, st, &t)) return rc;
    if (d_allowed) return launch_allowed(t, d_states, d_tokens, token_bits, d_states_out, n_rows, d_allowed, st);
    grammar_advance_kernel<<<(unsigned)((n_rows + GRAMMAR_THREADS - 1) / GRAMMAR_THREADS), GRAMMAR_THREADS, 0, st>>>(t, d_states, d_tokens, token_bits, n_rows, d_states_out);
    LAUNCH_CHECK("grammar_advance_kernel");
    return DNATOK_OK;
}

}  // extern "C"
