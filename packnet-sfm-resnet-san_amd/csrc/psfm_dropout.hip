// psfm_dropout.hip — dropout with a counter-based generator (include/psfm_dropout.h).
//
//   y[r, c] = [res[r, c] +] (word(mask row, c) < p 2^32 ? 0 : x[r, c] / (1 - p))
//
// One read of x and res, one write of y.  A thread takes chunks of 16 bytes (8 values of 16 bits: two Philox blocks),
// UNROLL of them with their loads first; a workgroup's chunks are consecutive, so that one 64-bit division a
// workgroup finds its first row and the threads go on in 32 bits.
#include "../../include/psfm_dropout.h"

#include <algorithm>
#include <string>

#include "psfm_philox.h"

using namespace psfm;

namespace {

thread_local std::string g_err;

int fail(int code, const char* msg) {
    g_err = msg;
    return code;
}
int status(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    g_err = std::string(what) + ": " + hipGetErrorString(e);
    return (int)e;
}

struct Args {
    const void* x;
    const void* res;
    void* y;
    int64_t ldx, ldr, rows, cols;
    DropArgs drop;
};

constexpr int UNROLL = 4, THREADS = 256;

template <typename T, bool RES, bool SHARED>
__global__ __launch_bounds__(THREADS) void k_dropout(const Args A) {
    constexpr int V = 16 / (int)sizeof(T);
    typedef T TV __attribute__((ext_vector_type(V)));
    const int64_t cpr = (A.cols + V - 1) / V, first = (int64_t)blockIdx.x * THREADS * UNROLL, row0 = first / cpr;
    const int64_t in0 = first - row0 * cpr;
    PhiloxKey key{};
    if (A.drop.rng) key = philox_key(A.drop.rng);
    int64_t row[UNROLL], col[UNROLL];
    TV x[UNROLL], res[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const int64_t at = in0 + u * THREADS + threadIdx.x;
        const int64_t down = (cpr >> 31) == 0 ? (uint32_t)at / (uint32_t)cpr : at / cpr;
        row[u] = row0 + down;
        col[u] = (at - down * cpr) * V;
        const bool whole = row[u] < A.rows && col[u] + V <= A.cols;
        if (whole) {
            __builtin_memcpy(&x[u], (const T*)A.x + row[u] * A.ldx + col[u], 16);
            if (RES) __builtin_memcpy(&res[u], (const T*)A.res + row[u] * A.ldr + col[u], 16);
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const bool in = row[u] < A.rows && col[u] + k < A.cols;
                x[u][k] = in ? ((const T*)A.x)[row[u] * A.ldx + col[u] + k] : (T)0.0f;
                if (RES) res[u][k] = in ? ((const T*)A.res)[row[u] * A.ldr + col[u] + k] : (T)0.0f;
            }
        }
    }
    KeepBits<V> keep;   // SHARED: a mask by channel
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        if (row[u] >= A.rows) return;
        TV y;
        float v[V];
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = (float)x[u][k];
        if (SHARED)
            drop_run(A.drop, key, keep, A.cols, mask_row(A.drop, row[u]), col[u], A.drop.scale, v);
        else if (A.drop.rng)
            drop_block(A.drop, key, mask_block(row[u], A.cols, col[u]), A.drop.scale, v);
#pragma unroll
        for (int k = 0; k < V; ++k) y[k] = (T)(RES ? v[k] + (float)res[u][k] : v[k]);
        T* p = (T*)A.y + row[u] * A.cols + col[u];
        if (col[u] + V <= A.cols) {
            __builtin_memcpy(p, &y, 16);
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (col[u] + k < A.cols) p[k] = y[k];
        }
    }
}

template <typename T>
int run(const Args& a, hipStream_t s) {
    constexpr int V = 16 / (int)sizeof(T), PER = THREADS * UNROLL;
    const int64_t blocks = (a.rows * ((a.cols + V - 1) / V) + PER - 1) / PER;
    if (blocks > 0xffffffffll / THREADS) return fail(-1, "psfm_dropout: more values than a launch holds");
    const dim3 grid((unsigned)blocks);
    if (a.drop.rng && a.drop.mask_rows > 1)
        a.res ? k_dropout<T, true, true><<<grid, THREADS, 0, s>>>(a) : k_dropout<T, false, true><<<grid, THREADS, 0, s>>>(a);
    else
        a.res ? k_dropout<T, true, false><<<grid, THREADS, 0, s>>>(a) : k_dropout<T, false, false><<<grid, THREADS, 0, s>>>(a);
    return status("psfm_dropout: launch");
}

__global__ void k_rng_next(int64_t* state, uint64_t add, int64_t* used) {
    const uint64_t seed = (uint64_t)state[0] + add, off = (uint64_t)state[1];
    used[0] = (int64_t)seed;
    used[1] = (int64_t)off;
    state[1] = (int64_t)(off + 1);
}

}  // namespace

extern "C" {

int psfm_dropout(const void* x, int64_t ldx, const void* res, int64_t ldr, int dtype, int64_t rows, int64_t cols,
                 int64_t mask_rows, double p, const int64_t* rng, void* y, void* stream) {
    const int64_t most = (int64_t)1 << 40;
    if (rows < 0 || cols < 0 || rows > most || cols > most || (double)rows * (double)std::max({cols, ldx, ldr}) > 1e18)
        return fail(-1, "psfm_dropout: rows and cols must be 0 .. 2^40, the whole below 10^18 values");
    if (dtype != PSFM_DTYPE_F32 && dtype != PSFM_DTYPE_F16 && dtype != PSFM_DTYPE_BF16)
        return fail(-2, "psfm_dropout: dtype must be PSFM_DTYPE_F32 / F16 / BF16");
    if (!(p >= 0.0 && p <= 1.0)) return fail(-3, "psfm_dropout: p must be in 0 .. 1");
    if (p > 0.0 && (!rng || mask_rows < 1)) return fail(-4, "psfm_dropout: needs rng and mask_rows >= 1");
    if (rows == 0 || cols == 0) return 0;
    if (!x || !y) return fail(-5, "psfm_dropout: null tensor");
    if (ldx < cols || (res && ldr < cols)) return fail(-6, "psfm_dropout: a row stride below the row's length");
    Args a{x, res, y, ldx, ldr, rows, cols, DropArgs{nullptr, 0, 1.0f, 1}};
    if (p > 0.0 && drop_threshold(p, &a.drop.last, &a.drop.scale)) a.drop.rng = rng, a.drop.mask_rows = mask_rows;
    const hipStream_t s = (hipStream_t)stream;
    return dtype == PSFM_DTYPE_F32 ? run<float>(a, s) : dtype == PSFM_DTYPE_F16 ? run<_Float16>(a, s) : run<__bf16>(a, s);
}

int psfm_rng_next(int64_t* state, int64_t add, int64_t* used, void* stream) {
    if (!state || !used) return fail(-1, "psfm_rng_next: null pointer");
    k_rng_next<<<1, 1, 0, (hipStream_t)stream>>>(state, (uint64_t)add, used);
    return status("psfm_rng_next: launch");
}

const char* psfm_dropout_last_error(void) { return g_err.c_str(); }

}  // extern "C"
