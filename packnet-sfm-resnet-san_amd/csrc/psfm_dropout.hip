// psfm_dropout.hip — dropout with a counter-based generator (include/psfm_dropout.h).
//
//   y[r, c] = [res[r, c] +] (word(mask row, c) < p 2^32 ? 0 : x[r, c] / (1 - p))
//
// One thread takes four columns of a row, one Philox block.
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

template <typename T>
__global__ __launch_bounds__(256) void k_dropout(const Args A) {
    const int64_t cb = (A.cols + 3) >> 2, total = A.rows * cb;
    PhiloxKey key{};
    if (A.drop.rng) key = philox_key(A.drop.rng);
    for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < total; id += (int64_t)gridDim.x * 256) {
        const int64_t r = id / cb, c = (id - r * cb) * 4;
        const T* x = (const T*)A.x + r * A.ldx + c;
        const T* res = A.res ? (const T*)A.res + r * A.ldr + c : nullptr;
        T* y = (T*)A.y + r * A.cols + c;
        uint32_t w[4];
        if (A.drop.rng) philox4(key, mask_block(mask_row(A.drop, r), A.cols, c), w);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (c + k >= A.cols) continue;
            float v = (float)x[k];
            if (A.drop.rng) v = w[k] <= A.drop.last ? 0.0f : v * A.drop.scale;
            y[k] = (T)(res ? v + (float)res[k] : v);
        }
    }
}

__global__ void k_rng_next(int64_t* state, int64_t* used) {
    const int64_t seed = state[0], off = state[1];
    used[0] = seed;
    used[1] = off;
    state[1] = (int64_t)((uint64_t)off + 1);
}

}  // namespace

extern "C" {

int psfm_dropout(const void* x, int64_t ldx, const void* res, int64_t ldr, int dtype, int64_t rows, int64_t cols,
                 int64_t mask_rows, double p, const int64_t* rng, void* y, void* stream) {
    const int64_t most = (int64_t)1 << 40;
    if (rows < 0 || cols < 0 || rows > most || cols > most || (double)rows * (double)cols > 1e18)
        return fail(-1, "psfm_dropout: rows and cols must be 0 .. 2^40");
    if (dtype != PSFM_DTYPE_F32 && dtype != PSFM_DTYPE_F16 && dtype != PSFM_DTYPE_BF16)
        return fail(-2, "psfm_dropout: dtype must be PSFM_DTYPE_F32 / F16 / BF16");
    if (!(p >= 0.0 && p <= 1.0)) return fail(-3, "psfm_dropout: p must be in 0 .. 1");
    if (p > 0.0 && (!rng || mask_rows < 1)) return fail(-4, "psfm_dropout: needs rng and mask_rows >= 1");
    if (rows == 0 || cols == 0) return 0;
    if (!x || !y) return fail(-5, "psfm_dropout: null tensor");
    if (ldx < cols || (res && ldr < cols)) return fail(-6, "psfm_dropout: a row stride below the row's length");
    Args a{x, res, y, ldx, ldr, rows, cols, DropArgs{nullptr, 0, 1.0f, 1}};
    if (p > 0.0 && drop_threshold(p, &a.drop.last, &a.drop.scale)) a.drop.rng = rng, a.drop.mask_rows = mask_rows;
    const int64_t groups = rows * ((cols + 3) / 4);
    const dim3 grid((unsigned)std::min<int64_t>((groups + 255) / 256, 16384));
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == PSFM_DTYPE_F32)
        k_dropout<float><<<grid, 256, 0, s>>>(a);
    else if (dtype == PSFM_DTYPE_F16)
        k_dropout<_Float16><<<grid, 256, 0, s>>>(a);
    else
        k_dropout<__bf16><<<grid, 256, 0, s>>>(a);
    return status("psfm_dropout: launch");
}

int psfm_rng_next(int64_t* state, int64_t* used, void* stream) {
    if (!state || !used) return fail(-1, "psfm_rng_next: null pointer");
    k_rng_next<<<1, 1, 0, (hipStream_t)stream>>>(state, used);
    return status("psfm_rng_next: launch");
}

const char* psfm_dropout_last_error(void) { return g_err.c_str(); }

}  // extern "C"
