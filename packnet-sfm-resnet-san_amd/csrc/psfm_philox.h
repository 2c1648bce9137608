// psfm_philox.h — the counter-based generator of the dropout masks (gfx950).
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011):
// ten rounds of two 32 x 32 -> 64 bit products over a 128-bit counter under a 64-bit key.  A mask is a
// [rows, cols] matrix; row r and columns 4b .. 4b + 3 take the four words of the counter
// (b' lo, b' hi, offset lo, offset hi), b' = r * ceil(cols / 4) + b, under the key (seed lo, seed hi).
// Every word is a function of its position alone: forward and backward make it again wherever they
// need it, in any order, and nothing of it is stored.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace psfm {

// One mask: `rng` = (seed, offset) on the device; a word at or below `last` drops its value, a kept one is
// scaled by `scale`; `mask_rows` consecutive data rows share a mask row (1: a mask by element).
struct DropArgs {
    const int64_t* rng;    // null: nothing is dropped
    uint32_t last;
    float scale;
    int64_t mask_rows;
};

struct PhiloxKey {
    uint32_t k0, k1, o0, o1;
};

__device__ __forceinline__ PhiloxKey philox_key(const int64_t* rng) {
    const uint64_t seed = (uint64_t)rng[0], off = (uint64_t)rng[1];
    return PhiloxKey{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)off, (uint32_t)(off >> 32)};
}

__device__ __forceinline__ void philox4(const PhiloxKey& key, uint64_t block, uint32_t out[4]) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = key.o0, c3 = key.o1, k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    out[0] = c0, out[1] = c1, out[2] = c2, out[3] = c3;
}

// The mask row of data row i, and the counter block of columns j .. j + 3 (j % 4 = 0) of a mask row.
__device__ __forceinline__ int64_t mask_row(const DropArgs& d, int64_t i) {
    if (!d.rng || d.mask_rows == 1) return i;
    if (((i | d.mask_rows) >> 32) == 0) return (uint32_t)i / (uint32_t)d.mask_rows;   // a 64-bit division is ten times this
    return i / d.mask_rows;
}
__device__ __forceinline__ uint64_t mask_block(int64_t mrow, int64_t cols, int64_t j) {
    return (uint64_t)mrow * (uint64_t)((cols + 3) >> 2) + (uint64_t)(j >> 2);
}

// v[k] = kept ? v[k] * scale : 0 for the N columns of the mask block `block` and the next ones.
template <int N>
__device__ __forceinline__ void drop_block(const DropArgs& d, const PhiloxKey& key, uint64_t block, float scale,
                                           float (&v)[N]) {
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        uint32_t w[4];
        philox4(key, block + q, w);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[4 * q + k] = w[k] <= d.last ? 0.0f : v[4 * q + k] * scale;
    }
}

// The keep bits of N columns, kept from call to call: a mask by channel is the same from row to row, and made anew only
// where the block is another.  A mask by element always is another, and goes by drop_block: the bits'
// packing and the branch cost a tenth of a pass there.
template <int N>
struct KeepBits {
    uint64_t block = ~0ull;
    uint32_t bits = 0;

    __device__ __forceinline__ uint32_t at(const DropArgs& d, const PhiloxKey& key, uint64_t b) {
        if (b != block) {
            block = b;
            bits = 0;
#pragma unroll
            for (int q = 0; q < N / 4; ++q) {
                uint32_t w[4];
                philox4(key, b + q, w);
#pragma unroll
                for (int k = 0; k < 4; ++k) bits |= (w[k] <= d.last ? 0u : 1u) << (4 * q + k);
            }
        }
        return bits;
    }
};

// The same of the columns j .. j + N - 1 (j % 4 = 0) of mask row mrow
template <int N>
__device__ __forceinline__ void drop_run(const DropArgs& d, const PhiloxKey& key, KeepBits<N>& keep, int64_t cols,
                                         int64_t mrow, int64_t j, float scale, float (&v)[N]) {
    const uint64_t block = mask_block(mrow, cols, j);
    if (d.mask_rows == 1) {
        drop_block(d, key, block, scale, v);
    } else {
        const uint32_t bits = keep.at(d, key, block);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = bits >> k & 1 ? v[k] * scale : 0.0f;
    }
}

// The host side of a mask: the words 0 .. last drop, so that round(p 2^32) of 2^32 do.  False where p drops
// nothing at that resolution.  p = 1 drops everything; its scale is never used and stays finite.
inline bool drop_threshold(double p, uint32_t* last, float* scale) {
    const double words = p * 4294967296.0;
    const uint64_t n = (uint64_t)(words + 0.5);
    if (n == 0) return false;
    *last = n >= 4294967296ull ? 0xffffffffu : (uint32_t)(n - 1);
    *scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
    return true;
}

}  // namespace psfm
