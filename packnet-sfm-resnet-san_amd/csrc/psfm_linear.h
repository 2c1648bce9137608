// psfm_linear.h (csrc) — what the translation units of the pointwise product share (gfx950).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/psfm_linear.h"
#include "psfm_philox.h"

namespace psfm {

// What follows a product's fp32 sums v[i, j].  Forward: z = v + bias, out = res + drop(act(z)).  Gradients:
// out = alpha v.
struct LinearEpi {
    void* out;             // [I, J] dense
    const void* bias;      // [J] or null
    const void* res;       // rows ldr apart, or null
    int64_t ldr;
    void* z;               // [I, J] dense, or null
    int act;
    float alpha;
    DropArgs drop;
};

// dz = drop(dy) act'(z), made where dy is staged (z null: act' = 1).  `cols` receives the sums over m of each split of the
// weight gradient, [splits, N], or `db` them scaled where there is one split.
struct DzArgs {
    const void* z;
    int act;
    DropArgs drop;
    float* cols;
    void* db;
};

// out[i, j] = sum over r of P[i, r] Q[j, r].  A "turned" operand is stored with r as its row.
struct GemmArgs {
    const void* P;
    const void* Q;
    int64_t ldp, ldq;
    int64_t I, J, R;
    int64_t rsplit;        // reduction elements of one split, whole LDS stages
    uint32_t ti, tj;       // tiles
    int splits;
    float* part;           // [splits, I, J] where splits > 1
    LinearEpi e;
    DzArgs dz;
    uint32_t blocks() const { return ti * tj * (uint32_t)splits; }
};

// A few rows times W, no tiles: y of 16 columns a workgroup
struct SkinnyArgs {
    const void* x;
    const void* w;
    int64_t ldx, M, N, K;
    LinearEpi e;
};

// Both gradients' products in one launch: workgroups 0 .. ndw - 1 make dw (long reductions first), the rest dx.
struct PairArgs {
    GemmArgs dx, dw;
    uint32_t ndx, ndw;
};

// What follows them in one launch: the joins of split products, then the column sums' parts.
struct FinishArgs {
    GemmArgs dx, dw;
    uint32_t ndx, ndw, ncol;
    const float* cols;
    int64_t parts, N;
    float alpha;
    void* db;
};

// dz as a pass of its own
struct DzPassArgs {
    const void* dy;
    void* out;             // null: column sums only
    int64_t M, N, rows;    // rows of one workgroup
    DzArgs dz;             // cols: [gridDim.y, N] or null
};

// One set per type (psfm_linear_<type>.hip).  Each launches and returns a hipError_t; `variant` is an index into
// LINEAR_TILES, `vec`: rows and runs of whole aligned 16-byte chunks.
struct LinearOps {
    int (*forward)(int variant, bool vec, const GemmArgs& a, hipStream_t s);
    int (*join)(const GemmArgs& a, hipStream_t s);          // of a split forward
    int (*skinny)(bool vec, const SkinnyArgs& a, hipStream_t s);
    int (*pair)(int variant, bool vec, bool dz, const PairArgs& a, hipStream_t s);
    int (*finish)(FinishArgs& a, hipStream_t s);
    int (*dz)(const DzPassArgs& a, int64_t gx, int64_t gy, hipStream_t s);
};

const LinearOps& linear_ops_f32();
const LinearOps& linear_ops_f16();
const LinearOps& linear_ops_bf16();

struct Tile {
    int bi, bj, threads;
};
constexpr Tile LINEAR_TILES[] = {{64, 64, 256}, {128, 128, 256}, {256, 256, 512}};
constexpr int LINEAR_NTILES = 3;   // 32-bit types: the first two
constexpr int DZ_THREADS = 256, SKINNY_THREADS = 512, FINISH_THREADS = 256;
// Chunks of columns in a k_dz workgroup: all of a narrow layer's, 32 of a wide one's (184320 x 64 bf16: 15.1 us with 8, 32.8
// with 32; 100000 x 8: 11.0, 20.0; 4096 x 24: 6.1, 6.3).
constexpr int DZ_NARROW = 8, DZ_WIDE = 32;
constexpr int SKINNY_ROWS = 32;    // at most
// Workgroups of one launch: the runtime counts a dimension's threads in 32 bits
constexpr int64_t most_blocks(int threads) { return 0xffffffffll / threads; }

}  // namespace psfm
