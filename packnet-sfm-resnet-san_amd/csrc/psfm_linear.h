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
};

enum GemmRole { GEMM_FWD = 0, GEMM_DX = 1, GEMM_DW = 2 };   // (P, Q): (x, W), (dz, W turned), (dz turned, x turned)

struct DzArgs {
    const void* dy;
    const void* z;         // null: act' = 1
    void* dz;              // null: column sums only
    float* part;           // [gridDim.y, N] column sums, or null
    int64_t M, N, rows;    // rows of one workgroup
    int act;
    DropArgs drop;
};

// One set per type (psfm_linear_<type>.hip).  Each returns a hipError_t.
struct LinearOps {
    // variant: an index into LINEAR_TILES
    int (*gemm)(int role, int variant, bool vec, const GemmArgs& a, hipStream_t s);
    int (*join)(const GemmArgs& a, bool full, hipStream_t s);
    int (*dz)(const DzArgs& a, int64_t gx, int64_t gy, hipStream_t s);
    int (*colsum)(const float* part, int64_t parts, int64_t N, float alpha, void* db, hipStream_t s);
};

const LinearOps& linear_ops_f32();
const LinearOps& linear_ops_f16();
const LinearOps& linear_ops_bf16();

struct Tile {
    int bi, bj;
};
// the tiles that every type is built for
constexpr Tile LINEAR_TILES[] = {{64, 64}, {128, 128}};
constexpr int LINEAR_NTILES = 2;
constexpr int DZ_THREADS = 256;
// chunks of columns in a k_dz workgroup: all of a narrow layer's, 32 of a wide one's
constexpr int DZ_NARROW = 8, DZ_WIDE = 32;

}  // namespace psfm
