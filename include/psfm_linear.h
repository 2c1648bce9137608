/*
 * psfm_linear.h — C-ABI of the pointwise product with its epilogue, and its gradients (gfx950).
 *
 *     z = x W^T + bias          x [M, K], W [N, K], bias [N]
 *     y = res + drop(act(z))    res, y [M, N]
 *
 * a 1x1 convolution over the pixels of a channels_last activation (M = N*H*W rows of K channels: the
 * residual blocks' shortcut, packnet_sfm/networks/layers/packnet/layers01.py:40-61), or a dense layer over
 * rows.  The mask of `drop` is psfm_dropout.h's over the [M, N] matrix: dropping y afterwards
 * with the same (seed, offset) is the same mask.
 *
 * Types: x, W, bias, res, y and the gradients share one of PSFM_DTYPE_F32 / F16 / BF16.  Products are
 * accumulated, and the epilogue is computed, in fp32; y is rounded once.
 *
 * Conventions as include/psfm.h: device pointers, caller-owned buffers, stream-ordered,
 * graph-capturable; return 0 / <0 bad argument / >0 hipError_t, message from psfm_linear_last_error().
 * Sums run in a fixed order: equal calls give equal bits.
 */
#ifndef PSFM_LINEAR_H
#define PSFM_LINEAR_H

#include <stddef.h>
#include <stdint.h>

#include "psfm_dropout.h"
#include "psfm_netops.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Activations: PSFM_ACT_NONE / RELU / SIGMOID / ELU (psfm_netops.h) and */
#define PSFM_ACT_SILU 4    /* z / (1 + exp(-z))             */
#define PSFM_ACT_GELU 5    /* z (1 + erf(z / sqrt(2))) / 2  */

typedef struct psfm_linear {
    int64_t M, N, K;       /* sizes >= 0; K = 0 is an empty sum.  What one launch does not hold returns -8: over
                              2^31 - 256 rows of a few columns or columns of a few rows, over 2.5 10^8 columns
                              where db is wanted                                              */
    int64_t ldx, ldr;      /* row strides of x and res in values (W, y, z, dy, dx, dw are dense) */
    int32_t dtype, act;
    double p;              /* dropout probability, 0: none                                     */
    int64_t mask_rows;     /* data rows that share a mask row (psfm_dropout)                   */
    const int64_t* rng;    /* (seed, offset) on the device; may be NULL where p = 0            */
} psfm_linear;

/* Workspace of the forward pass in bytes (0: none needed), or -1 (bad descriptor). */
int64_t psfm_linear_fwd_ws_bytes(const psfm_linear* d);
/* bias, res and z may be NULL.  z [M, N] receives the values before the activation, which the backward pass
 * differentiates at: in x's type for PSFM_ACT_RELU, else in fp16 (clamped to its range) for bf16 and in fp32
 * for fp16 and fp32 tensors. */
int psfm_linear_fwd(const psfm_linear* d, const void* x, const void* w, const void* bias, const void* res, void* y,
                    void* z, void* ws, void* stream);

/* Workspace of the backward pass for the wanted gradients in bytes, or -1. */
int64_t psfm_linear_bwd_ws_bytes(const psfm_linear* d, int want_dx, int want_dw, int want_db);
/* With dz = drop(dy) act'(z):  dx = dz W [M, K], dw = dz^T x [N, K], db = sum over rows of dz [N]; each may
 * be NULL.  dz is fp32 where db sums it.  The products take it in the tensors' type: in 16 bits with an activation other than
 * ReLU, small layers add a second product of what that rounding leaves (dx and dw are off by one rounding), the others
 * do not (by up to 1.5 roundings).  In fp16 a dz, before dropout's scale, below 2^-25 is lost and one beyond 65504 is infinite.  dy [M, N] dense.  z as the forward pass stored it (NULL for PSFM_ACT_NONE); for
 * PSFM_ACT_RELU any tensor of its sign will do (y, where neither residual nor dropout touched it).
 * The gradient of res is dy itself. */
int psfm_linear_bwd(const psfm_linear* d, const void* dy, const void* x, const void* w, const void* z, void* dx,
                    void* dw, void* db, void* ws, void* stream);

const char* psfm_linear_last_error(void);

#ifdef __cplusplus
}
#endif
#endif /* PSFM_LINEAR_H */
