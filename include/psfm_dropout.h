/*
 * psfm_dropout.h — C-ABI of dropout with a counter-based generator (gfx950).
 *
 * The reference's residual block drops whole channels of its shortcut (nn.Dropout2d,
 * packnet_sfm/networks/layers/packnet/layers01.py:40-61) with torch's generator, whose mask autograd
 * keeps for the backward pass.  Here the mask is a function of (seed, offset, position), Philox4x32-10,
 * made again by whoever needs it: the forward pass, the backward pass, and the product of
 * psfm_linear.h, which applies it in its epilogue.  Nothing of it is stored.
 *
 * A mask is a [mask rows, cols] matrix of 32-bit words; the words of row r, columns 4b .. 4b + 3 are the
 * four outputs of Philox4x32-10 at the counter (b' lo, b' hi, offset lo, offset hi),
 * b' = r * ceil(cols / 4) + b, under the key (seed lo, seed hi).  A value is dropped (becomes 0, whatever
 * it was) where its word is below round(p * 2^32), and multiplied by 1 / (1 - p) otherwise.
 *
 * Conventions as include/psfm.h: device pointers, caller-owned buffers, stream-ordered,
 * graph-capturable; return 0 / <0 bad argument / >0 hipError_t, message from psfm_dropout_last_error().
 */
#ifndef PSFM_DROPOUT_H
#define PSFM_DROPOUT_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PSFM_DTYPE_F32 0
#define PSFM_DTYPE_F16 1
#define PSFM_DTYPE_BF16 2

/* y[r, c] = [res[r, c] +] (dropped ? 0 : x[r, c] / (1 - p)) over `rows` x `cols` values; rows of x and res
 * start ldx / ldr values apart, y is dense.  Data rows q * mask_rows .. (q + 1) * mask_rows - 1 share
 * mask row q (1: by element; the pixels of an image: by channel).  rng: int64 [2] on the device, (seed, offset).
 * res may be NULL.  One rounding to the type.  Any size, any alignment that the type has.
 * The backward pass is the same call on dy with res = NULL. */
int psfm_dropout(const void* x, int64_t ldx, const void* res, int64_t ldr, int dtype, int64_t rows, int64_t cols,
                 int64_t mask_rows, double p, const int64_t* rng, void* y, void* stream);

/* used = (state.seed + add, state.offset); state.offset += 1 (both int64 [2] on the device, wrapping): one mask's
 * (seed, offset), drawn in stream order, so that every replay of a captured graph draws the next.  `add`: the
 * rank of a data-parallel job, whose ranks hold the same state. */
int psfm_rng_next(int64_t* state, int64_t add, int64_t* used, void* stream);

const char* psfm_dropout_last_error(void);

#ifdef __cplusplus
}
#endif
#endif /* PSFM_DROPOUT_H */
