// psfm_linear_bf16.hip — the pointwise product's kernels for __bf16 (psfm_linear_kernels.h).
#include "psfm_linear_kernels.h"

namespace psfm {
const LinearOps& linear_ops_bf16() {
    static const LinearOps o = ops<__bf16>();
    return o;
}
}  // namespace psfm
