// psfm_linear_f16.hip — the pointwise product's kernels for _Float16 (psfm_linear_kernels.h).
#include "psfm_linear_kernels.h"

namespace psfm {
const LinearOps& linear_ops_f16() {
    static const LinearOps o = ops<_Float16>();
    return o;
}
}  // namespace psfm
