// psfm_linear_f32.hip — the pointwise product's kernels for float (psfm_linear_kernels.h).
#include "psfm_linear_kernels.h"

namespace psfm {
const LinearOps& linear_ops_f32() {
    static const LinearOps o = ops<float>();
    return o;
}
}  // namespace psfm
