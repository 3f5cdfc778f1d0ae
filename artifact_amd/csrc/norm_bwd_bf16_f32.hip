// Layer-norm backward kernels for rows of type bf16_t whose normalised rows are of type float (see norm_rows.h).
#include "norm_rows.h"

namespace rofn {

int norm_bwd_bf16_f32(const NormArgs &a, const NormShape &s, int blocks, hipStream_t st) {
    return launch_norm_backward<bf16_t, float, false>(a, s, blocks, st);
}

}  // namespace rofn
