// Layer-norm forward kernels for rows of type float whose normalised rows are of type bf16_t (see norm_rows.h).
#include "norm_rows.h"

namespace rofn {

int norm_fwd_f32_bf16(const NormArgs &a, const NormShape &s, int blocks, hipStream_t st) {
    return launch_norm_forward<float, bf16_t>(a, s, blocks, st);
}

}  // namespace rofn
