// Layer-norm backward kernels with a ReLU for rows of type bf16_t whose normalised rows are of type float (see norm_rows.h).
#include "norm_rows.h"

namespace rofn {

int norm_bwd_relu_bf16_f32(const NormArgs &a, const NormShape &s, int blocks, hipStream_t st) {
    return launch_norm_backward<bf16_t, float, true>(a, s, blocks, st);
}

}  // namespace rofn
