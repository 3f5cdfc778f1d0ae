// Layer-norm backward kernels with a ReLU for rows of type float whose normalised rows are of type bf16_t (see norm_rows.h).
#include "norm_rows.h"

namespace rofn {

int norm_bwd_relu_f32_bf16(const NormArgs &a, const NormShape &s, int blocks, hipStream_t st) {
    return launch_norm_backward<float, bf16_t, true>(a, s, blocks, st);
}

}  // namespace rofn
