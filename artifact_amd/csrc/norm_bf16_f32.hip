// Layer-norm kernels for rows of type bf16_t whose normalised rows are of type float (see norm_rows.h).
#include "norm_rows.h"

namespace rofn {

int launch_norm_bf16_f32(const NormArgs &a, bool backward, const NormShape &s, int blocks, hipStream_t st) {
    return launch_norm<bf16_t, float>(a, backward, s, blocks, st);
}

}  // namespace rofn
