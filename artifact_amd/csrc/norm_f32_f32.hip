// Layer-norm kernels for rows of type float whose normalised rows are of type float (see norm_rows.h).
#include "norm_rows.h"

namespace rofn {

int launch_norm_f32_f32(const NormArgs &a, bool backward, const NormShape &s, int blocks, hipStream_t st) {
    return launch_norm<float, float>(a, backward, s, blocks, st);
}

}  // namespace rofn
