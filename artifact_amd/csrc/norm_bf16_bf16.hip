// Layer-norm kernels for rows of type bf16_t whose normalised rows are of type bf16_t (see norm_rows.h).
#include "norm_rows.h"

namespace rofn {

int launch_norm_bf16_bf16(const NormArgs &a, bool backward, const NormShape &s, int blocks, hipStream_t st) {
    return launch_norm<bf16_t, bf16_t>(a, backward, s, blocks, st);
}

}  // namespace rofn
