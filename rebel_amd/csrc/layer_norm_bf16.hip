// rebel_amd/csrc/layer_norm_bf16.hip -- the layer norm kernels for rows of type __bf16.
#include "layer_norm_kernel.h"

namespace rbl {
template void layer_norm_forward<__bf16>(const NormArgs&, int, hipStream_t);
template void layer_norm_backward<__bf16>(const NormArgs&, const BackwardPlan&, int, hipStream_t);
}  // namespace rbl
