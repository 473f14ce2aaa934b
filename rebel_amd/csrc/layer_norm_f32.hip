// rebel_amd/csrc/layer_norm_f32.hip -- the layer norm kernels for rows of type float.
#include "layer_norm_kernel.h"

namespace rbl {
template void layer_norm_forward<float>(const NormArgs&, int, hipStream_t);
template void layer_norm_backward<float>(const NormArgs&, const BackwardPlan&, int, hipStream_t);
}  // namespace rbl
