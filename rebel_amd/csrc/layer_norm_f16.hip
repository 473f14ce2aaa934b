// rebel_amd/csrc/layer_norm_f16.hip -- the layer norm kernels for rows of type _Float16.
#include "layer_norm_kernel.h"

namespace rbl {
template void layer_norm_forward<_Float16>(const NormArgs&, int, hipStream_t);
template void layer_norm_backward<_Float16>(const NormArgs&, const BackwardPlan&, int, hipStream_t);
}  // namespace rbl
