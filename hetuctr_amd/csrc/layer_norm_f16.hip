#include "layer_norm_backward.h"
#include "layer_norm_forward.h"

namespace hctr {
template void launch_norm<f16_t, f16_t>(const NormForward &, bool, bool, hipStream_t);
template unsigned launch_norm_grad<f16_t, f16_t>(const NormBackward &, bool, bool, hipStream_t);
} // namespace hctr
