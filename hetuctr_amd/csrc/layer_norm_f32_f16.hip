#include "layer_norm_backward.h"
#include "layer_norm_forward.h"

namespace hctr {
template void launch_norm<float, f16_t>(const NormForward &, bool, bool, hipStream_t);
template unsigned launch_norm_grad<float, f16_t>(const NormBackward &, bool, bool, hipStream_t);
} // namespace hctr
