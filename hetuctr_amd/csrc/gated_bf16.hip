#include "gated_kernels.h"

namespace hctr {
template void launch_gated<bf16_t>(GatedForward &, int, hipStream_t);
template void launch_gated_few<bf16_t>(const GatedForward &, hipStream_t);
template void launch_slopes<bf16_t>(const GatedSlopes &, hipStream_t);
} // namespace hctr
