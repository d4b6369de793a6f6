#include "gated_kernels.h"

namespace hctr {
template void launch_gated<float>(GatedForward &, int, hipStream_t);
template void launch_gated_few<float>(const GatedForward &, hipStream_t);
template void launch_slopes<float>(const GatedSlopes &, hipStream_t);
} // namespace hctr
