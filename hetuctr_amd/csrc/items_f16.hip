#include "items_kernels.h"

namespace hctr {
template void launch_items_forward<f16_t>(ItemsProduct &, int, hipStream_t);
template void launch_items_gradient<f16_t>(ItemsProduct &, int, hipStream_t);
template void launch_take_rows<f16_t>(const TakeRows &, hipStream_t);
} // namespace hctr
