#include "items_kernels.h"

namespace hctr {
template void launch_items_forward<float>(ItemsProduct &, int, hipStream_t);
template void launch_items_gradient<float>(ItemsProduct &, int, hipStream_t);
template void launch_take_rows<float>(const TakeRows &, hipStream_t);
} // namespace hctr
