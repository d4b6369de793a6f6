#include "items_kernels.h"

namespace hctr {
template void launch_items_forward<bf16_t>(ItemsProduct &, int, hipStream_t);
template void launch_items_gradient<bf16_t>(ItemsProduct &, int, hipStream_t);
template void launch_take_rows<bf16_t>(const TakeRows &, hipStream_t);
} // namespace hctr
