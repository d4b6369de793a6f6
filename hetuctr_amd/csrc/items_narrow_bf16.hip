#include "items_narrow.h"

namespace hctr {
template void launch_narrow_forward<bf16_t>(ItemsNarrow &, hipStream_t);
template void launch_narrow_dx<bf16_t>(ItemsNarrow &, hipStream_t);
template void launch_narrow_dweight<bf16_t>(ItemsNarrow &, hipStream_t);
} // namespace hctr
