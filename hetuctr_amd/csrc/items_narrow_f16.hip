#include "items_narrow.h"

namespace hctr {
template void launch_narrow_forward<f16_t>(ItemsNarrow &, hipStream_t);
template void launch_narrow_dx<f16_t>(ItemsNarrow &, hipStream_t);
template void launch_narrow_dweight<f16_t>(ItemsNarrow &, hipStream_t);
} // namespace hctr
