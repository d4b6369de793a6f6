#include "products_kernels.h"

namespace hctr {
template void launch_forward_product<f16_t>(ProductArgs &, int, hipStream_t);
template void launch_across_product<f16_t>(ProductArgs &, int, hipStream_t);
template void launch_join<f16_t>(const ProductArgs &, hipStream_t);
template void launch_copy_rows<f16_t>(const hctr_matrix &, size_t, size_t, char *, size_t, hipStream_t);
} // namespace hctr
