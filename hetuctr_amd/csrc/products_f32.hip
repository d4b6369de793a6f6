#include "products_kernels.h"

namespace hctr {
template void launch_forward_product<float>(ProductArgs &, int, hipStream_t);
template void launch_across_product<float>(ProductArgs &, int, hipStream_t);
template void launch_join<float>(const ProductArgs &, hipStream_t);
template void launch_copy_rows<float>(const hctr_matrix &, size_t, size_t, char *, size_t, hipStream_t);
} // namespace hctr
