// The product kernels for fp16 payloads.
#include "product_kernels.hpp"

namespace xp {

template struct ProductKernels<F16Payload>;

}  // namespace xp
