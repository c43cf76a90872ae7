// The product kernels for fp32 payloads.
#include "product_kernels.hpp"

namespace xp {

template struct ProductKernels<F32Payload>;

}  // namespace xp
