// The product kernels for bf16 payloads.
#include "product_kernels.hpp"

namespace xp {

template struct ProductKernels<Bf16Payload>;

}  // namespace xp
