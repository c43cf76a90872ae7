// The adapter kernels for fp16 payloads.
#include "adapter_tables.hpp"

namespace xp {

template struct AdapterKernels<F16Payload>;

}  // namespace xp
