// The adapter kernels for fp32 payloads.
#include "adapter_tables.hpp"

namespace xp {

template struct AdapterKernels<F32Payload>;

}  // namespace xp
