// The adapter kernels for bf16 payloads.
#include "adapter_tables.hpp"

namespace xp {

template struct AdapterKernels<Bf16Payload>;

}  // namespace xp
