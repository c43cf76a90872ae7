// Definitions of the adapter kernel tables, for the translation units that instantiate them.
#pragma once

#include "adapter_kernels.hpp"

namespace xp {

template <class P>
const void *AdapterKernels<P>::shrink(int rank_tiles) {
  switch (rank_tiles) {
    case 1:
      return reinterpret_cast<const void *>(&adapter_shrink_kernel<P, 1>);
    case 2:
      return reinterpret_cast<const void *>(&adapter_shrink_kernel<P, 2>);
    case 4:
      return reinterpret_cast<const void *>(&adapter_shrink_kernel<P, 4>);
    default:
      return reinterpret_cast<const void *>(&adapter_shrink_kernel<P, 8>);
  }
}

template <class P, bool ACT>
const void *adapter_expand_for(int rank_tiles) {
  switch (rank_tiles) {
    case 1:
      return reinterpret_cast<const void *>(&adapter_expand_kernel<P, 1, ACT>);
    case 2:
      return reinterpret_cast<const void *>(&adapter_expand_kernel<P, 2, ACT>);
    case 4:
      return reinterpret_cast<const void *>(&adapter_expand_kernel<P, 4, ACT>);
    default:
      return reinterpret_cast<const void *>(&adapter_expand_kernel<P, 8, ACT>);
  }
}

template <class P>
const void *AdapterKernels<P>::expand(int rank_tiles, bool activation) {
  return activation ? adapter_expand_for<P, true>(rank_tiles) : adapter_expand_for<P, false>(rank_tiles);
}

template <class P>
const void *AdapterKernels<P>::outer(int rank_tiles) {
  switch (rank_tiles) {
    case 1:
      return reinterpret_cast<const void *>(&adapter_outer_kernel<P, 1>);
    case 2:
      return reinterpret_cast<const void *>(&adapter_outer_kernel<P, 2>);
    case 4:
      return reinterpret_cast<const void *>(&adapter_outer_kernel<P, 4>);
    default:
      return reinterpret_cast<const void *>(&adapter_outer_kernel<P, 8>);
  }
}

}  // namespace xp
