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

template <class P, AdapterAct ACT, bool DIRECT>
const void *adapter_expand_for(int rank_tiles) {
  switch (rank_tiles) {
    case 1:
      return reinterpret_cast<const void *>(&adapter_expand_kernel<P, 1, ACT, DIRECT>);
    case 2:
      return reinterpret_cast<const void *>(&adapter_expand_kernel<P, 2, ACT, DIRECT>);
    case 4:
      return reinterpret_cast<const void *>(&adapter_expand_kernel<P, 4, ACT, DIRECT>);
    default:
      return reinterpret_cast<const void *>(&adapter_expand_kernel<P, 8, ACT, DIRECT>);
  }
}

template <class P, AdapterAct ACT>
const void *adapter_expand_for(int rank_tiles, bool direct) {
  return direct ? adapter_expand_for<P, ACT, true>(rank_tiles) : adapter_expand_for<P, ACT, false>(rank_tiles);
}

template <class P>
const void *AdapterKernels<P>::expand(int rank_tiles, AdapterAct activation, bool direct) {
  switch (activation) {
    case AdapterAct::None:
      return adapter_expand_for<P, AdapterAct::None>(rank_tiles, direct);
    case AdapterAct::GatedSilu:
      return adapter_expand_for<P, AdapterAct::GatedSilu>(rank_tiles, direct);
    default:
      return adapter_expand_for<P, AdapterAct::Any>(rank_tiles, direct);
  }
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
