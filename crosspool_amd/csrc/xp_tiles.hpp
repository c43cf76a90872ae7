// What the kernels that stage LDS tiles with direct buffer-to-LDS loads share.
#pragma once

#include "xp_common.hpp"

#include <type_traits>
#include <utility>

// Lambdas of these kernels are forced inline: a lambda left out of line takes the
// accumulator array by reference, which then lives in scratch memory instead of registers.
#define XP_INLINE __attribute__((always_inline))

namespace xp {
namespace {

// Offset that is always past a buffer resource's end (resources stay below 2^31 bytes, and
// adding a row's byte offset keeps it below 2^32).
constexpr uint32_t kOutOfRange = 0x7ffffff0u;

using lds_void_t = __attribute__((address_space(3))) void *;

// Direct global -> LDS load of 16 bytes per lane through a buffer resource: lane i's
// data lands at `lds_row_base + 16 i`; offsets past the resource's end write zeros.
template <int POLICY = 0>
__device__ __forceinline__ void buffer_load_lds16(__amdgpu_buffer_rsrc_t rsrc, void *lds_base, uint32_t voffset,
                                                  uint32_t soffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_t)(lds_base), 16, static_cast<int>(voffset),
                                           static_cast<int>(soffset), 0, POLICY);
}

// s_waitcnt with vmcnt <= N and the LDS / export counters left unconstrained (gfx9 encoding:
// vmcnt bits [3:0] and [15:14], expcnt [6:4], lgkmcnt [11:8]).
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt is a 6-bit counter");
  __builtin_amdgcn_s_waitcnt((N & 0xf) | ((N >> 4) << 14) | (0x7 << 4) | (0xf << 8));
}

// LDS tiles are rows of 64 bf16 (128 bytes = eight 16-byte chunks).  gfx950 serves
// ds_read_b128 sixteen lanes at a time from a 256-byte bank line, i.e. two tile rows, so
// the 16 rows one MFMA fragment read touches must occupy 16 distinct 16-byte slots:
// logical chunk c of row r is stored at physical chunk c ^ ((r / 2) % 8).
__device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }

// Calls f(std::integral_constant<int, 0>{}) .. f(std::integral_constant<int, N - 1>{}).
template <class F, int... I>
__device__ __forceinline__ void static_for_impl(F &&f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void static_for(F &&f) {
  static_for_impl(f, std::make_integer_sequence<int, N>{});
}

}  // namespace
}  // namespace xp
