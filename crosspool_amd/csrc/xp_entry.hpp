// What the C entry points share: errors, argument checks and the operands' ranges.
#pragma once

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <string>

#include "../../include/xpool_amd.h"
#include "xp_kernels.hpp"

namespace xp {

// Keeps `message` for xp_last_error and returns `code`.
int fail(int code, const std::string &message);

// The activation descriptor of the C ABI as the kernels take it (checked).
int activation_record(const xp_activation_desc *desc, ActivationArgs &out);

#define XP_HIP_CHECK(expr)                                                                   \
  do {                                                                                       \
    const hipError_t xp_error_ = (expr);                                                     \
    if (xp_error_ != hipSuccess) {                                                           \
      return fail(XP_ERROR_HIP, std::string(#expr) + " failed: " + hipGetErrorString(xp_error_)); \
    }                                                                                        \
  } while (0)

#define XP_REQUIRE(condition, message)                  \
  do {                                                  \
    if (!(condition)) {                                 \
      return fail(XP_ERROR_INVALID_ARGUMENT, message);  \
    }                                                   \
  } while (0)

inline bool aligned16(const void *pointer) { return (reinterpret_cast<uintptr_t>(pointer) & 15u) == 0; }

inline size_t dtype_bytes(int dtype) {
  switch (dtype) {
    case XP_DTYPE_BF16:
    case XP_DTYPE_F16:
      return 2;
    case XP_DTYPE_F32:
      return 4;
    default:
      return 0;
  }
}

inline bool aligned_to(const void *pointer, size_t bytes) { return (reinterpret_cast<uintptr_t>(pointer) % bytes) == 0; }

// A call's operand: `rows` runs of `width` bytes, `stride` bytes from one's begin to the next's.
struct Span {
  int64_t begin;
  int64_t stride;
  int64_t width;
  int64_t rows;
  int64_t end() const { return begin + (rows - 1) * stride + width; }
};
inline Span span_of(const void *p, size_t bytes) {
  const int64_t width = static_cast<int64_t>(bytes);
  return {reinterpret_cast<intptr_t>(p), width, width, p == nullptr || bytes == 0 ? 0 : 1};
}
inline Span span_of_rows(const void *p, int64_t ld, int64_t width, int64_t rows, size_t element) {
  const int64_t bytes = static_cast<int64_t>(element);
  return {reinterpret_cast<intptr_t>(p), ld * bytes, width * bytes, p == nullptr ? 0 : rows};
}
// Quotient rounded down.
inline int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b != 0 && (a < 0) != (b < 0) ? 1 : 0); }

// Whether two operands share a byte: not where the rows of one lie between those of the other, as columns of
// one wider tensor do.
inline bool overlaps(const Span &p, const Span &q) {
  if (p.rows == 0 || q.rows == 0 || p.begin >= q.end() || q.begin >= p.end()) {
    return false;
  }
  if (p.rows > 1 && q.rows > 1 && p.stride != q.stride) {
    // Row by row of the operand of fewer rows; the ranges have to overlap for this to be reached.
    const Span &few = p.rows <= q.rows ? p : q;
    const Span &many = p.rows <= q.rows ? q : p;
    for (int64_t row = 0; row < few.rows; ++row) {
      if (overlaps({few.begin + row * few.stride, few.width, few.width, 1}, many)) {
        return true;
      }
    }
    return false;
  }
  // Row i of p and row j of q meet where -q.width < (q.begin - p.begin) + (j - i) stride < p.width.
  const int64_t stride = p.rows > 1 ? p.stride : q.stride;
  const int64_t distance = q.begin - p.begin;
  const int64_t least = std::max(floor_div(-q.width - distance, stride) + 1, 1 - p.rows);
  const int64_t most = std::min(-floor_div(distance - p.width, stride) - 1, q.rows - 1);
  return least <= most;
}
inline bool touches(const Span &span, std::initializer_list<Span> others) {
  return std::any_of(others.begin(), others.end(), [&](const Span &other) { return overlaps(span, other); });
}

}  // namespace xp
