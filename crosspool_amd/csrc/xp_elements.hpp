// Elements of any payload dtype (bf16, fp16, fp32) at any alignment, and the activations: shared by
// the general projection, the standalone activation and its gradient, and the adapters.
#pragma once

#include "xp_kernels.hpp"

#include <hip/hip_fp16.h>

#include <type_traits>

namespace xp {

__device__ __forceinline__ float load_value(const void *base, int64_t index, int dtype) {
  switch (dtype) {
    case kDtypeF16:
      return __half2float(reinterpret_cast<const __half *>(base)[index]);
    case kDtypeF32:
      return reinterpret_cast<const float *>(base)[index];
    default:
      return bf16_to_float(reinterpret_cast<const uint16_t *>(base)[index]);
  }
}

// Nearest-even rounding to the payload dtype, back in fp32.
__device__ __forceinline__ float round_to(float value, int dtype) {
  switch (dtype) {
    case kDtypeF16:
      return __half2float(__float2half_rn(f32_rounding_point(value)));
    case kDtypeF32:
      return value;
    default:
      return round_bf16(value);
  }
}

__device__ __forceinline__ void store_value(void *base, int64_t index, float value, int dtype) {
  switch (dtype) {
    case kDtypeF16:
      reinterpret_cast<__half *>(base)[index] = __float2half_rn(f32_rounding_point(value));
      break;
    case kDtypeF32:
      reinterpret_cast<float *>(base)[index] = value;
      break;
    default:
      reinterpret_cast<uint16_t *>(base)[index] = static_cast<uint16_t>(float_to_bf16(value));
      break;
  }
}

// ReLU that keeps NaN payloads: x for x > 0 or NaN, +0 otherwise.
__device__ __forceinline__ float relu_keep_nan(float value) { return (value > 0.0f || value != value) ? value : 0.0f; }

__device__ __forceinline__ float apply_function(float value, const ActivationArgs &act) {
  switch (act.function) {
    case kActivationRelu:
      return relu_keep_nan(value);
    case kActivationGelu:
      if (act.approximate_tanh) {
        const float inner = 0.7978845608028654f * (value + 0.044715f * value * value * value);
        return 0.5f * value * (1.0f + tanhf(inner));
      }
      return 0.5f * value * (1.0f + erff(value * 0.7071067811865476f));
    default:  // SiLU: v / (1 + exp(-alpha v)), IEEE divide
      return value / (1.0f + expf(-act.alpha * value));
  }
}

__device__ __forceinline__ float apply_gated(float gate, float up, const ActivationArgs &act) {
  if (act.has_limit) {
    gate = fminf(gate, act.limit);
    up = fminf(fmaxf(up, -act.limit), act.limit);
  }
  return apply_function(gate, act) * (up + act.up_offset);
}

// A gated pair within the limit.  NaN is past no limit and stays (fminf and fmaxf, which the projections'
// and the standalone activation's epilogues above take, would make the limit of it).
__device__ __forceinline__ void clip_keep_nan(float &gate, float &up, float limit) {
  gate = gate > limit ? limit : gate;
  up = up > limit ? limit : up < -limit ? -limit : up;
}

// The fp32 element type beside Bf16Payload / F16Payload: a 16-byte chunk holds 4 columns, and
// its MFMA step covers 8 (lane half h multiplies columns 4 h + j of both operands at step j).
struct F32Payload {
  __device__ static __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    }
    return c;
  }
  // The 16 x 16 form: chunk lane / 16 of a row holds columns 4 (lane / 16) + j of step j.
  __device__ static __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    }
    return c;
  }
};

template <class T>
constexpr int kElementBytes = std::is_same_v<T, F32Payload> ? 4 : 2;
template <class T>
constexpr int kDtypeOf = std::is_same_v<T, F32Payload> ? kDtypeF32 : std::is_same_v<T, F16Payload> ? kDtypeF16 : kDtypeBf16;

// 16 (or 8) bytes from an address aligned to an element only.
__device__ __forceinline__ u32x4 load16_any(const unsigned char *address) {
  u32x4 value;
  __builtin_memcpy(&value, address, 16);
  return value;
}
__device__ __forceinline__ u32x2 load8_any(const unsigned char *address) {
  u32x2 value;
  __builtin_memcpy(&value, address, 8);
  return value;
}

// One LDS chunk (16 bytes of T) of a row at `source` (XT elements).
template <class XT, class T>
__device__ __forceinline__ u32x4 load_chunk(const unsigned char *source) {
  if constexpr (kElementBytes<XT> == kElementBytes<T>) {
    return load16_any(source);
  } else {
    const u32x2 packed = load8_any(source);
    return u32x4{__float_as_uint(XT::widen(packed[0] & 0xffffu)), __float_as_uint(XT::widen(packed[0] >> 16)),
                 __float_as_uint(XT::widen(packed[1] & 0xffffu)), __float_as_uint(XT::widen(packed[1] >> 16))};
  }
}

// The same where only `valid` (fewer than a chunk's) columns are left: zeros past them.
template <class XT, class T>
__device__ __forceinline__ u32x4 load_chunk_tail(const unsigned char *source, int64_t valid) {
  u32x4 chunk = {0u, 0u, 0u, 0u};
  if constexpr (kElementBytes<T> == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j < valid) {
        chunk[j] = kElementBytes<XT> == 4 ? reinterpret_cast<const uint32_t *>(source)[j]
                                          : __float_as_uint(load_value(source, j, kDtypeOf<XT>));
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j < valid) {
        chunk[j / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(source)[j]) << (16 * (j % 2));
      }
    }
  }
  return chunk;
}

}  // namespace xp
