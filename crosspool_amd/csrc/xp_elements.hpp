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

// A gated pair within the limit.  NaN is past no limit and stays (fminf and fmaxf, which the projections'
// and the standalone activation's epilogues below take, would make the limit of it).
__device__ __forceinline__ void clip_keep_nan(float &gate, float &up, float limit) {
  gate = gate > limit ? limit : gate;
  up = up > limit ? limit : up < -limit ? -limit : up;
}

template <bool KEEP_NAN = false>
__device__ __forceinline__ float apply_gated(float gate, float up, const ActivationArgs &act) {
  if (act.has_limit) {
    if constexpr (KEEP_NAN) {
      clip_keep_nan(gate, up, act.limit);
    } else {
      gate = fminf(gate, act.limit);
      up = fminf(fmaxf(up, -act.limit), act.limit);
    }
  }
  return apply_function(gate, act) * (up + act.up_offset);
}

// ------------------------------------------------------------------ gradient of the activation
// f(v) and f'(v) of one activation, in fp32 with the hardware's exp and reciprocal.  f is off by at most
// 2^-15 of itself, f' by 2^-15 of its two terms' magnitudes (next to its root they cancel, so its relative error
// has no bound there), against the store's 2^-9 or 2^-12: exponents x are off by a few 2^-24 |x| with |x| < 90.
// A sigmoid or density below 2^-126 may be 0.  The tails keep this: the sigmoid forms by themselves,
// 0.5 (1 + tanh(y)) as sigmoid(2 y), and Phi(v) by a form of its own, where 0.5 (1 + erff) cancels (nothing is
// left of that from v = -5.5) and erfcf takes longer than the memory (4096 rows of 12288 INTERLEAVED bf16 pairs:
// 106-112 us with it, 88 so; ungated 80 and 46-48).  PRECISE, for fp32 payloads, calls the library's exp and erfc and
// divides: a few steps of fp32 off.
enum class Slope : int { Silu = 1, Relu = 2, GeluErf = 3, GeluTanh = 4 };

template <Slope KIND, bool PRECISE = false>
__device__ __forceinline__ void value_and_slope(float v, float alpha, float &value, float &slope) {
  if constexpr (PRECISE && KIND != Slope::Relu) {
    if constexpr (KIND == Slope::GeluErf) {
      const float share = 0.5f * erfcf(v * -0.7071067811865476f);
      value = v * share;
      // Past 16 the density is 0 (and v may be infinite).
      const float near = fminf(fmaxf(v, -16.0f), 16.0f);
      slope = share + near * 0.3989422804014327f * expf(-0.5f * near * near);
    } else if constexpr (KIND == Slope::GeluTanh) {
      const float near = fminf(fmaxf(v, -16.0f), 16.0f);
      const float square = near * near;
      const float twice = 2.0f * 0.7978845608028654f * near * (1.0f + 0.044715f * square);
      const float share = v != v ? v : 1.0f / (1.0f + expf(-twice));
      value = v * share;
      slope = share + near * share * (1.0f - share) * (2.0f * 0.7978845608028654f) * (1.0f + 3.0f * 0.044715f * square);
    } else {
      const float share = 1.0f / (1.0f + expf(-alpha * v));
      value = v * share;
      const float near = fminf(fmaxf(alpha * v, -128.0f), 128.0f);
      slope = share * (1.0f + near * (1.0f - share));
    }
  } else if constexpr (KIND == Slope::Relu) {
    value = relu_keep_nan(v);
    slope = v != v ? v : v > 0.0f ? 1.0f : 0.0f;
  } else if constexpr (KIND == Slope::GeluErf) {
    // Phi(-x) = exp(-x^2 / 2) t P(t) for x >= 0, t = 1 / (1 + 0.3 x) (Hastings' form of approximation): it shares
    // the density's exp.  P has the least largest relative error over 0..16, found by reweighted least squares
    // against the scaled complementary error function; 2^-21 in fp32.  Past 16 all of it is 0.
    const float near = v > 16.0f ? 16.0f : v < -16.0f ? -16.0f : v;
    const float t = __builtin_amdgcn_rcpf(1.0f + 0.3f * fabsf(near));
    float ratio = 0.0347050946f;
    ratio = ratio * t - 0.153187922f;
    ratio = ratio * t + 0.199489063f;
    ratio = ratio * t - 0.0474273508f;
    ratio = ratio * t + 0.125292216f;
    ratio = ratio * t + 0.100889168f;
    ratio = ratio * t + 0.120600548f;
    ratio = ratio * t + 0.119639082f;
    const float density = __expf(-0.5f * near * near);
    const float tail = density * t * ratio;
    const float share = v > 0.0f ? 1.0f - tail : tail;
    value = v * share;
    slope = share + near * 0.3989422804014327f * density;
  } else if constexpr (KIND == Slope::GeluTanh) {
    // Past 16 the sigmoid is 0 or 1 and its slope 0 (and v^3 may overflow).
    const float near = fminf(fmaxf(v, -16.0f), 16.0f);
    const float square = near * near;
    const float twice = 2.0f * 0.7978845608028654f * near * (1.0f + 0.044715f * square);
    const float share = v != v ? v : __builtin_amdgcn_rcpf(1.0f + __expf(-twice));
    value = v * share;
    slope = share + near * share * (1.0f - share) * (2.0f * 0.7978845608028654f) * (1.0f + 3.0f * 0.044715f * square);
  } else {
    const float share = __builtin_amdgcn_rcpf(1.0f + __expf(-alpha * v));
    value = v * share;
    // Past 128 one of the two factors is 0 (and alpha v may overflow).
    const float near = fminf(fmaxf(alpha * v, -128.0f), 128.0f);
    slope = share * (1.0f + near * (1.0f - share));
  }
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
