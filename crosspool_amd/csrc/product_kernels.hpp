// The products' kernels: LDS-staged MFMA tiles over operands of either storage order, with the training
// operators' epilogues, and the sum of split K ranges.
//
// Layout.  A slab is 128 bytes of the reduction axis (64 columns of 16 bits, 32 of fp32).  An operand whose
// reduction axis runs along its rows is staged as in the projections' tile kernel: LDS rows of eight 16-byte
// chunks, chunk c of row r at c ^ (r / 2 % 8), fragments by ds_read_b128.  One whose reduction axis runs
// across its rows is staged as it lies in memory, a slab's 64 (32) rows of the tile's columns, and transposed
// by the read: ds_read_b64_tr_b16 hands each group of 16 lanes four reduction rows of 16 neighbouring columns
// as one column's four values per lane, so two of them make the 8-value fragment of v_mfma_f32_32x32x16.  No
// transposed copy of weights, activations or gradients is ever made.  (fp32 fragments of
// v_mfma_f32_32x32x2 are four ds_read_b32.)  The 64-byte groups that the four rows of one read touch lie in
// distinct quarters of LDS's 256-byte bank line: reduction row k keeps its 64-byte group g at g ^ (k % 4).
//
// The MFMA's M operand is B, so that a lane's sums are four neighbouring columns n of one row m.
//
// What bounds them.  Large products: the matrix cores, at the rate the card's power allows on random operands (bf16
// 4096 x 4096 x 24576 625 us, 1.32 PFLOP/s; 4096 x 12288 x 4096 311 us, 1.32; fp16 649 and 331; a loop without loads 1.5 to
// 1.75).  The epilogues of kActivate (bf16 4096 x 24576 x 4096 678 us against 628 without its activation and 100 MB of stores)
// and kGradient (4096 x 12288 x 4096 460 us against 311 without its 400 MB) move their bytes while the CU's matrix cores wait, since
// 256 x 256 accumulators leave no registers for a second tile.  Few rows: the operands' bytes (five rows of 2048 x 6144 8.8
// us, 2.9 TB/s).
//
// Registers.  kStore and kActivate use no scratch memory.  kGradient's small arrays take 12 or 24 bytes a lane of it, and its
// 256 x 256 tiles, which hold a block's kept values beside the accumulators, spill 126 registers in fp16 (132 bytes) and 6
// in bf16 (48 bytes).
#pragma once

#include "product.hpp"
#include "xp_elements.hpp"
#include "xp_tiles.hpp"

namespace xp {
namespace {

// ------------------------------------------------------------------ eight values of a row
// Runtime dtypes are wave-uniform: branches, not selects.
template <class P>
__device__ __forceinline__ void widen_chunk(u32x4 chunk, float (&value)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    value[j] = P::widen(j % 2 == 0 ? chunk[j / 2] & 0xffffu : chunk[j / 2] >> 16);
  }
}
template <class P>
__device__ __forceinline__ u32x4 pack_chunk(const float (&value)[8]) {
  return u32x4{P::pack2(value[0], value[1]), P::pack2(value[2], value[3]), P::pack2(value[4], value[5]),
               P::pack2(value[6], value[7])};
}

__device__ __forceinline__ void load_values(const void *source, int64_t index, int dtype, int count, float (&value)[8]) {
  if (dtype == kDtypeF32) {
    const float *from = static_cast<const float *>(source) + index;
    if (count >= 8) {
      __builtin_memcpy(value, from, 32);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        value[j] = j < count ? from[j] : 0.0f;
      }
    }
    return;
  }
  const uint16_t *from = static_cast<const uint16_t *>(source) + index;
  const unsigned char *bytes = reinterpret_cast<const unsigned char *>(from);
  const u32x4 chunk = count >= 8 ? load16_any(bytes) : load_chunk_tail<Bf16Payload, Bf16Payload>(bytes, count);
  if (dtype == kDtypeF16) {
    widen_chunk<F16Payload>(chunk, value);
  } else {
    widen_chunk<Bf16Payload>(chunk, value);
  }
}

__device__ __forceinline__ void store_values(void *target, int64_t index, int dtype, int count, const float (&value)[8]) {
  if (dtype == kDtypeF32) {
    float *to = static_cast<float *>(target) + index;
    if (count >= 8) {
      __builtin_memcpy(to, value, 32);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j < count) {
          to[j] = value[j];
        }
      }
    }
    return;
  }
  uint16_t *to = static_cast<uint16_t *>(target) + index;
  u32x4 packed;
  if (dtype == kDtypeF16) {
    packed = pack_chunk<F16Payload>(value);
  } else {
    packed = pack_chunk<Bf16Payload>(value);
  }
  if (count >= 8) {
    __builtin_memcpy(to, &packed, 16);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j < count) {
      to[j] = static_cast<uint16_t>(packed[j / 2] >> (16 * (j % 2)));
    }
  }
}

// Calls use with the activation as a compile-time constant (it is the same for the whole launch).
template <class F>
__device__ __forceinline__ void with_function(const ActivationArgs &act, F &&use) {
  switch (act.function) {
    case kActivationRelu:
      use(std::integral_constant<Slope, Slope::Relu>{});
      break;
    case kActivationGelu:
      if (act.approximate_tanh) {
        use(std::integral_constant<Slope, Slope::GeluTanh>{});
      } else {
        use(std::integral_constant<Slope, Slope::GeluErf>{});
      }
      break;
    default:
      use(std::integral_constant<Slope, Slope::Silu>{});
      break;
  }
}

// Where eight columns of a row lie: elements from the begin of the output, the base and the extra operand.
struct ChunkPlace {
  int64_t out;
  int64_t base;
  int64_t extra;
};
// Columns of the output, base and extra operands that one column of the sums stands for.
template <ProductEpilogue EPI>
__device__ __forceinline__ ChunkPlace chunk_place(const ProductArgs &a, int64_t matrix, int64_t row, int64_t col) {
  if constexpr (EPI == ProductEpilogue::kStore) {
    return {matrix * a.batch_out + row * a.ld_out + col, matrix * a.batch_base + row * a.ld_base + col,
            matrix * a.batch_extra + row * a.ld_extra + col};
  } else if constexpr (EPI == ProductEpilogue::kActivate) {
    return {row * a.ld_out + (a.halves != 0 ? col / 2 : col), 0, row * a.ld_extra + (a.act.gated ? col / 2 : col)};
  } else {
    const int64_t wide = a.act.gated && a.interleaved ? 2 * col : col;
    return {row * a.ld_out + wide, row * a.ld_base + wide, row * a.ld_extra + col};
  }
}

// What an epilogue reads beside the sums, as it lies in memory: requested for a whole block of rows before the first of
// them is used, since a workgroup in its epilogue has no other work to hide that latency under.
template <class P, ProductEpilogue EPI>
struct Beside {
  u32x4 base[2];
  u32x4 extra[2];
};
__device__ __forceinline__ void request_values(const void *source, int64_t index, int dtype, int count, u32x4 (&raw)[2]) {
  if (dtype == kDtypeF32) {
    const unsigned char *from = reinterpret_cast<const unsigned char *>(static_cast<const float *>(source) + index);
    if (count >= 8) {
      raw[0] = load16_any(from);
      raw[1] = load16_any(from + 16);
    } else {
      raw[0] = count >= 4 ? load16_any(from) : load_chunk_tail<F32Payload, F32Payload>(from, count);
      raw[1] = load_chunk_tail<F32Payload, F32Payload>(from + 16, count - 4);
    }
    return;
  }
  const unsigned char *from = reinterpret_cast<const unsigned char *>(static_cast<const uint16_t *>(source) + index);
  raw[0] = count >= 8 ? load16_any(from) : load_chunk_tail<Bf16Payload, Bf16Payload>(from, count);
}
__device__ __forceinline__ void take_values(const u32x4 (&raw)[2], int dtype, float (&value)[8]) {
  if (dtype == kDtypeF32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      value[j] = __uint_as_float(raw[j / 4][j % 4]);
    }
  } else if (dtype == kDtypeF16) {
    widen_chunk<F16Payload>(raw[0], value);
  } else {
    widen_chunk<Bf16Payload>(raw[0], value);
  }
}

// Four values of a row, as they lie in memory.
template <class P>
__device__ __forceinline__ void request_four(const void *source, int64_t index, int count, u32x4 &raw) {
  if constexpr (kElementBytes<P> == 4) {
    const unsigned char *from = reinterpret_cast<const unsigned char *>(static_cast<const float *>(source) + index);
    raw = count >= 4 ? load16_any(from) : load_chunk_tail<P, P>(from, count);
  } else {
    const unsigned char *from = reinterpret_cast<const unsigned char *>(static_cast<const uint16_t *>(source) + index);
    if (count >= 4) {
      const u32x2 packed = load8_any(from);
      raw = u32x4{packed[0], packed[1], 0u, 0u};
    } else {
      raw = load_chunk_tail<P, P>(from, count);
    }
  }
}
template <class P>
__device__ __forceinline__ void take_four(const u32x4 &raw, float (&value)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (kElementBytes<P> == 4) {
      value[j] = __uint_as_float(raw[j]);
    } else {
      value[j] = P::widen(j % 2 == 0 ? raw[j / 2] & 0xffffu : raw[j / 2] >> 16);
    }
  }
}

template <class P, ProductEpilogue EPI>
__device__ __forceinline__ void request(const ProductArgs &a, const ChunkPlace &at, int64_t col, Beside<P, EPI> &beside) {
  if constexpr (EPI == ProductEpilogue::kStore) {
    const int count = a.n - col < 8 ? static_cast<int>(a.n - col) : 8;
    if (a.beta != 0.0f) {
      request_values(a.base, at.base, a.base_dtype, count, beside.base);
    }
    if (a.extra != nullptr) {
      request_values(a.extra, at.extra, a.extra_dtype, count, beside.extra);
    }
  } else if constexpr (EPI == ProductEpilogue::kGradient) {
    const int count = a.n - col < 4 ? static_cast<int>(a.n - col) : 4;
    constexpr int dtype = kDtypeOf<P>;
    if (a.act.gated != 0 && a.interleaved != 0) {
      request_values(a.base, at.base, dtype, 2 * count, beside.base);
    } else {
      request_four<P>(a.base, at.base, count, beside.base[0]);
      if (a.act.gated) {
        request_four<P>(a.base, at.base + a.n, count, beside.base[1]);
      }
    }
  }
}

template <class P>
__device__ __forceinline__ void store_four(void *target, int64_t index, int count, const float (&value)[4]) {
  if constexpr (kElementBytes<P> == 4) {
    float *to = static_cast<float *>(target) + index;
    if (count >= 4) {
      __builtin_memcpy(to, value, 16);
      return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j < count) {
        to[j] = value[j];
      }
    }
  } else {
    uint16_t *to = static_cast<uint16_t *>(target) + index;
    const u32x2 packed = {P::pack2(value[0], value[1]), P::pack2(value[2], value[3])};
    if (count >= 4) {
      __builtin_memcpy(to, &packed, 8);
      return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j < count) {
        to[j] = static_cast<uint16_t>(packed[j / 2] >> (16 * (j % 2)));
      }
    }
  }
}

// The activation of a Gate and an Up.  NaN is past no limit, as in the backward pass of the same values.
template <Slope KIND, bool PRECISE>
__device__ __forceinline__ float gated_value(const ActivationArgs &act, float gate, float up) {
  if (act.has_limit) {
    clip_keep_nan(gate, up, act.limit);
  }
  float f;
  float unused;
  value_and_slope<KIND, PRECISE>(gate, act.alpha, f, unused);
  return f * (up + act.up_offset);
}

// The epilogue (but kGradient's) of columns col .. col + 7, those below n, of one row.
template <class P, ProductEpilogue EPI>
__device__ __forceinline__ void finish(const ProductArgs &a, const ChunkPlace &at, int64_t col, const Beside<P, EPI> &beside,
                                       float (&value)[8]) {
  constexpr int dtype = kDtypeOf<P>;
  constexpr bool PRECISE = kElementBytes<P> == 4;
  const int count = a.n - col < 8 ? static_cast<int>(a.n - col) : 8;
  if constexpr (EPI == ProductEpilogue::kStore) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      value[j] *= a.alpha;
    }
    if (a.beta != 0.0f) {
      float other[8];
      take_values(beside.base, a.base_dtype, other);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        value[j] += a.beta * other[j];
      }
    }
    if (a.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        value[j] += j < count ? a.bias[col + j] : 0.0f;
      }
    }
    if (a.extra != nullptr) {
      float other[8];
      take_values(beside.extra, a.extra_dtype, other);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        value[j] = a.keep * other[j] - a.step * value[j];
      }
    }
    store_values(a.out, at.out, a.out_dtype, a.padded_out ? 8 : count, value);
  } else if (a.halves != 0) {
    // Gate and Up of four outputs, which lie in two runs.
    float gate[4];
    float up[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool with_bias = a.bias != nullptr && 2 * j < count;
      gate[j] = value[2 * j] + (with_bias ? a.bias[col / 2 + j] : 0.0f);
      up[j] = value[2 * j + 1] + (with_bias ? a.bias[a.halves + col / 2 + j] : 0.0f);
    }
    store_four<P>(a.out, at.out, count / 2, gate);
    store_four<P>(a.out, at.out + a.halves, count / 2, up);
    float activated[4];
    with_function(a.act, [&](auto kind) XP_INLINE {
      constexpr Slope KIND = decltype(kind)::value;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        activated[j] = gated_value<KIND, PRECISE>(a.act, gate[j], up[j]);
      }
    });
    store_four<P>(a.extra, at.extra, count / 2, activated);
  } else {
    if (a.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        value[j] += j < count ? a.bias[col + j] : 0.0f;
      }
    }
    store_values(a.out, at.out, dtype, count, value);
    with_function(a.act, [&](auto kind) XP_INLINE {
      constexpr Slope KIND = decltype(kind)::value;
      float unused;
      if (!a.act.gated) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          value_and_slope<KIND, PRECISE>(value[j], a.act.alpha, value[j], unused);
        }
        return;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        value[j] = gated_value<KIND, PRECISE>(a.act, value[2 * j], value[2 * j + 1]);
      }
    });
    if (!a.act.gated) {
      store_values(a.extra, at.extra, dtype, count, value);
    } else if (count == 8) {
      if constexpr (PRECISE) {
        __builtin_memcpy(static_cast<float *>(a.extra) + at.extra, value, 16);
      } else {
        const u32x2 packed = {P::pack2(value[0], value[1]), P::pack2(value[2], value[3])};
        __builtin_memcpy(static_cast<uint16_t *>(a.extra) + at.extra, &packed, 8);
      }
    } else {
      // n is even: a pair is whole or absent.
      store_values(a.extra, at.extra, dtype, count / 2, value);
    }
  }
}

// kGradient for columns col .. col + 3: four pairs of INTERLEAVED Gate/Up are one 16-byte chunk of 16-bit values, so
// that neighbouring lanes read and write neighbouring chunks.  `sums` gathers the gradients by column: [0, 4) of
// Gate (or of ungated values), [4, 8) of Up.
template <class P>
__device__ __forceinline__ void finish_gradient(const ProductArgs &a, const ChunkPlace &at, int64_t col,
                                                const Beside<P, ProductEpilogue::kGradient> &beside, const float (&through)[4],
                                                float (&sums)[8]) {
  constexpr int dtype = kDtypeOf<P>;
  constexpr bool PRECISE = kElementBytes<P> == 4;
  const int count = a.n - col < 4 ? static_cast<int>(a.n - col) : 4;
  float gate[4];
  float up[4];
  const bool pairs = a.act.gated != 0 && a.interleaved != 0;
  if (pairs) {
    float both[8];
    take_values(beside.base, dtype, both);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      gate[j] = both[2 * j];
      up[j] = both[2 * j + 1];
    }
  } else {
    take_four<P>(beside.base[0], gate);
    take_four<P>(beside.base[1], up);
  }
  float activated[4];
  with_function(a.act, [&](auto kind) XP_INLINE {
    constexpr Slope KIND = decltype(kind)::value;
    if (!a.act.gated) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float slope;
        value_and_slope<KIND, PRECISE>(gate[j], a.act.alpha, activated[j], slope);
        gate[j] = through[j] * slope;
        up[j] = 0.0f;
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float clipped = gate[j];
      float factor = up[j];
      bool gate_on = true;
      bool up_on = true;
      if (a.act.has_limit) {
        clip_keep_nan(clipped, factor, a.act.limit);
        gate_on = !(gate[j] > a.act.limit);
        up_on = !(fabsf(up[j]) > a.act.limit);
      }
      float f;
      float slope;
      value_and_slope<KIND, PRECISE>(clipped, a.act.alpha, f, slope);
      factor += a.act.up_offset;
      gate[j] = gate_on ? through[j] * slope * factor : 0.0f;
      up[j] = up_on ? through[j] * f : 0.0f;
      activated[j] = f * factor;
    }
  });
  if (a.column_sums != nullptr) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sums[j] += gate[j];
      sums[4 + j] += up[j];
    }
  }
  store_four<P>(a.extra, at.extra, count, activated);
  if (pairs) {
    const float both[8] = {gate[0], up[0], gate[1], up[1], gate[2], up[2], gate[3], up[3]};
    store_values(a.out, at.out, dtype, 2 * count, both);
  } else {
    store_four<P>(a.out, at.out, count, gate);
    if (a.act.gated) {
      store_four<P>(a.out, at.out + a.n, count, up);
    }
  }
}

// Column sums of a wave's band: lanes with one chunk (lane % LANES) hold parts of the same columns.
template <int LANES>
__device__ __forceinline__ void store_column_sums(const ProductArgs &a, int64_t band, int64_t col, float (&sums)[8], int lane) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int offset = LANES; offset < 64; offset *= 2) {
      sums[j] += __shfl_xor(sums[j], offset, kWave);
    }
  }
  if (lane >= LANES) {
    return;
  }
  const int64_t wide = a.act.gated ? 2 * a.n : a.n;
  float *to = a.column_sums + band * wide;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (col + j < a.n) {
      if (!a.act.gated) {
        to[col + j] = sums[j];
      } else if (a.interleaved) {
        to[2 * (col + j)] = sums[j];
        to[2 * (col + j) + 1] = sums[4 + j];
      } else {
        to[col + j] = sums[j];
        to[a.n + col + j] = sums[4 + j];
      }
    }
  }
}

// ------------------------------------------------------------------ operands in LDS
using lds_bytes_t = __attribute__((address_space(3))) unsigned char *;
using i16x4 = short __attribute__((ext_vector_type(4)));

__device__ __forceinline__ u32x2 read_transposed(lds_bytes_t at) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)at));
}
__device__ __forceinline__ u32x4 read_chunk(lds_bytes_t at) {
  return *(const __attribute__((address_space(3))) u32x4 *)at;
}
__device__ __forceinline__ uint32_t read_word(lds_bytes_t at) {
  return *(const __attribute__((address_space(3))) uint32_t *)at;
}

// Direct global -> LDS load of 16 bytes per lane: lane i's data lands at LDS byte `to` + 16 i; offsets past the
// resource's `bytes` write zeros.  Written as an instruction because the compiler, which does not know the stages
// apart, waits for every load in flight before a ds_read_b64_tr (64 x 64 tiles: 0.57 us a slab instead of 0.27).  It
// has no result in a register; the kernel waits for its arrival itself, before a barrier that is a memory clobber.
// The compiler does not see a memory instruction here and adds no wait states: a load needs one behind the write of M0
// that it takes its LDS address from, and five behind a vector instruction that wrote one of its scalar registers (a
// readlane that brings a spilled one back).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // M0 among the clobbers: the compiler keeps nothing in it
__device__ __forceinline__ void load_lds16(u32x4 rsrc, uint32_t to, uint32_t voffset, uint32_t soffset) {
  __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                   :
                   : "s"(to), "v"(voffset), "s"(rsrc), "s"(soffset)
                   : "m0");
}
#pragma clang diagnostic pop
// The words of a raw buffer resource (make_rsrc), in scalar registers.
__device__ __forceinline__ u32x4 resource_words(const void *base, uint32_t bytes) {
  const uint64_t address = reinterpret_cast<uint64_t>(base);
  return u32x4{static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(address))),
               static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>((address >> 32) & 0xffffu))),
               static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(bytes))), 0x00020000u};
}

// The loads of one operand's tile of ROWS rows (columns, for COLS) into the stages.
template <class P, int ROWS, bool COLS, int LOAD_WAVES>
struct OperandLoads {
  static constexpr int ES = kElementBytes<P>;
  static constexpr int BK = 128 / ES;
  static constexpr int LOADS = ROWS / 8 / LOAD_WAVES;    // 1 KB load instructions per loading wave and slab
  static constexpr int LANES_PER_ROW = COLS ? ROWS * ES / 16 : 8;  // 16-byte chunks of one LDS row
  static constexpr int ROWS_PER_LOAD = 64 / LANES_PER_ROW;
  static_assert(ROWS % (8 * LOAD_WAVES) == 0, "stage rows must split evenly");
  static_assert(!COLS || LANES_PER_ROW <= 32, "a load covers two rows at least");

  const unsigned char *origin;  // the tile's first row (COLS: first column of reduction row 0)
  uint32_t ld_bytes;
  uint32_t span;                // bytes of the rows that a resource covers
  uint32_t lane_offset[2];
  uint32_t eight_bytes;         // between a load's rows and the next one's, and
  uint32_t lane_row;            // from there to this lane's row (rows along the reduction axis)
  int first;                    // this wave's first load of a slab

  // `rows_left` counts what is left of the operand from the tile's first row (column).  `halves`: not 0, rows 2 j and
  // 2 j + 1 are the operand's rows j and halves + j (rows along the reduction axis; 2 halves rows in 31 bits of bytes).
  __device__ __forceinline__ void setup(const void *data, int64_t ld, int64_t tile_first, int64_t rows_left, int wave, int lane,
                                        int64_t halves = 0) {
    ld_bytes = static_cast<uint32_t>(ld * ES);
    first = (wave % LOAD_WAVES) * LOADS;
    const int row = lane / LANES_PER_ROW;
    const int place = lane % LANES_PER_ROW;
    if constexpr (COLS) {
      origin = static_cast<const unsigned char *>(data) + tile_first * ES;
      span = 0;
#pragma unroll
      for (int variant = 0; variant < 2; ++variant) {
        const int chunk = place ^ scramble(variant, row);
        lane_offset[variant] = chunk * (16 / ES) < rows_left
                                   ? static_cast<uint32_t>(row) * ld_bytes + static_cast<uint32_t>(chunk * 16)
                                   : kOutOfRange;
      }
    } else {
      if (halves != 0) {
        origin = static_cast<const unsigned char *>(data) + tile_first / 2 * ld * ES;
        span = static_cast<uint32_t>(2 * halves - tile_first / 2) * ld_bytes;
        eight_bytes = 4 * ld_bytes;
        lane_row = static_cast<uint32_t>(row >> 1) * ld_bytes + (row % 2 != 0 ? static_cast<uint32_t>(halves) * ld_bytes : 0u);
      } else {
        origin = static_cast<const unsigned char *>(data) + tile_first * ld * ES;
        span = static_cast<uint32_t>(rows_left < ROWS ? rows_left : ROWS) * ld_bytes;
        eight_bytes = 8 * ld_bytes;
        lane_row = static_cast<uint32_t>(row) * ld_bytes;
      }
      // Eight rows a load: swizzle(8 g + row) = (row / 2) ^ (4 if g is odd), g = first + q.
      lane_offset[0] = static_cast<uint32_t>(place ^ (row >> 1) ^ (LOADS % 2 != 0 ? 4 * (first & 1) : 0));
      lane_offset[1] = lane_offset[0] ^ 4;
    }
  }

  // COLS: what the chunk index of reduction row k is xor-ed with; k's low bits follow from the load's variant
  // and the lane's row in it.
  __device__ static __forceinline__ int scramble(int variant, int row) {
    if constexpr (ROWS == 32) {
      return 0;                                       // four (16-bit) rows are a bank line
    } else if constexpr (ES == 4) {
      return variant << 3;                            // bit 2 of k
    } else if constexpr (ROWS >= 256) {
      return ((2 * variant + row) & 3) << 2;          // k % 4, two rows a load
    } else if constexpr (ROWS == 128) {
      return (row & 3) << 2;                          // four rows a load
    } else {
      return ((row >> 1) & 1) << 2;                   // two rows share a bank line
    }
  }
  // The variant of load q of a wave (its loads start at a multiple of LOADS, which is even or 1).
  static constexpr int variant(int q) {
    if constexpr (!COLS) {
      return q & 1;
    } else if constexpr (ES == 4) {
      return ROWS == 128 ? (q >> 1) & 1 : q & 1;
    } else {
      return ROWS >= 256 ? q & 1 : 0;
    }
  }

  // Load q of the slab at column k_pos of a range that ends at k_end, into the stage at LDS byte `stage`; a slab past
  // the end loads zeros.
  struct Slab {
    u32x4 rsrc;
    uint32_t k_bytes;
    int chunks_left;
  };
  __device__ __forceinline__ Slab slab(int64_t k_pos, int64_t k_end) const {
    Slab found;
    const int64_t left = k_end - k_pos;
    if constexpr (COLS) {
      const uint32_t rows = left <= 0 ? 0u : left < BK ? static_cast<uint32_t>(left) : static_cast<uint32_t>(BK);
      found.rsrc = resource_words(origin + k_pos * static_cast<int64_t>(ld_bytes), rows * ld_bytes);
      found.k_bytes = 0;
      found.chunks_left = 0;
    } else {
      found.rsrc = resource_words(origin, span);
      found.k_bytes = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(k_pos * ES)));
      // A chunk that the range's end cuts holds zeros past it (the operands' rows are whole chunks).
      const int64_t limit = left <= 0 ? 0 : left < BK ? left : BK;
      found.chunks_left = static_cast<int>((limit + 16 / ES - 1) / (16 / ES));
    }
    return found;
  }
  __device__ __forceinline__ void load(const Slab &from, int q, uint32_t stage) const {
    const uint32_t to = stage + static_cast<uint32_t>(first + q) * 1024u;
    if constexpr (COLS) {
      const uint32_t rows_before = static_cast<uint32_t>((first + q) * ROWS_PER_LOAD);
      load_lds16(from.rsrc, to, lane_offset[variant(q)] + rows_before * ld_bytes, 0);
    } else {
      const uint32_t chunk = lane_offset[variant(q)];
      const uint32_t offset = static_cast<uint32_t>(first + q) * eight_bytes + lane_row + chunk * 16;
      load_lds16(from.rsrc, to, static_cast<int>(chunk) < from.chunks_left ? offset : kOutOfRange, from.k_bytes);
    }
  }
};

// The fragments of a wave's TILES 32-row tiles, the first of them tile `first_tile` of the operand's region.
template <class P, int ROWS, bool COLS, int TILES, int STAGES>
struct OperandFragments {
  static constexpr int ES = kElementBytes<P>;
  static constexpr int STAGE_BYTES = ROWS * 128;
  static constexpr int LARGEST = (STAGES - 1) * STAGE_BYTES + (COLS ? STAGE_BYTES : (TILES - 1) * 4096);
  static constexpr int WINDOWS = LARGEST / 65536 + 1;
  static constexpr int BASES = COLS ? TILES : 4;
  uint32_t base[WINDOWS][BASES];

  // `step0`: the k step that read's step 0 stands for.
  __device__ __forceinline__ void setup(int region, int first_tile, int step0, int lane) {
    const int half = lane >> 5;
#pragma unroll
    for (int i = 0; i < BASES; ++i) {
      int at;
      if constexpr (!COLS) {
        const int row = lane & 31;
        at = (first_tile * 32 + row) * 128 + (((((step0 + i) & 3) * 2 + half) ^ swizzle(row)) << 4);
      } else if constexpr (ES == 4) {
        const int tile = ROWS == 32 ? 0 : (first_tile + i) ^ half;  // bit 2 of the reduction row is the lane's half
        at = (8 * step0 + 4 * half) * ROWS * 4 + tile * 128 + (lane & 31) * 4;
      } else {
        const int within = lane & 15;
        const int row = 16 * step0 + 8 * half + (within >> 2);
        const int tile = ROWS == 32    ? 0
                         : ROWS >= 128 ? (first_tile + i) ^ (within >> 2)
                                       : (first_tile + i) ^ ((within >> 3) & 1);
        at = row * ROWS * 2 + tile * 64 + ((lane >> 4) & 1) * 32 + (within & 3) * 8;
      }
#pragma unroll
      for (int w = 0; w < WINDOWS; ++w) {
        base[w][i] = static_cast<uint32_t>(region + at + w * 65536);
        __asm__ volatile("" : "+v"(base[w][i]));
      }
    }
  }

  // K step ks of the stage, 32-row tile `tile` (all compile-time after unrolling).
  __device__ __forceinline__ u32x4 read(lds_bytes_t lds, int stage, int ks, int tile) const {
    if constexpr (!COLS) {
      const int offset = stage * STAGE_BYTES + tile * 4096;
      return read_chunk(lds + base[offset >> 16][ks] + (offset & 0xffff));
    } else if constexpr (ES == 4) {
      u32x4 fragment;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int offset = stage * STAGE_BYTES + (8 * ks + j) * ROWS * 4;
        fragment[j] = read_word(lds + base[offset >> 16][tile] + (offset & 0xffff));
      }
      return fragment;
    } else {
      const int low = stage * STAGE_BYTES + 16 * ks * ROWS * 2;
      const int high = low + 4 * ROWS * 2;
      const u32x2 first = read_transposed(lds + base[low >> 16][tile] + (low & 0xffff));
      const u32x2 second = read_transposed(lds + base[high >> 16][tile] + (high & 0xffff));
      return u32x4{first[0], first[1], second[0], second[1]};
    }
  }
};

// ------------------------------------------------------------------ tiles of a launch
// Tile t of all matrices' tiles, in blocks of GROUP tile rows walked column by column, so that neighbouring tiles
// share the slabs of a few rows and columns.
struct ProductTile {
  uint32_t m;       // tile row
  uint32_t n;       // tile column
  uint32_t matrix;  // of the batch
};

// (32-bit divisions throughout: a 64-bit one is some hundred instructions, and a small product's workgroups spend as
// long finding their tile as multiplying it.)
template <int GROUP>
__device__ __forceinline__ ProductTile product_tile(const ProductArgs &a, uint32_t t) {
  const uint32_t rows = static_cast<uint32_t>(a.tile_rows);
  const uint32_t cols = static_cast<uint32_t>(a.tile_cols);
  const uint32_t tiles = a.symmetric ? rows * (rows + 1) / 2 : rows * cols;
  ProductTile found;
  found.matrix = a.batch == 1 ? 0 : t / tiles;
  const uint32_t within = t - found.matrix * tiles;
  if (a.symmetric) {
    uint32_t i = static_cast<uint32_t>((sqrtf(8.0f * static_cast<float>(within) + 1.0f) - 1.0f) * 0.5f);
    while (i * (i + 1) / 2 > within) {
      --i;
    }
    while ((i + 1) * (i + 2) / 2 <= within) {
      ++i;
    }
    found.m = i;
    found.n = within - i * (i + 1) / 2;
  } else {
    const uint32_t block = within / (GROUP * cols);
    const uint32_t in_block = within - block * GROUP * cols;
    const uint32_t height = rows - block * GROUP < GROUP ? rows - block * GROUP : GROUP;
    found.n = in_block / height;
    found.m = block * GROUP + in_block - found.n * height;
  }
  return found;
}

// Workgroups go to the 8 XCDs round robin by their number; XCD c takes one run of consecutive places among `count`,
// so that the tiles it works on together meet in its L2.
__device__ __forceinline__ uint32_t place_of(uint32_t number, uint32_t count) {
  const uint32_t xcd = number % 8;
  const uint32_t more = count % 8;
  return xcd * (count / 8) + (xcd < more ? xcd : more) + number / 8;
}

// The split tiles' slabs, all in one row, are shared out evenly: worker q takes [split_begin(q), split_begin(q + 1)),
// `share` slabs, the first `longer` workers one more.
__device__ __forceinline__ uint32_t split_begin(const ProductArgs &a, uint32_t q) {
  const uint32_t longer = static_cast<uint32_t>(a.longer);
  return q * static_cast<uint32_t>(a.share) + (q < longer ? q : longer);
}
// The worker that holds slab x.
__device__ __forceinline__ uint32_t split_worker(const ProductArgs &a, uint32_t x) {
  const uint32_t share = static_cast<uint32_t>(a.share);
  const uint32_t longer = static_cast<uint32_t>(a.longer);
  const uint32_t behind = longer * (share + 1);
  return x < behind ? x / (share + 1) : longer + (x - behind) / share;
}
template <int TILE>
constexpr int kTileGroup = TILE == 256 ? 4 : 8;

// ------------------------------------------------------------------ tile
// TILE x TILE tiles, WAVES_M x WAVES_N waves of 32x32 accumulators.  STAGES slabs of both operands live in LDS:
// while one is multiplied the loads of the next are in flight.  With eight waves only four load (a wave that
// issues loads stalls, and its SIMD's other wave keeps the matrix pipe busy).  The slab schedule is that of the
// projections' tile kernel: fragments are read one k step ahead of their MFMAs from two register sets, and the
// barrier sits where the slab's last fragments have been read.
template <int TILE, int STAGES>
constexpr int kStageBytes = 2 * STAGES * TILE * 128;
// Waves of a SIMD that the registers have to leave room for.
template <int TILE, int STAGES>
constexpr int kProductWaves = TILE == 32 ? 4 : TILE == 64 ? 3 : TILE == 128 && STAGES > 2 ? 1 : 2;
template <int TILE, int WAVES_M, int WAVES_N>
constexpr int kProductThreads = TILE == 32 ? 256 : 64 * WAVES_M * WAVES_N;

// Workgroup `block` of a product's.  MAY_SPLIT: tiles behind the whole ones may be shared by workers.
template <class P, int TILE, int WAVES_M, int WAVES_N, int STAGES, bool A_COLS, bool B_COLS, ProductEpilogue EPI, bool MAY_SPLIT>
__device__ __forceinline__ void product_body(const ProductArgs &a, uint32_t block, unsigned char *lds) {
  constexpr int ES = kElementBytes<P>;
  constexpr int BK = 128 / ES;
  // 32 x 32 tiles: the four waves take one k step of every slab each and add their sums in the epilogue.
  constexpr bool SPREAD = TILE == 32;
  constexpr int WAVES = SPREAD ? 4 : WAVES_M * WAVES_N;
  constexpr int STEPS = SPREAD ? 1 : 4;  // k steps of a slab that a wave multiplies
  constexpr int WTM = TILE / WAVES_M;
  constexpr int WTN = TILE / WAVES_N;
  constexpr int MT = WTM / 32;
  constexpr int NT = WTN / 32;
  constexpr int STAGE = TILE * 128;
  constexpr int REGION = STAGES * STAGE;
  constexpr int LOAD_WAVES = WAVES == 8 ? 4 : WAVES;
  using ALoads = OperandLoads<P, TILE, A_COLS, LOAD_WAVES>;
  using BLoads = OperandLoads<P, TILE, B_COLS, LOAD_WAVES>;
  constexpr int LOADS = ALoads::LOADS + BLoads::LOADS;
  static_assert(LOADS * (STAGES - 1) < 64, "in-flight loads must fit the vmcnt counter");
  static_assert(2 * REGION <= 160 * 1024, "stages must fit the CU's LDS");
  constexpr int PITCH = WTN + 4;  // floats of a staged row of the epilogue
  static_assert(WAVES * 32 * PITCH * 4 <= 2 * REGION, "the epilogue's rows must fit the stages");

  static_assert(kStageBytes<TILE, STAGES> == 2 * REGION, "the kernel's LDS");
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int wm = SPREAD ? 0 : wave % WAVES_M;
  const int wn = SPREAD ? 0 : wave / WAVES_M;
  const bool loading_wave = wave < LOAD_WAVES;

  const uint32_t tile_slabs = static_cast<uint32_t>((a.k + BK - 1) / BK);
  // Whole tiles first, one a workgroup; then the workers of the split tiles, each with one run of their slabs, the end
  // of one tile and the begin of the next among them (the host gives a worker at least one slab).
  // (What a split saves 256 x 256 tiles goes into their pieces' 256 KB, and 32 x 32 tiles are many as they are.)
  constexpr bool SPLITS = MAY_SPLIT && (TILE == 128 || TILE == 64);
  const uint32_t whole = static_cast<uint32_t>(a.whole);
  const bool worker = SPLITS && block >= whole;
  // Where every tile has the same number of workers, those of one part of K come one after another: they share slabs.
  uint32_t q = worker ? place_of(block - whole, static_cast<uint32_t>(a.workers)) : 0;
  if (worker && a.each > 1) {
    const uint32_t part = q / static_cast<uint32_t>(a.split);
    q = (q - part * static_cast<uint32_t>(a.split)) * static_cast<uint32_t>(a.each) + part;
  }
  uint32_t next = worker ? split_begin(a, q) : 0;
  const uint32_t stop = worker ? split_begin(a, q + 1) : tile_slabs;
  do {
    // Opaque, here and before the epilogue: what follows from it is computed where it is used, not kept in registers
    // around the loop (two workgroups of 128 x 128 no longer fit a CU then).
    int lane = threadIdx.x & 63;
    __asm__ volatile("" : "+v"(lane));
    OperandFragments<P, TILE, A_COLS, MT, STAGES> a_fragments;
    OperandFragments<P, TILE, B_COLS, NT, STAGES> b_fragments;
    a_fragments.setup(0, wm * MT, SPREAD ? wave : 0, lane);
    b_fragments.setup(REGION, wn * NT, SPREAD ? wave : 0, lane);
    const lds_bytes_t shared = (lds_bytes_t)lds;
    const uint32_t local = worker ? next / tile_slabs : 0;  // among the split tiles
    const ProductTile at = product_tile<kTileGroup<TILE>>(a, worker ? whole + local : place_of(block, whole));
    const uint32_t first_slab = next - local * tile_slabs;
    const int slabs = static_cast<int>(tile_slabs - first_slab < stop - next ? tile_slabs - first_slab : stop - next);
    next += static_cast<uint32_t>(slabs);
    const int64_t m0 = static_cast<int64_t>(at.m) * TILE;
    const int64_t n0 = static_cast<int64_t>(at.n) * TILE;
    const int64_t k_begin = static_cast<int64_t>(first_slab) * BK;
    const int64_t k_end = a.k - k_begin < static_cast<int64_t>(slabs) * BK ? a.k : k_begin + static_cast<int64_t>(slabs) * BK;
    ALoads a_loads;
    BLoads b_loads;
    a_loads.setup(static_cast<const unsigned char *>(a.a.data) + at.matrix * a.a.batch * ES, a.a.ld, m0, a.m - m0, wave, lane);
    b_loads.setup(static_cast<const unsigned char *>(a.b.data) + at.matrix * a.b.batch * ES, a.b.ld, n0, a.n - n0, wave, lane,
                EPI == ProductEpilogue::kActivate ? a.halves : 0);
    const uint32_t lds_begin = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>((uintptr_t)shared)));
    auto issue = [&](int number, int stage) XP_INLINE {
      const int64_t k_pos = k_begin + static_cast<int64_t>(number) * BK;
      const typename ALoads::Slab a_slab = a_loads.slab(k_pos, k_end);
      const typename BLoads::Slab b_slab = b_loads.slab(k_pos, k_end);
#pragma unroll
      for (int q = 0; q < ALoads::LOADS; ++q) {
        a_loads.load(a_slab, q, lds_begin + stage * STAGE);
      }
#pragma unroll
      for (int q = 0; q < BLoads::LOADS; ++q) {
        b_loads.load(b_slab, q, lds_begin + REGION + stage * STAGE);
      }
    };

    f32x16 acc[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          acc[mt][nt][r] = 0.0f;
        }
      }
    }
    // Wave tiles of up to four accumulators hold a whole slab's fragments twice: their few MFMAs a k step are shorter than
    // the LDS latency, so the next slab's are all read under this slab's MFMAs.  Larger ones read one k step ahead.
    constexpr bool WHOLE_SLABS = MT * NT == 1 || (MT * NT == 4 && STAGES > 2);
    u32x4 af[WHOLE_SLABS ? 2 * STEPS : 2][MT];
    u32x4 bf[WHOLE_SLABS ? 2 * STEPS : 2][NT];
    auto read_fragments = [&](int stage, int ks, int slot) XP_INLINE {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        af[slot][mt] = a_fragments.read(shared, stage, ks, mt);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        bf[slot][nt] = b_fragments.read(shared, stage, ks, nt);
      }
    };
    auto multiply = [&](int slot) XP_INLINE {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          acc[mt][nt] = P::mfma32(bf[slot][nt], af[slot][mt], acc[mt][nt]);
        }
      }
    };
    // Each wave waits for its loads of the next slab and for its own LDS reads; past the barrier every wave may
    // read the next slab and the stage just read may be refilled.
    auto stage_barrier = []() XP_INLINE {
      constexpr int N = LOADS * (STAGES - 2);
      __builtin_amdgcn_s_waitcnt((N & 0xf) | ((N >> 4) << 14) | (0x7 << 4));  // vmcnt(N) lgkmcnt(0)
      __builtin_amdgcn_sched_barrier(0);
      __asm__ volatile("s_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };

    if (loading_wave) {
#pragma unroll
      for (int s = 0; s < STAGES; ++s) {
        issue(s, s);
      }
    }
    wait_vmcnt<LOADS * (STAGES - 1)>();
    __syncthreads();
    auto read_slab = [&](int stage, int set) XP_INLINE {
#pragma unroll
      for (int ks = 0; ks < STEPS; ++ks) {
        read_fragments(stage, ks, set * STEPS + ks);
      }
    };
    auto multiply_slab = [&](int set) XP_INLINE {
#pragma unroll
      for (int ks = 0; ks < STEPS; ++ks) {
        multiply(set * STEPS + ks);
      }
    };
    if constexpr (WHOLE_SLABS) {
      read_slab(0, 0);
    } else {
      read_fragments(0, 0, 0);
    }

    constexpr int UNROLL = WHOLE_SLABS && STAGES % 2 != 0 ? 2 * STAGES : STAGES;
    auto slab = [&](auto index, auto loads, int number) XP_INLINE {
      constexpr int S = decltype(index)::value % STAGES;
      constexpr int NEXT = (S + 1) % STAGES;
      constexpr bool LOADING = decltype(loads)::value;
      if constexpr (WHOLE_SLABS) {
        constexpr int SET = decltype(index)::value % 2;
        stage_barrier();
        if constexpr (LOADING) {
          issue(number + STAGES, S);
        }
        read_slab(NEXT, 1 - SET);
        multiply_slab(SET);
        __builtin_amdgcn_sched_barrier(0);
        return;
      }
      read_fragments(S, 1, 1);
      multiply(0);
      __builtin_amdgcn_sched_barrier(0);
      read_fragments(S, 2, 0);
      multiply(1);
      __builtin_amdgcn_sched_barrier(0);
      read_fragments(S, 3, 1);
      multiply(0);
      stage_barrier();
      read_fragments(NEXT, 0, 0);
      if constexpr (LOADING) {
        issue(number + STAGES, S);
      }
      multiply(1);
      __builtin_amdgcn_sched_barrier(0);
    };
    int number = 0;
    auto main_loop = [&](auto loads) XP_INLINE {
      for (; number + UNROLL < slabs; number += UNROLL) {
        static_for<UNROLL>([&](auto j) XP_INLINE { slab(j, loads, number + decltype(j)::value); });
      }
      static_for<UNROLL - 1>([&](auto j) XP_INLINE {
        if (number + decltype(j)::value + 1 < slabs) {
          slab(j, loads, number + decltype(j)::value);
        }
      });
    };
    if constexpr (LOAD_WAVES == WAVES) {
      main_loop(std::true_type{});
    } else if (loading_wave) {
      main_loop(std::true_type{});
    } else {
      main_loop(std::false_type{});
    }
    static_for<UNROLL>([&](auto j) XP_INLINE {
      if ((slabs - 1) % UNROLL == decltype(j)::value) {
        if constexpr (WHOLE_SLABS) {
          multiply_slab(decltype(j)::value % 2);
        } else {
          constexpr int S = decltype(j)::value % STAGES;
          read_fragments(S, 1, 1);
          multiply(0);
          read_fragments(S, 2, 0);
          multiply(1);
          read_fragments(S, 3, 1);
          multiply(0);
          multiply(1);
        }
      }
    });
    // Refills past the end may still be landing in the stages that the epilogue reuses, and other waves reading.
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    __asm__ volatile("" : "+v"(lane));

    // 32 rows at a time go through a part of LDS of the wave's own, so that a lane then holds CHUNK neighbouring
    // columns of a row: whole 16-byte loads and stores, 128 contiguous bytes and more of each row.
    constexpr int CHUNK = EPI == ProductEpilogue::kGradient ? 4 : 8;
    constexpr int LANES = WTN / CHUNK;    // per row
    constexpr int ROWS_PER_PASS = 64 / LANES;
    float *rows = reinterpret_cast<float *>(lds) + wave * 32 * PITCH;
    const int64_t row0 = m0 + wm * WTM;
    const int64_t col0 = n0 + wn * WTN;
    // A worker's sums go to its piece of the tile, [TILE, TILE]: piece q + local, counted along the split tiles' slabs.
    float *partial = worker ? a.partials + static_cast<int64_t>(q + local) * (TILE * TILE) + (wm * WTM) * TILE + wn * WTN : nullptr;
    const bool mirrored = a.symmetric != 0 && at.m != at.n;
    const int chunk = lane % LANES;
    const int64_t col = col0 + chunk * CHUNK;
    if constexpr (SPREAD) {
      // The waves' sums side by side in LDS; each wave then finishes eight of the rows.
      const float *all = reinterpret_cast<const float *>(lds);
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const f32x4 four = {acc[0][0][4 * q4], acc[0][0][4 * q4 + 1], acc[0][0][4 * q4 + 2], acc[0][0][4 * q4 + 3]};
        *reinterpret_cast<f32x4 *>(rows + (lane & 31) * PITCH + 8 * q4 + 4 * (lane >> 5)) = four;
      }
      __syncthreads();
      const auto total = [&](int row, int column) __attribute__((always_inline)) {
        const float *from = all + row * PITCH + column;
        return (from[0] + from[32 * PITCH]) + (from[64 * PITCH] + from[96 * PITCH]);
      };
      [[maybe_unused]] float sums[8] = {};
      const int row = wave * 8 + lane / LANES;
      if (lane / LANES < 8 && row0 + row < a.m && col < a.n) {
        const ChunkPlace there = chunk_place<EPI>(a, at.matrix, row0 + row, col);
        Beside<P, EPI> beside;
        request<P, EPI>(a, there, col, beside);
        float value[CHUNK];
#pragma unroll
        for (int j = 0; j < CHUNK; ++j) {
          value[j] = total(row, chunk * CHUNK + j);
        }
        if constexpr (EPI == ProductEpilogue::kGradient) {
          finish_gradient<P>(a, there, col, beside, value, sums);
        } else {
          finish<P, EPI>(a, there, col, beside, value);
        }
      }
      if constexpr (EPI == ProductEpilogue::kStore) {
        const int64_t to_row = col0 + (threadIdx.x & 31);
        const int64_t to_col = row0 + (threadIdx.x >> 5) * 8;
        if (mirrored && threadIdx.x < 128 && to_row < a.n && to_col < a.m) {
          float value[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            value[j] = total(static_cast<int>(threadIdx.x >> 5) * 8 + j, static_cast<int>(threadIdx.x & 31));
          }
          const ChunkPlace across = chunk_place<EPI>(a, at.matrix, to_row, to_col);
          Beside<P, EPI> beside;
          request<P, EPI>(a, across, to_col, beside);
          finish<P, EPI>(a, across, to_col, beside, value);
        }
      }
      if constexpr (EPI == ProductEpilogue::kGradient) {
        if (a.column_sums != nullptr) {
          __syncthreads();
          float *bands = reinterpret_cast<float *>(lds);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            bands[wave * 512 + j * 64 + lane] = sums[j];
          }
          __syncthreads();
          if (wave == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int in = j * 64 + lane;
              sums[j] = (bands[in] + bands[512 + in]) + (bands[1024 + in] + bands[1536 + in]);
            }
            store_column_sums<LANES>(a, row0 / 32, col, sums, lane);
          }
        }
      }
      return;
    }
    ChunkPlace place = chunk_place<EPI>(a, at.matrix, row0 + lane / LANES, col);
    constexpr int PASSES = 32 / ROWS_PER_PASS;
    constexpr int AHEAD = EPI == ProductEpilogue::kGradient ? PASSES : PASSES < 2 ? PASSES : 2;  // passes whose loads are in flight
    Beside<P, EPI> beside[AHEAD];
    // One copy of this code for all blocks: it runs once a tile, and straight-line code of several times the size took
    // longer to fetch than to run (10 us a tile at 256 x 256).
#pragma unroll 1
    for (int mt = 0; mt < MT; ++mt) {
      if (row0 + mt * 32 >= a.m) {
        break;
      }
      [[maybe_unused]] float sums[8] = {};
      ChunkPlace there = place;
      auto request_pass = [&](int pass) XP_INLINE {
        if (partial == nullptr && row0 + mt * 32 + pass * ROWS_PER_PASS + lane / LANES < a.m && col < a.n) {
          request<P, EPI>(a, there, col, beside[pass % AHEAD]);
        }
        there.base += ROWS_PER_PASS * a.ld_base;
        there.extra += ROWS_PER_PASS * a.ld_extra;
      };
#pragma unroll
      for (int pass = 0; pass < AHEAD; ++pass) {
        request_pass(pass);
      }
      __builtin_amdgcn_wave_barrier();
      static_for<MT>([&](auto block) XP_INLINE {
        constexpr int B = decltype(block)::value;
        if (__builtin_amdgcn_readfirstlane(mt) == B) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const f32x4 four = {acc[B][nt][4 * q], acc[B][nt][4 * q + 1], acc[B][nt][4 * q + 2], acc[B][nt][4 * q + 3]};
              *reinterpret_cast<f32x4 *>(rows + (lane & 31) * PITCH + nt * 32 + 8 * q + 4 * (lane >> 5)) = four;
            }
          }
        }
      });
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int pass = 0; pass < PASSES; ++pass) {
        const int row = pass * ROWS_PER_PASS + lane / LANES;
        const int64_t to_row = row0 + mt * 32 + row;
        if (to_row < a.m && col < a.n) {
          float value[CHUNK];
#pragma unroll
          for (int part = 0; part < CHUNK / 4; ++part) {
            const f32x4 four = *reinterpret_cast<const f32x4 *>(rows + row * PITCH + chunk * CHUNK + part * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              value[part * 4 + j] = four[j];
            }
          }
          if (partial != nullptr) {
            __builtin_memcpy(__builtin_assume_aligned(partial + (mt * 32 + row) * TILE + chunk * CHUNK, 16), value, CHUNK * 4);
          } else if constexpr (EPI == ProductEpilogue::kGradient) {
            finish_gradient<P>(a, place, col, beside[pass % AHEAD], value, sums);
          } else {
            finish<P, EPI>(a, place, col, beside[pass % AHEAD], value);
          }
        }
        if (pass + AHEAD < PASSES) {
          request_pass(pass + AHEAD);
        }
        place.out += ROWS_PER_PASS * a.ld_out;
        place.base += ROWS_PER_PASS * a.ld_base;
        place.extra += ROWS_PER_PASS * a.ld_extra;
      }
      if constexpr (EPI == ProductEpilogue::kStore) {
        if (mirrored && partial == nullptr) {
          // The tile's transpose: eight rows of a column are eight neighbouring columns there.
          for (int pass = 0; pass < WTN * 4 / 64; ++pass) {
            const int column = (pass * 64 + lane) % WTN;
            const int group = (pass * 64 + lane) / WTN;
            const int64_t to_row = col0 + column;
            const int64_t to_col = row0 + mt * 32 + group * 8;
            if (to_row < a.n && to_col < a.m) {
              float value[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                value[j] = rows[(group * 8 + j) * PITCH + column];
              }
              const ChunkPlace across = chunk_place<EPI>(a, at.matrix, to_row, to_col);
              Beside<P, EPI> beside_it;
              request<P, EPI>(a, across, to_col, beside_it);
              finish<P, EPI>(a, across, to_col, beside_it, value);
            }
          }
        }
      }
      if constexpr (EPI == ProductEpilogue::kGradient) {
        if (partial == nullptr && a.column_sums != nullptr) {
          store_column_sums<LANES>(a, (row0 + mt * 32) / 32, col, sums, lane);
        }
      }
    }
    if constexpr (SPLITS) {
      __syncthreads();  // the next tile's loads land where the waves staged their rows
    }
  } while (SPLITS && next < stop);
}

template <class P, int TILE, int WAVES_M, int WAVES_N, int STAGES, bool A_COLS, bool B_COLS, ProductEpilogue EPI>
__global__ __launch_bounds__((kProductThreads<TILE, WAVES_M, WAVES_N>), (kProductWaves<TILE, STAGES>)) void product_kernel(ProductArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[kStageBytes<TILE, STAGES>];
  product_body<P, TILE, WAVES_M, WAVES_N, STAGES, A_COLS, B_COLS, EPI, true>(a, blockIdx.x, lds);
}

// Up to three products of one backward pass in one launch, whole tiles: their last rounds, which each by itself would leave
// most CUs idle in, are one.  The first (of an empty grid where there is none) is an inputs' gradient, the others
// weights' gradients.
template <class P, int TILE, int WAVES_M, int WAVES_N, int STAGES>
__global__ __launch_bounds__((kProductThreads<TILE, WAVES_M, WAVES_N>), (kProductWaves<TILE, STAGES>)) void product_group_kernel(ProductGroup g) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[kStageBytes<TILE, STAGES>];
  uint32_t block = blockIdx.x;
  if (block < static_cast<uint32_t>(g.blocks[0])) {
    product_body<P, TILE, WAVES_M, WAVES_N, STAGES, false, true, ProductEpilogue::kStore, false>(g.part[0], block, lds);
    return;
  }
  block -= static_cast<uint32_t>(g.blocks[0]);
  const int at = block < static_cast<uint32_t>(g.blocks[1]) ? 1 : 2;
  block -= at == 2 ? static_cast<uint32_t>(g.blocks[1]) : 0u;
  product_body<P, TILE, WAVES_M, WAVES_N, STAGES, true, true, ProductEpilogue::kStore, false>(g.part[at], block, lds);
}

// ------------------------------------------------------------------ split tiles
// The sum of a split tile's pieces in the order of their slabs, then the epilogue.  A workgroup takes 32 rows of 64
// columns, with the loads of four pieces in flight; the column sums of its band are added through LDS in wave order.
// Bound by the latency of its launch and loads: 6 to 8 us for 16 to 64 tiles of 128 x 128.
template <class P, int TILE, ProductEpilogue EPI>
__global__ __launch_bounds__(256) void product_join_kernel(ProductArgs a) {
  constexpr int CHUNK = EPI == ProductEpilogue::kGradient ? 4 : 8;
  constexpr int LANES = 64 / CHUNK;
  constexpr int ROWS_PER_PASS = 64 / LANES;
  constexpr int BLOCKS = TILE / 64 * (TILE / 32);  // of a tile
  constexpr int PITCH = 64 + 1;
  __shared__ float staged[EPI == ProductEpilogue::kStore ? 32 * PITCH : 4 * 64 * 8];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const uint32_t local = blockIdx.x / BLOCKS;
  const int block = static_cast<int>(blockIdx.x % BLOCKS);
  const int row_in = block / (TILE / 64) * 32;
  const int col_in = block % (TILE / 64) * 64;
  const ProductTile at = product_tile<kTileGroup<TILE>>(a, static_cast<uint32_t>(a.whole) + local);
  const int64_t row0 = static_cast<int64_t>(at.m) * TILE + row_in;
  const int64_t col0 = static_cast<int64_t>(at.n) * TILE + col_in;
  if (row0 >= a.m || col0 >= a.n) {
    return;
  }
  const uint32_t tile_slabs = static_cast<uint32_t>((a.k + 128 / kElementBytes<P> - 1) / (128 / kElementBytes<P>));
  const uint32_t first = split_worker(a, local * tile_slabs);
  const uint32_t last = split_worker(a, (local + 1) * tile_slabs - 1);
  const int64_t col = col0 + (lane % LANES) * CHUNK;
  const bool mirrored = a.symmetric != 0 && at.m != at.n;
  [[maybe_unused]] float sums[8] = {};
  for (int pass = 0; pass < 8 / ROWS_PER_PASS; ++pass) {
    const int row_at = wave * 8 + pass * ROWS_PER_PASS + lane / LANES;
    const int64_t row = row0 + row_at;
    const bool live = row < a.m && col < a.n;
    float value[CHUNK] = {};
    if (live) {
      const ChunkPlace place = chunk_place<EPI>(a, at.matrix, row, col);
      Beside<P, EPI> beside;
      request<P, EPI>(a, place, col, beside);
      const float *from = a.partials + static_cast<int64_t>(first + local) * (TILE * TILE) + (row_in + row_at) * TILE + col_in + (lane % LANES) * CHUNK;
      __builtin_memcpy(value, __builtin_assume_aligned(from, 16), CHUNK * 4);
      uint32_t more = last - first;
      for (; more >= 4; more -= 4) {
        float pieces[4][CHUNK];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          from += TILE * TILE;
          __builtin_memcpy(pieces[i], __builtin_assume_aligned(from, 16), CHUNK * 4);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int j = 0; j < CHUNK; ++j) {
            value[j] += pieces[i][j];
          }
        }
      }
      for (; more > 0; --more) {
        float piece[CHUNK];
        from += TILE * TILE;
        __builtin_memcpy(piece, __builtin_assume_aligned(from, 16), CHUNK * 4);
#pragma unroll
        for (int j = 0; j < CHUNK; ++j) {
          value[j] += piece[j];
        }
      }
      if constexpr (EPI == ProductEpilogue::kStore) {
        if (mirrored) {
#pragma unroll
          for (int j = 0; j < CHUNK; ++j) {
            staged[row_at * PITCH + (lane % LANES) * CHUNK + j] = value[j];
          }
        }
      }
      if constexpr (EPI == ProductEpilogue::kGradient) {
        finish_gradient<P>(a, place, col, beside, value, sums);
      } else {
        finish<P, EPI>(a, place, col, beside, value);
      }
    }
  }
  if constexpr (EPI == ProductEpilogue::kStore) {
    if (mirrored) {
      // The block's transpose, one chunk of eight a thread.  (Chunks past the operand's end are not stored.)
      __syncthreads();
      const int column = threadIdx.x & 63;
      const int group = threadIdx.x >> 6;
      const int64_t to_row = col0 + column;
      const int64_t to_col = row0 + group * 8;
      if (to_row < a.n && to_col < a.m) {
        float value[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          value[j] = to_col + j < a.m ? staged[(group * 8 + j) * PITCH + column] : 0.0f;
        }
        const ChunkPlace across = chunk_place<EPI>(a, at.matrix, to_row, to_col);
        Beside<P, EPI> beside;
        request<P, EPI>(a, across, to_col, beside);
        finish<P, EPI>(a, across, to_col, beside, value);
      }
    }
  }
  if constexpr (EPI == ProductEpilogue::kGradient) {
    if (a.column_sums != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        staged[wave * 512 + j * 64 + lane] = sums[j];
      }
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int at_lane = j * 64 + lane;
          sums[j] = (staged[at_lane] + staged[512 + at_lane]) + (staged[1024 + at_lane] + staged[1536 + at_lane]);
        }
        store_column_sums<LANES>(a, row0 / 32, col, sums, lane);
      }
    }
  }
}

}  // namespace

// ------------------------------------------------------------------ tables
template <class P, int TILE, int WAVES_M, int WAVES_N, int STAGES>
const void *product_tile_kernel(ProductEpilogue epilogue, bool a_cols, bool b_cols) {
  switch (epilogue) {
    case ProductEpilogue::kActivate:
      return reinterpret_cast<const void *>(
          &product_kernel<P, TILE, WAVES_M, WAVES_N, STAGES, false, false, ProductEpilogue::kActivate>);
    case ProductEpilogue::kGradient:
      return reinterpret_cast<const void *>(
          &product_kernel<P, TILE, WAVES_M, WAVES_N, STAGES, false, true, ProductEpilogue::kGradient>);
    default:
      return a_cols   ? reinterpret_cast<const void *>(
                          &product_kernel<P, TILE, WAVES_M, WAVES_N, STAGES, true, true, ProductEpilogue::kStore>)
             : b_cols ? reinterpret_cast<const void *>(
                            &product_kernel<P, TILE, WAVES_M, WAVES_N, STAGES, false, true, ProductEpilogue::kStore>)
                      : reinterpret_cast<const void *>(
                            &product_kernel<P, TILE, WAVES_M, WAVES_N, STAGES, false, false, ProductEpilogue::kStore>);
  }
}

template <class P, int TILE>
const void *product_join_for(ProductEpilogue epilogue) {
  switch (epilogue) {
    case ProductEpilogue::kActivate:
      return reinterpret_cast<const void *>(&product_join_kernel<P, TILE, ProductEpilogue::kActivate>);
    case ProductEpilogue::kGradient:
      return reinterpret_cast<const void *>(&product_join_kernel<P, TILE, ProductEpilogue::kGradient>);
    default:
      return reinterpret_cast<const void *>(&product_join_kernel<P, TILE, ProductEpilogue::kStore>);
  }
}

template <class P>
const void *ProductKernels<P>::main(ProductTiles tiles, ProductEpilogue epilogue, bool a_cols, bool b_cols) {
  if constexpr (kElementBytes<P> == 2) {  // fp32's matrix pipe is full with two 128 x 128 tiles on a CU
    if (tiles == ProductTiles::k256) {
      return product_tile_kernel<P, 256, 2, 4, 2>(epilogue, a_cols, b_cols);
    }
    if (tiles == ProductTiles::k128Deep) {
      return product_tile_kernel<P, 128, 2, 2, 4>(epilogue, a_cols, b_cols);
    }
  }
  switch (tiles) {
    case ProductTiles::k128Pairs:
      return product_tile_kernel<P, 128, 2, 2, 2>(epilogue, a_cols, b_cols);
    case ProductTiles::k64:
      return product_tile_kernel<P, 64, 2, 2, 3>(epilogue, a_cols, b_cols);
    default:
      return product_tile_kernel<P, 32, 1, 1, 4>(epilogue, a_cols, b_cols);
  }
}

template <class P>
const void *ProductKernels<P>::group(ProductTiles tiles) {
  return tiles == ProductTiles::k128Pairs ? reinterpret_cast<const void *>(&product_group_kernel<P, 128, 2, 2, 2>)
         : tiles == ProductTiles::k64     ? reinterpret_cast<const void *>(&product_group_kernel<P, 64, 2, 2, 3>)
                                          : reinterpret_cast<const void *>(&product_group_kernel<P, 32, 1, 1, 4>);
}

template <class P>
const void *ProductKernels<P>::join(int tile, ProductEpilogue epilogue) {
  return tile == 128 ? product_join_for<P, 128>(epilogue) : product_join_for<P, 64>(epilogue);
}

}  // namespace xp
