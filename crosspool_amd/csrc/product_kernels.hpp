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
#pragma once

#include "product.hpp"
#include "xp_elements.hpp"
#include "xp_tiles.hpp"

namespace xp {
namespace {

// ------------------------------------------------------------------ eight values of a row
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
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t bits = j % 2 == 0 ? chunk[j / 2] & 0xffffu : chunk[j / 2] >> 16;
    value[j] = dtype == kDtypeF16 ? F16Payload::widen(bits) : Bf16Payload::widen(bits);
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
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    packed[j] = dtype == kDtypeF16 ? F16Payload::pack2(value[2 * j], value[2 * j + 1])
                                   : Bf16Payload::pack2(value[2 * j], value[2 * j + 1]);
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

template <class P>
__device__ __forceinline__ void slope_of(float v, const ActivationArgs &act, float &value, float &slope) {
  constexpr bool PRECISE = kElementBytes<P> == 4;
  switch (act.function) {
    case kActivationRelu:
      value_and_slope<Slope::Relu, PRECISE>(v, act.alpha, value, slope);
      break;
    case kActivationGelu:
      if (act.approximate_tanh) {
        value_and_slope<Slope::GeluTanh, PRECISE>(v, act.alpha, value, slope);
      } else {
        value_and_slope<Slope::GeluErf, PRECISE>(v, act.alpha, value, slope);
      }
      break;
    default:
      value_and_slope<Slope::Silu, PRECISE>(v, act.alpha, value, slope);
      break;
  }
}

// The epilogue of columns col .. col + 7 (those below n) of one row.  `sums` gathers kGradient's gradients by
// column: [0, 8) of Gate (or of ungated values), [8, 16) of Up.
template <class P, ProductEpilogue EPI>
__device__ __forceinline__ void finish(const ProductArgs &a, int64_t matrix, int64_t row, int64_t col, float (&value)[8],
                                       float (&sums)[16]) {
  constexpr int dtype = kDtypeOf<P>;
  const int count = a.n - col < 8 ? static_cast<int>(a.n - col) : 8;
  if constexpr (EPI == ProductEpilogue::kStore) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      value[j] *= a.alpha;
    }
    if (a.beta != 0.0f) {
      float other[8];
      load_values(a.base, matrix * a.batch_base + row * a.ld_base + col, a.base_dtype, count, other);
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
      load_values(a.extra, matrix * a.batch_extra + row * a.ld_extra + col, a.extra_dtype, count, other);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        value[j] = a.keep * other[j] - a.step * value[j];
      }
    }
    store_values(a.out, matrix * a.batch_out + row * a.ld_out + col, a.out_dtype, a.padded_out ? 8 : count, value);
  } else if constexpr (EPI == ProductEpilogue::kActivate) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      value[j] += a.bias != nullptr && j < count ? a.bias[col + j] : 0.0f;
    }
    store_values(a.out, row * a.ld_out + col, dtype, count, value);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      value[j] = round_to(value[j], dtype);
    }
    if (a.act.gated) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        value[j] = apply_gated(value[2 * j], value[2 * j + 1], a.act);
      }
      // n is even: a pair is whole or absent.
      store_values(a.extra, row * a.ld_extra + col / 2, dtype, count / 2, value);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        value[j] = apply_function(value[j], a.act);
      }
      store_values(a.extra, row * a.ld_extra + col, dtype, count, value);
    }
  } else {
    if (!a.act.gated) {
      float input[8];
      load_values(a.base, row * a.ld_base + col, dtype, count, input);
      float activated[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float slope;
        slope_of<P>(input[j], a.act, activated[j], slope);
        value[j] *= slope;
        sums[j] += value[j];
      }
      store_values(a.extra, row * a.ld_extra + col, dtype, count, activated);
      store_values(a.out, row * a.ld_out + col, dtype, count, value);
      return;
    }
    float first[8];   // interleaved: the first four pairs; else Gate
    float second[8] = {};  // the other four pairs; Up
    const bool pairs = a.interleaved != 0;
    const int64_t gate_at = row * a.ld_base + (pairs ? 2 * col : col);
    const int64_t up_at = gate_at + (pairs ? 8 : a.n);
    const int gate_count = pairs ? (count >= 4 ? 8 : 2 * count) : count;
    const int up_count = pairs ? 2 * count - gate_count : count;
    load_values(a.base, gate_at, dtype, gate_count, first);
    if (up_count > 0) {
      load_values(a.base, up_at, dtype, up_count, second);
    }
    float activated[8];
    float grad_ups[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float gate = pairs ? (j < 4 ? first[(2 * j) & 7] : second[(2 * j) & 7]) : first[j];
      const float up = pairs ? (j < 4 ? first[(2 * j + 1) & 7] : second[(2 * j + 1) & 7]) : second[j];
      float clipped = gate;
      float factor = up;
      bool gate_on = true;
      bool up_on = true;
      if (a.act.has_limit) {
        clip_keep_nan(clipped, factor, a.act.limit);
        gate_on = !(gate > a.act.limit);
        up_on = !(fabsf(up) > a.act.limit);
      }
      float f;
      float slope;
      slope_of<P>(clipped, a.act, f, slope);
      factor += a.act.up_offset;
      activated[j] = f * factor;
      const float through = value[j];
      const float grad_gate = gate_on && j < count ? through * slope * factor : 0.0f;
      const float grad_up = up_on && j < count ? through * f : 0.0f;
      sums[j] += grad_gate;
      sums[8 + j] += grad_up;
      value[j] = grad_gate;
      grad_ups[j] = grad_up;
    }
    store_values(a.extra, row * a.ld_extra + col, dtype, count, activated);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int pair = j / 2;
      first[j] = pairs ? (j % 2 == 0 ? value[pair] : grad_ups[pair]) : value[j];
      second[j] = pairs ? (j % 2 == 0 ? value[4 + pair] : grad_ups[4 + pair]) : grad_ups[j];
    }
    const int64_t to = row * a.ld_out + (pairs ? 2 * col : col);
    store_values(a.out, to, dtype, gate_count, first);
    if (up_count > 0) {
      store_values(a.out, to + (pairs ? 8 : a.n), dtype, up_count, second);
    }
  }
}

// Column sums of a wave's band: lanes with one chunk (lane % LANES) hold parts of the same columns.
template <int LANES>
__device__ __forceinline__ void store_column_sums(const ProductArgs &a, int64_t band, int64_t col, float (&sums)[16], int lane) {
#pragma unroll
  for (int j = 0; j < 16; ++j) {
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
  for (int j = 0; j < 8; ++j) {
    if (col + j < a.n) {
      if (!a.act.gated) {
        to[col + j] = sums[j];
      } else if (a.interleaved) {
        to[2 * (col + j)] = sums[j];
        to[2 * (col + j) + 1] = sums[8 + j];
      } else {
        to[col + j] = sums[j];
        to[a.n + col + j] = sums[8 + j];
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

// The loads of one operand's tile of ROWS rows (columns, for COLS) into the stages.
template <class P, int ROWS, bool COLS, int LOAD_WAVES>
struct OperandLoads {
  static constexpr int ES = kElementBytes<P>;
  static constexpr int BK = 128 / ES;
  static constexpr int LOADS = ROWS / 8 / LOAD_WAVES;    // 1 KB load instructions per loading wave and slab
  static constexpr int LANES_PER_ROW = COLS ? ROWS * ES / 16 : 8;  // 16-byte chunks of one LDS row
  static constexpr int ROWS_PER_LOAD = 64 / LANES_PER_ROW;
  static_assert(ROWS % (8 * LOAD_WAVES) == 0, "stage rows must split evenly");
  static_assert(!COLS || LANES_PER_ROW <= 64, "a load covers whole rows");

  const unsigned char *origin;  // the tile's first row (COLS: first column of reduction row 0)
  uint32_t ld_bytes;
  uint32_t span;                // bytes of the rows that a resource covers
  uint32_t lane_offset[2];
  int first;                    // this wave's first load of a slab

  // `rows` counts what is left of the operand from the tile's first row (column).
  __device__ __forceinline__ void setup(const void *data, int64_t ld, int64_t tile_first, int64_t rows_left, int wave, int lane) {
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
      origin = static_cast<const unsigned char *>(data) + tile_first * ld * ES;
      span = static_cast<uint32_t>(rows_left < ROWS ? rows_left : ROWS) * ld_bytes;
      // Eight rows a load: swizzle(8 g + row) = (row / 2) ^ (4 if g is odd).
      lane_offset[0] = static_cast<uint32_t>(place ^ (row >> 1));
      lane_offset[1] = lane_offset[0] ^ 4;
    }
  }

  // COLS: what the chunk index of reduction row k is xor-ed with; k's low bits follow from the load's variant
  // and the lane's row in it.
  __device__ static __forceinline__ int scramble(int variant, int row) {
    if constexpr (ES == 4) {
      return variant << 3;                            // bit 2 of k
    } else if constexpr (ROWS >= 256) {
      return ((2 * variant + row) & 3) << 2;          // k % 4, two rows a load
    } else if constexpr (ROWS == 128) {
      return (row & 3) << 2;                          // four rows a load
    } else {
      return ((row >> 1) & 1) << 2;                   // two rows share a bank line
    }
  }
  // The variant of load q of a wave (its loads start at a multiple of LOADS).
  static constexpr int variant(int q) {
    if constexpr (!COLS) {
      return q & 1;
    } else if constexpr (ES == 4) {
      return ROWS >= 256 ? (q >> 2) & 1 : ROWS == 128 ? (q >> 1) & 1 : q & 1;
    } else {
      return ROWS >= 256 ? q & 1 : 0;
    }
  }

  // Slab at column k_pos of a range that ends at k_end into `stage`; a slab past the end loads zeros.
  __device__ __forceinline__ void issue(int64_t k_pos, int64_t k_end, unsigned char *stage) const {
    if constexpr (COLS) {
      const int64_t left = k_end - k_pos;
      const uint32_t rows = left <= 0 ? 0u : left < BK ? static_cast<uint32_t>(left) : static_cast<uint32_t>(BK);
      const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(origin + (left <= 0 ? 0 : k_pos * static_cast<int64_t>(ld_bytes)), rows * ld_bytes);
#pragma unroll
      for (int q = 0; q < LOADS; ++q) {
        const uint32_t rows_before = static_cast<uint32_t>((first + q) * ROWS_PER_LOAD);
        buffer_load_lds16(rsrc, stage + (first + q) * 1024, lane_offset[variant(q)] + rows_before * ld_bytes, 0);
      }
    } else {
      const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(origin, span);
      const uint32_t k_bytes = static_cast<uint32_t>(k_pos * ES);
      // A chunk that the range's end cuts holds zeros past it (the operands' rows are whole chunks).
      const int64_t chunks_left = (k_end - k_pos + 16 / ES - 1) / (16 / ES);
      const uint32_t row = static_cast<uint32_t>((threadIdx.x & 63) >> 3);
#pragma unroll
      for (int q = 0; q < LOADS; ++q) {
        const uint32_t chunk = lane_offset[variant(q)];
        const uint32_t offset = (static_cast<uint32_t>((first + q) * 8) + row) * ld_bytes + chunk * 16;
        buffer_load_lds16(rsrc, stage + (first + q) * 1024, static_cast<int64_t>(chunk) < chunks_left ? offset : kOutOfRange, k_bytes);
      }
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

  __device__ __forceinline__ void setup(int region, int first_tile, int lane) {
    const int half = lane >> 5;
#pragma unroll
    for (int i = 0; i < BASES; ++i) {
      int at;
      if constexpr (!COLS) {
        const int row = lane & 31;
        at = (first_tile * 32 + row) * 128 + (((i * 2 + half) ^ swizzle(row)) << 4);
      } else if constexpr (ES == 4) {
        const int tile = (first_tile + i) ^ half;  // bit 2 of the reduction row is the lane's half
        at = 4 * half * ROWS * 4 + tile * 128 + (lane & 31) * 4;
      } else {
        const int within = lane & 15;
        const int row = 8 * half + (within >> 2);
        const int tile = ROWS >= 128 ? (first_tile + i) ^ (within >> 2) : (first_tile + i) ^ ((within >> 3) & 1);
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
struct ProductTile {
  int64_t m;       // tile row
  int64_t n;       // tile column
  int64_t matrix;  // of the batch
  int64_t range;   // of K
};

// Workgroups go to the 8 XCDs round robin by their number; XCD c takes one run of consecutive tiles, and a run
// walks blocks of GROUP tile rows column by column, so that the tiles an XCD works on together share the slabs
// of a few rows and columns in its L2.
template <int GROUP>
__device__ __forceinline__ ProductTile product_tile(const ProductArgs &a, int tile) {
  const int64_t rows = (a.m + tile - 1) / tile;
  const int64_t cols = (a.n + tile - 1) / tile;
  const int64_t tiles = a.symmetric ? rows * (rows + 1) / 2 : rows * cols;
  const uint32_t all = gridDim.x;
  const uint32_t xcd = blockIdx.x % 8;
  const uint32_t run = all / 8;
  const uint32_t more = all % 8;
  const int64_t t = static_cast<int64_t>(xcd * run + (xcd < more ? xcd : more) + blockIdx.x / 8);
  ProductTile found;
  const int64_t z = t / tiles;
  const int64_t within = t - z * tiles;
  found.matrix = z / a.ranges;
  found.range = z - found.matrix * a.ranges;
  if (a.symmetric) {
    int64_t i = static_cast<int64_t>((sqrtf(8.0f * static_cast<float>(within) + 1.0f) - 1.0f) * 0.5f);
    while (i * (i + 1) / 2 > within) {
      --i;
    }
    while ((i + 1) * (i + 2) / 2 <= within) {
      ++i;
    }
    found.m = i;
    found.n = within - i * (i + 1) / 2;
  } else {
    const int64_t block = within / (GROUP * cols);
    const int64_t in_block = within - block * GROUP * cols;
    const int64_t height = rows - block * GROUP < GROUP ? rows - block * GROUP : GROUP;
    found.n = in_block / height;
    found.m = block * GROUP + in_block - found.n * height;
  }
  return found;
}

// ------------------------------------------------------------------ tile
// TILE x TILE tiles, WAVES_M x WAVES_N waves of 32x32 accumulators.  STAGES slabs of both operands live in LDS:
// while one is multiplied the loads of the next are in flight.  With eight waves only four load (a wave that
// issues loads stalls, and its SIMD's other wave keeps the matrix pipe busy).  The slab schedule is that of the
// projections' tile kernel: fragments are read one k step ahead of their MFMAs from two register sets, and the
// barrier sits where the slab's last fragments have been read.
template <class P, int TILE, int WAVES_M, int WAVES_N, int STAGES, bool A_COLS, bool B_COLS, ProductEpilogue EPI>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N) void product_kernel(ProductArgs a) {
  constexpr int ES = kElementBytes<P>;
  constexpr int BK = 128 / ES;
  constexpr int WAVES = WAVES_M * WAVES_N;
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

  __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * REGION];

  const ProductTile at = product_tile<(TILE == 256 ? 4 : 8)>(a, TILE);
  const int64_t m0 = at.m * TILE;
  const int64_t n0 = at.n * TILE;
  const int64_t k_begin = at.range * a.k_slice;
  const int64_t k_end = a.k - k_begin < a.k_slice ? a.k : k_begin + a.k_slice;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int wm = wave % WAVES_M;
  const int wn = wave / WAVES_M;
  const bool loading_wave = wave < LOAD_WAVES;

  ALoads a_loads;
  BLoads b_loads;
  a_loads.setup(static_cast<const unsigned char *>(a.a.data) + at.matrix * a.a.batch * ES, a.a.ld, m0, a.m - m0, wave, lane);
  b_loads.setup(static_cast<const unsigned char *>(a.b.data) + at.matrix * a.b.batch * ES, a.b.ld, n0, a.n - n0, wave, lane);
  OperandFragments<P, TILE, A_COLS, MT, STAGES> a_fragments;
  OperandFragments<P, TILE, B_COLS, NT, STAGES> b_fragments;
  a_fragments.setup(0, wm * MT, lane);
  b_fragments.setup(REGION, wn * NT, lane);
  const lds_bytes_t shared = (lds_bytes_t)lds;
  // The host makes no empty range: every workgroup runs at least one slab.
  const int64_t slabs = (k_end - k_begin + BK - 1) / BK;
  auto issue = [&](int64_t slab, int stage) XP_INLINE {
    a_loads.issue(k_begin + slab * BK, k_end, lds + stage * STAGE);
    b_loads.issue(k_begin + slab * BK, k_end, lds + REGION + stage * STAGE);
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
  u32x4 af[2][MT];
  u32x4 bf[2][NT];
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
  read_fragments(0, 0, 0);

  auto slab = [&](auto index, auto loads, int64_t number) XP_INLINE {
    constexpr int S = decltype(index)::value % STAGES;
    constexpr int NEXT = (S + 1) % STAGES;
    constexpr bool LOADING = decltype(loads)::value;
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
  int64_t number = 0;
  auto main_loop = [&](auto loads) XP_INLINE {
    for (; number + STAGES < slabs; number += STAGES) {
      static_for<STAGES>([&](auto j) XP_INLINE { slab(j, loads, number + decltype(j)::value); });
    }
    static_for<STAGES - 1>([&](auto j) XP_INLINE {
      if (number + decltype(j)::value + 1 < slabs) {
        slab(j, loads, number + decltype(j)::value);
      }
    });
  };
  if (loading_wave) {
    main_loop(std::true_type{});
  } else {
    main_loop(std::false_type{});
  }
  static_for<STAGES>([&](auto j) XP_INLINE {
    if ((slabs - 1) % STAGES == decltype(j)::value) {
      constexpr int S = decltype(j)::value;
      read_fragments(S, 1, 1);
      multiply(0);
      read_fragments(S, 2, 0);
      multiply(1);
      read_fragments(S, 3, 1);
      multiply(0);
      multiply(1);
    }
  });
  // Refills past the end may still be landing in the stages that the epilogue reuses, and other waves reading.
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();

  // 32 rows at a time go through a part of LDS of the wave's own, so that a lane then holds eight neighbouring
  // columns of a row: whole 16-byte loads and stores, 128 contiguous bytes and more of each row.
  float *rows = reinterpret_cast<float *>(lds) + wave * 32 * PITCH;
  constexpr int LANES = WTN / 8;        // per row
  constexpr int ROWS_PER_PASS = 64 / LANES;
  const int64_t row0 = m0 + wm * WTM;
  const int64_t col0 = n0 + wn * WTN;
  const int64_t pitch_n = (a.n + 7) / 8 * 8;
  float *partial = a.ranges > 1 ? a.partials + (at.matrix * a.ranges + at.range) * a.m * pitch_n : nullptr;
  const bool mirrored = a.symmetric != 0 && at.m != at.n;
  float sums[16] = {};
  auto put = [&](int64_t row, int64_t col, float (&value)[8]) XP_INLINE {
    if (partial != nullptr) {
      __builtin_memcpy(__builtin_assume_aligned(partial + row * pitch_n + col, 16), value, 32);
    } else {
      finish<P, EPI>(a, at.matrix, row, col, value, sums);
    }
  };
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if (row0 + mt * 32 >= a.m) {
      break;
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 four = {acc[mt][nt][4 * q], acc[mt][nt][4 * q + 1], acc[mt][nt][4 * q + 2], acc[mt][nt][4 * q + 3]};
        *reinterpret_cast<f32x4 *>(rows + (lane & 31) * PITCH + nt * 32 + 8 * q + 4 * (lane >> 5)) = four;
      }
    }
    __builtin_amdgcn_wave_barrier();
    const int chunk = lane % LANES;
    for (int pass = 0; pass < 32 / ROWS_PER_PASS; ++pass) {
      const int row = pass * ROWS_PER_PASS + lane / LANES;
      const int64_t to_row = row0 + mt * 32 + row;
      const int64_t to_col = col0 + chunk * 8;
      if (to_row < a.m && to_col < a.n) {
        float value[8];
        const f32x4 low = *reinterpret_cast<const f32x4 *>(rows + row * PITCH + chunk * 8);
        const f32x4 high = *reinterpret_cast<const f32x4 *>(rows + row * PITCH + chunk * 8 + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          value[j] = low[j];
          value[4 + j] = high[j];
        }
        put(to_row, to_col, value);
      }
    }
    if constexpr (EPI == ProductEpilogue::kStore) {
      if (mirrored) {
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
            put(to_row, to_col, value);
          }
        }
      }
    }
  }
  if constexpr (EPI == ProductEpilogue::kGradient) {
    if (partial == nullptr && a.column_sums != nullptr && row0 < a.m) {
      store_column_sums<LANES>(a, at.m * WAVES_M + wm, col0 + (lane % LANES) * 8, sums, lane);
    }
  }
}

// ------------------------------------------------------------------ sum of the K ranges
// In range order, then the epilogue.  A wave takes 32 rows of 64 columns (a band of the column sums).
template <class P, ProductEpilogue EPI>
__global__ __launch_bounds__(256) void product_reduce_kernel(ProductArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t band = static_cast<int64_t>(blockIdx.y) * 4 + (threadIdx.x >> 6);
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 64 + (lane & 7) * 8;
  const int64_t matrix = blockIdx.z;
  const int64_t pitch_n = (a.n + 7) / 8 * 8;
  const int64_t plane = a.m * pitch_n;
  const float *partial = a.partials + matrix * a.ranges * plane;
  float sums[16] = {};
  if (band * 32 >= a.m) {
    return;
  }
  for (int pass = 0; pass < 4; ++pass) {
    const int64_t row = band * 32 + pass * 8 + (lane >> 3);
    if (row < a.m && col < a.n) {
      const float *from = partial + row * pitch_n + col;
      float value[8];
      __builtin_memcpy(value, __builtin_assume_aligned(from, 16), 32);
      for (int64_t range = 1; range < a.ranges; ++range) {
        float more[8];
        __builtin_memcpy(more, __builtin_assume_aligned(from + range * plane, 16), 32);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          value[j] += more[j];
        }
      }
      finish<P, EPI>(a, matrix, row, col, value, sums);
    }
  }
  if constexpr (EPI == ProductEpilogue::kGradient) {
    if (a.column_sums != nullptr) {
      store_column_sums<8>(a, band, col, sums, lane);
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

template <class P>
const void *ProductKernels<P>::tile(int tile, ProductEpilogue epilogue, bool a_cols, bool b_cols) {
  return tile == 256   ? product_tile_kernel<P, 256, 2, 4, 2>(epilogue, a_cols, b_cols)
         : tile == 128 ? product_tile_kernel<P, 128, 2, 2, 2>(epilogue, a_cols, b_cols)
                       : product_tile_kernel<P, 64, 2, 2, 2>(epilogue, a_cols, b_cols);
}

template <class P>
const void *ProductKernels<P>::reduce(ProductEpilogue epilogue) {
  switch (epilogue) {
    case ProductEpilogue::kActivate:
      return reinterpret_cast<const void *>(&product_reduce_kernel<P, ProductEpilogue::kActivate>);
    case ProductEpilogue::kGradient:
      return reinterpret_cast<const void *>(&product_reduce_kernel<P, ProductEpilogue::kGradient>);
    default:
      return reinterpret_cast<const void *>(&product_reduce_kernel<P, ProductEpilogue::kStore>);
  }
}

}  // namespace xp
