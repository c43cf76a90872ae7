// Training a layer's projections: their gradients, the gated block's forward pass with what its backward pass
// reads, and that backward pass.  No counterpart in the reference.
//
// Every product is one of product_kernels.hpp: y = x w^T + b has dx = dy w, whose reduction runs along dy's rows
// and across w's, and dw = dy^T x, whose reduction runs across the rows of both.  The gradient of the
// activation's outputs is never written: its product's epilogue reads the kept projection and writes the
// projection's gradient and the activation's outputs, both of which the weights' gradients read next.
//
// Roundings.  Sums are fp32.  What a later product reads is rounded to the payload, as its matrix instructions take it: the
// activated values (forward and backward) and the gradient of the projection, half a step each.  In 16 bits the block's
// results are 1.4 times as far off as with both kept in fp32 (bf16 2.3e-3 against 1.7e-3 in the 2-norm, fp16 2.9e-4 against 2.1e-4),
// whose products would run at a tenth of the rate.
//
// Operands whose rows are not whole 16-byte chunks are first copied with padded rows into the workspace.

#include "product_kernels.hpp"
#include "xp_elements.hpp"
#include "xp_entry.hpp"

#include <cmath>

namespace xp {
namespace {

// ------------------------------------------------------------------ rows of whole chunks
struct PadJob {
  const void *source;
  void *target;
  int64_t rows;
  int64_t width;
  int64_t ld;
  int64_t padded;    // row length of the target, a whole number of chunks
  uint32_t blocks;
};
struct PadArgs {
  PadJob job[4];
  int32_t count;
};

// Workgroups of an operand's copy: all four together stay below a launch's 2^32 threads.
constexpr int64_t kPadBlocks = int64_t{1} << 21;

// Rows of any alignment into rows of whole 16-byte chunks, zeros behind them: up to four operands in one launch.  One
// thread a chunk (several chunks past 8 GiB of them).  Bound by latency at the sizes where it is a part of the whole (9 MB of fp16 weights, inputs and gradients of
// 777 rows of 1030 x 2053: 6.6 us).
template <class P>
__global__ __launch_bounds__(256) void pad_rows_kernel(PadArgs a) {
  constexpr int CHUNK = 16 / kElementBytes<P>;
  uint32_t block = blockIdx.x;
  int at = 0;
  while (at + 1 < a.count && block >= a.job[at].blocks) {
    block -= a.job[at].blocks;
    ++at;
  }
  const PadJob job = a.job[at];
  const uint32_t chunks = static_cast<uint32_t>(job.padded / CHUNK);
  const int64_t count = job.rows * chunks;
  for (int64_t index = static_cast<int64_t>(block) * 256 + threadIdx.x; index < count; index += static_cast<int64_t>(job.blocks) * 256) {
    const int64_t row = index < (int64_t{1} << 32) ? static_cast<uint32_t>(index) / chunks : index / chunks;
    const int64_t column = (index - row * chunks) * CHUNK;
    const unsigned char *from = static_cast<const unsigned char *>(job.source) + (row * job.ld + column) * kElementBytes<P>;
    const u32x4 chunk = job.width - column >= CHUNK ? load16_any(from) : load_chunk_tail<P, P>(from, job.width - column);
    store16(static_cast<unsigned char *>(job.target) + (row * job.padded + column) * kElementBytes<P>, chunk);
  }
}

// Zeros in columns [width, padded) of every row of the target.
__global__ __launch_bounds__(256) void clear_pad_kernel(PadJob job, int element) {
  const int64_t behind = (job.padded - job.width) * element / 2;  // 16-bit words
  const int64_t index = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = index / behind;
  if (row < job.rows) {
    uint16_t *words = reinterpret_cast<uint16_t *>(static_cast<unsigned char *>(job.target) + (row * job.padded + job.width) * element);
    words[index - row * behind] = 0;
  }
}

// ------------------------------------------------------------------ sums over rows
struct ColumnSumArgs {
  const void *source;  // [rows, n]
  float *bands;        // [bands, n]
  float *out;          // [n]
  int64_t rows;
  int64_t n;
  int64_t ld;
  int64_t band_rows;
  int64_t band_count;
  int32_t accumulate;
};

// fp32 sums of a band's rows, bound by memory (4096 fp16 rows of 12288 columns with the bands' sum 19.8 us, 5.1 TB/s).  A
// workgroup takes a chunk of columns per lane and the band's rows in turn over its four
// waves, eight of a wave's in flight, and adds the waves' sums through LDS in wave order.
constexpr int kBandRowsOfSum = 64;

template <class P>
__global__ __launch_bounds__(256) void column_sum_kernel(ColumnSumArgs a) {
  constexpr int ES = kElementBytes<P>;
  constexpr int CHUNK = 16 / ES;
  constexpr int AHEAD = 8;
  __shared__ float waves[4][CHUNK][64];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int64_t column = (static_cast<int64_t>(blockIdx.x) * 64 + lane) * CHUNK;
  const bool live = column < a.n;
  // The last chunk of a ragged row is read where it ends with the row (its first columns again, which another lane stores).
  const int64_t from_column = a.n - column >= CHUNK || a.n < CHUNK ? column : a.n - CHUNK;
  const bool whole = a.n >= CHUNK;
  const int64_t first = static_cast<int64_t>(blockIdx.y) * a.band_rows;
  const int64_t last = first + a.band_rows < a.rows ? first + a.band_rows : a.rows;
  const auto row_at = [&](int64_t row) __attribute__((always_inline)) {
    const unsigned char *from = static_cast<const unsigned char *>(a.source) + (row * a.ld + from_column) * ES;
    return whole ? load16_any(from) : load_chunk_tail<P, P>(from, a.n);
  };
  float sum[CHUNK] = {};
  const auto add = [&](const u32x4 &chunk) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < CHUNK; ++j) {
      if constexpr (ES == 4) {
        sum[j] += __uint_as_float(chunk[j]);
      } else {
        sum[j] += P::widen(j % 2 == 0 ? chunk[j / 2] & 0xffffu : chunk[j / 2] >> 16);
      }
    }
  };
  int64_t row = first + wave;
  if (live) {
    for (; row + 4 * (AHEAD - 1) < last; row += 4 * AHEAD) {
      u32x4 chunks[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        chunks[i] = row_at(row + 4 * i);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        add(chunks[i]);
      }
    }
    for (; row < last; row += 4) {
      add(row_at(row));
    }
  }
#pragma unroll
  for (int j = 0; j < CHUNK; ++j) {
    waves[wave][j][lane] = sum[j];
  }
  __syncthreads();
  if (wave != 0 || !live) {
    return;
  }
  float *to = a.bands + static_cast<int64_t>(blockIdx.y) * a.n + from_column;
#pragma unroll
  for (int j = 0; j < CHUNK; ++j) {
    if (from_column + j >= column && from_column + j < a.n) {
      to[j] = (waves[0][j][lane] + waves[1][j][lane]) + (waves[2][j][lane] + waves[3][j][lane]);
    }
  }
}

// All rows by one workgroup: sixteen waves take them in turn, four bytes a lane and sixteen rows in flight.  Bound by latency;
// up to kRowsAtOnce rows as short as bands and a launch that adds them, or shorter (777 fp16 rows of 2053 columns 6.2 us against
// 7.4, of 12288 5.2 against 7.7; 1024 rows 7.6 against 6.9 and 6.0 against 7.1).  It adds the bands' sums too.
constexpr int64_t kRowsAtOnce = 1024;
constexpr int kSumWaves = 16;

template <class P>
__device__ __forceinline__ void sum_rows(const ColumnSumArgs &a, uint32_t block, float (&waves)[kSumWaves][2][64]) {
  constexpr int ES = kElementBytes<P>;
  constexpr int COLS = 4 / ES;
  constexpr int AHEAD = 16;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int64_t column = (static_cast<int64_t>(block) * 64 + lane) * COLS;
  const bool live = column < a.n;
  const bool whole = a.n - column >= COLS;
  float sum[COLS] = {};
  const auto row_at = [&](int64_t row) __attribute__((always_inline)) {
    const unsigned char *from = static_cast<const unsigned char *>(a.source) + (row * a.ld + column) * ES;
    uint32_t word = 0;
    if (whole) {
      __builtin_memcpy(&word, from, 4);
    } else {
      word = *reinterpret_cast<const uint16_t *>(from);
    }
    return word;
  };
  const auto add = [&](uint32_t word) __attribute__((always_inline)) {
    if constexpr (ES == 4) {
      sum[0] += __uint_as_float(word);
    } else {
      sum[0] += P::widen(word & 0xffffu);
      sum[1] += P::widen(word >> 16);
    }
  };
  int64_t row = wave;
  if (live) {
    for (; row + kSumWaves * (AHEAD - 1) < a.rows; row += kSumWaves * AHEAD) {
      uint32_t words[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        words[i] = row_at(row + kSumWaves * i);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        add(words[i]);
      }
    }
#pragma unroll 4
    for (; row < a.rows; row += kSumWaves) {
      add(row_at(row));
    }
  }
#pragma unroll
  for (int j = 0; j < COLS; ++j) {
    waves[wave][j][lane] = sum[j];
  }
  __syncthreads();
  if (wave != 0 || !live) {
    return;
  }
#pragma unroll
  for (int j = 0; j < COLS; ++j) {
    if (column + j < a.n) {
      float total = 0.0f;
#pragma unroll
      for (int w = 0; w < kSumWaves; ++w) {
        total += waves[w][j][lane];
      }
      a.out[column + j] = a.accumulate ? a.out[column + j] + total : total;
    }
  }
}

// Sums of payload rows, and of fp32 bands' sums, in one launch.
struct RowSums {
  ColumnSumArgs rows;
  ColumnSumArgs bands;
  uint32_t row_blocks;
};

template <class P>
__global__ __launch_bounds__(64 * kSumWaves) void row_sums_kernel(RowSums a) {
  __shared__ float waves[kSumWaves][2][64];
  if (blockIdx.x < a.row_blocks) {
    sum_rows<P>(a.rows, blockIdx.x, waves);
  } else {
    sum_rows<F32Payload>(a.bands, blockIdx.x - a.row_blocks, waves);
  }
}

// ------------------------------------------------------------------ weights' gradients of few rows
struct ThinOuterArgs {
  const void *a;  // [rows, m]
  const void *b;  // [rows, n]
  void *out;      // [m, n]
  int64_t ld_a;
  int64_t ld_b;
  int64_t m;
  int64_t n;
  int32_t rows;
  int32_t out_dtype;
  int32_t accumulate;
  int32_t lanes = 0;     // threads that share a row of the output
  int32_t across = 0;    // workgroups that share one
  int32_t out_rows = 0;  // of a workgroup
};

// out (+)= a^T b over at most ROWS rows, in fp32 on the vector pipes, rows in order.  The output's bytes bound it; a
// matrix core tile has one slab to multiply here and spends its time on its first loads and its epilogue.  A thread keeps eight
// columns of b in registers and walks the output's rows, whose factors the workgroup holds in LDS: 16-byte stores,
// neighbouring lanes side by side.  Operands of any alignment.  2048 x 6144 of five bf16 rows: 9.4 us by itself (25 MB, 2.7
// TB/s), 12.9 with the inputs' gradient beside it (50 MB, 3.9 TB/s; one after the other 17.6).  From nine rows on 16-bit
// operands are faster on tiles (2048 x 6144 of sixteen 12.5 us against 18.8, 1030 x 2053 with the inputs' gradient 14 against
// 22.7), fp32 ones, whose tiles work longer, from seventeen (2048 x 6144 with the inputs' gradient 29.6 against 42).
constexpr int kThinRows = 16;
bool thin_rows(int64_t rows, size_t element) { return rows <= (element == 4 ? kThinRows : kThinRows / 2); }
constexpr int kThinOutRows = 32;

template <class P, int ROWS>
__device__ __forceinline__ void thin_outer(const ThinOuterArgs &a, uint32_t block, unsigned char *lds) {
  float (*factors)[ROWS] = reinterpret_cast<float (*)[ROWS]>(lds);
  const uint32_t down = block / static_cast<uint32_t>(a.across);
  const uint32_t along = block - down * static_cast<uint32_t>(a.across);
  const int64_t first = static_cast<int64_t>(down) * a.out_rows;
  for (int i = threadIdx.x; i < a.out_rows * ROWS; i += 256) {
    const int row = i % a.out_rows;
    const int t = i / a.out_rows;
    factors[row][t] = t < a.rows && first + row < a.m ? load_value(a.a, t * a.ld_a + first + row, kDtypeOf<P>) : 0.0f;
  }
  const int lane = static_cast<int>(threadIdx.x) % a.lanes;
  const int side = static_cast<int>(threadIdx.x) / a.lanes;
  const int sides = 256 / a.lanes;
  const int64_t column = (static_cast<int64_t>(along) * a.lanes + lane) * 8;
  const int count = a.n - column < 8 ? static_cast<int>(a.n - column) : 8;
  float b[ROWS][8] = {};
  if (count > 0) {
#pragma unroll
    for (int t = 0; t < ROWS; ++t) {
      if (t < a.rows) {
        load_values(a.b, t * a.ld_b + column, kDtypeOf<P>, count, b[t]);
      }
    }
  }
  __syncthreads();
  if (count <= 0 || side >= sides) {
    return;
  }
  for (int row = side; row < a.out_rows && first + row < a.m; row += sides) {
    float sum[8] = {};
#pragma unroll
    for (int t = 0; t < ROWS; t += 4) {
      const f32x4 four = *reinterpret_cast<const f32x4 *>(&factors[row][t]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sum[j] = fmaf(four[i], b[t + i][j], sum[j]);
        }
      }
    }
    const int64_t at = (first + row) * a.n + column;
    if (a.accumulate) {
      float held[8];
      load_values(a.out, at, a.out_dtype, count, held);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum[j] += held[j];
      }
    }
    store_values(a.out, at, a.out_dtype, count, sum);
  }
}

// The gradients of few rows in one launch: an inputs' gradient (32 x 32 tiles of product_kernels.hpp; it reads the weights) and
// up to two weights' gradients, which write as much.  Each by itself leaves half of the memory's directions idle.
struct ThinArgs {
  ProductArgs inputs;
  ThinOuterArgs outer[2];
  uint32_t blocks[3];
};

template <class P, int ROWS>
__global__ __launch_bounds__(256, (ROWS > 8 ? 2 : 4)) void thin_gradients_kernel(ThinArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[kStageBytes<32, 4>];
  static_assert(sizeof(float) * kThinOutRows * ROWS <= kStageBytes<32, 4>, "the factors fit the stages");
  uint32_t block = blockIdx.x;
  if (block < a.blocks[0]) {
    product_body<P, 32, 1, 1, 4, false, true, ProductEpilogue::kStore, false>(a.inputs, block, lds);
    return;
  }
  block -= a.blocks[0];
  const int at = block < a.blocks[1] ? 0 : 1;
  thin_outer<P, ROWS>(a.outer[at], at == 0 ? block : block - a.blocks[1], lds);
}

template <class P>
const void *thin_gradients_for(int rows) {
  if constexpr (kElementBytes<P> == 4) {
    if (rows > 8) {
      return reinterpret_cast<const void *>(&thin_gradients_kernel<P, kThinRows>);
    }
  }
  return rows <= 4 ? reinterpret_cast<const void *>(&thin_gradients_kernel<P, 4>)
                   : reinterpret_cast<const void *>(&thin_gradients_kernel<P, 8>);
}

// Zeros over whole rows of an output (its gradient over no rows).
__global__ __launch_bounds__(256) void clear_kernel(uint16_t *target, int64_t words) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t index = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; index < words; index += stride) {
    target[index] = 0;
  }
}

unsigned blocks_of(int64_t items, int64_t per_block) { return static_cast<unsigned>((items + per_block - 1) / per_block); }

constexpr size_t kAlign = 256;
constexpr int64_t kMaxRows = int64_t{1} << 24;
constexpr int64_t kMaxWidth = int64_t{1} << 20;
constexpr int64_t kMaxStride = int64_t{1} << 20;

size_t aligned_bytes(size_t bytes) { return (bytes + kAlign - 1) / kAlign * kAlign; }
int64_t padded_width(int64_t width, size_t element) {
  const int64_t chunk = static_cast<int64_t>(16 / element);
  return (width + chunk - 1) / chunk * chunk;
}
bool whole_rows(int64_t width, size_t element) { return width % static_cast<int64_t>(16 / element) == 0; }

// Regions of a workspace, one behind another.
struct Regions {
  unsigned char *base;
  size_t used = 0;
  void *take(size_t bytes) {
    void *at = base == nullptr ? nullptr : base + used;
    used += aligned_bytes(bytes);
    return at;
  }
};

// Partial sums of a product for every number of rows up to a capacity, at powers of two below it.
template <class Plan>
size_t scratch_upto(int64_t capacity, Plan &&plan) {
  size_t most = 0;
  for (int64_t rows = capacity; rows >= 1; rows /= 2) {
    most = std::max(most, plan(rows));
  }
  return most;
}

size_t unlimited_scratch(int64_t m, int64_t n, int64_t k, int element) {
  return product_scratch_bytes(plan_product(m, n, k, 1, element, false, SIZE_MAX));
}

// ------------------------------------------------------------------ launches
struct Caller {
  hipStream_t stream;
  int dtype;
  size_t element;
  float *scratch;
  size_t scratch_bytes;

  hipError_t product(ProductArgs &args, ProductEpilogue epilogue, bool a_cols, bool b_cols) const {
    args.partials = scratch;
    args.batch = 1;
    return launch_product(args, epilogue, a_cols, b_cols, dtype, scratch_bytes, stream);
  }

  hipError_t products(ProductGroup &group, const bool (&present)[3]) const {
    for (ProductArgs &part : group.part) {
      part.partials = scratch;
      part.batch = 1;
    }
    return launch_products(group, present, dtype, scratch_bytes, stream);
  }

  // `source` itself where its rows are whole chunks, else a padded copy in `target`, which `pads` then has to make.
  ProductOperand padded(const void *source, int64_t rows, int64_t width, int64_t ld, void *target, PadArgs &pads) const {
    if (whole_rows(width, element)) {
      return {source, ld, 0};
    }
    const int64_t length = padded_width(width, element);
    const int64_t chunks = rows * (length / static_cast<int64_t>(16 / element));
    const uint32_t blocks = static_cast<uint32_t>(std::min((chunks + 255) / 256, kPadBlocks));
    pads.job[pads.count++] = PadJob{source, target, rows, width, ld, length, blocks};
    return {target, length, 0};
  }

  hipError_t pad(const PadArgs &pads) const {
    KernelLaunch kernel;
    uint32_t blocks = 0;
    for (int i = 0; i < pads.count; ++i) {
      blocks += pads.job[i].blocks;
    }
    kernel.func = element == 4 ? reinterpret_cast<const void *>(&pad_rows_kernel<F32Payload>)
                               : reinterpret_cast<const void *>(&pad_rows_kernel<Bf16Payload>);
    kernel.grid = dim3(blocks);
    kernel.block = dim3(256);
    kernel.set_args(pads);
    return pads.count == 0 ? hipSuccess : launch(kernel, stream);
  }

  // Gradients of few rows (thin_rows); `inputs` and those of `outer` may be null.
  hipError_t thin_gradients(ProductArgs *inputs, std::initializer_list<const ThinOuterArgs *> outer, int rows) const {
    ThinArgs args{};
    if (inputs != nullptr) {
      inputs->batch = 1;
      inputs->partials = scratch;
      const ProductPlan plan = plan_product(inputs->m, inputs->n, inputs->k, 1, static_cast<int>(element), false, scratch_bytes);
      if (plan.tiles == ProductTiles::k32) {
        args.inputs = *inputs;
        args.inputs.tile_rows = static_cast<int32_t>((inputs->m + 31) / 32);
        args.inputs.tile_cols = static_cast<int32_t>((inputs->n + 31) / 32);
        args.inputs.whole = args.inputs.tile_rows * args.inputs.tile_cols;
        args.blocks[0] = static_cast<uint32_t>(args.inputs.whole);
      } else if (const hipError_t status = launch_product(*inputs, ProductEpilogue::kStore, false, true, dtype, scratch_bytes, stream);
                 status != hipSuccess) {
        return status;
      }
    }
    int count = 0;
    for (const ThinOuterArgs *each : outer) {
      if (each == nullptr) {
        continue;
      }
      ThinOuterArgs &part = args.outer[count];
      part = *each;
      const int64_t chunks = (part.n + 7) / 8;
      part.lanes = static_cast<int32_t>(std::min<int64_t>(chunks, 256));
      part.across = static_cast<int32_t>((chunks + part.lanes - 1) / part.lanes);
      // Enough workgroups for the chip, each with as many rows as that leaves.
      part.out_rows = static_cast<int32_t>(std::clamp<int64_t>(part.m * part.across / (rows > 8 ? 512 : 1024), 4, kThinOutRows));
      args.blocks[++count] = static_cast<uint32_t>(part.across) * blocks_of(part.m, part.out_rows);
    }
    const uint32_t blocks = args.blocks[0] + args.blocks[1] + args.blocks[2];
    if (blocks == 0) {
      return hipSuccess;
    }
    const void *func = dtype == kDtypeF32   ? thin_gradients_for<F32Payload>(rows)
                       : dtype == kDtypeF16 ? thin_gradients_for<F16Payload>(rows)
                                            : thin_gradients_for<Bf16Payload>(rows);
    void *params[] = {&args};
    return hipLaunchKernel(func, dim3(blocks), dim3(256), params, 0, stream);
  }

  hipError_t clear(void *target, size_t bytes) const {
    const int64_t words = static_cast<int64_t>(bytes / 2);
    clear_kernel<<<std::min(blocks_of(words, 256), 4096u), 256, 0, stream>>>(static_cast<uint16_t *>(target), words);
    return hipGetLastError();
  }

  // Either may be null.
  hipError_t row_sums(const ColumnSumArgs *rows, const ColumnSumArgs *bands) const {
    RowSums args{};
    uint32_t blocks = 0;
    if (rows != nullptr) {
      args.rows = *rows;
      args.row_blocks = blocks = blocks_of(rows->n, 64 * static_cast<int64_t>(4 / element));
    }
    if (bands != nullptr) {
      args.bands = *bands;
      blocks += blocks_of(bands->n, 64);
    }
    KernelLaunch kernel;
    kernel.func = dtype == kDtypeF32   ? reinterpret_cast<const void *>(&row_sums_kernel<F32Payload>)
                  : dtype == kDtypeF16 ? reinterpret_cast<const void *>(&row_sums_kernel<F16Payload>)
                                       : reinterpret_cast<const void *>(&row_sums_kernel<Bf16Payload>);
    kernel.grid = dim3(blocks);
    kernel.block = dim3(64 * kSumWaves);
    kernel.set_args(args);
    return blocks == 0 ? hipSuccess : launch(kernel, stream);
  }

  hipError_t column_sums(const void *source, int64_t rows, int64_t n, int64_t ld, float *bands, float *out, bool accumulate) const;
};

// Bands of a column sum: 64 rows, or more where that makes over 64 of them.
int64_t column_sum_bands(int64_t rows) { return std::min<int64_t>((rows + kBandRowsOfSum - 1) / kBandRowsOfSum, 64); }

hipError_t Caller::column_sums(const void *source, int64_t rows, int64_t n, int64_t ld, float *bands, float *out,
                               bool accumulate) const {
  ColumnSumArgs args{source, bands, out, rows, n, ld, 0, 0, accumulate};
  const int64_t wanted = column_sum_bands(rows);
  args.band_rows = (rows + wanted - 1) / wanted;
  args.band_count = (rows + args.band_rows - 1) / args.band_rows;
  KernelLaunch kernel;
  if (rows <= kRowsAtOnce) {
    return row_sums(&args, nullptr);
  }
  kernel.func = dtype == kDtypeF32   ? reinterpret_cast<const void *>(&column_sum_kernel<F32Payload>)
                : dtype == kDtypeF16 ? reinterpret_cast<const void *>(&column_sum_kernel<F16Payload>)
                                     : reinterpret_cast<const void *>(&column_sum_kernel<Bf16Payload>);
  kernel.grid = dim3(blocks_of(n, 64 * static_cast<int64_t>(16 / element)), static_cast<unsigned>(args.band_count));
  kernel.block = dim3(256);
  kernel.set_args(args);
  if (const hipError_t status = launch(kernel, stream); status != hipSuccess) {
    return status;
  }
  const ColumnSumArgs sums{bands, nullptr, out, args.band_count, n, n, 0, 0, accumulate};
  return row_sums(nullptr, &sums);
}

// out (+)= sum over rows t of a[t][i] b[t][j]: a weight's gradient.
ProductArgs outer_args(const ProductOperand &a, int64_t m, const ProductOperand &b, int64_t n, int64_t rows, void *out,
                       int out_dtype, bool accumulate) {
  ProductArgs args{};
  args.a = a;
  args.b = b;
  args.m = m;
  args.n = n;
  args.k = rows;
  args.out = out;
  args.ld_out = n;
  args.base = out;
  args.ld_base = n;
  args.out_dtype = args.base_dtype = static_cast<int8_t>(out_dtype);
  args.alpha = 1.0f;
  args.beta = accumulate ? 1.0f : 0.0f;
  return args;
}

// out = a w: the gradient of a projection's inputs.
ProductArgs inputs_args(const ProductOperand &a, const ProductOperand &w, int64_t rows, int64_t n, int64_t k, void *out,
                        int64_t ld_out, int dtype) {
  ProductArgs args{};
  args.a = a;
  args.b = w;
  args.m = rows;
  args.n = k;
  args.k = n;
  args.out = out;
  args.ld_out = ld_out;
  args.out_dtype = static_cast<int8_t>(dtype);
  args.alpha = 1.0f;
  return args;
}

// ------------------------------------------------------------------ workspaces
struct ProjectionRegions {
  void *x;
  void *w;
  void *grad;
  float *bands;
  float *scratch;
  size_t scratch_bytes;
  size_t bytes;
};

ProjectionRegions projection_regions(unsigned char *base, int64_t rows, int64_t n, int64_t k, size_t element) {
  Regions regions{base};
  ProjectionRegions found{};
  const size_t padded_k = static_cast<size_t>(padded_width(k, element)) * element;
  if (!whole_rows(k, element)) {
    found.x = regions.take(static_cast<size_t>(rows) * padded_k);
    found.w = regions.take(static_cast<size_t>(n) * padded_k);
  }
  if (!whole_rows(n, element)) {
    found.grad = regions.take(static_cast<size_t>(rows * padded_width(n, element)) * element);
  }
  found.bands = static_cast<float *>(regions.take(static_cast<size_t>(column_sum_bands(rows) * n) * 4));
  found.scratch_bytes = scratch_upto(rows, [&](int64_t live) {
    return std::max(unlimited_scratch(live, k, n, static_cast<int>(element)),
                    unlimited_scratch(n, k, live, static_cast<int>(element)));
  });
  found.scratch = static_cast<float *>(regions.take(found.scratch_bytes));
  found.bytes = regions.used;
  return found;
}

struct KeepRegions {
  void *x;
  void *w;
  float *scratch;
  size_t scratch_bytes;
  size_t bytes;
};

KeepRegions keep_regions(unsigned char *base, int64_t rows, int64_t n, int64_t k, size_t element) {
  Regions regions{base};
  KeepRegions found{};
  const size_t padded_k = static_cast<size_t>(padded_width(k, element)) * element;
  if (!whole_rows(k, element)) {
    found.x = regions.take(static_cast<size_t>(rows) * padded_k);
    found.w = regions.take(static_cast<size_t>(n) * padded_k);
  }
  found.scratch_bytes =
      scratch_upto(rows, [&](int64_t live) { return unlimited_scratch(live, n, k, static_cast<int>(element)); });
  found.scratch = static_cast<float *>(regions.take(found.scratch_bytes));
  found.bytes = regions.used;
  return found;
}

struct DenseRegions {
  void *x;
  void *w_in;
  void *w_out;
  void *grad;
  void *through;    // [rows, wide padded]: the projection's gradient
  void *activated;  // [rows, width padded]
  float *bands;
  float *scratch;
  size_t scratch_bytes;
  size_t bytes;
};

DenseRegions dense_regions(unsigned char *base, int64_t rows, int64_t hidden, int64_t width, int64_t wide, size_t element) {
  Regions regions{base};
  DenseRegions found{};
  const size_t padded_hidden = static_cast<size_t>(padded_width(hidden, element)) * element;
  const size_t padded_inner = static_cast<size_t>(padded_width(width, element)) * element;
  if (!whole_rows(hidden, element)) {
    found.x = regions.take(static_cast<size_t>(rows) * padded_hidden);
    found.w_in = regions.take(static_cast<size_t>(wide) * padded_hidden);
    found.grad = regions.take(static_cast<size_t>(rows) * padded_hidden);
  }
  if (!whole_rows(width, element)) {
    found.w_out = regions.take(static_cast<size_t>(hidden) * padded_inner);
  }
  found.through = regions.take(static_cast<size_t>(rows * padded_width(wide, element)) * element);
  found.activated = regions.take(static_cast<size_t>(rows) * padded_inner);
  found.bands = static_cast<float *>(
      regions.take(static_cast<size_t>(std::max((rows + kBandRows - 1) / kBandRows * wide, column_sum_bands(rows) * hidden)) * 4));
  found.scratch_bytes = scratch_upto(rows, [&](int64_t live) {
    const int es = static_cast<int>(element);
    return std::max(std::max(unlimited_scratch(live, width, hidden, es), unlimited_scratch(live, hidden, wide, es)),
                    std::max(unlimited_scratch(wide, hidden, live, es), unlimited_scratch(hidden, width, live, es)));
  });
  found.scratch = static_cast<float *>(regions.take(found.scratch_bytes));
  found.bytes = regions.used;
  return found;
}

bool extents_valid(int64_t rows, int64_t a, int64_t b) {
  return rows >= 0 && rows <= kMaxRows && a >= 1 && a <= kMaxWidth && b >= 1 && b <= kMaxWidth;
}
constexpr const char *kExtents = "training operators take up to 2^24 rows and widths of 1 to 2^20";

// A matrix [rows, width]: non-null, aligned to an element, and where its rows are whole 16-byte chunks and the
// kernels load it (`loaded`), every row on a 16-byte boundary.
int check_rows(const char *name, const void *pointer, int64_t ld, int64_t width, size_t element, bool loaded) {
  XP_REQUIRE(pointer != nullptr && aligned_to(pointer, element), std::string(name) + " must be non-null and aligned to its element size");
  XP_REQUIRE(ld >= width && ld <= kMaxStride, std::string(name) + " has a row stride below its width or above 2^20");
  XP_REQUIRE(!loaded || !whole_rows(width, element) || (aligned16(pointer) && whole_rows(ld, element)),
             std::string(name) + " has rows of whole 16 bytes that do not start on 16-byte boundaries");
  return XP_OK;
}

#define XP_TRY(expr)                                  \
  do {                                                \
    if (const int xp_status_ = (expr); xp_status_ != XP_OK) { \
      return xp_status_;                              \
    }                                                 \
  } while (0)

int check_weight_gradient(const char *name, const void *pointer, int grad_dtype, int dtype) {
  XP_REQUIRE(grad_dtype == dtype || grad_dtype == XP_DTYPE_F32, "weight gradients are of the payload dtype or fp32");
  XP_REQUIRE(aligned_to(pointer, dtype_bytes(grad_dtype)), std::string(name) + " must be aligned to its element size");
  return XP_OK;
}

bool apart(std::initializer_list<Span> written, std::initializer_list<Span> read) {
  for (auto at = written.begin(); at != written.end(); ++at) {
    for (auto other = at + 1; other != written.end(); ++other) {
      if (overlaps(*at, *other)) {
        return false;
      }
    }
    if (touches(*at, read)) {
      return false;
    }
  }
  return true;
}

}  // namespace

}  // namespace xp

using namespace xp;

extern "C" {

size_t xp_projection_backward_workspace_bytes(int64_t rows, int64_t n, int64_t k, int dtype) {
  const size_t element = dtype_bytes(dtype);
  return element == 0 || !extents_valid(rows, n, k) || rows == 0 ? 0 : projection_regions(nullptr, rows, n, k, element).bytes;
}

int xp_projection_backward(const void *x, int64_t ld_x, int64_t rows, int64_t k, const void *w, int64_t n, const void *grad_out,
                           int64_t ld_grad, int dtype, void *grad_x, int64_t ld_grad_x, void *grad_w, int grad_w_dtype,
                           float *grad_bias, int accumulate, int64_t capacity, void *workspace, size_t workspace_bytes,
                           xp_stream_t stream) {
  const size_t element = dtype_bytes(dtype);
  XP_REQUIRE(element != 0, "payload dtype must be bf16, fp16 or fp32");
  XP_REQUIRE(extents_valid(rows, n, k) && rows <= capacity && capacity <= kMaxRows, kExtents);
  XP_TRY(check_rows("projection weights", w, k, k, element, true));
  if (grad_w != nullptr) {
    XP_TRY(check_weight_gradient("weight gradient", grad_w, grad_w_dtype, dtype));
  }
  XP_REQUIRE(aligned_to(grad_bias, 4), "the bias gradient must be 4-byte aligned");
  const size_t kept = grad_w == nullptr ? 0 : dtype_bytes(grad_w_dtype);
  Caller call{static_cast<hipStream_t>(stream), dtype, element, nullptr, 0};
  if (rows == 0) {
    if (accumulate == 0) {
      if (grad_w != nullptr) {
        XP_HIP_CHECK(call.clear(grad_w, static_cast<size_t>(n * k) * kept));
      }
      if (grad_bias != nullptr) {
        XP_HIP_CHECK(call.clear(grad_bias, static_cast<size_t>(n) * 4));
      }
    }
    return XP_OK;
  }
  XP_TRY(check_rows("output gradient", grad_out, ld_grad, n, element, true));
  if (grad_w != nullptr) {
    XP_TRY(check_rows("projection input", x, ld_x, k, element, true));
  }
  if (grad_x != nullptr) {
    XP_TRY(check_rows("input gradient", grad_x, ld_grad_x, k, element, false));
  }
  const ProjectionRegions at = projection_regions(static_cast<unsigned char *>(workspace), capacity, n, k, element);
  XP_REQUIRE(workspace != nullptr && aligned16(workspace) && workspace_bytes >= at.bytes,
             "workspace is missing, unaligned or smaller than xp_projection_backward_workspace_bytes");
  const Span read_x = span_of_rows(grad_w == nullptr ? nullptr : x, ld_x, k, rows, element);
  const Span read_grad = span_of_rows(grad_out, ld_grad, n, rows, element);
  const Span read_w = span_of(w, static_cast<size_t>(n * k) * element);
  XP_REQUIRE(apart({span_of_rows(grad_x, ld_grad_x, k, rows, element), span_of(grad_w, static_cast<size_t>(n * k) * kept),
                    span_of(grad_bias, static_cast<size_t>(n) * 4), span_of(workspace, at.bytes)},
                   {read_x, read_grad, read_w}),
             "gradients and workspace must overlap neither the operands nor each other");
  call.scratch = at.scratch;
  call.scratch_bytes = at.scratch_bytes;
  const bool thin = thin_rows(rows, element);
  PadArgs pads{};
  ProductOperand grad{};
  ProductOperand weights{};
  ProductOperand inputs{};
  if (grad_x != nullptr || (grad_w != nullptr && !thin)) {
    grad = call.padded(grad_out, rows, n, ld_grad, at.grad, pads);
  }
  if (grad_x != nullptr) {
    weights = call.padded(w, n, k, k, at.w, pads);
  }
  if (grad_w != nullptr && !thin) {
    inputs = call.padded(x, rows, k, ld_x, at.x, pads);
  }
  XP_HIP_CHECK(call.pad(pads));
  ProductGroup group{};
  const bool present[3] = {grad_x != nullptr, grad_w != nullptr && !thin, false};
  if (present[0]) {
    group.part[0] = inputs_args(grad, weights, rows, n, k, grad_x, ld_grad_x, dtype);
  }
  if (present[1]) {
    group.part[1] = outer_args(grad, n, inputs, k, rows, grad_w, grad_w_dtype, accumulate != 0);
  }
  if (thin) {
    const int few = static_cast<int>(rows);
    const ThinOuterArgs outer{grad_out, x, grad_w, ld_grad, ld_x, n, k, few, grad_w_dtype, accumulate};
    XP_HIP_CHECK(call.thin_gradients(present[0] ? &group.part[0] : nullptr, {grad_w == nullptr ? nullptr : &outer}, few));
  } else {
    XP_HIP_CHECK(call.products(group, present));
  }
  if (grad_bias != nullptr) {
    XP_HIP_CHECK(call.column_sums(grad_out, rows, n, ld_grad, at.bands, grad_bias, accumulate != 0));
  }
  return XP_OK;
}

size_t xp_projection_keep_workspace_bytes(int64_t rows, int64_t n, int64_t k, int dtype) {
  const size_t element = dtype_bytes(dtype);
  return element == 0 || !extents_valid(rows, n, k) || rows == 0 ? 0 : keep_regions(nullptr, rows, n, k, element).bytes;
}

int xp_projection_keep(const void *x, int64_t ld_x, int64_t rows, int64_t k, const void *w, int64_t n, const float *bias,
                       void *projected, int64_t ld_projected, void *activated, int dtype, int order,
                       const xp_activation_desc *activation, int64_t capacity, void *workspace, size_t workspace_bytes,
                       xp_stream_t stream) {
  const size_t element = dtype_bytes(dtype);
  XP_REQUIRE(element != 0, "payload dtype must be bf16, fp16 or fp32");
  XP_REQUIRE(extents_valid(rows, n, k) && rows <= capacity && capacity <= kMaxRows, kExtents);
  ProductArgs args{};
  XP_REQUIRE(activated == nullptr || activation != nullptr, "activated outputs need an activation");
  XP_TRY(activation_record(activation, args.act));
  XP_REQUIRE(args.act.gated == 0 || n % 2 == 0, "a gated projection needs an even number of weight rows");
  const bool halves = activated != nullptr && args.act.gated != 0 && order == XP_GATE_UP_CONCATENATED;
  XP_REQUIRE(activated == nullptr || args.act.gated == 0 || halves || order == XP_GATE_UP_INTERLEAVED,
             "gated activation requires a Gate/Up order");
  XP_REQUIRE(!halves || n * padded_width(k, element) * static_cast<int64_t>(element) < int64_t{1} << 31,
             "activated outputs of CONCATENATED weights need less than 2 GiB of weights");
  if (rows == 0) {
    return XP_OK;
  }
  XP_TRY(check_rows("projection weights", w, k, k, element, true));
  XP_TRY(check_rows("projection input", x, ld_x, k, element, true));
  XP_TRY(check_rows("kept projection", projected, ld_projected, n, element, false));
  XP_REQUIRE(aligned_to(bias, 4) && aligned_to(activated, element), "bias and activated outputs must be aligned to their element size");
  const KeepRegions at = keep_regions(static_cast<unsigned char *>(workspace), capacity, n, k, element);
  XP_REQUIRE(at.bytes == 0 || (workspace != nullptr && aligned16(workspace) && workspace_bytes >= at.bytes),
             "workspace is missing, unaligned or smaller than xp_projection_keep_workspace_bytes");
  const int64_t outputs = args.act.gated != 0 ? n / 2 : n;
  XP_REQUIRE(apart({span_of_rows(projected, ld_projected, n, rows, element),
                    span_of(activated, activated == nullptr ? 0 : static_cast<size_t>(rows * outputs) * element),
                    span_of(workspace, at.bytes)},
                   {span_of_rows(x, ld_x, k, rows, element), span_of(w, static_cast<size_t>(n * k) * element),
                    span_of(bias, bias == nullptr ? 0 : static_cast<size_t>(n) * 4)}),
             "outputs and workspace must overlap neither the operands nor each other");
  const Caller call{static_cast<hipStream_t>(stream), dtype, element, at.scratch, at.scratch_bytes};
  PadArgs pads{};
  args.a = call.padded(x, rows, k, ld_x, at.x, pads);
  args.b = call.padded(w, n, k, k, at.w, pads);
  XP_HIP_CHECK(call.pad(pads));
  args.m = rows;
  args.n = n;
  args.k = k;
  args.out = projected;
  args.ld_out = ld_projected;
  args.out_dtype = static_cast<int8_t>(dtype);
  args.bias = bias;
  args.alpha = 1.0f;
  if (activated != nullptr) {
    args.extra = activated;
    args.ld_extra = outputs;
    args.halves = halves ? n / 2 : 0;
  }
  XP_HIP_CHECK(call.product(args, activated != nullptr ? ProductEpilogue::kActivate : ProductEpilogue::kStore, false, false));
  return XP_OK;
}

size_t xp_dense_backward_workspace_bytes(int64_t rows, int64_t hidden, int64_t intermediate, int gated, int dtype) {
  const size_t element = dtype_bytes(dtype);
  const int64_t wide = gated != 0 ? 2 * intermediate : intermediate;
  return element == 0 || !extents_valid(rows, hidden, wide) || rows == 0
             ? 0
             : dense_regions(nullptr, rows, hidden, intermediate, wide, element).bytes;
}

int xp_dense_backward(const void *x, int64_t ld_x, int64_t rows, int64_t hidden, const void *w_in, const void *w_out,
                      int64_t intermediate, const void *projected, int64_t ld_projected, const void *grad_out, int64_t ld_grad,
                      int dtype, int order, const xp_activation_desc *activation, void *grad_x, int64_t ld_grad_x, void *grad_w_in,
                      void *grad_w_out, int grad_w_dtype, float *grad_bias_in, float *grad_bias_out, int accumulate,
                      int64_t capacity, void *workspace, size_t workspace_bytes, xp_stream_t stream) {
  const size_t element = dtype_bytes(dtype);
  XP_REQUIRE(element != 0, "payload dtype must be bf16, fp16 or fp32");
  XP_REQUIRE(activation != nullptr, "activation descriptor must be non-null");
  ProductArgs args{};
  XP_TRY(activation_record(activation, args.act));
  const bool gated = args.act.gated != 0;
  XP_REQUIRE(!gated || order == XP_GATE_UP_INTERLEAVED || order == XP_GATE_UP_CONCATENATED,
             "gated activation requires a Gate/Up order");
  const int64_t width = intermediate;
  XP_REQUIRE(width >= 1 && width <= kMaxWidth, kExtents);
  const int64_t wide = gated ? 2 * width : width;
  XP_REQUIRE(extents_valid(rows, hidden, wide) && rows <= capacity && capacity <= kMaxRows, kExtents);
  for (const void *gradient : {grad_w_in, grad_w_out}) {
    if (gradient != nullptr) {
      XP_TRY(check_weight_gradient("weight gradient", gradient, grad_w_dtype, dtype));
    }
  }
  XP_REQUIRE(aligned_to(grad_bias_in, 4) && aligned_to(grad_bias_out, 4), "bias gradients must be 4-byte aligned");
  const size_t kept = grad_w_in == nullptr && grad_w_out == nullptr ? 0 : dtype_bytes(grad_w_dtype);
  const size_t in_bytes = grad_w_in == nullptr ? 0 : static_cast<size_t>(wide * hidden) * kept;
  const size_t out_bytes = grad_w_out == nullptr ? 0 : static_cast<size_t>(hidden * width) * kept;
  Caller call{static_cast<hipStream_t>(stream), dtype, element, nullptr, 0};
  if (rows == 0) {
    if (accumulate == 0) {
      if (grad_w_in != nullptr) {
        XP_HIP_CHECK(call.clear(grad_w_in, in_bytes));
      }
      if (grad_w_out != nullptr) {
        XP_HIP_CHECK(call.clear(grad_w_out, out_bytes));
      }
      if (grad_bias_in != nullptr) {
        XP_HIP_CHECK(call.clear(grad_bias_in, static_cast<size_t>(wide) * 4));
      }
      if (grad_bias_out != nullptr) {
        XP_HIP_CHECK(call.clear(grad_bias_out, static_cast<size_t>(hidden) * 4));
      }
    }
    return XP_OK;
  }
  XP_TRY(check_rows("input projection's weights", w_in, hidden, hidden, element, true));
  XP_TRY(check_rows("output projection's weights", w_out, width, width, element, true));
  XP_TRY(check_rows("kept projection", projected, ld_projected, wide, element, false));
  XP_TRY(check_rows("output gradient", grad_out, ld_grad, hidden, element, true));
  if (grad_w_in != nullptr) {
    XP_TRY(check_rows("hidden states", x, ld_x, hidden, element, true));
  }
  if (grad_x != nullptr) {
    XP_TRY(check_rows("gradient of the hidden states", grad_x, ld_grad_x, hidden, element, false));
  }
  const DenseRegions at = dense_regions(static_cast<unsigned char *>(workspace), capacity, hidden, width, wide, element);
  XP_REQUIRE(workspace != nullptr && aligned16(workspace) && workspace_bytes >= at.bytes,
             "workspace is missing, unaligned or smaller than xp_dense_backward_workspace_bytes");
  XP_REQUIRE(apart({span_of_rows(grad_x, ld_grad_x, hidden, rows, element), span_of(grad_w_in, in_bytes),
                    span_of(grad_w_out, out_bytes), span_of(grad_bias_in, static_cast<size_t>(wide) * 4),
                    span_of(grad_bias_out, static_cast<size_t>(hidden) * 4), span_of(workspace, at.bytes)},
                   {span_of_rows(grad_w_in == nullptr ? nullptr : x, ld_x, hidden, rows, element),
                    span_of_rows(projected, ld_projected, wide, rows, element), span_of_rows(grad_out, ld_grad, hidden, rows, element),
                    span_of(w_in, static_cast<size_t>(wide * hidden) * element),
                    span_of(w_out, static_cast<size_t>(hidden * width) * element)}),
             "gradients and workspace must overlap neither the operands nor each other");
  call.scratch = at.scratch;
  call.scratch_bytes = at.scratch_bytes;

  const bool thin = thin_rows(rows, element);
  PadArgs pads{};
  const ProductOperand grad = call.padded(grad_out, rows, hidden, ld_grad, at.grad, pads);
  const ProductOperand w_out_rows = call.padded(w_out, hidden, width, width, at.w_out, pads);
  ProductOperand w_in_rows{};
  ProductOperand inputs{};
  if (grad_x != nullptr) {
    w_in_rows = call.padded(w_in, wide, hidden, hidden, at.w_in, pads);
  }
  if (grad_w_in != nullptr && !thin) {
    inputs = call.padded(x, rows, hidden, ld_x, at.x, pads);
  }
  XP_HIP_CHECK(call.pad(pads));
  const int64_t through_ld = padded_width(wide, element);
  const ProductOperand through{at.through, through_ld, 0};
  const ProductOperand activated{at.activated, padded_width(width, element), 0};
  if (grad_x != nullptr || grad_w_in != nullptr || grad_bias_in != nullptr || grad_w_out != nullptr) {
    args.a = grad;
    args.b = w_out_rows;
    args.m = rows;
    args.n = width;
    args.k = hidden;
    args.out = at.through;
    args.ld_out = through_ld;
    args.base = projected;
    args.ld_base = ld_projected;
    args.extra = at.activated;
    args.ld_extra = activated.ld;
    args.interleaved = order == XP_GATE_UP_INTERLEAVED;
    args.column_sums = grad_bias_in != nullptr ? at.bands : nullptr;
    args.alpha = 1.0f;
    XP_HIP_CHECK(call.product(args, ProductEpilogue::kGradient, false, true));
  }
  // The biases' gradients, together where the outputs' needs no bands of its own (they would share the kept ones' place).
  const ColumnSumArgs in_bands{at.bands, nullptr, grad_bias_in, (rows + kBandRows - 1) / kBandRows, wide, wide, 0, 0, accumulate};
  const ColumnSumArgs out_rows{grad_out, nullptr, grad_bias_out, rows, hidden, ld_grad, 0, 0, accumulate};
  const bool out_at_once = grad_bias_out != nullptr && rows <= kRowsAtOnce;
  XP_HIP_CHECK(call.row_sums(out_at_once ? &out_rows : nullptr, grad_bias_in != nullptr ? &in_bands : nullptr));
  if (grad_x != nullptr) {
    if (through_ld != wide) {
      const int64_t words = rows * (through_ld - wide) * static_cast<int64_t>(element) / 2;
      clear_pad_kernel<<<blocks_of(words, 256), 256, 0, call.stream>>>(
          PadJob{nullptr, at.through, rows, wide, 0, through_ld, 0}, static_cast<int>(element));
      XP_HIP_CHECK(hipGetLastError());
    }
  }
  ProductGroup group{};
  const bool present[3] = {grad_x != nullptr, grad_w_in != nullptr && !thin, grad_w_out != nullptr && !thin};
  if (present[0]) {
    group.part[0] = inputs_args(through, w_in_rows, rows, wide, hidden, grad_x, ld_grad_x, dtype);
  }
  if (present[1]) {
    group.part[1] = outer_args(through, wide, inputs, hidden, rows, grad_w_in, grad_w_dtype, accumulate != 0);
  }
  if (present[2]) {
    group.part[2] = outer_args(grad, hidden, activated, width, rows, grad_w_out, grad_w_dtype, accumulate != 0);
  }
  if (thin) {
    const int few = static_cast<int>(rows);
    const ThinOuterArgs in{at.through, x, grad_w_in, through_ld, ld_x, wide, hidden, few, grad_w_dtype, accumulate};
    const ThinOuterArgs out{grad_out, at.activated, grad_w_out, ld_grad, activated.ld, hidden, width, few, grad_w_dtype, accumulate};
    XP_HIP_CHECK(call.thin_gradients(present[0] ? &group.part[0] : nullptr,
                                     {grad_w_in == nullptr ? nullptr : &in, grad_w_out == nullptr ? nullptr : &out}, few));
  } else {
    XP_HIP_CHECK(call.products(group, present));
  }
  if (grad_bias_out != nullptr && !out_at_once) {
    XP_HIP_CHECK(call.column_sums(grad_out, rows, hidden, ld_grad, at.bands, grad_bias_out, accumulate != 0));
  }
  return XP_OK;
}

}  // extern "C"
