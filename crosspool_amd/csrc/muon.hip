// Orthogonal updates: U S V^T of an update becomes nearly U V^T by Newton-Schulz products, for batches of
// matrices, alone or inside an optimiser's step.  No counterpart in the reference.
//
//   X0 = G / (|G| + eps),  X <- a X + (b A + c A^2) X,  A = X X^T  (wide) or X <- a X + X (b A + c A^2), A = X^T X
//
// (Frobenius norm, a = 3.4445, b = -4.7750, c = 2.0315: the polynomial takes every singular value in (0, 1] to
// about [0.7, 1.2] within five steps.)  The Gram matrix is the short side's; it and its square are symmetric, so
// only tiles on and below their diagonals are computed.  A wide and a tall matrix differ in the storage orders of
// the products alone: nothing is transposed.
//
// Precision.  16-bit payloads run on fp16 matrix products with fp32 sums: X, A and b A + c A^2 are rounded to
// fp16 (2^-12 of a value), eight times finer than the bf16 results, and no product costs more for it.  |X| <= 1 in
// the Frobenius norm at first and singular values stay below 1.3, so every value of X and A is below 1.7 and of
// b A + c A^2 below 9: stored times 2^12 they stay below fp16's 65504, and what a typical element of a 16384 x
// 65536 matrix comes to, 2^-15, is at 2^-3, far above its subnormal numbers.  fp32 payloads stay in fp32.
// Iterating on the Gram matrices alone (X once at the end) needs fewer products where the long side is long, but
// squares singular values: a rounding of A, 2^-12 of its largest, grows by a^2 a step in the directions of small
// ones, past their true values.

#include "product_kernels.hpp"
#include "xp_entry.hpp"

#include <cmath>

namespace xp {
namespace {

constexpr float kA = 3.4445f;
constexpr float kB = -4.7750f;
constexpr float kC = 2.0315f;
constexpr float kFp16Scale = 4096.0f;

struct MuonTensor {
  void *data;
  int64_t matrix;  // elements between matrices
  int64_t row;     // between rows
  int32_t dtype;
};

struct MuonArgs {
  MuonTensor gradient;
  MuonTensor momentum;      // data null: orthogonalise the gradient itself
  MuonTensor new_momentum;  // fp32
  void *x;                  // [matrices, rows, padded]
  double *squares;          // [matrices, parts]
  int64_t rows;
  int64_t columns;
  int64_t padded;
  int64_t parts;            // workgroups of a matrix
  float factor;
  float eps;
  float scale;
  int32_t nesterov;
  int32_t x_dtype;
};

// The update's eight values at (row, column); with `fresh` the momentum is still the old one and its new value
// is stored.
__device__ __forceinline__ void update_values(const MuonArgs &a, int64_t matrix, int64_t row, int64_t column, int count, bool fresh,
                                              float (&value)[8]) {
  load_values(a.gradient.data, matrix * a.gradient.matrix + row * a.gradient.row + column, a.gradient.dtype, count, value);
  if (a.new_momentum.data == nullptr) {
    return;
  }
  const MuonTensor &source = fresh ? a.momentum : a.new_momentum;
  float momentum[8];
  load_values(source.data, matrix * source.matrix + row * source.row + column, kDtypeF32, count, momentum);
  if (fresh) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      momentum[j] = a.factor * momentum[j] + value[j];
    }
    store_values(a.new_momentum.data, matrix * a.new_momentum.matrix + row * a.new_momentum.row + column, kDtypeF32, count, momentum);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    value[j] = a.nesterov ? value[j] + a.factor * momentum[j] : momentum[j];
  }
}

__device__ __forceinline__ double wave_sum64(double value) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) {
    value += __shfl_xor(value, offset, kWave);
  }
  return value;
}

// The sum of a workgroup's values, in wave order, for all its threads.
__device__ __forceinline__ double group_sum(double value) {
  __shared__ double waves[4];
  value = wave_sum64(value);
  if ((threadIdx.x & 63) == 0) {
    waves[threadIdx.x >> 6] = value;
  }
  __syncthreads();
  return (waves[0] + waves[1]) + (waves[2] + waves[3]);
}

// New momentum, and the sum of the update's squares per workgroup, in 64 bits: an fp32 update's squares may
// pass fp32's range.  Bound by memory: 32 bf16 gradients of 2048 x 768 with their momentum, 503 MB, 108 us (4.7 TB/s).
__global__ __launch_bounds__(256) void muon_norm_kernel(MuonArgs a) {
  const int64_t groups = (a.columns + 7) / 8;
  const int64_t items = a.rows * groups;
  const int64_t matrix = blockIdx.y;
  double squares = 0.0;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; item < items; item += a.parts * 256) {
    const int64_t row = item / groups;
    const int64_t column = (item - row * groups) * 8;
    const int count = a.columns - column < 8 ? static_cast<int>(a.columns - column) : 8;
    float value[8];
    update_values(a, matrix, row, column, count, true, value);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      squares += j < count ? static_cast<double>(value[j]) * static_cast<double>(value[j]) : 0.0;
    }
  }
  const double sum = group_sum(squares);
  if (threadIdx.x == 0) {
    a.squares[matrix * a.parts + blockIdx.x] = sum;
  }
}

// X0 in rows of whole groups of eight columns, zeros behind the last column.  Bound by memory (the same matrices 403 MB,
// 80 us, 5 TB/s): the norm has to be known before the first value can be stored, so the update is read twice.
__global__ __launch_bounds__(256) void muon_scale_kernel(MuonArgs a) {
  const int64_t groups = (a.columns + 7) / 8;
  const int64_t items = a.rows * groups;
  const int64_t matrix = blockIdx.y;
  double squares = 0.0;
  for (int64_t part = threadIdx.x; part < a.parts; part += 256) {
    squares += a.squares[matrix * a.parts + part];
  }
  const double norm = sqrt(group_sum(squares));
  // A norm near the ends of fp32's range has a reciprocal past them (of a zero matrix and a tiny eps infinite: NaN): 64 bits.
  const double exact = static_cast<double>(a.scale) / (norm + static_cast<double>(a.eps));
  const float factor = static_cast<float>(exact);
  const bool normal = factor >= 0x1p-126f && factor <= 0x1.fffffep127f;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; item < items; item += a.parts * 256) {
    const int64_t row = item / groups;
    const int64_t column = (item - row * groups) * 8;
    const int count = a.columns - column < 8 ? static_cast<int>(a.columns - column) : 8;
    float value[8];
    update_values(a, matrix, row, column, count, false, value);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      value[j] = j >= count ? 0.0f : normal ? value[j] * factor : static_cast<float>(static_cast<double>(value[j]) * exact);
    }
    store_values(a.x, (matrix * a.rows + row) * a.padded + column, a.x_dtype, 8, value);
  }
}

constexpr int64_t kMaxMatrices = 4096;
constexpr int64_t kMaxShort = int64_t{1} << 16;
constexpr int64_t kMaxLong = int64_t{1} << 20;
constexpr int64_t kMaxElements = int64_t{1} << 36;
constexpr int64_t kMaxSteps = 16;
constexpr const char *kMuonExtents =
    "orthogonal updates take 1 to 4096 matrices with a short side of 1 to 65536 and a long side of at most 1048576, 2^36 values in all";

struct MuonShape {
  int64_t matrices;
  int64_t rows;
  int64_t columns;
  int dtype;
  bool tall() const { return rows > columns; }
  int64_t shorter() const { return std::min(rows, columns); }
  int64_t longer() const { return std::max(rows, columns); }
};

bool muon_shape_valid(const MuonShape &shape) {
  return dtype_bytes(shape.dtype) != 0 && shape.matrices >= 1 && shape.matrices <= kMaxMatrices && shape.rows >= 1 &&
         shape.columns >= 1 && shape.shorter() <= kMaxShort && shape.longer() <= kMaxLong &&
         shape.rows * shape.columns <= kMaxElements / shape.matrices;
}

int64_t eights(int64_t value) { return (value + 7) / 8 * 8; }

struct MuonRegions {
  void *x[2];
  void *gram;
  void *polynomial;
  double *squares;
  float *scratch;
  size_t scratch_bytes;
  size_t bytes;
  int64_t parts;
};

MuonRegions muon_regions(unsigned char *base, const MuonShape &shape) {
  MuonRegions found{};
  size_t used = 0;
  const auto take = [&](size_t bytes) -> void * {
    void *at = base == nullptr ? nullptr : base + used;
    used += (bytes + 255) / 256 * 256;
    return at;
  };
  const size_t element = shape.dtype == XP_DTYPE_F32 ? 4 : 2;
  const int64_t s = shape.shorter();
  const size_t x_bytes = static_cast<size_t>(shape.matrices * shape.rows * eights(shape.columns)) * element;
  const size_t gram_bytes = static_cast<size_t>(shape.matrices * s * eights(s)) * element;
  found.x[0] = take(x_bytes);
  found.x[1] = take(x_bytes);
  found.gram = take(gram_bytes);
  found.polynomial = take(gram_bytes);
  // Workgroups of the element-wise kernels: a few rounds of the chip over all matrices.
  const int64_t items = shape.rows * ((shape.columns + 7) / 8);
  found.parts = std::max<int64_t>(1, std::min((items + 255) / 256, std::max<int64_t>(1, 2048 / shape.matrices)));
  found.squares = static_cast<double *>(take(static_cast<size_t>(shape.matrices * found.parts) * sizeof(double)));
  const int es = static_cast<int>(element);
  const auto scratch = [&](int64_t m, int64_t n, int64_t k, bool symmetric) {
    return product_scratch_bytes(plan_product(m, n, k, shape.matrices, es, symmetric, SIZE_MAX));
  };
  found.scratch_bytes = std::max({scratch(s, s, shape.longer(), true), scratch(s, s, s, true),
                                  scratch(shape.rows, shape.columns, s, false)});
  found.scratch = static_cast<float *>(take(found.scratch_bytes));
  found.bytes = used;
  return found;
}

// Rows of a batch of matrices lie apart: matrices one behind another, or their rows between one another's.
bool rows_apart(const xp_matrices &tensor, const MuonShape &shape) {
  const int64_t inner = (shape.rows - 1) * tensor.row_stride + shape.columns;
  const bool behind = tensor.row_stride >= shape.columns && (shape.matrices == 1 || tensor.matrix_stride >= inner);
  const bool between = tensor.matrix_stride >= shape.columns &&
                       (shape.rows == 1 || tensor.row_stride >= (shape.matrices - 1) * tensor.matrix_stride + shape.columns);
  return behind || between;
}

int check_matrices(const char *name, const xp_matrices *tensor, const MuonShape &shape, size_t element) {
  XP_REQUIRE(tensor != nullptr && tensor->data != nullptr && aligned_to(tensor->data, element),
             std::string(name) + " must be non-null and aligned to their element size");
  XP_REQUIRE(tensor->row_stride >= 0 && tensor->matrix_stride >= 0 && tensor->row_stride <= (int64_t{1} << 32) &&
                 tensor->matrix_stride <= (int64_t{1} << 40) && rows_apart(*tensor, shape),
             std::string(name) + " must have contiguous, separate rows");
  return XP_OK;
}

Span matrices_span(const xp_matrices *tensor, const MuonShape &shape, size_t element) {
  if (tensor == nullptr) {
    return span_of(nullptr, 0);
  }
  const int64_t elements = (shape.matrices - 1) * tensor->matrix_stride + (shape.rows - 1) * tensor->row_stride + shape.columns;
  return span_of(tensor->data, static_cast<size_t>(elements) * element);
}

bool same_matrices(const xp_matrices &a, const xp_matrices &b) {
  return a.data == b.data && a.matrix_stride == b.matrix_stride && a.row_stride == b.row_stride;
}

// What a step of the optimiser adds to the orthogonalisation.
struct MuonStep {
  const xp_matrices *weights = nullptr;
  int weights_dtype = 0;
  float keep = 0.0f;
  float step = 0.0f;
};

int muon_run(const MuonShape &shape, MuonArgs args, int steps, const xp_matrices &out, int out_dtype, const MuonStep &step,
             const MuonRegions &at, hipStream_t stream) {
  const bool fp32 = shape.dtype == XP_DTYPE_F32;
  const int dtype = fp32 ? kDtypeF32 : kDtypeF16;
  const float scale = fp32 ? 1.0f : kFp16Scale;
  const int64_t s = shape.shorter();
  const int64_t padded = eights(shape.columns);
  const int64_t gram_ld = eights(s);
  args.x = at.x[0];
  args.squares = at.squares;
  args.rows = shape.rows;
  args.columns = shape.columns;
  args.padded = padded;
  args.parts = at.parts;
  args.scale = scale;
  args.x_dtype = dtype;
  KernelLaunch kernel;
  kernel.grid = dim3(static_cast<unsigned>(at.parts), static_cast<unsigned>(shape.matrices));
  kernel.block = dim3(256);
  kernel.set_args(args);
  kernel.func = reinterpret_cast<const void *>(&muon_norm_kernel);
  XP_HIP_CHECK(launch(kernel, stream));
  kernel.func = reinterpret_cast<const void *>(&muon_scale_kernel);
  XP_HIP_CHECK(launch(kernel, stream));

  ProductArgs common{};
  common.batch = static_cast<int32_t>(shape.matrices);
  common.partials = at.scratch;
  const auto stored = [&](void *data, int64_t rows, int64_t ld) { return ProductOperand{data, ld, rows * ld}; };
  for (int i = 0; i < steps; ++i) {
    const ProductOperand x = stored(at.x[i % 2], shape.rows, padded);
    const ProductOperand gram = stored(at.gram, s, gram_ld);
    const ProductOperand polynomial = stored(at.polynomial, s, gram_ld);
    ProductArgs product = common;
    product.m = product.n = s;
    product.symmetric = 1;
    product.padded_out = 1;
    product.ld_out = gram_ld;
    product.batch_out = gram.batch;
    product.out_dtype = static_cast<int8_t>(dtype);
    // A
    product.a = product.b = x;
    product.k = shape.longer();
    product.out = at.gram;
    product.alpha = 1.0f / scale;
    XP_HIP_CHECK(launch_product(product, ProductEpilogue::kStore, shape.tall(), shape.tall(), dtype, at.scratch_bytes, stream));
    // b A + c A A
    product.a = product.b = gram;
    product.k = s;
    product.out = at.polynomial;
    product.alpha = kC / scale;
    product.beta = kB;
    product.base = at.gram;
    product.ld_base = gram_ld;
    product.batch_base = gram.batch;
    product.base_dtype = static_cast<int8_t>(dtype);
    XP_HIP_CHECK(launch_product(product, ProductEpilogue::kStore, false, false, dtype, at.scratch_bytes, stream));
    // a X + (b A + c A A) X
    product = common;
    const bool last = i + 1 == steps;
    product.m = shape.rows;
    product.n = shape.columns;
    product.k = s;
    product.a = shape.tall() ? x : polynomial;
    product.b = shape.tall() ? polynomial : x;
    product.base = x.data;
    product.ld_base = padded;
    product.batch_base = x.batch;
    product.base_dtype = static_cast<int8_t>(dtype);
    product.alpha = last ? 1.0f / (scale * scale) : 1.0f / scale;
    product.beta = last ? kA / scale : kA;
    if (last) {
      product.out = out.data;
      product.ld_out = out.row_stride;
      product.batch_out = out.matrix_stride;
      product.out_dtype = static_cast<int8_t>(out_dtype);
      if (step.weights != nullptr) {
        product.extra = step.weights->data;
        product.ld_extra = step.weights->row_stride;
        product.batch_extra = step.weights->matrix_stride;
        product.extra_dtype = static_cast<int8_t>(step.weights_dtype);
        product.keep = step.keep;
        product.step = step.step;
      }
    } else {
      product.out = at.x[(i + 1) % 2];
      product.ld_out = padded;
      product.batch_out = x.batch;
      product.out_dtype = static_cast<int8_t>(dtype);
      product.padded_out = 1;
    }
    XP_HIP_CHECK(launch_product(product, ProductEpilogue::kStore, false, !shape.tall(), dtype, at.scratch_bytes, stream));
  }
  return XP_OK;
}

MuonTensor muon_tensor(const xp_matrices &tensor, int dtype) {
  return {tensor.data, tensor.matrix_stride, tensor.row_stride, dtype};
}

int check_muon(const MuonShape &shape, int steps, float eps) {
  XP_REQUIRE(muon_shape_valid(shape), kMuonExtents);
  XP_REQUIRE(steps >= 1 && steps <= kMaxSteps, "orthogonal updates take 1 to 16 steps");
  XP_REQUIRE(eps > 0.0f && std::isfinite(eps), "eps must be positive and finite");
  return XP_OK;
}

}  // namespace
}  // namespace xp

using namespace xp;

extern "C" {

size_t xp_muon_workspace_bytes(int64_t matrices, int64_t rows, int64_t columns, int dtype) {
  const MuonShape shape{matrices, rows, columns, dtype};
  return muon_shape_valid(shape) ? muon_regions(nullptr, shape).bytes : 0;
}

int xp_muon_orthogonalize(const xp_matrices *updates, int64_t matrices, int64_t rows, int64_t columns, int dtype, int steps,
                          float eps, const xp_matrices *output, void *workspace, size_t workspace_bytes, xp_stream_t stream) {
  const MuonShape shape{matrices, rows, columns, dtype};
  if (const int status = check_muon(shape, steps, eps); status != XP_OK) {
    return status;
  }
  const size_t element = dtype_bytes(dtype);
  if (const int status = check_matrices("updates", updates, shape, element); status != XP_OK) {
    return status;
  }
  if (const int status = check_matrices("orthogonal updates", output, shape, element); status != XP_OK) {
    return status;
  }
  const MuonRegions at = muon_regions(static_cast<unsigned char *>(workspace), shape);
  XP_REQUIRE(workspace != nullptr && aligned16(workspace) && workspace_bytes >= at.bytes,
             "workspace is missing, unaligned or smaller than xp_muon_workspace_bytes");
  const Span read = matrices_span(updates, shape, element);
  const Span written = matrices_span(output, shape, element);
  XP_REQUIRE(same_matrices(*updates, *output) || !overlaps(read, written), "the output may be the updates only whole");
  XP_REQUIRE(!touches(span_of(workspace, at.bytes), {read, written}), "the workspace must not overlap the operands");
  MuonArgs args{};
  args.gradient = muon_tensor(*updates, dtype);
  args.eps = eps;
  return muon_run(shape, args, steps, *output, dtype, MuonStep{}, at, static_cast<hipStream_t>(stream));
}

int xp_muon_step(const xp_matrices *weights, const xp_matrices *gradients, const xp_matrices *momentum,
                 const xp_matrices *new_weights, const xp_matrices *new_momentum, int64_t matrices, int64_t rows, int64_t columns,
                 int dtype, int weights_dtype, int steps, float eps, float learning_rate, float weight_decay, float momentum_factor,
                 int nesterov, float update_scale, void *workspace, size_t workspace_bytes, xp_stream_t stream) {
  const MuonShape shape{matrices, rows, columns, dtype};
  if (const int status = check_muon(shape, steps, eps); status != XP_OK) {
    return status;
  }
  XP_REQUIRE(weights_dtype == dtype || weights_dtype == XP_DTYPE_F32, "weights are of the gradients' dtype or fp32");
  XP_REQUIRE(std::isfinite(learning_rate) && std::isfinite(weight_decay) && std::isfinite(update_scale) && momentum_factor >= 0.0f &&
                 momentum_factor < 1.0f,
             "learning rate, decay and scale must be finite, and the momentum factor in [0, 1)");
  const size_t element = dtype_bytes(dtype);
  const size_t kept = dtype_bytes(weights_dtype);
  struct {
    const char *name;
    const xp_matrices *tensor;
    size_t element;
  } const tensors[] = {{"gradients", gradients, element}, {"momentum", momentum, 4}, {"new momentum", new_momentum, 4},
                       {"weights", weights, kept}, {"new weights", new_weights, kept}};
  for (const auto &each : tensors) {
    if (const int status = check_matrices(each.name, each.tensor, shape, each.element); status != XP_OK) {
      return status;
    }
  }
  const MuonRegions at = muon_regions(static_cast<unsigned char *>(workspace), shape);
  XP_REQUIRE(workspace != nullptr && aligned16(workspace) && workspace_bytes >= at.bytes,
             "workspace is missing, unaligned or smaller than xp_muon_workspace_bytes");
  const Span read_gradients = matrices_span(gradients, shape, element);
  const Span read_momentum = matrices_span(momentum, shape, 4);
  const Span read_weights = matrices_span(weights, shape, kept);
  const Span write_momentum = matrices_span(new_momentum, shape, 4);
  const Span write_weights = matrices_span(new_weights, shape, kept);
  XP_REQUIRE((same_matrices(*momentum, *new_momentum) || !overlaps(read_momentum, write_momentum)) &&
                 (same_matrices(*weights, *new_weights) || !overlaps(read_weights, write_weights)),
             "new momentum and weights may be the old ones only whole");
  XP_REQUIRE(!touches(write_momentum, {read_gradients, read_weights, write_weights}) &&
                 !touches(write_weights, {read_gradients, read_momentum}) &&
                 !touches(span_of(workspace, at.bytes),
                          {read_gradients, read_momentum, read_weights, write_momentum, write_weights}),
             "new momentum, new weights and workspace must overlap neither the operands nor each other");
  MuonArgs args{};
  args.gradient = muon_tensor(*gradients, dtype);
  args.momentum = muon_tensor(*momentum, kDtypeF32);
  args.new_momentum = muon_tensor(*new_momentum, kDtypeF32);
  args.eps = eps;
  args.factor = momentum_factor;
  args.nesterov = nesterov != 0;
  const MuonStep step{weights, weights_dtype, 1.0f - learning_rate * weight_decay, learning_rate * update_scale};
  return muon_run(shape, args, steps, *new_weights, weights_dtype, step, at, static_cast<hipStream_t>(stream));
}

}  // extern "C"
