// Matrix products of the training operators: out[m][n] = epilogue(sum over k of A(m, k) B(n, k)), every
// operand stored with its reduction axis along its rows or across them.  Argument records and plans; the
// kernels are in product_kernels.hpp, instantiated for one payload in product_{bf16,f16,f32}.hip.
#pragma once

#include "xp_kernels.hpp"

namespace xp {

// What a product does with its fp32 sums.
enum class ProductEpilogue : int {
  kStore = 0,     // out = alpha sum + beta base + bias; or keep extra - step (alpha sum + beta base)
  kActivate = 1,  // out = sum + bias rounded to the payload, extra = the activation of the unrounded value
  kGradient = 2,  // a gradient of an activation's outputs: out = the gradient of its inputs (base), extra = its outputs
};

// One operand [rows, k]: element (r, k) at data[r ld + k], or where the reduction axis runs across its rows
// (`cols` of a kernel) at data[k ld + r].
struct ProductOperand {
  const void *data;
  int64_t ld;
  int64_t batch;  // elements between the matrices of a batch
};

struct ProductArgs {
  ProductOperand a;
  ProductOperand b;
  int64_t m;
  int64_t n;
  int64_t k;
  float *partials;     // [workers + split, tile, tile]: sums of the split tiles' pieces
  void *out;
  int64_t ld_out;
  int64_t batch_out;
  const void *base;
  int64_t ld_base;
  int64_t batch_base;
  void *extra;         // kStore: values read (weights), may be null; else written
  int64_t ld_extra;
  int64_t batch_extra;
  const float *bias;   // fp32 [n] or null
  float *column_sums;  // kGradient: sums of the unrounded gradients over bands of rows [bands, 2 n or n], or null
  int64_t halves;      // kActivate: not 0, B's rows and the output's columns are all Gates, then as many Ups; a tile works on pairs
  float alpha;
  float beta;          // 0: base is not read
  float keep;
  float step;
  int32_t batch;
  int32_t tile_rows;   // tiles down and across one matrix
  int32_t tile_cols;
  int32_t whole;       // tiles that one workgroup computes each
  int32_t split;       // the tiles behind them, shared by
  int32_t workers;     // as many workgroups,
  int32_t share;       // `share` slabs each,
  int32_t longer;      // the first `longer` of them one more
  int32_t each;        // workers of a tile, where all have the same number
  int8_t out_dtype;
  int8_t base_dtype;
  int8_t extra_dtype;
  int8_t symmetric;    // A and B are one operand: tiles below the diagonal are computed and mirrored
  int8_t padded_out;   // kStore: the output's rows are whole groups of eight columns, zeros behind column n
  int8_t interleaved;  // kGradient: Gate/Up pairs in neighbouring columns, else in halves
  ActivationArgs act;
};
static_assert(sizeof(ProductArgs) <= 288, "a kernel's argument record");

// Tile sizes, stages of LDS and workgroups that a CU holds (fp32: k128Pairs, k64 and k32).
enum class ProductTiles : int { k256 = 0, k128Pairs = 1, k128Deep = 2, k64 = 3, k32 = 4 };
constexpr int tile_size(ProductTiles tiles) {
  return tiles == ProductTiles::k256 ? 256 : tiles == ProductTiles::k64 ? 64 : tiles == ProductTiles::k32 ? 32 : 128;
}

struct ProductPlan {
  ProductTiles tiles;
  int64_t whole;
  int64_t split;
  int64_t workers;
  double us;  // as modelled
};

// The fastest plan for a product in a workspace of `scratch` bytes for its split tiles' sums; `us` below 0 where no launch
// holds all tiles.
ProductPlan plan_product(int64_t m, int64_t n, int64_t k, int64_t batch, int element_bytes, bool symmetric, size_t scratch);
size_t product_scratch_bytes(const ProductPlan &plan);

// Rows of a band of ProductArgs::column_sums.
constexpr int64_t kBandRows = 32;

struct ProductLaunch {
  KernelLaunch main;
  KernelLaunch join;  // empty without split tiles
};
// `dtype` is that of the operands.  Fills the tiles' and workers' counts of the record from the plan.
ProductLaunch make_product(const ProductArgs &args, const ProductPlan &plan, ProductEpilogue epilogue, bool a_cols, bool b_cols,
                           int dtype);

// The product as planned for its sizes, a batch of too many tiles for one launch in several.
hipError_t launch_product(const ProductArgs &args, ProductEpilogue epilogue, bool a_cols, bool b_cols, int dtype,
                          size_t scratch_bytes, hipStream_t stream);

// Products of one backward pass that do not depend on each other, kStore: an inputs' gradient (part 0, blocks 0 where there
// is none) and up to two weights' gradients.
struct ProductGroup {
  ProductArgs part[3];
  int32_t blocks[3];
};
// All of them, in one launch where that is modelled as faster than one after another.  `present` says which there are.
hipError_t launch_products(ProductGroup &group, const bool (&present)[3], int dtype, size_t scratch_bytes, hipStream_t stream);

template <class P>
struct ProductKernels {
  static const void *group(ProductTiles tiles);
  static const void *main(ProductTiles tiles, ProductEpilogue epilogue, bool a_cols, bool b_cols);
  static const void *join(int tile, ProductEpilogue epilogue);
};

}  // namespace xp
