// Plans and launches of the training operators' products.
#include "product.hpp"
#include "xp_elements.hpp"

#include <algorithm>
#include <cmath>

namespace xp {

// A product's time in microseconds.  A CU's workgroups share its throughput: `slab[i]` is the time of one slab in
// each of i + 1 workgroups on it (as many as fit), and a tile costs `tile` besides (first loads, epilogue), a split
// piece `piece` (its sums go out in fp32).  Measured on MI355X with 12 and 48 slabs on 128 to 1024 workgroups, for the
// three storage orders, whose times differ by less than 10 %.
namespace {
struct ProductCost {
  ProductTiles tiles;
  int together;
  double slab[3];
  double tile;
  double piece;
};
constexpr ProductCost kCosts16[] = {{ProductTiles::k256, 1, {1.36, 0.0, 0.0}, 9.5, 14.0},
                                    {ProductTiles::k128Pairs, 2, {0.72, 0.87, 0.0}, 5.0, 6.0},
                                    {ProductTiles::k128Deep, 1, {0.49, 0.0, 0.0}, 5.0, 6.0},
                                    {ProductTiles::k64, 3, {0.25, 0.41, 0.57}, 1.5, 2.0}};
constexpr ProductCost kCosts32[] = {{ProductTiles::k256, 1, {7.45, 0.0, 0.0}, 13.0, 16.0},
                                    {ProductTiles::k128Pairs, 2, {2.03, 3.8, 0.0}, 7.0, 8.0},
                                    {ProductTiles::k128Deep, 1, {2.0, 0.0, 0.0}, 7.0, 8.0},
                                    {ProductTiles::k64, 3, {0.59, 1.02, 1.5}, 2.0, 2.5}};
constexpr int64_t kCus = 256;
constexpr double kLaunchUs = 3.5;
constexpr double kJoinUs = 3.0;
constexpr double kBytesPerUs = 4e6;
constexpr int64_t kMinSlabs = 2;  // of a worker

// `groups` workgroups of `slabs` slabs each, all of one kind, on the chip.
double rounds_us(const ProductCost &cost, int64_t groups, double slabs, double each) {
  const int64_t full = groups / (kCus * cost.together);
  const int64_t rest = (groups - full * kCus * cost.together + kCus - 1) / kCus;
  return static_cast<double>(full) * (slabs * cost.slab[cost.together - 1] + each) +
         (rest > 0 ? slabs * cost.slab[rest - 1] + each : 0.0);
}
}  // namespace

size_t product_scratch_bytes(const ProductPlan &plan) {
  const size_t size = static_cast<size_t>(tile_size(plan.tiles));
  return plan.split > 0 ? static_cast<size_t>(plan.workers + plan.split) * size * size * sizeof(float) : 0;
}

ProductPlan plan_product(int64_t m, int64_t n, int64_t k, int64_t batch, int element_bytes, bool symmetric, size_t scratch) {
  const int64_t slab = 128 / element_bytes;
  const int64_t slabs = (k + slab - 1) / slab;
  ProductPlan best{};
  best.us = -1.0;
  for (const ProductCost &cost : element_bytes == 4 ? kCosts32 : kCosts16) {
    const int64_t size = tile_size(cost.tiles);
    const int64_t rows = (m + size - 1) / size;
    const int64_t cols = (n + size - 1) / size;
    const int64_t tiles = batch * (symmetric ? rows * (rows + 1) / 2 : rows * cols);
    const auto consider = [&](int64_t whole, int64_t workers) {
      ProductPlan plan{cost.tiles, whole, tiles - whole, workers, kLaunchUs};
      const int64_t together = plan.split * slabs;
      if (plan.split > 0 && (workers < plan.split || workers * kMinSlabs > together || product_scratch_bytes(plan) > scratch)) {
        return;
      }
      if (whole > 0) {
        plan.us += rounds_us(cost, whole, static_cast<double>(slabs), cost.tile);
      }
      if (plan.split > 0) {
        // A worker whose run crosses a tile's end stores twice.
        const double pieces = workers % plan.split == 0 ? 1.0 : 2.0;
        plan.us += rounds_us(cost, workers, std::ceil(static_cast<double>(together) / static_cast<double>(workers)), cost.piece * pieces) +
                   kJoinUs + static_cast<double>(product_scratch_bytes(plan)) / kBytesPerUs;
      }
      if (best.us < 0.0 || plan.us < best.us) {
        best = plan;
      }
    };
    consider(tiles, 0);
    const int64_t slots = kCus * cost.together;
    const int64_t full = tiles / slots * slots;
    if (full == tiles || cost.tiles == ProductTiles::k256) {
      continue;
    }
    const int64_t split = tiles - full;
    for (int64_t per_cu = 1; per_cu <= cost.together; ++per_cu) {
      consider(full, kCus * per_cu);
      // The same number of workers for every tile: none crosses a tile's end.
      consider(full, kCus * per_cu / split * split);
    }
    for (int64_t each = 2; each * split < kCus; ++each) {
      consider(full, each * split);
    }
  }
  return best;
}

ProductLaunch make_product(const ProductArgs &args, const ProductPlan &plan, ProductEpilogue epilogue, bool a_cols, bool b_cols,
                           int dtype) {
  ProductLaunch launches;
  ProductArgs record = args;
  record.whole = static_cast<int32_t>(plan.whole);
  record.split = static_cast<int32_t>(plan.split);
  record.workers = static_cast<int32_t>(plan.workers);
  const int size = tile_size(plan.tiles);
  launches.main.func = dtype == kDtypeF32   ? ProductKernels<F32Payload>::main(plan.tiles, epilogue, a_cols, b_cols)
                       : dtype == kDtypeF16 ? ProductKernels<F16Payload>::main(plan.tiles, epilogue, a_cols, b_cols)
                                            : ProductKernels<Bf16Payload>::main(plan.tiles, epilogue, a_cols, b_cols);
  launches.main.grid = dim3(static_cast<unsigned>(plan.whole + plan.workers));
  launches.main.block = dim3(size == 256 ? 512 : 256);
  launches.main.set_args(record);
  if (plan.split > 0) {
    launches.join.func = dtype == kDtypeF32   ? ProductKernels<F32Payload>::join(size, epilogue)
                         : dtype == kDtypeF16 ? ProductKernels<F16Payload>::join(size, epilogue)
                                              : ProductKernels<Bf16Payload>::join(size, epilogue);
    launches.join.grid = dim3(static_cast<unsigned>(plan.split * (size / 64) * (size / 32)));
    launches.join.block = dim3(256);
    launches.join.set_args(record);
  }
  return launches;
}

hipError_t launch_product(const ProductArgs &args, ProductEpilogue epilogue, bool a_cols, bool b_cols, int dtype,
                          size_t scratch_bytes, hipStream_t stream) {
  const ProductPlan plan =
      plan_product(args.m, args.n, args.k, args.batch, dtype == kDtypeF32 ? 4 : 2, args.symmetric != 0, scratch_bytes);
  const ProductLaunch launches = make_product(args, plan, epilogue, a_cols, b_cols, dtype);
  if (const hipError_t status = launch(launches.main, stream); status != hipSuccess) {
    return status;
  }
  return launch(launches.join, stream);
}

}  // namespace xp
