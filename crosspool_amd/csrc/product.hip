// Plans and launches of the training operators' products.
#include "product.hpp"
#include "xp_elements.hpp"

#include <algorithm>
#include <cmath>

namespace xp {

// A product's time in microseconds: a CU's workgroups share its throughput and a workgroup's slabs follow one
// another at no less than the slab latency; a K split adds the reduction's launch and its sums' traffic.
namespace {
struct ProductCost {
  int tile;
  double latency;     // us per slab of a workgroup alone on its CU
  double throughput;  // us per slab and workgroup of a full CU
  double together;    // workgroups that a CU holds
};
constexpr ProductCost kCosts16[] = {{256, 1.55, 1.55, 1}, {128, 0.62, 0.48, 2}, {64, 0.33, 0.17, 5}};
constexpr ProductCost kCosts32[] = {{256, 7.0, 7.0, 1}, {128, 2.2, 1.9, 2}, {64, 0.9, 0.55, 5}};
constexpr double kCus = 256.0;
constexpr double kLaunchUs = 4.0;
constexpr double kReduceUs = 3.0;
constexpr double kPartialBytesPerUs = 8e6;
constexpr int64_t kMaxRanges = 32;
}  // namespace

size_t product_scratch_bytes(const ProductPlan &plan, int64_t m, int64_t n, int64_t batch) {
  return plan.ranges > 1 ? static_cast<size_t>(batch * plan.ranges * m * ((n + 7) / 8 * 8)) * 4 : 0;
}

ProductPlan plan_product(int64_t m, int64_t n, int64_t k, int64_t batch, int element_bytes, bool symmetric, size_t scratch) {
  const int64_t slab = 128 / element_bytes;
  const int64_t slabs = (k + slab - 1) / slab;
  ProductPlan best{};
  double best_us = -1.0;
  for (const ProductCost &cost : element_bytes == 4 ? kCosts32 : kCosts16) {
    const int64_t rows = (m + cost.tile - 1) / cost.tile;
    const int64_t cols = (n + cost.tile - 1) / cost.tile;
    const int64_t tiles = batch * (symmetric ? rows * (rows + 1) / 2 : rows * cols);
    for (int64_t ranges = 1; ranges <= kMaxRanges; ++ranges) {
      const int64_t per_range = (slabs + ranges - 1) / ranges;
      if (ranges > 1 && (per_range < 2 || (ranges - 1) * per_range >= slabs)) {
        continue;
      }
      const ProductPlan plan{cost.tile, ranges, ranges > 1 ? per_range * slab : k, 0};
      const size_t bytes = product_scratch_bytes(plan, m, n, batch);
      if (bytes > scratch) {
        continue;
      }
      const double groups = static_cast<double>(tiles * ranges);
      const double full = std::floor(groups / (kCus * cost.together));
      const double rest = std::ceil((groups - full * kCus * cost.together) / kCus);
      const double us = static_cast<double>(per_range) *
                            (full * cost.together * cost.throughput + (rest > 0.0 ? std::max(cost.latency, rest * cost.throughput) : 0.0)) +
                        (ranges > 1 ? kReduceUs + 2.0 * static_cast<double>(bytes) / kPartialBytesPerUs : 0.0);
      if (best_us < 0.0 || us < best_us) {
        best = plan;
        best_us = us;
      }
    }
  }
  best.bands = best.ranges > 1 ? (m + 31) / 32 : (m + best.tile / 2 - 1) / (best.tile / 2);
  return best;
}

ProductLaunch make_product(const ProductArgs &args, const ProductPlan &plan, ProductEpilogue epilogue, bool a_cols, bool b_cols,
                           int dtype) {
  ProductLaunch launches;
  ProductArgs record = args;
  record.ranges = static_cast<int32_t>(plan.ranges);
  record.k_slice = plan.k_slice;
  const int64_t rows = (args.m + plan.tile - 1) / plan.tile;
  const int64_t cols = (args.n + plan.tile - 1) / plan.tile;
  const int64_t tiles = (args.symmetric != 0 ? rows * (rows + 1) / 2 : rows * cols) * args.batch * plan.ranges;
  launches.main.func = dtype == kDtypeF32   ? ProductKernels<F32Payload>::tile(plan.tile, epilogue, a_cols, b_cols)
                       : dtype == kDtypeF16 ? ProductKernels<F16Payload>::tile(plan.tile, epilogue, a_cols, b_cols)
                                            : ProductKernels<Bf16Payload>::tile(plan.tile, epilogue, a_cols, b_cols);
  launches.main.grid = dim3(static_cast<unsigned>(tiles));
  launches.main.block = dim3(plan.tile == 256 ? 512 : 256);
  launches.main.set_args(record);
  if (plan.ranges > 1) {
    launches.reduce.func = dtype == kDtypeF32   ? ProductKernels<F32Payload>::reduce(epilogue)
                           : dtype == kDtypeF16 ? ProductKernels<F16Payload>::reduce(epilogue)
                                                : ProductKernels<Bf16Payload>::reduce(epilogue);
    launches.reduce.grid = dim3(static_cast<unsigned>((args.n + 63) / 64), static_cast<unsigned>((args.m + 127) / 128),
                                static_cast<unsigned>(args.batch));
    launches.reduce.block = dim3(256);
    launches.reduce.set_args(record);
  }
  return launches;
}

hipError_t launch_product(const ProductArgs &args, ProductEpilogue epilogue, bool a_cols, bool b_cols, int dtype,
                          size_t scratch_bytes, hipStream_t stream, ProductPlan *chosen) {
  const ProductPlan plan = plan_product(args.m, args.n, args.k, args.batch, dtype == kDtypeF32 ? 4 : 2, args.symmetric != 0, scratch_bytes);
  if (chosen != nullptr) {
    *chosen = plan;
  }
  const ProductLaunch launches = make_product(args, plan, epilogue, a_cols, b_cols, dtype);
  if (const hipError_t status = launch(launches.main, stream); status != hipSuccess) {
    return status;
  }
  return launch(launches.reduce, stream);
}

}  // namespace xp
