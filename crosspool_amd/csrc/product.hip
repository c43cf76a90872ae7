// Plans and launches of the training operators' products.
#include "product.hpp"
#include "xp_elements.hpp"

#include <algorithm>
#include <cmath>
#include <iterator>
#include <type_traits>

namespace xp {

// A product's time in microseconds.  A CU's workgroups share its throughput: with i + 1 of them on it (as many as fit),
// a slab in each takes `slab[i]`, and the first loads and the epilogue `around[i]`.  Fitted on MI355X to 1, 4, 12 and 48
// slabs on 64 to 2048 workgroups; the three storage orders differ by less than 10 %.  Model and measured, us, of a product
// repeated by itself: bf16 4096 x 12288 x 4096 289 / 311, fp16 1000 x 2048 x 12288 65 / 63 (its join among them),
// 12288 x 2048 x 1000 61 / 62, 1000 x 6144 x 2048 37 / 35.  Among other launches, whose data it follows, the second takes 81
// and the third 64.  The model knows kStore's plain epilogue alone: kGradient's loads and stores (1000 x 6144 x 2048 37 / 75),
// mirrored tiles (fp16 symmetric 4096 x 12288 197 / 220, 32 of 768 x 768 26 / 45) and a base read back (32 of
// 2048 x 768 x 768 74 / 99) come on top.
namespace {
struct ProductCost {
  ProductTiles tiles;
  int together;
  double slab[4];
  double around[4];
};
constexpr ProductCost kCosts16[] = {{ProductTiles::k256, 1, {1.38}, {7.2}},
                                    {ProductTiles::k128Pairs, 2, {0.73, 0.85}, {4.7, 7.0}},
                                    {ProductTiles::k128Deep, 1, {0.5}, {6.3}},
                                    {ProductTiles::k64, 3, {0.245, 0.38, 0.52}, {2.3, 3.0, 3.9}},
                                    {ProductTiles::k32, 4, {0.155, 0.22, 0.36, 0.46}, {0.8, 1.1, 1.4, 1.7}}};
constexpr ProductCost kCosts32[] = {{ProductTiles::k128Pairs, 2, {1.95, 3.67}, {7.0, 7.5}},
                                    {ProductTiles::k64, 3, {0.62, 1.05, 1.49}, {2.4, 3.4, 4.6}},
                                    {ProductTiles::k32, 4, {0.235, 0.345, 0.48, 0.6}, {0.9, 1.3, 1.6, 2.0}}};
struct ProductCosts {
  const ProductCost *first;
  const ProductCost *last;
  const ProductCost *begin() const { return first; }
  const ProductCost *end() const { return last; }
};
ProductCosts costs_of(int element_bytes) {
  return element_bytes == 4 ? ProductCosts{std::begin(kCosts32), std::end(kCosts32)}
                            : ProductCosts{std::begin(kCosts16), std::end(kCosts16)};
}
constexpr int64_t kCus = 256;
constexpr double kLaunchUs = 2.3;
constexpr double kJoinUs = 3.0;       // its launch,
constexpr double kPieceUs = 0.25;     // what a piece of a tile adds to its latency,
constexpr double kBytesPerUs = 4e6;   // and the pieces' way out and back
constexpr int64_t kMinSlabs = 2;      // of a worker
// A launch holds fewer than 2^32 threads.
bool launchable(int64_t groups, ProductTiles tiles) {
  return groups < (int64_t{1} << 32) / (tiles == ProductTiles::k256 ? 512 : 256);
}

// `groups` workgroups of `slabs` slabs each in `pieces` tiles, all of one kind, on the chip; `apart`: no two of them work
// on the same slabs, which then come from beyond the L2 caches.
constexpr double kApartBytesPerUs = 10e6;
double rounds_us(const ProductCost &cost, int64_t groups, double slabs, double pieces, bool apart) {
  const int64_t full = groups / (kCus * cost.together);
  const int64_t rest = (groups - full * kCus * cost.together + kCus - 1) / kCus;
  const auto round = [&](int64_t count) {
    const double load = apart ? static_cast<double>(count * kCus * 256 * tile_size(cost.tiles)) / kApartBytesPerUs : 0.0;
    return slabs * std::max(cost.slab[count - 1], load) + pieces * cost.around[count - 1];
  };
  return static_cast<double>(full) * round(cost.together) + (rest > 0 ? round(rest) : 0.0);
}
}  // namespace

size_t product_scratch_bytes(const ProductPlan &plan) {
  const size_t size = static_cast<size_t>(tile_size(plan.tiles));
  return plan.split > 0 ? static_cast<size_t>(plan.workers + plan.split) * size * size * sizeof(float) : 0;
}

namespace {
ProductPlan find_plan(int64_t m, int64_t n, int64_t k, int64_t batch, int element_bytes, bool symmetric, size_t scratch) {
  const int64_t slab = 128 / element_bytes;
  const int64_t slabs = (k + slab - 1) / slab;
  ProductPlan best{};
  best.us = -1.0;
  for (const ProductCost &cost : costs_of(element_bytes)) {
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
      if (!launchable(whole + workers, cost.tiles)) {
        return;
      }
      if (whole > 0) {
        plan.us += rounds_us(cost, whole, static_cast<double>(slabs), 1.0, false);
      }
      if (plan.split > 0) {
        // A worker whose run crosses a tile's end has two pieces.
        const bool even = workers % plan.split == 0 && together % workers == 0;
        const double pieces = even ? 1.0 : 1.7;
        const double each = std::ceil(static_cast<double>(together) / static_cast<double>(workers));
        plan.us += rounds_us(cost, workers, each, pieces, !even) + kJoinUs +
                   kPieceUs * static_cast<double>(workers) / static_cast<double>(plan.split) +
                   static_cast<double>(product_scratch_bytes(plan)) / kBytesPerUs;
      }
      if (best.us < 0.0 || plan.us < best.us) {
        best = plan;
      }
    };
    consider(tiles, 0);
    const int64_t slots = kCus * cost.together;
    const int64_t full = tiles / slots * slots;
    if (full == tiles || cost.tiles == ProductTiles::k256 || cost.tiles == ProductTiles::k32) {
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

struct PlanKey {
  int64_t m;
  int64_t n;
  int64_t k;
  int64_t batch;
  size_t scratch;
  int64_t kind;
  bool operator==(const PlanKey &) const = default;
};
struct KnownPlan {
  PlanKey key;
  ProductPlan plan;
};
constexpr size_t kKnownPlans = 512;
}  // namespace

// A plan follows from its arguments alone.  A small call asks for some ten of them, workspace sizes among them, whose search
// took longer than its launches (a backward pass of three rows of 256 x 256 17 us of host time): each thread keeps the last ones.
ProductPlan plan_product(int64_t m, int64_t n, int64_t k, int64_t batch, int element_bytes, bool symmetric, size_t scratch) {
  static thread_local KnownPlan known[kKnownPlans];  // (no product has m = 0)
  const PlanKey key{m, n, k, batch, scratch, element_bytes * 2 + (symmetric ? 1 : 0)};
  uint64_t hash = 0;
  for (const uint64_t part : {static_cast<uint64_t>(m), static_cast<uint64_t>(n), static_cast<uint64_t>(k), static_cast<uint64_t>(batch),
                              static_cast<uint64_t>(scratch), static_cast<uint64_t>(key.kind)}) {
    hash = (hash ^ part) * 0x9e3779b97f4a7c15ull;
    hash ^= hash >> 29;
  }
  KnownPlan &place = known[hash % kKnownPlans];
  if (!(place.key == key)) {
    place.plan = find_plan(m, n, k, batch, element_bytes, symmetric, scratch);
    place.key = key;
  }
  return place.plan;
}

ProductLaunch make_product(const ProductArgs &args, const ProductPlan &plan, ProductEpilogue epilogue, bool a_cols, bool b_cols,
                           int dtype) {
  ProductLaunch launches;
  ProductArgs record = args;
  record.whole = static_cast<int32_t>(plan.whole);
  record.split = static_cast<int32_t>(plan.split);
  record.workers = static_cast<int32_t>(plan.workers);
  const int size = tile_size(plan.tiles);
  record.tile_rows = static_cast<int32_t>((args.m + size - 1) / size);
  record.tile_cols = static_cast<int32_t>((args.n + size - 1) / size);
  if (plan.split > 0) {
    const int64_t slab = dtype == kDtypeF32 ? 32 : 64;
    const int64_t together = plan.split * ((args.k + slab - 1) / slab);
    record.share = static_cast<int32_t>(together / plan.workers);
    record.longer = static_cast<int32_t>(together % plan.workers);
    record.each = together % plan.workers == 0 && plan.workers % plan.split == 0 ? static_cast<int32_t>(plan.workers / plan.split) : 0;
  }
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

namespace {
// `matrices` matrices further in an operand of `dtype`.
template <class T>
void advance(T *&data, int64_t matrices, int64_t batch, int dtype) {
  using Byte = std::conditional_t<std::is_const_v<T>, const unsigned char, unsigned char>;
  data = data == nullptr ? nullptr : static_cast<Byte *>(data) + matrices * batch * (dtype == kDtypeF32 ? 4 : 2);
}
}  // namespace

hipError_t launch_product(const ProductArgs &args, ProductEpilogue epilogue, bool a_cols, bool b_cols, int dtype,
                          size_t scratch_bytes, hipStream_t stream) {
  const ProductPlan plan =
      plan_product(args.m, args.n, args.k, args.batch, dtype == kDtypeF32 ? 4 : 2, args.symmetric != 0, scratch_bytes);
  if (plan.us < 0.0) {
    // More tiles than one launch holds (over a thousand matrices of 1 x 2^20): in two halves.
    if (args.batch < 2) {
      return hipErrorInvalidConfiguration;
    }
    ProductArgs half = args;
    half.batch = args.batch / 2;
    if (const hipError_t status = launch_product(half, epilogue, a_cols, b_cols, dtype, scratch_bytes, stream); status != hipSuccess) {
      return status;
    }
    const int64_t done = half.batch;
    half.batch = args.batch - half.batch;
    advance(half.a.data, done, half.a.batch, dtype);
    advance(half.b.data, done, half.b.batch, dtype);
    advance(half.out, done, half.batch_out, half.out_dtype);
    advance(half.base, done, half.batch_base, half.base_dtype);
    advance(half.extra, done, half.batch_extra, half.extra_dtype);
    return launch_product(half, epilogue, a_cols, b_cols, dtype, scratch_bytes, stream);
  }
  const ProductLaunch launches = make_product(args, plan, epilogue, a_cols, b_cols, dtype);
  if (const hipError_t status = launch(launches.main, stream); status != hipSuccess) {
    return status;
  }
  return launch(launches.join, stream);
}

hipError_t launch_products(ProductGroup &group, const bool (&present)[3], int dtype, size_t scratch_bytes, hipStream_t stream) {
  const int element = dtype == kDtypeF32 ? 4 : 2;
  const int64_t slab = 128 / element;
  double apart_us = 0.0;
  int count = 0;
  for (int i = 0; i < 3; ++i) {
    if (present[i]) {
      const ProductArgs &part = group.part[i];
      apart_us += plan_product(part.m, part.n, part.k, 1, element, false, scratch_bytes).us;
      ++count;
    }
  }
  // Together: the tiles in their order on a chip that is full to the last of them, or the longest tile's time.
  double best_us = apart_us;
  ProductTiles best = ProductTiles::k256;
  for (const ProductCost &cost : costs_of(element)) {
    if (count < 2 || cost.tiles == ProductTiles::k256 || cost.tiles == ProductTiles::k128Deep) {
      continue;
    }
    const int64_t size = tile_size(cost.tiles);
    int64_t groups = 0;
    double work = 0.0;
    double longest = 0.0;
    for (int i = 0; i < 3; ++i) {
      if (present[i]) {
        const ProductArgs &part = group.part[i];
        const double slabs = static_cast<double>((part.k + slab - 1) / slab);
        const int64_t part_tiles = ((part.m + size - 1) / size) * ((part.n + size - 1) / size);
        const double tiles = static_cast<double>(part_tiles);
        const double each = slabs * cost.slab[cost.together - 1] + cost.around[cost.together - 1];
        groups += part_tiles;
        work += tiles * each / static_cast<double>(kCus * cost.together);
        longest = std::max(longest, each);
      }
    }
    const double us = kLaunchUs + std::max(longest, work + 0.5 * cost.around[cost.together - 1]);
    if (us < best_us && launchable(groups, cost.tiles)) {
      best_us = us;
      best = cost.tiles;
    }
  }
  if (best == ProductTiles::k256) {
    for (int i = 0; i < 3; ++i) {
      if (present[i]) {
        if (const hipError_t status = launch_product(group.part[i], ProductEpilogue::kStore, i > 0, true, dtype, scratch_bytes, stream);
            status != hipSuccess) {
          return status;
        }
      }
    }
    return hipSuccess;
  }
  int64_t blocks = 0;
  for (int i = 0; i < 3; ++i) {
    ProductArgs &part = group.part[i];
    group.blocks[i] = 0;
    if (present[i]) {
      const int64_t size = tile_size(best);
      part.tile_rows = static_cast<int32_t>((part.m + size - 1) / size);
      part.tile_cols = static_cast<int32_t>((part.n + size - 1) / size);
      part.whole = part.tile_rows * part.tile_cols;
      group.blocks[i] = part.whole;
      blocks += part.whole;
    }
  }
  const void *kernel = dtype == kDtypeF32   ? ProductKernels<F32Payload>::group(best)
                       : dtype == kDtypeF16 ? ProductKernels<F16Payload>::group(best)
                                            : ProductKernels<Bf16Payload>::group(best);
  void *params[] = {&group};
  return hipLaunchKernel(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), params, 0, stream);
}

}  // namespace xp
