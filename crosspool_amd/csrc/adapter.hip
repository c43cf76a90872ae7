// Low-rank adapters: the sort of a batch's rows by adapter, the small kernels of the backward pass
// and the launches of all of them (the products are in adapter_kernels.hpp).

#include "adapter_kernels.hpp"

#include <algorithm>

namespace xp {
namespace {

// ------------------------------------------------------------------ rows by adapter
constexpr int kRouteThreads = 1024;
constexpr int kRouteWaves = kRouteThreads / kWave;
constexpr int kRouteGroups = kAdapterMaxCount + 2;

// Rows, tiles, runs and, in one value, slots of partial sums (at most 2^17) and adapters with rows of some
// groups, added up.
struct RouteSums {
  int value[4];
};
constexpr int kRouteAdapter = 1 << 20;

__device__ __forceinline__ RouteSums wave_inclusive_scan(RouteSums sums) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int offset = 1; offset < kWave; offset <<= 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int other = __shfl_up(sums.value[i], offset, kWave);
      sums.value[i] += lane >= offset ? other : 0;
    }
  }
  return sums;
}

// A stable counting sort by one workgroup: every wave counts a contiguous sixteenth of the rows 64 at a
// time, a row's place among the 64 being the number of earlier lanes of its group; the counts are scanned
// over groups and waves, and the rows are placed.  Stable and free of racing increments, so the sums of
// the gradients have one order.  Bound by the latency of its steps: one read of the ids (kept in registers
// with their places up to 8192 rows), four barriers, one wave's scan where two groups per lane hold all of
// them.  One increment per group and 64 rows: with one per row the LDS took a cycle for each (8192 rows of
// 8 adapters: 14 us, 9.8 so).  Past 8192 rows the ids are read twice and the time grows with the rows: 20 us
// for 16384 of 8 adapters, 72 for 65536 and 1.4 ms for 2^20 (512 adapters: 32, 114 and 2.0 ms).
constexpr int kRouteKept = 8;

struct RouteLds {
  int counts[kRouteWaves * kRouteGroups];
  int starts[kRouteGroups + 1];
  int tile_starts[kRouteGroups + 1];
  int run_starts[kRouteGroups + 1];
  int slot_starts[kRouteGroups];
  int transposes[kRouteGroups];
  RouteSums wave_sums[kRouteWaves];
};

__device__ __forceinline__ void route_rows(const AdapterRouteArgs &a, RouteLds &lds) {
  int *counts = lds.counts;
  int *starts = lds.starts;
  int *tile_starts = lds.tile_starts;
  int *run_starts = lds.run_starts;
  int *slot_starts = lds.slot_starts;
  RouteSums *wave_sums = lds.wave_sums;
  const AdapterBatch &batch = a.batch;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int count = batch.count;
  const int groups = count + 2;
  const int rows = static_cast<int>(batch.rows);
  const int share = ((rows + kRouteWaves - 1) / kRouteWaves + kWave - 1) / kWave * kWave;
  const int first = wave * share;
  const int last = first + share < rows ? first + share : rows;
  int kept[kRouteKept];
#pragma unroll
  for (int i = 0; i < kRouteKept; ++i) {
    const int row = first + i * kWave + lane;
    kept[i] = row < last ? batch.ids[row] : -1;
  }
  for (int index = tid; index < kRouteWaves * groups; index += kRouteThreads) {
    counts[index] = 0;
  }
  __syncthreads();
  int *own = counts + wave * groups;
  bool bad = false;
  // The lanes with a row of the lane's group, by ballots over the bits of the group.
  auto same_group = [&](bool live, int group) __attribute__((always_inline)) {
    unsigned long long same = __ballot(live);
    for (int bit = 1; bit < groups; bit <<= 1) {
      const unsigned long long set = __ballot((group & bit) != 0);
      same &= (group & bit) != 0 ? set : ~set;
    }
    return same;
  };
  // Rows' places among the wave's rows of their group; a group's first lane counts for all of them.
  int place_of[kRouteKept];
#pragma unroll
  for (int i = 0; i < kRouteKept; ++i) {
    place_of[i] = 0;
    if (first + i * kWave < last) {
      const bool live = first + i * kWave + lane < last;
      const int group = live ? adapter_group(kept[i], count) : 0;
      bad |= group > count;
      const unsigned long long same = same_group(live, group);
      const int earlier = __popcll(same & ((1ull << lane) - 1));
      int added = 0;
      if (live && earlier == 0) {
        added = atomicAdd(&own[group], __popcll(same));
      }
      place_of[i] = __shfl(added, __ffsll(same) - 1, kWave) + earlier;
    }
  }
  const bool all_kept = first + kRouteKept * kWave >= last;
  for (int row = first + kRouteKept * kWave; row < last; row += kWave) {
    const bool live = row + lane < last;
    const int group = live ? adapter_group(batch.ids[row + lane], count) : 0;
    bad |= group > count;
    const unsigned long long same = same_group(live, group);
    if (live && (same & ((1ull << lane) - 1)) == 0) {
      atomicAdd(&own[group], __popcll(same));
    }
  }
  if (__ballot(bad) != 0 && lane == 0) {
    raise_fault(a.fault, kFaultAdapterOutOfRange);
  }
  __syncthreads();
  // Two groups per thread.
  RouteSums mine[2] = {};
  RouteSums both = {};
  if (2 * tid < groups) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int group = 2 * tid + i;
      if (group < groups) {
        int length = 0;
#pragma unroll
        for (int w = 0; w < kRouteWaves; ++w) {
          const int part = counts[w * groups + group];
          counts[w * groups + group] = length;
          length += part;
        }
        const bool runs = group < count && batch.run_rows > 0;
        const int pieces = runs ? (length + batch.run_rows - 1) / batch.run_rows : 0;
        mine[i] = {{length, (length + kAdapterTileRows - 1) / kAdapterTileRows, pieces,
                    (pieces > 1 ? pieces : 0) + (length > 0 ? kRouteAdapter : 0)}};
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          both.value[v] += mine[i].value[v];
        }
      }
    }
  }
  RouteSums before = {};
  if (groups <= 2 * kWave) {
    if (wave == 0) {
      const RouteSums inclusive = wave_inclusive_scan(both);
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        before.value[v] = inclusive.value[v] - both.value[v];
      }
    }
  } else {
    const RouteSums inclusive = wave_inclusive_scan(both);
    if (lane == kWave - 1) {
      wave_sums[wave] = inclusive;
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      before.value[v] = inclusive.value[v] - both.value[v];
      for (int w = 0; w < wave; ++w) {
        before.value[v] += wave_sums[w].value[v];
      }
    }
  }
  if (2 * tid < groups) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int group = 2 * tid + i;
      if (group < groups) {
        starts[group] = before.value[0];
        tile_starts[group] = before.value[1];
        run_starts[group] = before.value[2];
        const int first_slot = before.value[3] % kRouteAdapter;
        slot_starts[group] = mine[i].value[2] > 1 ? first_slot : -1;
        lds.transposes[group] = batch.transposes != nullptr ? before.value[3] / kRouteAdapter : group;
        if (group <= count) {
          batch.starts[group] = before.value[0];
        }
        if (group < count && batch.transposes != nullptr) {
          batch.transposes[group] = lds.transposes[group];
        }
        if (group < count && batch.run_rows > 0) {
          batch.run_slots[2 * group] = first_slot;
          batch.run_slots[2 * group + 1] = mine[i].value[2];
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          before.value[v] += mine[i].value[v];
        }
        if (group == groups - 1) {
          starts[groups] = before.value[0];
          tile_starts[groups] = before.value[1];
          run_starts[groups] = before.value[2];
        }
      }
    }
  }
  __syncthreads();
  // Placement.
  if (all_kept) {
#pragma unroll
    for (int i = 0; i < kRouteKept; ++i) {
      const int row = first + i * kWave + lane;
      if (row < last) {
        const int group = adapter_group(kept[i], count);
        batch.perm[starts[group] + own[group] + place_of[i]] = row;
      }
    }
  } else {
    for (int row = first; row < last; row += kWave) {
      const bool live = row + lane < last;
      const int group = live ? adapter_group(batch.ids[row + lane], count) : 0;
      const unsigned long long same = same_group(live, group);
      if (live) {
        const int earlier = __popcll(same & ((1ull << lane) - 1));
        batch.perm[starts[group] + own[group] + earlier] = row + lane;
        // Every lane of the wave has read the count before it moves on: one wave runs in order.
        __builtin_amdgcn_wave_barrier();
        if (earlier == 0) {
          atomicAdd(&own[group], __popcll(same));
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
  // The group of a tile (run): the last that starts at or before it (an empty one starts where the
  // next does).
  auto find = [&](const int *table, int value) {
    int low = 0;
    int high = groups;
    while (high - low > 1) {
      const int middle = (low + high) / 2;
      if (table[middle] <= value) {
        low = middle;
      } else {
        high = middle;
      }
    }
    return low;
  };
  for (int tile = tid; tile < batch.max_tiles; tile += kRouteThreads) {
    int *entry = batch.tiles + 4 * tile;
    if (tile >= tile_starts[groups]) {
      entry[0] = -1;
      continue;
    }
    const int group = find(tile_starts, tile);
    const int begin = starts[group] + (tile - tile_starts[group]) * kAdapterTileRows;
    const int left = starts[group + 1] - begin;
    entry[0] = group;
    entry[1] = begin;
    entry[2] = left < kAdapterTileRows ? left : kAdapterTileRows;
    entry[3] = group < count ? adapter_rank_of(a.ranks, group, a.max_rank) + 256 * lds.transposes[group] : 0;
  }
  for (int run = tid; run < batch.max_runs; run += kRouteThreads) {
    int *entry = batch.runs + 8 * run;
    if (run >= run_starts[groups]) {
      entry[0] = -1;
      continue;
    }
    const int group = find(run_starts, run);
    const int begin = starts[group] + (run - run_starts[group]) * batch.run_rows;
    entry[0] = group;
    entry[1] = begin;
    entry[2] = begin + batch.run_rows < starts[group + 1] ? begin + batch.run_rows : starts[group + 1];
    entry[3] = slot_starts[group] < 0 ? -1 : slot_starts[group] + run - run_starts[group];
    entry[4] = tile_starts[group] + (run - run_starts[group]) * (batch.run_rows / kAdapterTileRows);
  }
}

__global__ __launch_bounds__(kRouteThreads) void adapter_route_kernel(AdapterRouteArgs a) {
  __shared__ RouteLds lds;
  route_rows(a, lds);
}

// ------------------------------------------------------------------ transposes
// at[a][k][r] = A_a[r][k] and bt[a][r][n] = B_a[n][r] for the adapters that have rows: 64 columns of
// A (rows of B) per workgroup through LDS.  Ranks past the adapter's are left unwritten.  Pools of more
// than kTransposeGroups adapters have places for those with rows only (a batch of one row would ask for
// gigabytes beside a large pool), in the pool's order.
template <class E>
struct TransposeLds {
  E tile[kAdapterMaxRank][64 + 1];
};

template <class E, bool SORTED>
__device__ __forceinline__ void transpose_columns(const AdapterTransposeArgs &a, int64_t block, int group0, int groups,
                                                  TransposeLds<E> &lds) {
  auto &tile = lds.tile;
  const int64_t blocks0 = a.at != nullptr ? (a.k + 63) / 64 : 0;
  const bool second = block >= blocks0;
  const int64_t c0 = (block - (second ? blocks0 : 0)) * 64;
  const int64_t length = second ? a.n : a.k;
  const int columns = length - c0 < 64 ? static_cast<int>(length - c0) : 64;
  for (int group = group0; group < a.batch.count; group += groups) {
    const int rank = adapter_rank(a.ranks, group, a.max_rank);
    if (rank == 0) {
      continue;
    }
    if constexpr (SORTED) {
      if (a.batch.starts[group + 1] == a.batch.starts[group]) {
        continue;
      }
    } else {
      int found = 0;
#pragma unroll 4
      for (int64_t row = threadIdx.x; row < a.batch.rows; row += kRouteThreads) {
        found |= a.batch.ids[row] == group ? 1 : 0;
      }
      if (__syncthreads_or(found) == 0) {
        continue;
      }
    }
    const int64_t place = SORTED && a.batch.transposes != nullptr ? a.batch.transposes[group] : group;
    if (second) {
      const E *source = static_cast<const E *>(a.b) + (group * a.n + c0) * a.max_rank;
      E *target = static_cast<E *>(a.bt) + place * a.rp * a.n + c0;
      for (int index = threadIdx.x; index < columns * rank; index += kRouteThreads) {
        const int column = index / rank;
        const int r = index - column * rank;
        tile[r][column] = source[static_cast<int64_t>(column) * a.max_rank + r];
      }
      __syncthreads();
      for (int index = threadIdx.x; index < 64 * rank; index += kRouteThreads) {
        const int column = index & 63;
        if (column < columns) {
          target[(index >> 6) * a.n + column] = tile[index >> 6][column];
        }
      }
    } else {
      const E *source = static_cast<const E *>(a.a) + static_cast<int64_t>(group) * a.max_rank * a.k + c0;
      E *target = static_cast<E *>(a.at) + (place * a.k + c0) * a.rp;
      for (int index = threadIdx.x; index < 64 * rank; index += kRouteThreads) {
        const int column = index & 63;
        if (column < columns) {
          tile[index >> 6][column] = source[(index >> 6) * a.k + column];
        }
      }
      __syncthreads();
      for (int index = threadIdx.x; index < columns * rank; index += kRouteThreads) {
        const int column = index / rank;
        const int r = index - column * rank;
        target[static_cast<int64_t>(column) * a.rp + r] = tile[r][column];
      }
    }
    __syncthreads();
  }
}

// Few rows and adapters: the sort is the first workgroup of the transposes' launch, and the others look
// for their adapter's rows in the ids themselves.  Both are bound by latency: one after the other they
// took 13 us where they take 9 together (4096 rows, an adapter of rank 16 of 4096 x 24576).  With more,
// reading the ids once per workgroup and adapter would cost more than a launch.
constexpr int kTransposeGroups = 32;
constexpr int64_t kRoutesBesideRows = 8192;

template <class E>
__global__ __launch_bounds__(kRouteThreads) void adapter_transpose_kernel(AdapterRouteTransposeArgs a) {
  __shared__ TransposeLds<E> lds;
  transpose_columns<E, true>(a.transpose, blockIdx.x, blockIdx.y, gridDim.y, lds);
}

template <class E>
__global__ __launch_bounds__(kRouteThreads) void adapter_route_transpose_kernel(
    AdapterRouteTransposeArgs a) {
  __shared__ union {
    RouteLds route;
    TransposeLds<E> transpose;
  } lds;
  if (blockIdx.x == 0) {
    if (blockIdx.y == 0) {
      route_rows(a.route, lds.route);
    }
    return;
  }
  transpose_columns<E, false>(a.transpose, blockIdx.x - 1, blockIdx.y, gridDim.y, lds.transpose);
}

// ------------------------------------------------------------------ terms
// The K ranges' sums of t (u) in range order as the coefficient operands of the outer products: for each
// tile of 64 positions, step of 32 (fp32: 16) positions and 16 ranks, lane l's 16 bytes are those of rank
// l % 16 and the 8 (4) positions from 8 (4) (l / 16), 16-bit payloads' as two planes of bf16 terms;
// positions past the tile are zero.  One workgroup per tile.  Bound by latency (4.8 us at 4096 rows); the
// outer products' many workgroups of a tile read the result as often as there are column blocks.
__global__ __launch_bounds__(256) void adapter_terms_kernel(AdapterTermsArgs a) {
  __shared__ int list[kAdapterTileRows];
  __shared__ float values[kAdapterTileRows][kAdapterMaxRank + 1];
  const int planes = a.f32 != 0 ? 1 : 2;
  const int per_lane = a.f32 != 0 ? 4 : 8;
  const int steps = kAdapterTileRows / (4 * per_lane);
  const int rank_tiles = a.rp / 16;
  for (int64_t slot = blockIdx.x;; slot += gridDim.x) {
    const AdapterTile tile = adapter_tile(a.batch, a.ranks, a.max_rank, slot, false);
    if (tile.group < 0) {
      return;
    }
    if (threadIdx.x < kAdapterTileRows) {
      list[threadIdx.x] = tile.row;
    }
    __syncthreads();
    int columns = 16;
    while (columns < tile.rank) {
      columns *= 2;
    }
    if (tile.rank > 0) {
      const int job = blockIdx.y;
      const int64_t plane = a.batch.rows * a.rp;
      const int quads = columns / 4;
      for (int index = threadIdx.x; index < kAdapterTileRows * quads; index += 256) {
        const int row = index / quads;
        const int r = 4 * (index & (quads - 1));
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        if (row < tile.rows) {
          const float *source = a.partials[job] + static_cast<int64_t>(list[row]) * a.rp + r;
#pragma unroll 8
          for (int64_t range = 0; range < a.ranges[job]; ++range) {
            sum += *reinterpret_cast<const f32x4 *>(source + range * plane);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          values[row][r + j] = sum[j];
        }
      }
      __syncthreads();
      unsigned char *out = static_cast<unsigned char *>(a.terms[job]) + slot * steps * rank_tiles * planes * 1024;
      for (int index = threadIdx.x; index < steps * (columns / 16) * kWave; index += 256) {
        const int lane = index & 63;
        const int r = index / kWave % (columns / 16);
        const int step = index / kWave / (columns / 16);
        const int rank = r * 16 + (lane & 15);
        const int row = (step * 4 + (lane >> 4)) * per_lane;
        unsigned char *target = out + ((step * rank_tiles + r) * planes * kWave + lane) * 16;
        u32x4 high;
        u32x4 low;
        if (a.f32 != 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            high[j] = __float_as_uint(values[row + j][rank]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t h;
            uint32_t l;
            split_pair(values[row + 2 * j][rank], values[row + 2 * j + 1][rank], h, l);
            high[j] = h;
            low[j] = l;
          }
          *reinterpret_cast<u32x4 *>(target + 1024) = low;
        }
        *reinterpret_cast<u32x4 *>(target) = high;
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ gradients of several runs
// The runs' sums of an adapter's gradients in run order, times its scale; zeros for an adapter without
// rows.  Reads what the outer products wrote just before: 5.8 us for two runs of 28672 columns
// of rank 16, 2 to 4 where there is nothing to add.
__global__ __launch_bounds__(256) void adapter_reduce_kernel(AdapterReduceArgs a) {
  const bool second = static_cast<int64_t>(blockIdx.x) >= a.blocks0;
  const AdapterOuterJob &job = a.job[second ? 1 : 0];
  const int64_t block = blockIdx.x - (second ? a.blocks0 : 0);
  const uint32_t elements = static_cast<uint32_t>(job.columns * a.max_rank);
  for (int group = blockIdx.y; group < a.batch.count; group += gridDim.y) {
    const int slot = a.batch.run_slots[2 * group];
    const int runs = a.batch.run_slots[2 * group + 1];
    if (runs == 1) {
      continue;
    }
    const int rank = adapter_rank(a.ranks, group, a.max_rank);
    const float scale = a.scales != nullptr ? a.scales[group] : 1.0f;
    const int64_t plane = static_cast<int64_t>(a.rp) * job.columns;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t index = static_cast<uint32_t>(block * 1024) + i * 256 + threadIdx.x;
      if (index >= elements) {
        continue;
      }
      const uint32_t width = second ? static_cast<uint32_t>(a.max_rank) : static_cast<uint32_t>(job.columns);
      const uint32_t major = index / width;
      const uint32_t minor = index - major * width;
      const int r = static_cast<int>(second ? minor : major);
      float sum = 0.0f;
      if (r < rank) {
        const float *source = job.partials + slot * plane +
                              (second ? static_cast<int64_t>(major) * a.rp + r
                                      : static_cast<int64_t>(r) * job.columns + minor);
#pragma unroll 4
        for (int run = 0; run < runs; ++run) {
          sum += source[run * plane];
        }
        // No rows: zero whatever the scale.
        sum = runs > 0 ? sum * scale : 0.0f;
      }
      store_value(job.grad, static_cast<int64_t>(group) * elements + index, sum, a.dtype);
    }
  }
}

int rank_tiles(int64_t max_rank) { return max_rank <= 16 ? 1 : max_rank <= 32 ? 2 : max_rank <= 64 ? 4 : 8; }

// Workgroups of the shrink kernel that fill the chip: two per CU.
constexpr int64_t kShrinkWorkgroups = 512;
constexpr int64_t kMaxRanges = 8;
constexpr int64_t kStepsPerWorkgroup = 16;  // the least: four steps per wave
constexpr int64_t kExpandWorkgroups = 512;
// Decode has a tile per adapter at most, of a few rows each: three workgroups per CU, were each row its
// own tile (48 rows of 32 adapters of rank 32 x 24576 columns: 13.8 us; with half or twice as many 17.5).
constexpr int64_t kDirectWorkgroups = 768;
constexpr int64_t kOuterWorkgroups = 512;
constexpr int64_t kMinRunRows = 256;
// Tiles of adapters with few rows come on top of the whole ones; workgroups past this many walk on.
constexpr int64_t kExtraSlots = 64;

int64_t align16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

unsigned tile_slots(const AdapterBatch &batch) {
  if (batch.tiles == nullptr) {
    return static_cast<unsigned>(batch.rows);
  }
  const int64_t whole = (batch.rows + kAdapterTileRows - 1) / kAdapterTileRows;
  return static_cast<unsigned>(std::min<int64_t>({whole + kExtraSlots, batch.max_tiles, 65535}));
}

template <class Args>
KernelLaunch launch_of(const void *func, dim3 grid, unsigned block, const Args &args) {
  KernelLaunch kernel;
  kernel.func = func;
  kernel.grid = grid;
  kernel.block = dim3(block, 1, 1);
  kernel.set_args(args);
  return kernel;
}

dim3 transpose_grid(const AdapterTransposeArgs &a) {
  const int64_t blocks = (a.at != nullptr ? (a.k + 63) / 64 : 0) + (a.n + 63) / 64;
  return dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(std::min(a.batch.count, kTransposeGroups)), 1);
}

// Whether transposes have places for the adapters with rows only.
bool transposes_compact(const AdapterShape &shape) { return shape.backward && shape.count > kTransposeGroups; }

}  // namespace

AdapterPlan plan_adapter(const AdapterShape &shape) {
  AdapterPlan plan{};
  const int64_t element = shape.dtype == kDtypeF32 ? 4 : 2;
  const int64_t rows = shape.rows;
  plan.rp = 16 * rank_tiles(shape.max_rank);
  const bool routed = shape.backward || rows > kAdapterDirectRows;
  const int64_t tiles = std::max<int64_t>(1, (rows + kAdapterTileRows - 1) / kAdapterTileRows);
  const int64_t widths[2] = {shape.input_width, shape.output_width};
  int64_t at = 0;
  if (routed) {
    plan.max_tiles = rows / kAdapterTileRows + std::min(rows, shape.count + 2);
    int64_t ints = 4 * plan.max_tiles + shape.count + 1 + rows;
    if (shape.backward) {
      const int64_t blocks = (widths[0] + 63) / 64 + (widths[1] + 63) / 64;
      const int64_t wanted = std::max<int64_t>(1, (kOuterWorkgroups + blocks - 1) / blocks);
      const int64_t run_rows = ((rows + wanted - 1) / wanted + kAdapterTileRows - 1) / kAdapterTileRows * kAdapterTileRows;
      plan.run_rows = std::max(kMinRunRows, run_rows);
      // At least rows / run_rows, and growing with the rows as the workspace's size has to.
      plan.max_runs = std::min(rows / kMinRunRows, wanted) + std::min(rows, shape.count);
      // An adapter of several runs has more than run_rows rows.
      plan.run_slots = std::min(2 * rows / kMinRunRows, 2 * wanted);
      ints += 8 * plan.max_runs + 2 * shape.count + (transposes_compact(shape) ? shape.count : 0);
    }
    at = align16(ints * 4);
  }
  for (int p = 0; p < (shape.backward ? 2 : 1); ++p) {
    const int64_t steps = (widths[p] * element + 63) / 64;
    const int64_t most = std::max<int64_t>(1, std::min(kMaxRanges, steps / kStepsPerWorkgroup));
    const int64_t wanted = routed ? (kShrinkWorkgroups + tiles - 1) / tiles : kMaxRanges;
    const int64_t ranges = std::min(most, wanted);
    plan.steps_per_range[p] = ((steps + ranges - 1) / ranges + 3) / 4 * 4;
    plan.ranges[p] = (steps + plan.steps_per_range[p] - 1) / plan.steps_per_range[p];
    plan.partials[p] = static_cast<size_t>(at);
    at += align16(plan.ranges[p] * rows * plan.rp * 4);
  }
  if (shape.backward) {
    for (int p = 0; p < 2; ++p) {
      plan.terms[p] = static_cast<size_t>(at);
      at += plan.max_tiles * kAdapterTileRows * plan.rp * 4;
      plan.sums[p] = static_cast<size_t>(at);
      at += align16(plan.run_slots * plan.rp * widths[p] * 4);
    }
    const int64_t transposes = transposes_compact(shape) ? std::min(rows, shape.count) : shape.count;
    plan.at = static_cast<size_t>(at);
    at += align16(transposes * shape.input_width * plan.rp * element);
    plan.bt = static_cast<size_t>(at);
    at += align16(transposes * shape.output_width * plan.rp * element);
  }
  plan.bytes = static_cast<size_t>(at);
  return plan;
}

size_t adapter_workspace_bytes(const AdapterShape &shape) {
  AdapterShape smaller = shape;
  if (shape.backward) {
    smaller.rows = std::max<int64_t>(shape.rows, 1);  // no rows are planned as one
  }
  size_t most = plan_adapter(smaller).bytes;
  // The number of K ranges depends on the tiles alone, up to one range, and falls as they grow.
  for (int64_t tiles = 1; tiles <= kShrinkWorkgroups && tiles * kAdapterTileRows < shape.rows; ++tiles) {
    smaller.rows = tiles * kAdapterTileRows;
    most = std::max(most, plan_adapter(smaller).bytes);
  }
  return most;
}

AdapterBatch adapter_batch(const AdapterShape &shape, const AdapterPlan &plan, const int32_t *ids,
                           unsigned char *workspace) {
  AdapterBatch batch{};
  batch.ids = ids;
  batch.rows = shape.rows;
  batch.count = static_cast<int32_t>(shape.count);
  if (plan.max_tiles > 0) {
    batch.tiles = reinterpret_cast<int32_t *>(workspace + plan.route);
    batch.runs = batch.tiles + 4 * plan.max_tiles;
    batch.run_slots = batch.runs + 8 * plan.max_runs;
    batch.starts = batch.run_slots + (plan.run_rows > 0 ? 2 * shape.count : 0);
    batch.perm = batch.starts + shape.count + 1;
    batch.transposes = transposes_compact(shape) ? batch.perm + shape.rows : nullptr;
    batch.max_tiles = static_cast<int32_t>(plan.max_tiles);
    batch.max_runs = static_cast<int32_t>(plan.max_runs);
    batch.run_rows = static_cast<int32_t>(plan.run_rows);
  }
  return batch;
}

KernelLaunch make_adapter_route(const AdapterRouteArgs &args) {
  return launch_of(reinterpret_cast<const void *>(&adapter_route_kernel), dim3(1, 1, 1), kRouteThreads, args);
}

KernelLaunch make_adapter_shrink(const AdapterShrinkArgs &args, const AdapterPlan &plan, int dtype) {
  const int tiles = static_cast<int>(plan.rp / 16);
  const void *func = dtype == kDtypeF32   ? AdapterKernels<F32Payload>::shrink(tiles)
                     : dtype == kDtypeF16 ? AdapterKernels<F16Payload>::shrink(tiles)
                                          : AdapterKernels<Bf16Payload>::shrink(tiles);
  AdapterShrinkArgs record = args;
  record.slots = tile_slots(args.batch);
  return launch_of(func, dim3(static_cast<unsigned>((args.job[0].ranges + args.job[1].ranges) * record.slots), 1, 1),
                   kAdapterShrinkWaves * kWave, record);
}

KernelLaunch make_adapter_expand(const AdapterExpandArgs &args, const AdapterPlan &plan, int dtype) {
  const int tiles = static_cast<int>(plan.rp / 16);
  const bool direct = args.batch.tiles == nullptr;
  const AdapterAct act = args.act.function == kActivationNone                                       ? AdapterAct::None
                         : args.act.gated != 0 && args.act.function == kActivationSilu ? AdapterAct::GatedSilu
                                                                                       : AdapterAct::Any;
  const void *func = dtype == kDtypeF32   ? AdapterKernels<F32Payload>::expand(tiles, act, direct)
                     : dtype == kDtypeF16 ? AdapterKernels<F16Payload>::expand(tiles, act, direct)
                                          : AdapterKernels<Bf16Payload>::expand(tiles, act, direct);
  AdapterExpandArgs record = args;
  const int64_t unit = dtype == kDtypeF32 ? 64 : 128;  // columns of a turn; in decode of each wave
  const int64_t turn = direct ? kAdapterExpandWaves * unit : unit;
  const int64_t turns = (args.n + turn - 1) / turn;
  const int64_t row_tiles = direct ? args.batch.rows : (args.batch.rows + kAdapterTileRows - 1) / kAdapterTileRows;
  const int64_t wanted = direct ? kDirectWorkgroups : kExpandWorkgroups;
  const int64_t groups = std::min(turns, std::max<int64_t>(1, (wanted + row_tiles - 1) / row_tiles));
  record.columns = (turns + groups - 1) / groups * turn;
  return launch_of(func,
                   dim3(static_cast<unsigned>((args.n + record.columns - 1) / record.columns), tile_slots(args.batch), 1),
                   kAdapterExpandWaves * kWave, record);
}

bool adapter_routes_beside_transpose(const AdapterBatch &batch) {
  return batch.count <= kTransposeGroups && batch.rows <= kRoutesBesideRows;
}

KernelLaunch make_adapter_route_transpose(const AdapterRouteTransposeArgs &args) {
  const void *func = args.transpose.element == 4
                         ? reinterpret_cast<const void *>(&adapter_route_transpose_kernel<uint32_t>)
                         : reinterpret_cast<const void *>(&adapter_route_transpose_kernel<uint16_t>);
  dim3 grid = transpose_grid(args.transpose);
  grid.x += 1;
  return launch_of(func, grid, kRouteThreads, args);
}

KernelLaunch make_adapter_transpose(const AdapterRouteTransposeArgs &args) {
  const void *func = args.transpose.element == 4 ? reinterpret_cast<const void *>(&adapter_transpose_kernel<uint32_t>)
                                                 : reinterpret_cast<const void *>(&adapter_transpose_kernel<uint16_t>);
  return launch_of(func, transpose_grid(args.transpose), kRouteThreads, args);
}

KernelLaunch make_adapter_terms(const AdapterTermsArgs &args) {
  return launch_of(reinterpret_cast<const void *>(&adapter_terms_kernel), dim3(tile_slots(args.batch), 2, 1), 256, args);
}

KernelLaunch make_adapter_outer(const AdapterOuterArgs &args, const AdapterPlan &plan, int dtype) {
  const int tiles = static_cast<int>(plan.rp / 16);
  const void *func = dtype == kDtypeF32   ? AdapterKernels<F32Payload>::outer(tiles)
                     : dtype == kDtypeF16 ? AdapterKernels<F16Payload>::outer(tiles)
                                          : AdapterKernels<Bf16Payload>::outer(tiles);
  const int64_t columns = dtype == kDtypeF32 || tiles > 2 ? 64 : 128;  // of a workgroup (kOuterColumns)
  const int64_t blocks = (args.job[0].columns + columns - 1) / columns + (args.job[1].columns + columns - 1) / columns;
  const int64_t runs = std::min<int64_t>(plan.max_runs, args.batch.rows / plan.run_rows + kExtraSlots);
  return launch_of(func,
                   dim3(static_cast<unsigned>(blocks),
                        static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(runs, 1), 65535)), 1),
                   kAdapterOuterWaves * kWave, args);
}

KernelLaunch make_adapter_reduce(const AdapterReduceArgs &args) {
  AdapterReduceArgs record = args;
  record.blocks0 = (args.job[0].columns * args.max_rank + 1023) / 1024;
  const int64_t blocks1 = (args.job[1].columns * args.max_rank + 1023) / 1024;
  return launch_of(reinterpret_cast<const void *>(&adapter_reduce_kernel),
                   dim3(static_cast<unsigned>(record.blocks0 + blocks1),
                        static_cast<unsigned>(std::min(args.batch.count, 1024)), 1),
                   256, record);
}

}  // namespace xp
