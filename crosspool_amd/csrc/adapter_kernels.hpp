// Low-rank adapters of many requests beside a shared projection, and their gradients, on gfx950.
//
//   t[i] = A_a x[i]                     (shrink:  r = the adapter's rank, up to 128)
//   y[i] = act(base[i] + s_a B_a t[i])  (expand;  without an activation y = base + s_a B_a t)
// for every token row i, a = ids[i]; ids[i] = -1 leaves base alone.  With dy the gradient of y
// (no activation), u[i] = B_a^T dy[i]:
//   dx[i] = base[i] + s_a A_a^T u[i],  dA_a = s_a sum_i u[i] x[i]^T,  dB_a = s_a sum_i dy[i] t[i]^T,
// sums over the rows of adapter a.  u is shrink over B_a^T, dx is expand over A_a^T, so the
// backward pass transposes the weights of the adapters in use once and runs the same two kernels;
// dA and dB are the outer-product kernel.
//
// Rows are worked on by adapter, in tiles of up to 64 rows that share one.  Up to 64 rows the tiles
// are found with ballots inside every workgroup (no launch of its own); above, one workgroup sorts
// the rows by adapter first (stable, so sums have one order and repeated calls the same bits).
//
// Everything here is bound by memory or, at few rows, by latency: with r <= 128 the matrix cores
// need a fraction of the time that the rows' bytes do.  t, u and all sums are fp32.  16-bit
// payloads multiply t (u) as two bf16 terms, its leading 16 bits truncated and the rest rounded
// (relative error 2^-17, below the 2^-9 of the output's rounding); fp16 weights and rows beside it
// are split the same way (within 2^-133), because fp16 terms of t would overflow or lose the small ones.
#pragma once

#include "xp_elements.hpp"
#include "xp_kernels.hpp"

namespace xp {

constexpr int kAdapterShrinkWaves = 4;

// Elements of P in 16 bytes, and columns in one 16 x 16 MFMA step over four such chunks.
template <class P>
constexpr int kChunk = 16 / kElementBytes<P>;
template <class P>
constexpr int kStep = 4 * kChunk<P>;

// A uniform value that the compiler takes as made here: what is computed from it is not moved ahead of
// this point (out of the loop over a workgroup's tiles, where addresses of every load would take
// registers from the loads themselves).
__device__ __forceinline__ int64_t made_here(int64_t value) {
  __asm__ volatile("" : "+s"(value));
  return value;
}
__device__ __forceinline__ int lane_here() {
  int lane = static_cast<int>(threadIdx.x & 63);
  __asm__ volatile("" : "+v"(lane));
  return lane;
}

// A run of rows whose outer products one workgroup sums.
struct AdapterRun {
  int group;
  int first;  // positions first .. end - 1
  int end;
  int slot;   // of its partial sums, or -1: the adapter's only run
  int tile;   // its first tile
};

struct AdapterTile {
  int group;  // the adapter; count: rows without one; count + 1: rows whose id is out of range; -1: no tile
  int rows;
  int rank;   // 0 without an adapter
  int place;  // of its weights: the adapter, or in a backward pass its transposes' place
  int row;    // lane i: the tile's row i (past the tile: any row of the batch)
};

__device__ __forceinline__ int adapter_group(int id, int count) {
  return id >= 0 && id < count ? id : id == -1 ? count : count + 1;
}

__device__ __forceinline__ int adapter_rank_of(const int32_t *ranks, int group, int max_rank) {
  const int rank = ranks != nullptr ? ranks[group] : max_rank;
  return rank < 0 ? 0 : rank > max_rank ? max_rank : rank;
}
// The same for a group that all lanes share.
__device__ __forceinline__ int adapter_rank(const int32_t *ranks, int group, int max_rank) {
  return __builtin_amdgcn_readfirstlane(adapter_rank_of(ranks, group, max_rank));
}

// Tile `slot` of the batch, the same in every wave of a workgroup.  `all`: tiles of rows without an
// adapter too.
__device__ __forceinline__ AdapterTile adapter_tile(const AdapterBatch &batch, const int32_t *ranks, int max_rank,
                                                    int64_t slot, bool all) {
  const int lane = lane_here();
  AdapterTile tile{-1, 0, 0, 0, 0};
  if (batch.tiles == nullptr) {
    // One slot per row: the first row of each adapter leads its tile.
    if (slot >= batch.rows) {
      return tile;
    }
    const bool live = lane < batch.rows;
    const int group = live ? adapter_group(batch.ids[lane], batch.count) : -1;
    const int mine = __builtin_amdgcn_readlane(group, static_cast<int>(slot));
    const unsigned long long mask = __ballot(live && group == mine);
    if (__builtin_ctzll(mask) != slot || (!all && mine >= batch.count)) {
      return tile;
    }
    tile.group = mine;
    tile.place = mine;
    tile.rows = __popcll(mask);
    tile.rank = mine < batch.count ? adapter_rank(ranks, mine, max_rank) : 0;
    // Every row of the tile sends its number to the lane of its place, the others to the last lanes.
    const unsigned long long below = (1ull << lane) - 1;
    const int place = (mask >> lane & 1) != 0 ? __popcll(mask & below) : tile.rows + __popcll(~mask & below);
    const int row = __builtin_amdgcn_ds_permute(4 * place, lane);
    tile.row = lane < tile.rows ? row : static_cast<int>(slot);
  } else {
    // Tiles of adapters come first, then those of rows without one, then entries of group -1.
    if (slot >= batch.max_tiles) {
      return tile;
    }
    const u32x4 entry = *reinterpret_cast<const u32x4 *>(batch.tiles + 4 * slot);
    const int group = __builtin_amdgcn_readfirstlane(static_cast<int>(entry[0]));
    if (group < 0 || (!all && group >= batch.count)) {
      return tile;
    }
    const int first = __builtin_amdgcn_readfirstlane(static_cast<int>(entry[1]));
    tile.group = group;
    tile.rows = __builtin_amdgcn_readfirstlane(static_cast<int>(entry[2]));
    const int rank_and_place = __builtin_amdgcn_readfirstlane(static_cast<int>(entry[3]));
    tile.rank = rank_and_place % 256;
    tile.place = rank_and_place / 256;
    tile.row = batch.perm[first + (lane < tile.rows ? lane : 0)];
  }
  return tile;
}

// The two bf16 terms of a pair of values: leading bits truncated, the rest to nearest even.  Both have the
// value's sign, and neither is zero unless the value is: a rest of zero would make NaN of an infinite factor, so
// bf16's smallest number (2^-133; the matrix cores keep subnormal operands) is added to every rest, far
// below the rest's own rounding where the value is above 2^-110.
__device__ __forceinline__ float leading_term(float value) {
  const uint32_t bits = __float_as_uint(value);
  return __uint_as_float((bits & 0xffff0000u) | (value != value ? 0x00400000u : 0u));
}
__device__ __forceinline__ float rest_term(float value, float leading) {
  constexpr float kLeast = 0x1p-133f;
  const float rest = (__float_as_uint(value) & 0x7f800000u) == 0x7f800000u ? 0.0f : value - leading;
  return rest + __builtin_amdgcn_fmed3f(value, -kLeast, kLeast);
}
__device__ __forceinline__ void split_pair(float a, float b, uint32_t &high, uint32_t &low) {
  const float ha = leading_term(a);
  const float hb = leading_term(b);
  high = (__float_as_uint(ha) >> 16) | (__float_as_uint(hb) & 0xffff0000u);
  low = Bf16Payload::pack2(rest_term(a, ha), rest_term(b, hb));
}

// A chunk of P as bf16 terms: itself (bf16), or two terms (fp16).
template <class P>
__device__ __forceinline__ void chunk_terms(u32x4 chunk, u32x4 &high, u32x4 &low) {
  if constexpr (std::is_same_v<P, F16Payload>) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t h;
      uint32_t l;
      split_pair(P::widen(chunk[w] & 0xffffu), P::widen(chunk[w] >> 16), h, l);
      high[w] = h;
      low[w] = l;
    }
  } else {
    high = chunk;
  }
}

// Word w of a mask that keeps a chunk's first `count` elements of P.
template <class P>
__device__ __forceinline__ uint32_t chunk_mask(int w, int count) {
  if constexpr (kElementBytes<P> == 4) {
    return w < count ? 0xffffffffu : 0u;
  } else {
    return 2 * w + 1 < count ? 0xffffffffu : 2 * w < count ? 0x0000ffffu : 0u;
  }
}

template <class P>
__device__ __forceinline__ float element(const void *base, int64_t index) {
  return load_value(base, index, kDtypeOf<P>);
}

// ------------------------------------------------------------------ shrink
// One tile of rows against all of its adapter's A rows over one K range.  The workgroup's four waves
// take the range's groups of U steps in turn; a step is 64 bytes of every row.  Loads have four
// neighbouring lanes on a row's 64 bytes and go through 1 KB of LDS per operand, the wave's own, to the
// lanes that the MFMA wants them in: loaded in those, with rows along the lanes, every lane is an access of
// its own (8192 x 12288 of one adapter of rank 64 in bf16: 59 us, 53 to 55 so).  Partial sums
// of the waves meet in LDS, those of the ranges in `partials` [range][row][rp].  Bound by the rows' bytes:
// 4096 rows of 24576 and of 4096 columns at rank 16 take 53 us (4.4 TB/s); at rank 64 every tile of 64 rows
// reads as many bytes of A, from the L2, as of the rows (8192 x 12288, eight adapters: 57 to 59 us, 3.5 TB/s).
template <int RT>
constexpr int kShrinkRegion = (4 + RT) * 1024;  // bytes of LDS per wave

template <class P, int NRT, int TT, int U, int REGION>
__device__ __forceinline__ void shrink_body(const AdapterShrinkArgs &a, const AdapterShrinkJob &job, int64_t range,
                                            const AdapterTile &tile, int place, unsigned char *lds) {
  constexpr int ES = kElementBytes<P>;
  constexpr int STEP = kStep<P>;
  const int64_t k = made_here(job.k);
  const int lane = lane_here();
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  unsigned char *own = lds + wave * REGION;
  // Loading, lane l has chunk l % 4 of row l / 4; multiplying, chunk l / 16 of row l % 16.  A row's chunks
  // are exchanged by its number so that 16 lanes reading one chunk of 16 rows use all banks.
  const int put = (lane >> 2) * 64 + (((lane & 3) ^ (lane >> 4)) << 4);
  const int get = (lane & 15) * 64 + (((lane >> 4) ^ (lane >> 2 & 3)) << 4);
  // Rows past the tile read another, ranks past the adapter's the first: their sums go nowhere.
  const unsigned char *x[TT];
  const unsigned char *w = static_cast<const unsigned char *>(job.w) + static_cast<int64_t>(place) * job.w_rows * k * ES;
  uint32_t w_offset[NRT];
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const int64_t row = __shfl(tile.row, t * 16 + (lane >> 2), kWave);
    x[t] = static_cast<const unsigned char *>(job.x) + row * job.ldx * ES + (lane & 3) * 16;
  }
#pragma unroll
  for (int r = 0; r < NRT; ++r) {
    const int at = r * 16 + (lane >> 2);
    w_offset[r] = static_cast<uint32_t>((at < tile.rank ? at : 0) * k * ES + (lane & 3) * 16);
  }
  f32x4 acc[NRT][TT];
#pragma unroll
  for (int r = 0; r < NRT; ++r) {
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      acc[r][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
  auto multiply = [&](const u32x4 (&xs)[TT], const u32x4 (&ws)[NRT]) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      *reinterpret_cast<u32x4 *>(own + t * 1024 + put) = xs[t];
    }
#pragma unroll
    for (int r = 0; r < NRT; ++r) {
      *reinterpret_cast<u32x4 *>(own + (TT + r) * 1024 + put) = ws[r];
    }
    u32x4 rows[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      rows[t] = *reinterpret_cast<const u32x4 *>(own + t * 1024 + get);
    }
#pragma unroll
    for (int r = 0; r < NRT; ++r) {
      const u32x4 weights = *reinterpret_cast<const u32x4 *>(own + (TT + r) * 1024 + get);
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        acc[r][t] = P::mfma16(weights, rows[t], acc[r][t]);
      }
    }
  };
  const int64_t steps = (k + STEP - 1) / STEP;
  const int64_t begin = range * job.steps_per_range;
  const int64_t end = begin + job.steps_per_range < steps ? begin + job.steps_per_range : steps;
  const int64_t whole_end = end < k / STEP ? end : k / STEP;
  const int64_t groups = whole_end > begin ? (whole_end - begin) / U : 0;
  for (int64_t at = wave; at < groups; at += kAdapterShrinkWaves) {
    const int64_t offset = (begin + at * U) * (STEP * ES);
    u32x4 xs[U][TT];
    u32x4 ws[U][NRT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        xs[u][t] = load16_any(x[t] + offset + u * (STEP * ES));
      }
#pragma unroll
      for (int r = 0; r < NRT; ++r) {
        ws[u][r] = load16_any(w + offset + u * (STEP * ES) + w_offset[r]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      multiply(xs[u], ws[u]);
    }
  }
  // The steps past the last whole group, one per wave (at most U <= 4).  A chunk that the width cuts is
  // the row's last whole one with the columns before the cut cleared in both operands (added one column at a
  // time instead, six columns of 777 rows at rank 24 took 5 of 12 us).
  if (const int64_t step = begin + groups * U + wave; step < end) {
    const int64_t chunk = step * 4 + (lane & 3);
    const int before = kChunk<P> - static_cast<int>(k % kChunk<P>);
    const bool whole = (chunk + 1) * kChunk<P> <= k;
    const bool cut = !whole && chunk * kChunk<P> < k && k >= kChunk<P>;
    const int64_t offset = step * (STEP * ES) - (cut ? before * ES : 0);
    u32x4 keep;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      keep[j] = cut ? ~chunk_mask<P>(j, before) : ~0u;
    }
    u32x4 xs[TT];
    u32x4 ws[NRT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      xs[t] = u32x4{0u, 0u, 0u, 0u};
      if (whole || cut) {
        xs[t] = load16_any(x[t] + offset) & keep;
      }
    }
#pragma unroll
    for (int r = 0; r < NRT; ++r) {
      ws[r] = u32x4{0u, 0u, 0u, 0u};
      if (whole || cut) {
        ws[r] = load16_any(w + offset + w_offset[r]) & keep;
      }
    }
    multiply(xs, ws);
  }
  // Rows shorter than a chunk are added one column at a time.
  const int64_t width = made_here(job.k);
  const int64_t cut = width < kChunk<P> ? 0 : width;
  // Lane holds t[row lane % 16][4 (lane / 16) + j] of every 16 x 16 tile.
  const int out_lane = lane_here();
#pragma unroll
  for (int r = 0; r < NRT; ++r) {
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      *reinterpret_cast<f32x4 *>(own + (t * kWave + out_lane) * 16) = acc[r][t];
    }
    __syncthreads();
    const int at = static_cast<int>(threadIdx.x >> 6) * 16 + (out_lane & 15);
    const int64_t row = __shfl(tile.row, at, kWave);
    if (threadIdx.x < TT * kWave) {
      f32x4 sum = *reinterpret_cast<const f32x4 *>(lds + threadIdx.x * 16);
#pragma unroll
      for (int v = 1; v < kAdapterShrinkWaves; ++v) {
        sum += *reinterpret_cast<const f32x4 *>(lds + v * REGION + threadIdx.x * 16);
      }
      const int first = r * 16 + 4 * (out_lane >> 4);
      if (at < tile.rows) {
        for (int64_t column = cut; column < width; ++column) {
          const float value = element<P>(job.x, row * job.ldx + column);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sum[j] += first + j < tile.rank ? value * element<P>(w, (first + j) * width + column) : 0.0f;
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sum[j] = first + j < tile.rank ? sum[j] : 0.0f;
        }
        *reinterpret_cast<f32x4 *>(job.partials + (range * a.batch.rows + row) * a.rp + first) = sum;
      }
    }
    __syncthreads();
  }
}

template <class P, int RT, int TT, int REGION>
__device__ __forceinline__ void shrink_ranks(const AdapterShrinkArgs &a, const AdapterShrinkJob &job, int64_t range,
                                             const AdapterTile &tile, int place, unsigned char *lds) {
  if constexpr (RT > 1) {
    if (tile.rank <= 8 * RT) {
      return shrink_ranks<P, RT / 2, TT, REGION>(a, job, range, tile, place, lds);
    }
  }
  // U steps of TT row and RT weight operands, 16 bytes per lane each, beside the sums: within the 128
  // registers of two workgroups a CU up to two rank tiles, the 256 of one above.  Not of TT: a row's sums
  // have one order however many rows share its adapter (four steps of one operand each would save 0.2 us).
  constexpr int U = RT <= 4 ? 2 : 1;
  shrink_body<P, RT, TT, U, REGION>(a, job, range, tile, place, lds);
}

template <class P, int RT>
__global__ __launch_bounds__(kAdapterShrinkWaves *kWave, RT <= 2 ? 4 : 2) void adapter_shrink_kernel(AdapterShrinkArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[kAdapterShrinkWaves * kShrinkRegion<RT>];
  // A tile's ranges follow one another, so that whole rows are read at about one time (ranges of one
  // part of all rows first: 63 us instead of 48 for 4096 x 24576 in bf16).  The second job comes after
  // the first: side by side, the dispatcher's round over the CUs gave half of them the longer ranges only.
  const int64_t first_job = a.job[0].ranges * a.slots;
  const bool second = blockIdx.x >= first_job;
  const AdapterShrinkJob &job = a.job[second ? 1 : 0];
  const int64_t place = second ? blockIdx.x - first_job : blockIdx.x;
  const int64_t range = place % job.ranges;
  for (int64_t slot = place / job.ranges;; slot += a.slots) {
    const AdapterTile tile = adapter_tile(a.batch, a.ranks, a.max_rank, slot, false);
    if (tile.group < 0) {
      return;
    }
    if (tile.rank > 0) {
      const int place = second ? tile.group : tile.place;  // the second job's weights are the pool's own
      if (tile.rows <= 16) {
        shrink_ranks<P, RT, 1, kShrinkRegion<RT>>(a, job, range, tile, place, lds);
      } else {
        shrink_ranks<P, RT, 4, kShrinkRegion<RT>>(a, job, range, tile, place, lds);
      }
    }
  }
}

// ------------------------------------------------------------------ expand
// One tile of rows against a range of its adapter's B rows (output columns): t is summed over its K
// ranges once per workgroup into LDS as MFMA operands ([leading terms | rests] of 16-bit payloads:
// one product over 2 r columns).  Rows are the MFMA's M operand and output columns its N, column
// CH i + j of a unit of 16 CH being column i of MFMA tile j: a lane's sums over the CH tiles are then 16
// bytes of consecutive columns of one row, and 16 lanes hold 256 contiguous bytes of it, so that base is
// read and the result stored in whole lines by neighbouring lanes.  (With rows along the lanes, as the
// products' natural layout has them, every lane of a load or store is an access of its own: 60 us instead
// of 39 for 8192 x 4096 at rank 64 in bf16.)
//
// Sorted batches give each wave 16 rows of a tile and stage a unit's B rows in LDS, read from memory
// once and in order, one unit ahead.  Small ones (decode) give each wave a unit of its own and turn the B
// rows in its LDS as shrink does (48 rows of 32 adapters of rank 32 x 24576: 16.4 us, 13.8 so, 4 TB/s of B's
// 64-byte rows).  Bound by base and output, whose 256-byte pieces of 64 rows read and write
// below a plain copy's rate: 2048 x 24576 with a gated SiLU at rank 32 40.7 us (3.8 TB/s), 8192 x 4096 at
// rank 64 39 us (3.4 TB/s).  A second unit in flight, two to three times the workgroups and nontemporal
// stores changed nothing or cost up to a fifth.
constexpr int kAdapterExpandWaves = 4;

// The epilogue's activation: none, a gated SiLU, or any.
enum class AdapterAct : int { None = 0, GatedSilu = 1, Any = 2 };

template <class P, int RT>
constexpr int kAdapterTermStride = std::is_same_v<P, F32Payload> ? 4 * (RT * 16 + 4) : 2 * (2 * RT * 16 + 8);  // bytes

// Consecutive values to an element-aligned address.
template <class P, int N>
__device__ __forceinline__ void store_values(unsigned char *out, const float (&value)[N]) {
  constexpr int WORDS = N * kElementBytes<P> / 4;
  using Words = uint32_t __attribute__((ext_vector_type(WORDS), aligned(kElementBytes<P>)));
  Words packed;
#pragma unroll
  for (int j = 0; j < WORDS; ++j) {
    if constexpr (kElementBytes<P> == 4) {
      packed[j] = __float_as_uint(value[j]);
    } else {
      packed[j] = P::pack2(value[2 * j], value[2 * j + 1]);
    }
  }
  *reinterpret_cast<Words *>(out) = packed;
}

// f(g) (u + offset) of the sum, any f.
__device__ __forceinline__ float gated_value(float gate, float up, ActivationArgs act) {
  if (act.has_limit) {
    clip_keep_nan(gate, up, act.limit);
  }
  act.has_limit = 0;
  return apply_gated(gate, up, act);
}

// silu(g) (u + offset).  16-bit results take the hardware's exp and reciprocal (relative error below
// 2^-16, under the store's 2^-9 or 2^-12), fp32 ones expf and an IEEE divide as elsewhere.
template <class P>
__device__ __forceinline__ float gated_silu_value(float gate, float up, const ActivationArgs &act) {
  if (act.has_limit) {
    clip_keep_nan(gate, up, act.limit);
  }
  if constexpr (kElementBytes<P> == 4) {
    return gate / (1.0f + expf(-act.alpha * gate)) * (up + act.up_offset);
  } else {
    return gate * __builtin_amdgcn_rcpf(1.0f + __expf(-act.alpha * gate)) * (up + act.up_offset);
  }
}

// t of the tile's rows: the K ranges' sums, in range order, as the operands that the products read
// (zero past the rank).  The workgroup meets after it.
template <class P, int RT>
__device__ __forceinline__ void stage_terms(const AdapterExpandArgs &a, const AdapterTile &tile, unsigned char *terms) {
  constexpr int kBatch = 8;
  constexpr int kQuads = 4 * RT;
  const int64_t plane = a.batch.rows * a.rp;
  for (int first = 0; first < tile.rows * kQuads; first += kAdapterExpandWaves * kWave) {
    const int index = first + static_cast<int>(threadIdx.x);
    const int at = index / kQuads;
    const int quad = index % kQuads;
    const int64_t row = __shfl(tile.row, at & 63, kWave);  // of every lane, before some have no part
    if (at >= tile.rows) {
      continue;
    }
    const float *source = a.partials + row * a.rp + 4 * quad;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (4 * quad < tile.rank) {
      for (int64_t batch = 0; batch < a.ranges; batch += kBatch) {
        f32x4 part[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          if (batch + j < a.ranges) {
            part[j] = *reinterpret_cast<const f32x4 *>(source + (batch + j) * plane);
          }
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          if (batch + j < a.ranges) {
            sum += part[j];
          }
        }
      }
    }
    unsigned char *target = terms + at * kAdapterTermStride<P, RT>;
    if constexpr (std::is_same_v<P, F32Payload>) {
      *reinterpret_cast<f32x4 *>(target + 16 * quad) = sum;
    } else {
      uint32_t h0;
      uint32_t h1;
      uint32_t l0;
      uint32_t l1;
      split_pair(sum[0], sum[1], h0, l0);
      split_pair(sum[2], sum[3], h1, l1);
      *reinterpret_cast<u32x2 *>(target + 8 * quad) = u32x2{h0, h1};
      *reinterpret_cast<u32x2 *>(target + 32 * RT + 8 * quad) = u32x2{l0, l1};
    }
  }
}

// The columns from `first` on, one (a gated pair) per thread: those past the last whole chunk.
template <class P, int RT, AdapterAct ACT>
__device__ __forceinline__ void expand_columns(const AdapterExpandArgs &a, const AdapterTile &tile,
                                               const unsigned char *terms, float scale, int64_t first) {
  const bool gated = ACT == AdapterAct::GatedSilu || (ACT == AdapterAct::Any && a.act.gated != 0);
  const int columns = static_cast<int>(a.n - first) / (gated ? 2 : 1);
  const int64_t weights = static_cast<int64_t>(tile.place) * a.n * a.ld_w;
  for (int start = 0; start < tile.rows * columns; start += kAdapterExpandWaves * kWave) {
    const int index = start + static_cast<int>(threadIdx.x);
    const int at = index / columns;
    const int64_t row = __shfl(tile.row, at & 63, kWave);
    if (at >= tile.rows) {
      continue;
    }
    const unsigned char *t = terms + at * kAdapterTermStride<P, RT>;
    auto column = [&](int64_t n) __attribute__((always_inline)) {
      float sum = 0.0f;
#pragma unroll 4
      for (int r = 0; r < tile.rank; ++r) {
        float coefficient;
        if constexpr (std::is_same_v<P, F32Payload>) {
          coefficient = reinterpret_cast<const float *>(t)[r];
        } else {
          const uint16_t *parts = reinterpret_cast<const uint16_t *>(t);
          coefficient = bf16_to_float(parts[r]) + bf16_to_float(parts[RT * 16 + r]);
        }
        sum += coefficient * element<P>(a.w, weights + n * a.ld_w + r);
      }
      const float from_base = a.base != nullptr ? element<P>(a.base, row * a.ld_base + n) : 0.0f;
      return tile.rank > 0 ? from_base + scale * sum : from_base;
    };
    const int64_t n = index - at * columns;
    if (gated) {
      const float gate = column(first + 2 * n);
      const float up = column(first + 2 * n + 1);
      float value;
      if constexpr (ACT == AdapterAct::GatedSilu) {
        value = gated_silu_value<P>(gate, up, a.act);
      } else {
        value = gated_value(gate, up, a.act);
      }
      store_value(a.out, row * a.ld_out + first / 2 + n, value, kDtypeOf<P>);
    } else {
      const float value = column(first + n);
      store_value(a.out, row * a.ld_out + first + n, ACT == AdapterAct::Any ? apply_function(value, a.act) : value,
                  kDtypeOf<P>);
    }
  }
}

template <class P, int RT, AdapterAct ACT>
struct AdapterExpand {
  static constexpr int ES = kElementBytes<P>;
  static constexpr int CH = kChunk<P>;
  static constexpr bool F32 = std::is_same_v<P, F32Payload>;
  static constexpr bool F16 = std::is_same_v<P, F16Payload>;
  static constexpr int UNIT = 16 * CH;                     // columns
  static constexpr int C = RT * 16 / CH;                   // chunks of a B row
  static constexpr int STEPS = F32 ? C / 4 : C / 2;        // MFMA steps: r columns, or 2 r
  static constexpr int FRAGS = F32 ? C / 4 : (C + 3) / 4;  // distinct B operands among them
  static constexpr int STAGED = UNIT * C / (kAdapterExpandWaves * kWave);  // chunks per thread: RT
  static constexpr int PLANES = F16 ? 2 : 1;               // fp16 is staged as its two bf16 terms
  static constexpr int PLANE_BYTES = UNIT * C * 16;
  static constexpr int TERM_BYTES = kAdapterTileRows * kAdapterTermStride<P, RT>;
  static constexpr int TURN_BYTES = kAdapterExpandWaves * CH * 1024;
  static constexpr int LDS_BYTES = 2 * PLANES * PLANE_BYTES > TERM_BYTES ? 2 * PLANES * PLANE_BYTES : TERM_BYTES;

  const AdapterExpandArgs &a;
  const unsigned char *w;
  int64_t whole;  // columns before it are stored here
  int rank;
  int lane16;
  int quarter;
  int row[4];     // the lane's rows; past the tile: another, which is not stored
  bool live[4];
  u32x4 ts[STEPS];
  u32x4 base[4];       // of this turn
  u32x4 next_base[4];  // of the next

  // Rows first .. first + 15 of the tile.
  __device__ __forceinline__ AdapterExpand(const AdapterExpandArgs &args, int64_t whole_columns, const AdapterTile &tile,
                                           int first)
      : a(args),
        w(static_cast<const unsigned char *>(args.w) + static_cast<int64_t>(tile.place) * args.n * args.ld_w * ES),
        whole(whole_columns),
        rank(tile.rank),
        lane16(lane_here() & 15),
        quarter(lane_here() >> 4) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int at = first + 4 * quarter + q;
      row[q] = __shfl(tile.row, at, kWave);
      live[q] = at < tile.rows;
    }
  }

  // Columns past the whole ones read the last of those; they are not stored.
  __device__ __forceinline__ void load_base(int64_t c0) {
    if (a.base != nullptr) {
      const int64_t n = c0 + CH * lane16;
      const int64_t column = n < whole ? n : whole - CH;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        next_base[q] = load16_any(static_cast<const unsigned char *>(a.base) + (row[q] * a.ld_base + column) * ES);
      }
    }
  }

  __device__ __forceinline__ void load_terms(const unsigned char *terms, int first) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      ts[s] = *reinterpret_cast<const u32x4 *>(terms + (first + lane16) * kAdapterTermStride<P, RT> + (s * 4 + quarter) * 16);
    }
  }

  // A chunk of a B row with what lies past the rank cleared (the pool may hold anything there).
  __device__ __forceinline__ u32x4 within_rank(u32x4 value, int chunk) const {
    if (rank != RT * 16) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        value[j] &= chunk_mask<P>(j, rank - chunk * CH);
      }
    }
    return value;
  }
  // Its bytes: chunks past the rank read the row's first, rows past the whole columns the last of those.
  __device__ __forceinline__ u32x4 load_chunk_of(int64_t n, int chunk) const {
    const uint32_t row_offset = static_cast<uint32_t>(n < whole ? n : whole - 1) * static_cast<uint32_t>(a.ld_w * ES);
    return load16_any(w + (row_offset + (chunk * CH < rank ? chunk * 16 : 0)));
  }

  __device__ __forceinline__ void add_products(f32x4 (&acc)[CH], int j, int s, u32x4 high, u32x4 low) const {
    if constexpr (F32) {
      acc[j] = F32Payload::mfma16(ts[s], high, acc[j]);
    } else {
      acc[j] = Bf16Payload::mfma16(ts[s], high, acc[j]);
      if constexpr (F16) {
        acc[j] = Bf16Payload::mfma16(ts[s], low, acc[j]);
      }
    }
  }

  // B rows of a unit in LDS: row CH i + j at place 16 j + i, whose chunks are exchanged so that the 16
  // lanes that read one chunk of neighbouring places use all banks.
  __device__ static __forceinline__ int staged_offset(int place, int chunk) {
    const int exchange = C >= 16 ? place & 15 : place * C / 16 & (C - 1);
    return (place * C + (chunk ^ exchange)) * 16;
  }
  __device__ __forceinline__ void fetch(int64_t c0, u32x4 (&staged)[STAGED]) const {
#pragma unroll
    for (int i = 0; i < STAGED; ++i) {
      const int e = i * kAdapterExpandWaves * kWave + static_cast<int>(threadIdx.x);
      staged[i] = load_chunk_of(c0 + e / C, e % C);
    }
  }
  __device__ __forceinline__ void stage(const u32x4 (&staged)[STAGED], unsigned char *lds) const {
#pragma unroll
    for (int i = 0; i < STAGED; ++i) {
      const int e = i * kAdapterExpandWaves * kWave + static_cast<int>(threadIdx.x);
      const int n = e / C;
      const int offset = staged_offset(n % CH * 16 + n / CH, e % C);
      u32x4 high;
      u32x4 low;
      chunk_terms<P>(within_rank(staged[i], e % C), high, low);
      *reinterpret_cast<u32x4 *>(lds + offset) = high;
      if constexpr (F16) {
        *reinterpret_cast<u32x4 *>(lds + PLANE_BYTES + offset) = low;
      }
    }
  }
  __device__ __forceinline__ void multiply_staged(const unsigned char *lds, f32x4 (&acc)[CH]) const {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
#pragma unroll
      for (int f = 0; f < FRAGS; ++f) {
        const int offset = staged_offset(16 * j + lane16, (f * 4 + quarter) % C);
        const u32x4 high = *reinterpret_cast<const u32x4 *>(lds + offset);
        u32x4 low = high;
        if constexpr (F16) {
          low = *reinterpret_cast<const u32x4 *>(lds + PLANE_BYTES + offset);
        }
#pragma unroll
        for (int s = f; s < STEPS; s += FRAGS) {
          add_products(acc, j, s, high, low);
        }
      }
    }
  }

  // Whether the limit holds is decided once per unit, not by a selection per value.
  __device__ __forceinline__ void store(int64_t c0, float scale, const f32x4 (&acc)[CH]) const {
    if (ACT != AdapterAct::None && a.act.has_limit) {
      store_rows<true>(c0, scale, acc);
    } else {
      store_rows<false>(c0, scale, acc);
    }
  }
  template <bool LIMIT>
  __device__ __forceinline__ void store_rows(int64_t c0, float scale, const f32x4 (&acc)[CH]) const {
    ActivationArgs act = a.act;
    act.has_limit = LIMIT ? 1 : 0;
    const bool gated = ACT == AdapterAct::GatedSilu || (ACT == AdapterAct::Any && act.gated != 0);
    const int64_t n = c0 + CH * lane16;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (!live[q] || n >= whole) {
        continue;
      }
      float value[CH];
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        float from_base = 0.0f;
        if (a.base != nullptr) {
          if constexpr (F32) {
            from_base = __uint_as_float(base[q][j]);
          } else {
            from_base = P::widen(j % 2 == 0 ? base[q][j / 2] & 0xffffu : base[q][j / 2] >> 16);
          }
        }
        value[j] = fmaf(scale, acc[j][q], from_base);
      }
      unsigned char *out = static_cast<unsigned char *>(a.out);
      if (gated) {
        float activated[CH / 2];
#pragma unroll
        for (int j = 0; j < CH / 2; ++j) {
          if constexpr (ACT == AdapterAct::GatedSilu) {
            activated[j] = gated_silu_value<P>(value[2 * j], value[2 * j + 1], act);
          } else {
            activated[j] = gated_value(value[2 * j], value[2 * j + 1], act);
          }
        }
        store_values<P>(out + (row[q] * a.ld_out + n / 2) * ES, activated);
      } else {
        if constexpr (ACT == AdapterAct::Any) {
#pragma unroll
          for (int j = 0; j < CH; ++j) {
            value[j] = apply_function(value[j], act);
          }
        }
        store_values<P>(out + (row[q] * a.ld_out + n) * ES, value);
      }
    }
  }

  __device__ __forceinline__ void take_base() {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      base[q] = next_base[q];
    }
  }
};

template <int CH>
__device__ __forceinline__ void clear(f32x4 (&acc)[CH]) {
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
}

// The units of columns go to the waves (decode), for each 16 of the tile's rows.
template <class P, int RT, AdapterAct ACT>
__device__ __forceinline__ void expand_by_columns(const AdapterExpandArgs &a, const AdapterTile &tile, unsigned char *lds,
                                                  float scale, int64_t whole, int64_t begin, int64_t stop,
                                                  bool stage_here) {
  using Work = AdapterExpand<P, RT, ACT>;
  constexpr int CH = Work::CH;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = lane_here();
  // Loading, lane l has chunk l % 4 of the l / 4-th row; multiplying, chunk l / 16 of the l % 16-th (shrink's
  // exchange of chunks).
  unsigned char *own = lds + Work::TERM_BYTES + wave * CH * 1024;
  const int put = (lane >> 2) * 64 + (((lane & 3) ^ (lane >> 4)) << 4);
  const int get = (lane & 15) * 64 + (((lane >> 4) ^ (lane >> 2 & 3)) << 4);
#pragma unroll 1
  for (int first = 0; first < tile.rows; first += 16) {
    Work work(a, whole, tile, first);
#pragma unroll 1
    for (int64_t c0 = begin + wave * Work::UNIT; c0 < stop; c0 += kAdapterExpandWaves * Work::UNIT) {
      work.load_base(c0);
      f32x4 acc[CH];
      clear(acc);
      if (tile.rank > 0) {
        u32x4 ws[CH][Work::FRAGS];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
#pragma unroll
          for (int f = 0; f < Work::FRAGS; ++f) {
            ws[j][f] = work.load_chunk_of(c0 + CH * (lane >> 2) + j, (f * 4 + (lane & 3)) % Work::C);
          }
        }
        if (stage_here && first == 0 && c0 == begin + wave * Work::UNIT) {
          // Every wave has columns: t is summed while B is on its way.
          stage_terms<P, RT>(a, tile, lds);
          __syncthreads();
        }
        work.load_terms(lds, first);
#pragma unroll
        for (int f = 0; f < Work::FRAGS; ++f) {
#pragma unroll
          for (int j = 0; j < CH; ++j) {
            *reinterpret_cast<u32x4 *>(own + j * 1024 + put) = ws[j][f];
          }
#pragma unroll
          for (int j = 0; j < CH; ++j) {
            const u32x4 turned = *reinterpret_cast<const u32x4 *>(own + j * 1024 + get);
            u32x4 high;
            u32x4 low;
            chunk_terms<P>(work.within_rank(turned, (f * 4 + work.quarter) % Work::C), high, low);
#pragma unroll
            for (int s = f; s < Work::STEPS; s += Work::FRAGS) {
              work.add_products(acc, j, s, high, low);
            }
          }
        }
      }
      work.take_base();
      work.store(c0, scale, acc);
    }
  }
}

// The rows of a tile go to the waves, 16 each: B rows through LDS, the next unit's on their way while
// this one's results leave.
template <class P, int RT, AdapterAct ACT>
__device__ __forceinline__ void expand_by_rows(const AdapterExpandArgs &a, const AdapterTile &tile, unsigned char *lds,
                                               float scale, int64_t whole, int64_t begin, int64_t stop) {
  using Work = AdapterExpand<P, RT, ACT>;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int first = 16 * wave;
  Work work(a, whole, tile, first);
  int64_t c0 = begin;
  u32x4 staged[Work::STAGED];
  if (c0 < stop) {
    work.load_base(c0);
    if (tile.rank > 0) {
      work.fetch(c0, staged);
    }
  }
  if (tile.rank > 0) {
    stage_terms<P, RT>(a, tile, lds);
    __syncthreads();
    work.load_terms(lds, first);
    __syncthreads();  // the terms' place is B's now
  }
  unsigned char *now = lds;
  unsigned char *then = lds + Work::PLANES * Work::PLANE_BYTES;
  if (tile.rank > 0 && c0 < stop) {
    work.stage(staged, now);
    __syncthreads();
  }
#pragma unroll 1
  while (c0 < stop) {
    const int64_t next = c0 + Work::UNIT;
    work.take_base();
    if (next < stop) {
      if (tile.rank > 0) {
        work.fetch(next, staged);
      }
      work.load_base(next);
    }
    if (first < tile.rows) {
      f32x4 acc[Work::CH];
      clear(acc);
      if (tile.rank > 0) {
        work.multiply_staged(now, acc);
      }
      work.store(c0, scale, acc);
    }
    if (tile.rank > 0 && next < stop) {
      work.stage(staged, then);
      __syncthreads();
      unsigned char *other = now;
      now = then;
      then = other;
    }
    c0 = next;
  }
}

// Rows with an id out of range: NaN past the activation.
template <class P, AdapterAct ACT>
__device__ __forceinline__ void fill_with_nan(const AdapterExpandArgs &a, const AdapterTile &tile, int64_t begin,
                                              int64_t end) {
  const int per_value = ACT == AdapterAct::GatedSilu || (ACT == AdapterAct::Any && a.act.gated != 0) ? 2 : 1;
  for (int at = 0; at < tile.rows; ++at) {
    const int64_t row = __shfl(tile.row, at, kWave);
    for (int64_t n = begin / per_value + threadIdx.x; n < end / per_value; n += kAdapterExpandWaves * kWave) {
      store_value(a.out, row * a.ld_out + n, __builtin_nanf(""), kDtypeOf<P>);
    }
  }
}

// DIRECT: batches of up to kAdapterDirectRows rows.
template <class P, int RT, AdapterAct ACT, bool DIRECT>
__device__ __forceinline__ void expand_tile(const AdapterExpandArgs &a, const AdapterTile &tile, unsigned char *lds,
                                            int64_t begin, int64_t end) {
  constexpr int CH = kChunk<P>;
  const bool own = tile.group < a.batch.count;
  const float scale = own && a.scales != nullptr ? a.scales[tile.group] : 1.0f;
  // A row without an adapter has sums of +0 and keeps its base through base + -1 * 0 (-0 too).
  const float factor = tile.rank > 0 ? scale : -1.0f;
  // Whole chunks of columns go a unit at a time, the rest one by one; so do the last B rows of a pool whose
  // rows are not whole chunks, since a row's last chunk passes its end, by less than a chunk.
  const int64_t within = a.n - (a.ld_w % CH != 0 ? (CH - 1 + a.ld_w - 1) / a.ld_w : 0);
  const int64_t whole = within < CH ? 0 : within - within % CH;
  const int64_t stop = end < whole ? end : whole;
  if constexpr (DIRECT) {
    const bool all = stop > begin + (kAdapterExpandWaves - 1) * AdapterExpand<P, RT, ACT>::UNIT;
    if (tile.rank > 0 && !all) {
      // Some waves have no columns to load first.
      stage_terms<P, RT>(a, tile, lds);
      __syncthreads();
    }
    expand_by_columns<P, RT, ACT>(a, tile, lds, factor, whole, begin, stop, all);
  } else {
    if (begin < stop) {
      expand_by_rows<P, RT, ACT>(a, tile, lds, factor, whole, begin, stop);
    }
    if (tile.rank > 0 && whole < a.n && end == a.n) {
      __syncthreads();  // B's place is the terms' again for the columns left over
      stage_terms<P, RT>(a, tile, lds);
      __syncthreads();
    }
  }
  if (end == a.n && whole < a.n) {
    expand_columns<P, RT, ACT>(a, tile, lds, scale, whole);
  }
}

template <class P, int RT, AdapterAct ACT, bool DIRECT>
constexpr int kExpandLds = DIRECT ? AdapterExpand<P, RT, ACT>::TERM_BYTES + AdapterExpand<P, RT, ACT>::TURN_BYTES
                                  : AdapterExpand<P, RT, ACT>::LDS_BYTES;

// Workgroups per CU: what the registers hold, or one where the LDS (160 KB) holds no second.
template <class P, int RT, AdapterAct ACT, bool DIRECT>
constexpr int kExpandPerCu = (2 * kExpandLds<P, RT, ACT, DIRECT> > 160 * 1024) ? 1 : RT <= 2 ? 3 : 2;

template <class P, int RT, AdapterAct ACT, bool DIRECT>
__global__ __launch_bounds__(kAdapterExpandWaves *kWave, (kExpandPerCu<P, RT, ACT, DIRECT>))
void adapter_expand_kernel(AdapterExpandArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[kExpandLds<P, RT, ACT, DIRECT>];
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * a.columns;
  const int64_t end = begin + a.columns < a.n ? begin + a.columns : a.n;
  for (int64_t slot = blockIdx.y;; slot += gridDim.y) {
    const AdapterTile tile = adapter_tile(a.batch, a.ranks, a.max_rank, slot, true);
    if (tile.group < 0) {
      return;
    }
    if (tile.group > a.batch.count) {
      if (DIRECT && threadIdx.x == 0) {
        raise_fault(a.fault, kFaultAdapterOutOfRange);
      }
      fill_with_nan<P, ACT>(a, tile, begin, end);
    } else if (tile.rank > 0 || !a.in_place) {
      expand_tile<P, RT, ACT, DIRECT>(a, tile, lds, begin, end);
    }
    __syncthreads();  // the terms are rewritten
  }
}

// ------------------------------------------------------------------ outer products
// dA_a = s sum_i u[i] x[i]^T and dB_a = s sum_i dy[i] t[i]^T over one run of an adapter's rows and 16 CL
// columns of x (dy): the rows are the MFMA's K.  A lane loads CL columns of eight rows (fp32: of four),
// neighbouring lanes neighbouring columns, and pairs of rows' words give, by one byte permutation each,
// the operand of every CL-th column; which 16 columns an MFMA holds is free, so no LDS transposition is
// needed.  The coefficients (u or t) come from adapter_terms_kernel as the operands themselves, a
// kilobyte per load.  Four waves take the run's tiles of 64 rows in turn and meet in LDS; a run that is
// its adapter's only one stores the gradient, others their sums, which adapter_reduce_kernel adds in
// run order.  Bound by the rows' bytes: 4096 rows of 4096 and 24576 columns at rank 16 take 37 us in two
// runs per column block (6.4 TB/s, more than a copy's rate: the pass before read the same rows), 44 us in one, 38 to 39 in three
// or four, whose sums cost the reduction more as well.
constexpr int kAdapterOuterWaves = 4;

template <class P>
constexpr int kOuterRows = std::is_same_v<P, F32Payload> ? 4 : 8;  // rows per lane and step
// Columns per lane: 16 bytes, or half where the sums of four and eight rank tiles take the registers.
template <class P, int RT>
constexpr int kOuterColumns = std::is_same_v<P, F32Payload> || RT > 2 ? 4 : 8;

template <class P, int RT, int NRT, bool SWAP>
__device__ __forceinline__ void outer_body(const AdapterOuterArgs &a, const AdapterOuterJob &job, int64_t block,
                                           const AdapterRun &run, int rank, float scale, unsigned char *lds) {
  constexpr bool F32 = std::is_same_v<P, F32Payload>;
  constexpr bool F16 = std::is_same_v<P, F16Payload>;
  constexpr int ES = kElementBytes<P>;
  constexpr int ROWS = kOuterRows<P>;
  constexpr int BLOCKS = kAdapterTileRows / (4 * ROWS);  // steps per tile
  constexpr int CL = kOuterColumns<P, RT>;
  constexpr int WORDS = CL * ES / 4;
  constexpr int PLANES = F32 ? 1 : 2;
  using Words = uint32_t __attribute__((ext_vector_type(WORDS)));
  const int lane = lane_here();
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane16 = lane & 15;
  const int quarter = lane >> 4;
  const int64_t columns = made_here(job.columns);
  const int64_t c0 = block * 16 * CL;
  // The last lane of a width that CL does not divide takes its last CL columns, some of them twice.
  const bool narrow = columns < CL;
  auto column_of = [&](int index) __attribute__((always_inline)) {
    const int64_t column = c0 + CL * index;
    return narrow ? 0 : column + CL <= columns ? column : columns - CL;
  };
  const unsigned char *data = static_cast<const unsigned char *>(job.data) + column_of(lane16) * ES;
  f32x4 acc[NRT][CL];
#pragma unroll
  for (int r = 0; r < NRT; ++r) {
#pragma unroll
    for (int j = 0; j < CL; ++j) {
      acc[r][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
#pragma unroll 1
  for (int tile = wave; run.first + tile * kAdapterTileRows < run.end; tile += kAdapterOuterWaves) {
    const int position = run.first + tile * kAdapterTileRows;
    const int rows = run.end - position < kAdapterTileRows ? run.end - position : kAdapterTileRows;
    const int mine = a.batch.perm[position + (lane < rows ? lane : 0)];
    const unsigned char *terms = static_cast<const unsigned char *>(job.terms) +
                                 static_cast<int64_t>(run.tile + tile) * (BLOCKS * PLANES * 1024) * (a.rp / 16) + lane * 16;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      if (b * 4 * ROWS >= rows) {
        continue;
      }
      u32x4 coefficient[NRT][PLANES];
#pragma unroll
      for (int r = 0; r < NRT; ++r) {
#pragma unroll
        for (int plane = 0; plane < PLANES; ++plane) {
          coefficient[r][plane] =
              *reinterpret_cast<const u32x4 *>(terms + ((b * (a.rp / 16) + r) * PLANES + plane) * 1024);
        }
      }
      Words words[ROWS];
#pragma unroll
      for (int e = 0; e < ROWS; ++e) {
        const int64_t row = __shfl(mine, b * 4 * ROWS + quarter * ROWS + e, kWave);
        const unsigned char *source = data + row * job.ld * ES;
        if (!narrow) {
          __builtin_memcpy(&words[e], source, sizeof(Words));
        } else {
#pragma unroll
          for (int j = 0; j < WORDS; ++j) {
            words[e][j] = 0u;
          }
#pragma unroll
          for (int j = 0; j < CL - 1; ++j) {
            if (j < columns) {
              if constexpr (F32) {
                words[e][j] = reinterpret_cast<const uint32_t *>(source)[j];
              } else {
                words[e][j / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(source)[j]) << (16 * (j % 2));
              }
            }
          }
        }
      }
      if ((b + 1) * 4 * ROWS > rows) {
        // Rows past the tile have coefficients of zero, which an infinity or NaN would turn into NaN.
#pragma unroll
        for (int e = 0; e < ROWS; ++e) {
          if (b * 4 * ROWS + quarter * ROWS + e >= rows) {
#pragma unroll
            for (int j = 0; j < WORDS; ++j) {
              words[e][j] = 0u;
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < CL; ++j) {
        // Column CL (lane % 16) + j of the lane's rows.
        u32x4 operand;
        u32x4 rest;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (F32) {
            operand[q] = words[q][j];
          } else {
            operand[q] = __builtin_amdgcn_perm(words[2 * q + 1][j / 2], words[2 * q][j / 2],
                                               j % 2 == 0 ? 0x05040100u : 0x07060302u);
          }
        }
        if constexpr (F16) {
          const u32x4 both = operand;
          chunk_terms<P>(both, operand, rest);
        }
#pragma unroll
        for (int r = 0; r < NRT; ++r) {
          auto add = [&](u32x4 with, u32x4 rows_of) __attribute__((always_inline)) {
            using M = std::conditional_t<F32, F32Payload, Bf16Payload>;
            acc[r][j] = SWAP ? M::mfma16(rows_of, with, acc[r][j]) : M::mfma16(with, rows_of, acc[r][j]);
          };
#pragma unroll
          for (int plane = 0; plane < PLANES; ++plane) {
            add(coefficient[r][plane], operand);
            if constexpr (F16) {
              add(coefficient[r][plane], rest);
            }
          }
        }
      }
    }
  }
  // SWAP: lane holds rank lane % 16 and, of column group 4 (lane / 16) + q, column j; otherwise ranks
  // 4 (lane / 16) + q and column group lane % 16.
  const int q = wave;
  const int out_lane = lane_here();
  const int group = SWAP ? 4 * (out_lane >> 4) + q : out_lane & 15;
  const int64_t first = c0 + CL * group;  // as if CL divided the width
  const int64_t column = column_of(group);
  // The group's columns that are its own: from CL - valid on.
  const int skip = first + CL <= columns ? 0 : first < columns ? static_cast<int>(first - column) : CL;
  const int limit = narrow ? static_cast<int>(columns) : CL;
  const int begin_j = narrow ? (group == 0 && block == 0 ? 0 : CL) : skip;
#pragma unroll
  for (int r = 0; r < NRT; ++r) {
#pragma unroll
    for (int j = 0; j < CL; ++j) {
      *reinterpret_cast<f32x4 *>(lds + ((wave * CL + j) * kWave + out_lane) * 16) = acc[r][j];
    }
    __syncthreads();
    float total[CL];
#pragma unroll
    for (int j = 0; j < CL; ++j) {
      const float *flat = reinterpret_cast<const float *>(lds) + (j * kWave + out_lane) * 4 + q;
      total[j] = flat[0];
#pragma unroll
      for (int v = 1; v < kAdapterOuterWaves; ++v) {
        total[j] += flat[v * CL * kWave * 4];
      }
    }
    const int at = r * 16 + (SWAP ? out_lane & 15 : 4 * (out_lane >> 4) + q);
    if (run.slot >= 0) {
      float *target = SWAP ? job.partials + (run.slot * columns + column) * a.rp + at
                           : job.partials + (static_cast<int64_t>(run.slot) * a.rp + at) * columns + column;
      const int64_t stride = SWAP ? a.rp : 1;
#pragma unroll
      for (int j = 0; j < CL; ++j) {
        if (j >= begin_j && j < limit) {
          target[j * stride] = total[j];
        }
      }
    } else if (at < a.max_rank) {
      const int64_t index = SWAP ? (run.group * columns + column) * a.max_rank + at
                                 : (static_cast<int64_t>(run.group) * a.max_rank + at) * columns + column;
      const int64_t stride = SWAP ? a.max_rank : 1;
#pragma unroll
      for (int j = 0; j < CL; ++j) {
        if (j >= begin_j && j < limit) {
          store_value(job.grad, index + j * stride, at < rank ? scale * total[j] : 0.0f, kDtypeOf<P>);
        }
      }
    }
    __syncthreads();
  }
  if (run.slot < 0) {
    // Ranks past the tiles above: no gradient.
    for (int at = NRT * 16 + wave; at < a.max_rank; at += kAdapterOuterWaves) {
      for (int64_t n = c0 + out_lane; n < c0 + 16 * CL && n < columns; n += kWave) {
        store_value(job.grad, SWAP ? (run.group * columns + n) * a.max_rank + at
                                   : (static_cast<int64_t>(run.group) * a.max_rank + at) * columns + n,
                    0.0f, kDtypeOf<P>);
      }
    }
  }
}

template <class P, int RT, int NRT, bool SWAP>
__device__ __forceinline__ void outer_ranks(const AdapterOuterArgs &a, const AdapterOuterJob &job, int64_t block,
                                            const AdapterRun &run, int rank, float scale, unsigned char *lds) {
  if constexpr (NRT > 1) {
    if (rank <= 8 * NRT) {
      return outer_ranks<P, RT, NRT / 2, SWAP>(a, job, block, run, rank, scale, lds);
    }
  }
  outer_body<P, RT, NRT, SWAP>(a, job, block, run, rank, scale, lds);
}

template <class P, int RT>
__global__ __launch_bounds__(kAdapterOuterWaves *kWave) void adapter_outer_kernel(AdapterOuterArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[kAdapterOuterWaves * kOuterColumns<P, RT> * 1024];
  constexpr int kColumns = 16 * kOuterColumns<P, RT>;
  // The blocks of job 0, then those of job 1.
  const int64_t blocks0 = (a.job[0].columns + kColumns - 1) / kColumns;
  const bool second = static_cast<int64_t>(blockIdx.x) >= blocks0;
  const int64_t block = blockIdx.x - (second ? blocks0 : 0);
  for (int64_t index = blockIdx.y; index < a.batch.max_runs; index += gridDim.y) {
    const u32x4 entry = *reinterpret_cast<const u32x4 *>(a.batch.runs + 8 * index);
    AdapterRun run;
    run.group = __builtin_amdgcn_readfirstlane(static_cast<int>(entry[0]));
    if (run.group < 0) {
      return;
    }
    run.first = __builtin_amdgcn_readfirstlane(static_cast<int>(entry[1]));
    run.end = __builtin_amdgcn_readfirstlane(static_cast<int>(entry[2]));
    run.slot = __builtin_amdgcn_readfirstlane(static_cast<int>(entry[3]));
    run.tile = __builtin_amdgcn_readfirstlane(a.batch.runs[8 * index + 4]);
    const int rank = adapter_rank(a.ranks, run.group, a.max_rank);
    const float scale = a.scales != nullptr ? a.scales[run.group] : 1.0f;
    if (second) {
      outer_ranks<P, RT, RT, true>(a, a.job[1], block, run, rank, scale, lds);
    } else {
      outer_ranks<P, RT, RT, false>(a, a.job[0], block, run, rank, scale, lds);
    }
  }
}

// The kernels of payload P, by the number of 16-rank tiles of the largest rank (1, 2, 4 or 8).
template <class P>
struct AdapterKernels {
  static const void *shrink(int rank_tiles);
  static const void *expand(int rank_tiles, AdapterAct activation, bool direct);
  static const void *outer(int rank_tiles);
};
extern template struct AdapterKernels<Bf16Payload>;
extern template struct AdapterKernels<F16Payload>;
extern template struct AdapterKernels<F32Payload>;

}  // namespace xp
