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
// are split the same way, exactly, because fp16 terms of t would overflow or lose the small ones.
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

struct AdapterTile {
  int group;  // the adapter; count: rows without one; count + 1: rows whose id is out of range; -1: no tile
  int rows;
  int rank;   // 0 without an adapter
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
  AdapterTile tile{-1, 0, 0, 0};
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
    tile.rank = __builtin_amdgcn_readfirstlane(static_cast<int>(entry[3]));
    tile.row = batch.perm[first + (lane < tile.rows ? lane : 0)];
  }
  return tile;
}

// The two bf16 terms of a pair of values: leading bits truncated, the rest to nearest even.  An
// infinite or NaN value has no rest.
__device__ __forceinline__ float leading_term(float value) {
  const uint32_t bits = __float_as_uint(value);
  return __uint_as_float((bits & 0xffff0000u) | (value != value ? 0x00400000u : 0u));
}
__device__ __forceinline__ float rest_term(float value, float leading) {
  return (__float_as_uint(value) & 0x7f800000u) == 0x7f800000u ? 0.0f : value - leading;
}
__device__ __forceinline__ void split_pair(float a, float b, uint32_t &high, uint32_t &low) {
  const float ha = leading_term(a);
  const float hb = leading_term(b);
  high = (__float_as_uint(ha) >> 16) | (__float_as_uint(hb) & 0xffff0000u);
  low = Bf16Payload::pack2(rest_term(a, ha), rest_term(b, hb));
}

// A chunk of P as bf16 terms: itself (bf16), or the exact pair (fp16).
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
// One tile of rows against all of its adapter's A rows over one K range.  The workgroup's four
// waves take the range's groups of U steps in turn (a step is 64 bytes of every row: full lines
// when U is even), rows straight from global memory as MFMA operands: a row is read by one wave
// only, so LDS would add a copy and no reuse; A comes from L2.  Partial sums of the waves meet in
// LDS, those of the ranges in `partials` [range][row][rp].
template <class P, int NRT, int TT, int U>
__device__ __forceinline__ void shrink_body(const AdapterShrinkArgs &a, const AdapterShrinkJob &job, int64_t range,
                                            const AdapterTile &tile, f32x4 (*sums)[4 * kWave]) {
  constexpr int ES = kElementBytes<P>;
  constexpr int STEP = kStep<P>;
  const int64_t k = made_here(job.k);
  const int lane = lane_here();
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int row16 = lane & 15;
  const int quarter = lane >> 4;
  // Rows past the tile read another, ranks past the adapter's the first: their sums go nowhere.
  const unsigned char *x[TT];
  const unsigned char *w = static_cast<const unsigned char *>(job.w) + static_cast<int64_t>(tile.group) * job.w_rows * k * ES;
  uint32_t w_offset[NRT];
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const int64_t row = __shfl(tile.row, t * 16 + row16, kWave);
    x[t] = static_cast<const unsigned char *>(job.x) + (row * job.ldx + quarter * kChunk<P>) * ES;
  }
#pragma unroll
  for (int r = 0; r < NRT; ++r) {
    const int at = r * 16 + row16;
    w_offset[r] = static_cast<uint32_t>(((at < tile.rank ? at : 0) * k + quarter * kChunk<P>) * ES);
  }
  f32x4 acc[NRT][TT];
#pragma unroll
  for (int r = 0; r < NRT; ++r) {
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      acc[r][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
  const int64_t steps = (k + STEP - 1) / STEP;
  const int64_t begin = range * job.steps_per_range;
  const int64_t end = begin + job.steps_per_range < steps ? begin + job.steps_per_range : steps;
  // Groups of U whole steps.  Sixteen waves a CU keep enough loads in flight; a second buffer per wave
  // would halve them.
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
#pragma unroll
      for (int r = 0; r < NRT; ++r) {
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          acc[r][t] = P::mfma16(ws[u][r], xs[u][t], acc[r][t]);
        }
      }
    }
  }
  // The steps past the last whole group, one per wave (at most U <= 4).  Chunks that the width
  // cuts are zero here: their columns are added one by one below.
  if (const int64_t step = begin + groups * U + wave; step < end) {
    const bool whole = (step * 4 + quarter + 1) * kChunk<P> <= k;
    const int64_t offset = step * (STEP * ES);
    u32x4 tail[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      tail[t] = u32x4{0u, 0u, 0u, 0u};
      if (whole) {
        tail[t] = load16_any(x[t] + offset);
      }
    }
#pragma unroll
    for (int r = 0; r < NRT; ++r) {
      u32x4 weights = {0u, 0u, 0u, 0u};
      if (whole) {
        weights = load16_any(w + offset + w_offset[r]);
      }
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        acc[r][t] = P::mfma16(weights, tail[t], acc[r][t]);
      }
    }
  }
  // This range's columns that are added one by one.
  const int64_t width = made_here(job.k);
  const int64_t cut = end == steps ? width - width % kChunk<P> : width;
  // Lane holds t[row lane % 16][4 (lane / 16) + j] of every 16 x 16 tile.
  const int out_lane = lane_here();
#pragma unroll
  for (int r = 0; r < NRT; ++r) {
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      sums[wave][t * kWave + out_lane] = acc[r][t];
    }
    __syncthreads();
    const int at = static_cast<int>(threadIdx.x >> 6) * 16 + (out_lane & 15);
    const int64_t row = __shfl(tile.row, at, kWave);
    if (threadIdx.x < TT * kWave) {
      f32x4 sum = sums[0][threadIdx.x];
#pragma unroll
      for (int v = 1; v < kAdapterShrinkWaves; ++v) {
        sum += sums[v][threadIdx.x];
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

template <class P, int RT, int TT>
__device__ __forceinline__ void shrink_ranks(const AdapterShrinkArgs &a, const AdapterShrinkJob &job, int64_t range,
                                             const AdapterTile &tile, f32x4 (*sums)[4 * kWave]) {
  if constexpr (RT > 1) {
    if (tile.rank <= 8 * RT) {
      return shrink_ranks<P, RT / 2, TT>(a, job, range, tile, sums);
    }
  }
  // U steps of TT row and RT weight operands, 16 bytes per lane each, beside the sums: within the 128
  // registers of two workgroups a CU up to two rank tiles, the 256 of one above.
  constexpr int U = RT + TT <= 2 ? 4 : RT <= 4 ? 2 : 1;
  shrink_body<P, RT, TT, U>(a, job, range, tile, sums);
}

template <class P, int RT>
__global__ __launch_bounds__(kAdapterShrinkWaves *kWave, RT <= 2 ? 4 : 2) void adapter_shrink_kernel(AdapterShrinkArgs a) {
  __shared__ f32x4 sums[kAdapterShrinkWaves][4 * kWave];
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
      if (tile.rows <= 16) {
        shrink_ranks<P, RT, 1>(a, job, range, tile, sums);
      } else {
        shrink_ranks<P, RT, 4>(a, job, range, tile, sums);
      }
    }
  }
}

// ------------------------------------------------------------------ expand
// One tile of rows against a range of its adapter's B rows (output columns): t is summed over its K
// ranges once per workgroup into LDS as MFMA operands ([leading terms | rests] of 16-bit payloads:
// one product over 2 r columns), then each wave takes 64 columns at a time (of half the rows where a
// tile has more than 32).  B rows are the MFMA's M operand in an order that leaves every lane 16
// bytes of consecutive output columns of one row: base is added, and the row written, in 64-byte
// runs straight from the accumulators.  The next columns' B rows are in flight while the last ones'
// results are converted and stored.
constexpr int kAdapterExpandWaves = 4;
constexpr int kAdapterExpandColumns = 64;  // per wave and turn

// The epilogue's activation: none, a gated SiLU, or any.
enum class AdapterAct : int { None = 0, GatedSilu = 1, Any = 2 };

template <class P, int RT>
constexpr int kAdapterTermStride = std::is_same_v<P, F32Payload> ? 4 * (RT * 16 + 4) : 2 * (2 * RT * 16 + 8);  // bytes

// `count` consecutive values to an element-aligned address.
template <class P, int N>
__device__ __forceinline__ void store_values(unsigned char *out, const float (&value)[N], int count) {
  if constexpr (kElementBytes<P> == 4) {
    if (count == N) {
      __builtin_memcpy(out, value, sizeof(value));
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (j < count) {
          reinterpret_cast<float *>(out)[j] = value[j];
        }
      }
    }
  } else {
    uint32_t packed[N / 2];
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      packed[j] = P::pack2(value[2 * j], value[2 * j + 1]);
    }
    if (count == N) {
      __builtin_memcpy(out, packed, sizeof(packed));
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (j < count) {
          reinterpret_cast<uint16_t *>(out)[j] = static_cast<uint16_t>(packed[j / 2] >> (16 * (j % 2)));
        }
      }
    }
  }
}

// silu(g) (u + offset).  16-bit results take the hardware's exp and reciprocal (relative error below
// 2^-16, under the store's 2^-9 or 2^-12), fp32 ones expf and an IEEE divide as elsewhere.
template <class P>
__device__ __forceinline__ float gated_silu_value(float gate, float up, const ActivationArgs &act) {
  if (act.has_limit) {
    gate = fminf(gate, act.limit);
    up = fminf(fmaxf(up, -act.limit), act.limit);
  }
  if constexpr (kElementBytes<P> == 4) {
    return gate / (1.0f + expf(-act.alpha * gate)) * (up + act.up_offset);
  } else {
    return gate * __builtin_amdgcn_rcpf(1.0f + __expf(-act.alpha * gate)) * (up + act.up_offset);
  }
}

template <class P, int RT, int TT, AdapterAct ACT>
struct AdapterExpand {
  static constexpr int ES = kElementBytes<P>;
  static constexpr int CH = kChunk<P>;
  static constexpr bool F32 = std::is_same_v<P, F32Payload>;
  static constexpr int CHUNKS = kAdapterExpandColumns / (4 * CH);  // 16-byte runs per lane and row
  static constexpr int PER = CH / 4;                               // MFMA tiles per run
  static constexpr int C = RT * 16 / CH;                           // B chunks of a row
  static constexpr int STEPS = F32 ? C / 4 : C / 2;                // MFMA steps: r columns, or 2 r
  static constexpr int FRAGS = F32 ? C / 4 : (C + 3) / 4;          // distinct B operands among them

  const AdapterExpandArgs &a;
  const unsigned char *w;
  int64_t whole;  // columns before it are stored here
  int rank;
  int row16;
  int quarter;
  int row[TT];    // past the tile: another, which is not stored
  bool live[TT];
  u32x4 ws[4][FRAGS];
  u32x4 base[TT][CHUNKS];

  __device__ __forceinline__ AdapterExpand(const AdapterExpandArgs &args, int64_t whole_columns, int group, int tile_rank,
                                           int first_row, int rows, int tile_row)
      : a(args),
        w(static_cast<const unsigned char *>(args.w) + static_cast<int64_t>(group) * args.n * args.ld_w * ES),
        whole(whole_columns),
        rank(tile_rank),
        row16(lane_here() & 15),
        quarter(lane_here() >> 4) {
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int at = first_row + t * 16 + row16;
      live[t] = at < rows;
      row[t] = __shfl(tile_row, at, kWave);
    }
  }

  // The lane's part of base and of B rows for the 64 columns from c0, with no branch per load: columns
  // past the whole ones read the last of those, chunks past the rank the row's first, neither of which
  // is used.
  __device__ __forceinline__ void load_base(int64_t c0) {
    if (a.base != nullptr) {
#pragma unroll
      for (int t = 0; t < TT; ++t) {
#pragma unroll
        for (int p = 0; p < CHUNKS; ++p) {
          const int64_t n = c0 + p * 4 * CH + quarter * CH;
          base[t][p] = load16_any(static_cast<const unsigned char *>(a.base) +
                                  (row[t] * a.ld_base + (n < whole ? n : whole - CH)) * ES);
        }
      }
    }
  }
  __device__ __forceinline__ void load_weights(int64_t c0) {
    if (rank > 0) {
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int64_t n = c0 + (m / PER) * 4 * CH + (row16 >> 2) * CH + (m % PER) * 4 + (row16 & 3);
        const uint32_t row_offset = static_cast<uint32_t>(n < whole ? n : whole - 1) * static_cast<uint32_t>(a.ld_w * ES);
#pragma unroll
        for (int f = 0; f < FRAGS; ++f) {
          const int chunk = (f * 4 + quarter) % C;
          ws[m][f] = load16_any(w + (row_offset + (chunk * CH < rank ? chunk * 16 : 0)));
        }
      }
    }
  }

  __device__ __forceinline__ void multiply(const unsigned char *terms, f32x4 (&acc)[4][TT]) {
    if (rank != RT * 16) {
      // Columns past the rank may hold anything.
#pragma unroll
      for (int f = 0; f < FRAGS; ++f) {
        const int within = rank - (f * 4 + quarter) % C * CH;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t mask = chunk_mask<P>(j, within);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            ws[m][f][j] &= mask;
          }
        }
      }
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      if (RT > 2 && (s * 4 % C) * CH >= rank) {
        continue;  // a pool of larger ranks: nothing there
      }
      u32x4 ts[TT];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        ts[t] = *reinterpret_cast<const u32x4 *>(terms + (t * 16 + row16) * kAdapterTermStride<P, RT> + (s * 4 + quarter) * 16);
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        if constexpr (F32) {
#pragma unroll
          for (int t = 0; t < TT; ++t) {
            acc[m][t] = F32Payload::mfma16(ws[m][s % FRAGS], ts[t], acc[m][t]);
          }
        } else {
          u32x4 high;
          u32x4 low;
          chunk_terms<P>(ws[m][s % FRAGS], high, low);
#pragma unroll
          for (int t = 0; t < TT; ++t) {
            acc[m][t] = Bf16Payload::mfma16(high, ts[t], acc[m][t]);
            if constexpr (std::is_same_v<P, F16Payload>) {
              acc[m][t] = Bf16Payload::mfma16(low, ts[t], acc[m][t]);
            }
          }
        }
      }
    }
  }

  // Lane holds columns 4 (lane / 16) + j of every B tile for row lane % 16.
  __device__ __forceinline__ void store(int64_t c0, float scale, bool poison, const f32x4 (&acc)[4][TT]) {
    const bool gated = ACT == AdapterAct::GatedSilu || (ACT == AdapterAct::Any && a.act.gated != 0);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
#pragma unroll
      for (int p = 0; p < CHUNKS; ++p) {
        const int64_t n = c0 + p * 4 * CH + quarter * CH;
        if (!live[t] || n >= whole) {
          continue;
        }
        float value[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          float from_base = 0.0f;
          if (a.base != nullptr) {
            const u32x4 &chunk = base[t][p];
            if constexpr (F32) {
              from_base = __uint_as_float(chunk[j]);
            } else {
              from_base = P::widen(j % 2 == 0 ? chunk[j / 2] & 0xffffu : chunk[j / 2] >> 16);
            }
          }
          // A row without an adapter keeps base's bits (-0 among them).
          value[j] = rank > 0 ? from_base + scale * acc[p * PER + j / 4][t][j % 4] : from_base;
          value[j] = poison ? __builtin_nanf("") : value[j];
        }
        unsigned char *out = static_cast<unsigned char *>(a.out);
        if (gated) {
          float activated[CH / 2];
#pragma unroll
          for (int j = 0; j < CH / 2; ++j) {
            if constexpr (ACT == AdapterAct::GatedSilu) {
              activated[j] = gated_silu_value<P>(value[2 * j], value[2 * j + 1], a.act);
            } else {
              activated[j] = apply_gated(value[2 * j], value[2 * j + 1], a.act);
            }
          }
          store_values<P>(out + (row[t] * a.ld_out + n / 2) * ES, activated, CH / 2);
        } else {
          if constexpr (ACT == AdapterAct::Any) {
#pragma unroll
            for (int j = 0; j < CH; ++j) {
              value[j] = apply_function(value[j], a.act);
            }
          }
          store_values<P>(out + (row[t] * a.ld_out + n) * ES, value, CH);
        }
      }
    }
  }
};

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
                                               const unsigned char *terms, float scale, bool poison, int64_t first) {
  const bool gated = ACT == AdapterAct::GatedSilu || (ACT == AdapterAct::Any && a.act.gated != 0);
  const int columns = static_cast<int>(a.n - first) / (gated ? 2 : 1);
  const int64_t weights = static_cast<int64_t>(tile.group) * a.n * a.ld_w;
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
      return poison ? __builtin_nanf("") : tile.rank > 0 ? from_base + scale * sum : from_base;
    };
    const int64_t n = index - at * columns;
    if (gated) {
      const float gate = column(first + 2 * n);
      const float up = column(first + 2 * n + 1);
      float value;
      if constexpr (ACT == AdapterAct::GatedSilu) {
        value = gated_silu_value<P>(gate, up, a.act);
      } else {
        value = apply_gated(gate, up, a.act);
      }
      store_value(a.out, row * a.ld_out + first / 2 + n, value, kDtypeOf<P>);
    } else {
      const float value = column(first + n);
      store_value(a.out, row * a.ld_out + first + n, ACT == AdapterAct::Any ? apply_function(value, a.act) : value,
                  kDtypeOf<P>);
    }
  }
}

template <class P, int RT, int TT, AdapterAct ACT>
__device__ __forceinline__ void expand_tile(const AdapterExpandArgs &a, const AdapterTile &tile, unsigned char *terms,
                                            int64_t begin, int64_t end) {
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  // Tiles of more than 16 TT rows: the waves' halves take a half each.
  const int halves = tile.rows > 16 * TT ? 2 : 1;
  const int half = halves > 1 ? wave & 1 : 0;
  const bool poison = tile.group > a.batch.count;
  const bool own = tile.group < a.batch.count;
  const float scale = own && a.scales != nullptr ? a.scales[tile.group] : 1.0f;
  const int64_t stride = kAdapterExpandWaves / halves * kAdapterExpandColumns;
  // Whole chunks of columns go 64 at a time, the rest one by one; so do the last B rows of a pool whose
  // rows are not whole chunks, since a row's last chunk passes its end, by less than a chunk.
  constexpr int CH = kChunk<P>;
  const int64_t within = a.n - (a.ld_w % CH != 0 ? (CH - 1 + a.ld_w - 1) / a.ld_w : 0);
  const int64_t whole = within < CH ? 0 : within - within % CH;
  const int64_t stop = end < whole ? end : whole;
  AdapterExpand<P, RT, TT, ACT> work(a, whole, tile.group, tile.rank, half * 16 * TT, tile.rows, tile.row);
  int64_t c0 = begin + wave / halves * kAdapterExpandColumns;
  if (c0 < stop) {
    work.load_base(c0);
    work.load_weights(c0);
  }
  if (tile.rank > 0) {
    stage_terms<P, RT>(a, tile, terms);
    __syncthreads();
  }
  const unsigned char *operands = terms + half * 16 * TT * kAdapterTermStride<P, RT>;
#pragma unroll 1
  while (c0 < stop) {
    f32x4 acc[4][TT];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        acc[m][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
    }
    if (tile.rank > 0) {
      work.multiply(operands, acc);
    }
    // The next B rows are in flight while this turn's results leave.
    const int64_t next = c0 + stride;
    if (next < stop) {
      work.load_weights(next);
    }
    work.store(c0, scale, poison, acc);
    if (next < stop) {
      work.load_base(next);
    }
    c0 = next;
  }
  if (end == a.n && whole < a.n) {
    expand_columns<P, RT, ACT>(a, tile, terms, scale, poison, whole);
  }
}

template <class P, int RT, AdapterAct ACT>
__global__ __launch_bounds__(kAdapterExpandWaves *kWave, RT <= 2 ? 4 : RT <= 4 ? 3 : 2) void adapter_expand_kernel(AdapterExpandArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned char terms[kAdapterTileRows * kAdapterTermStride<P, RT>];
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * a.columns;
  const int64_t end = begin + a.columns < a.n ? begin + a.columns : a.n;
  for (int64_t slot = blockIdx.y;; slot += gridDim.y) {
    const AdapterTile tile = adapter_tile(a.batch, a.ranks, a.max_rank, slot, true);
    if (tile.group < 0) {
      return;
    }
    const bool poison = tile.group > a.batch.count;
    if (poison && a.batch.tiles == nullptr && threadIdx.x == 0) {
      raise_fault(a.fault, kFaultAdapterOutOfRange);
    }
    if (tile.rank > 0 || poison || !a.in_place) {
      if (tile.rows <= 16) {
        expand_tile<P, RT, 1, ACT>(a, tile, terms, begin, end);
      } else {
        expand_tile<P, RT, 2, ACT>(a, tile, terms, begin, end);
      }
    }
    __syncthreads();  // the terms are rewritten
  }
}

// ------------------------------------------------------------------ outer products
// dA_a = s sum_i u[i] x[i]^T and dB_a = s sum_i dy[i] t[i]^T over one run of an adapter's rows and 64
// columns of x (dy): the rows are the MFMA's K.  A lane loads four columns of eight rows (fp32: of
// four), and pairs of rows' words give, by one byte permutation each, the operand of every fourth
// column; which 16 columns an MFMA holds is free, so no LDS transposition is needed.  The
// coefficients (u or t) come transposed and split into terms from adapter_terms_kernel.  Four waves
// take the run's rows in turn and meet in LDS; a run that is its adapter's only one stores the
// gradient, others their sums, which adapter_reduce_kernel adds in run order.
constexpr int kAdapterOuterWaves = 4;

template <class P, int NRT, bool SWAP>
__device__ __forceinline__ void outer_body(const AdapterOuterArgs &a, const AdapterOuterJob &job, int64_t c0, int first,
                                           int end, int rank, float scale, int64_t slot, int group,
                                           f32x4 (*sums)[4 * kWave]) {
  constexpr bool F32 = std::is_same_v<P, F32Payload>;
  constexpr bool F16 = std::is_same_v<P, F16Payload>;
  constexpr int ES = kElementBytes<P>;
  constexpr int ROWS = F32 ? 4 : 8;  // rows per lane and step
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int col16 = lane & 15;
  const int quarter = lane >> 4;
  f32x4 acc[NRT][4];
#pragma unroll
  for (int r = 0; r < NRT; ++r) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc[r][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
  const int64_t column = c0 + 4 * col16;
  const int64_t valid = job.columns - column;
  const unsigned char *data = static_cast<const unsigned char *>(job.data) + column * ES;
  const int64_t terms_plane = static_cast<int64_t>(a.rp) * a.stride;
  for (int p0 = first + wave * 4 * ROWS; p0 < end; p0 += kAdapterOuterWaves * 4 * ROWS) {
    const int p = p0 + quarter * ROWS;
    // words[e]: columns 0..3 of row e (16-bit payloads: two words).
    uint32_t words[ROWS][F32 ? 4 : 2];
#pragma unroll
    for (int e = 0; e < ROWS; ++e) {
#pragma unroll
      for (int j = 0; j < (F32 ? 4 : 2); ++j) {
        words[e][j] = 0u;
      }
      if (p + e < end && valid > 0) {
        const unsigned char *source = data + a.batch.perm[p + e] * job.ld * ES;
        if (valid >= 4) {
          __builtin_memcpy(words[e], source, sizeof(words[e]));
        } else {
#pragma unroll
          for (int j = 0; j < 3; ++j) {
            if (j < valid) {
              if constexpr (F32) {
                words[e][j] = reinterpret_cast<const uint32_t *>(source)[j];
              } else {
                words[e][j / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(source)[j]) << (16 * (j % 2));
              }
            }
          }
        }
      }
    }
    // Coefficients of the lane's rows for rank 16 r + lane % 16; rows past the run count zero.
    auto coefficients = [&](int r, int term) __attribute__((always_inline)) {
      u32x4 value = {0u, 0u, 0u, 0u};
      if (p < end) {
        const unsigned char *source =
            reinterpret_cast<const unsigned char *>(job.terms) +
            (term * terms_plane + static_cast<int64_t>(r * 16 + col16) * a.stride + p) * (F32 ? 4 : 2);
        value = load16_any(source);
        if (p + ROWS > end) {
#pragma unroll
          for (int e = 0; e < ROWS; ++e) {
            if (p + e >= end) {
              if constexpr (F32) {
                value[e] = 0u;
              } else {
                value[e / 2] &= e % 2 == 0 ? 0xffff0000u : 0x0000ffffu;
              }
            }
          }
        }
      }
      return value;
    };
    // operand[j]: column 4 (lane % 16) + j of the lane's rows.
    u32x4 operand[4];
    u32x4 rest[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if constexpr (F32) {
          operand[j][q] = words[q][j];
        } else {
          operand[j][q] = __builtin_amdgcn_perm(words[2 * q + 1][j / 2], words[2 * q][j / 2],
                                                j % 2 == 0 ? 0x05040100u : 0x07060302u);
        }
      }
      if constexpr (F16) {
        u32x4 high;
        chunk_terms<P>(operand[j], high, rest[j]);
        operand[j] = high;
      }
    }
#pragma unroll
    for (int r = 0; r < NRT; ++r) {
      const u32x4 high = coefficients(r, 0);
      if constexpr (F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[r][j] = SWAP ? F32Payload::mfma16(operand[j], high, acc[r][j])
                           : F32Payload::mfma16(high, operand[j], acc[r][j]);
        }
      } else {
        const u32x4 low = coefficients(r, 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          auto add = [&](u32x4 coefficient, u32x4 rows) __attribute__((always_inline)) {
            acc[r][j] = SWAP ? Bf16Payload::mfma16(rows, coefficient, acc[r][j])
                             : Bf16Payload::mfma16(coefficient, rows, acc[r][j]);
          };
          add(high, operand[j]);
          add(low, operand[j]);
          if constexpr (F16) {
            add(high, rest[j]);
            add(low, rest[j]);
          }
        }
      }
    }
  }
  // SWAP: lane holds rank lane % 16 and columns 16 (lane / 16) + 4 q + j; otherwise ranks
  // 4 (lane / 16) + q and columns 4 (lane % 16) + j.
  const int q = wave;
  unsigned char *grad = static_cast<unsigned char *>(job.grad);
#pragma unroll
  for (int r = 0; r < NRT; ++r) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sums[wave][j * kWave + lane] = acc[r][j];
    }
    __syncthreads();
    float total[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float *flat = reinterpret_cast<const float *>(&sums[0][j * kWave + lane]) + q;
      total[j] = flat[0];
#pragma unroll
      for (int v = 1; v < kAdapterOuterWaves; ++v) {
        total[j] += flat[v * 16 * kWave];
      }
    }
    const int at = r * 16 + (SWAP ? col16 : 4 * quarter + q);
    const int64_t n = c0 + (SWAP ? 16 * quarter + 4 * q : 4 * col16);
    const int count = job.columns - n < 4 ? static_cast<int>(job.columns - n) : 4;
    if (slot >= 0) {
      if (SWAP) {
        float *target = job.partials + (slot * job.columns + n) * a.rp + at;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j < count) {
            target[static_cast<int64_t>(j) * a.rp] = total[j];
          }
        }
      } else {
        float *target = job.partials + (slot * a.rp + at) * job.columns + n;
        if (count == 4) {
          __builtin_memcpy(target, total, sizeof(total));
        } else {
#pragma unroll
          for (int j = 0; j < 3; ++j) {
            if (j < count) {
              target[j] = total[j];
            }
          }
        }
      }
    } else if (at < a.max_rank) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        total[j] = at < rank ? scale * total[j] : 0.0f;
      }
      if (SWAP) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j < count) {
            const float one[2] = {total[j], 0.0f};
            store_values<P>(grad + ((group * job.columns + n + j) * a.max_rank + at) * ES, one, 1);
          }
        }
      } else if (count > 0) {
        store_values<P>(grad + ((static_cast<int64_t>(group) * a.max_rank + at) * job.columns + n) * ES, total, count);
      }
    }
    __syncthreads();
  }
  if (slot < 0) {
    // Ranks past the tiles above: no gradient.
    for (int at = NRT * 16 + wave; at < a.max_rank; at += kAdapterOuterWaves) {
      const int64_t n = c0 + lane;
      if (n < job.columns) {
        const float zero[2] = {0.0f, 0.0f};
        const int64_t index = SWAP ? (group * job.columns + n) * a.max_rank + at
                                   : (static_cast<int64_t>(group) * a.max_rank + at) * job.columns + n;
        store_values<P>(grad + index * ES, zero, 1);
      }
    }
  }
}

template <class P, int RT, bool SWAP>
__device__ __forceinline__ void outer_ranks(const AdapterOuterArgs &a, const AdapterOuterJob &job, int64_t c0, int first,
                                            int end, int rank, float scale, int64_t slot, int group,
                                            f32x4 (*sums)[4 * kWave]) {
  if constexpr (RT > 1) {
    if (rank <= 8 * RT) {
      return outer_ranks<P, RT / 2, SWAP>(a, job, c0, first, end, rank, scale, slot, group, sums);
    }
  }
  outer_body<P, RT, SWAP>(a, job, c0, first, end, rank, scale, slot, group, sums);
}

template <class P, int RT>
__global__ __launch_bounds__(kAdapterOuterWaves *kWave) void adapter_outer_kernel(AdapterOuterArgs a) {
  __shared__ f32x4 sums[kAdapterOuterWaves][4 * kWave];
  const bool second = static_cast<int64_t>(blockIdx.x) >= a.blocks0;
  const int64_t c0 = (blockIdx.x - (second ? a.blocks0 : 0)) * 64;
  for (int64_t run = blockIdx.y; run < a.batch.max_runs; run += gridDim.y) {
    const int group = __builtin_amdgcn_readfirstlane(a.batch.runs[4 * run]);
    if (group < 0) {
      return;
    }
    const int first = __builtin_amdgcn_readfirstlane(a.batch.runs[4 * run + 1]);
    const int end = __builtin_amdgcn_readfirstlane(a.batch.runs[4 * run + 2]);
    const int slot = __builtin_amdgcn_readfirstlane(a.batch.runs[4 * run + 3]);
    const int rank = adapter_rank(a.ranks, group, a.max_rank);
    const float scale = a.scales != nullptr ? a.scales[group] : 1.0f;
    if (second) {
      outer_ranks<P, RT, true>(a, a.job[1], c0, first, end, rank, scale, slot, group, sums);
    } else {
      outer_ranks<P, RT, false>(a, a.job[0], c0, first, end, rank, scale, slot, group, sums);
    }
  }
}

// The kernels of payload P, by the number of 16-rank tiles of the largest rank (1, 2, 4 or 8).
template <class P>
struct AdapterKernels {
  static const void *shrink(int rank_tiles);
  static const void *expand(int rank_tiles, AdapterAct activation);
  static const void *outer(int rank_tiles);
};
extern template struct AdapterKernels<Bf16Payload>;
extern template struct AdapterKernels<F16Payload>;
extern template struct AdapterKernels<F32Payload>;

}  // namespace xp
