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

constexpr int kAdapterShrinkWaves = 8;

// Elements of P in 16 bytes, and columns in one 16 x 16 MFMA step over four such chunks.
template <class P>
constexpr int kChunk = 16 / kElementBytes<P>;
template <class P>
constexpr int kStep = 4 * kChunk<P>;

struct AdapterTile {
  int group;  // adapter, kAdapterNone / kAdapterBad offsets past the count, or -1: no tile
  int rows;
};

__device__ __forceinline__ int adapter_group(int id, int count) {
  return id >= 0 && id < count ? id : id == -1 ? count : count + 1;
}

// Tile `slot` of the batch and its rows (list[0, rows), in LDS).  All threads of the workgroup call
// it; it ends with a barrier when there is a tile.  `all`: tiles of rows without an adapter too.
__device__ __forceinline__ AdapterTile adapter_tile(const AdapterBatch &batch, int64_t slot, bool all, int *list) {
  const int lane = threadIdx.x & 63;
  AdapterTile tile{-1, 0};
  if (batch.head == nullptr) {
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
    if (threadIdx.x < 64 && (mask >> lane & 1) != 0) {
      list[__popcll(mask & ((1ull << lane) - 1))] = lane;
    }
    tile.group = mine;
    tile.rows = __popcll(mask);
  } else {
    if (slot >= batch.head[all ? 1 : 0]) {
      return tile;
    }
    tile.group = __builtin_amdgcn_readfirstlane(batch.tiles[2 * slot]);
    const int first = __builtin_amdgcn_readfirstlane(batch.tiles[2 * slot + 1]);
    const int left = __builtin_amdgcn_readfirstlane(batch.starts[tile.group + 1]) - first;
    tile.rows = left < kAdapterTileRows ? left : kAdapterTileRows;
    if (static_cast<int>(threadIdx.x) < tile.rows) {
      list[threadIdx.x] = batch.perm[first + threadIdx.x];
    }
  }
  __syncthreads();
  return tile;
}

__device__ __forceinline__ int adapter_rank(const int32_t *ranks, int group, int max_rank) {
  if (ranks == nullptr) {
    return max_rank;
  }
  const int rank = __builtin_amdgcn_readfirstlane(ranks[group]);
  return rank < 0 ? 0 : rank > max_rank ? max_rank : rank;
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

// ------------------------------------------------------------------ shrink
// One tile of rows against all of its adapter's A rows over one K range.  The workgroup's eight
// waves take the range's groups of U steps in turn (a step is 64 bytes of every row: full lines
// when U is even), rows straight from global memory as MFMA operands: a row is read by one wave
// only, so LDS would add a copy and no reuse; A comes from L2.  Partial sums of the waves meet in
// LDS, those of the ranges in `partials` [range][row][rp].
template <class P, int NRT, int TT, int U>
__device__ __forceinline__ void shrink_body(const AdapterShrinkArgs &a, const AdapterShrinkJob &job, int64_t range,
                                            int group, int rank, int rows, const int *list,
                                            f32x4 (*sums)[4 * kWave]) {
  constexpr int ES = kElementBytes<P>;
  constexpr int STEP = kStep<P>;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int row16 = lane & 15;
  const int quarter = lane >> 4;
  // Rows past the tile or the rank read the first one: their sums go nowhere.
  const unsigned char *x[TT];
  const unsigned char *w[NRT];
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const int at = t * 16 + row16;
    x[t] = static_cast<const unsigned char *>(job.x) + (list[at < rows ? at : 0] * job.ldx + quarter * kChunk<P>) * ES;
  }
#pragma unroll
  for (int r = 0; r < NRT; ++r) {
    const int at = r * 16 + row16;
    w[r] = static_cast<const unsigned char *>(job.w) +
           ((static_cast<int64_t>(group) * job.w_rows + (at < rank ? at : 0)) * job.k + quarter * kChunk<P>) * ES;
  }
  f32x4 acc[NRT][TT];
#pragma unroll
  for (int r = 0; r < NRT; ++r) {
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      acc[r][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
  const int64_t steps = (job.k + STEP - 1) / STEP;
  const int64_t begin = range * job.steps_per_range;
  const int64_t end = begin + job.steps_per_range < steps ? begin + job.steps_per_range : steps;
#pragma unroll 1
  for (int64_t step = begin + wave * U; step < end; step += kAdapterShrinkWaves * U) {
    if (step + U <= end && (step + U) * STEP <= job.k) {
      u32x4 xs[U][TT];
      u32x4 ws[U][NRT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          xs[u][t] = load16_any(x[t] + (step + u) * (STEP * ES));
        }
#pragma unroll
        for (int r = 0; r < NRT; ++r) {
          ws[u][r] = load16_any(w[r] + (step + u) * (STEP * ES));
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
    } else {
      const int64_t last = step + U < end ? step + U : end;
#pragma unroll 1
      for (int64_t s = step; s < last; ++s) {
        const int64_t valid = job.k - s * STEP - quarter * kChunk<P>;
        auto load = [&](const unsigned char *source) __attribute__((always_inline)) {
          return valid >= kChunk<P> ? load16_any(source + s * (STEP * ES))
                                    : load_chunk_tail<P, P>(source + s * (STEP * ES), valid);
        };
        u32x4 xs[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          xs[t] = load(x[t]);
        }
#pragma unroll
        for (int r = 0; r < NRT; ++r) {
          const u32x4 ws = load(w[r]);
#pragma unroll
          for (int t = 0; t < TT; ++t) {
            acc[r][t] = P::mfma16(ws, xs[t], acc[r][t]);
          }
        }
      }
    }
  }
  // Lane holds t[row lane % 16][4 (lane / 16) + j] of every 16 x 16 tile.
#pragma unroll
  for (int r = 0; r < NRT; ++r) {
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      sums[wave][t * kWave + lane] = acc[r][t];
    }
    __syncthreads();
    if (threadIdx.x < TT * kWave) {
      f32x4 sum = sums[0][threadIdx.x];
#pragma unroll
      for (int v = 1; v < kAdapterShrinkWaves; ++v) {
        sum += sums[v][threadIdx.x];
      }
      const int at = static_cast<int>(threadIdx.x >> 6) * 16 + row16;
      const int first = r * 16 + 4 * quarter;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sum[j] = first + j < rank ? sum[j] : 0.0f;
      }
      if (at < rows) {
        *reinterpret_cast<f32x4 *>(job.partials + (range * a.batch.rows + list[at]) * a.rp + first) = sum;
      }
    }
    __syncthreads();
  }
}

template <class P, int RT, int TT, int U>
__device__ __forceinline__ void shrink_ranks(const AdapterShrinkArgs &a, const AdapterShrinkJob &job, int64_t range,
                                             int group, int rank, int rows, const int *list,
                                             f32x4 (*sums)[4 * kWave]) {
  if constexpr (RT > 1) {
    if (rank <= 8 * RT) {
      return shrink_ranks<P, RT / 2, TT, (U < 4 ? 2 * U : U)>(a, job, range, group, rank, rows, list, sums);
    }
  }
  shrink_body<P, RT, TT, U>(a, job, range, group, rank, rows, list, sums);
}

template <class P, int RT>
__global__ __launch_bounds__(kAdapterShrinkWaves *kWave) void adapter_shrink_kernel(AdapterShrinkArgs a) {
  __shared__ int list[kAdapterTileRows];
  __shared__ f32x4 sums[kAdapterShrinkWaves][4 * kWave];
  const bool second = static_cast<int64_t>(blockIdx.x) >= a.job[0].ranges;
  const AdapterShrinkJob &job = a.job[second ? 1 : 0];
  const int64_t range = blockIdx.x - (second ? a.job[0].ranges : 0);
  for (int64_t slot = blockIdx.y;; slot += gridDim.y) {
    const AdapterTile tile = adapter_tile(a.batch, slot, false, list);
    if (tile.group < 0) {
      return;
    }
    const int rank = adapter_rank(a.ranks, tile.group, a.max_rank);
    if (rank > 0) {
      if (tile.rows <= 16) {
        shrink_ranks<P, RT, 1, (RT >= 4 ? 2 : 4)>(a, job, range, tile.group, rank, tile.rows, list, sums);
      } else {
        shrink_ranks<P, RT, 4, (RT >= 8 ? 1 : RT >= 4 ? 2 : 4)>(a, job, range, tile.group, rank, tile.rows, list, sums);
      }
    }
    __syncthreads();  // the list is rewritten
  }
}

// ------------------------------------------------------------------ expand
// One tile of rows against a range of its adapter's B rows (output columns): t is summed over its K
// ranges once per workgroup into LDS as MFMA operands ([leading terms | rests] of 16-bit payloads:
// one product over 2 r columns), then each wave takes 64 columns at a time.  B rows are the MFMA's M
// operand in an order that leaves every lane 16 bytes of consecutive output columns of one row:
// base is added, and the row written, in 64-byte runs straight from the accumulators.
constexpr int kAdapterExpandWaves = 4;
constexpr int kAdapterExpandColumns = 64;  // per wave and turn

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

// acc += (64 B rows from column c0) x (t of the tile's rows), for up to 16 NRT ranks.
template <class P, int NRT, int TT>
__device__ __forceinline__ void expand_products(const unsigned char *w, int64_t c0, int64_t n_end, int ld_w, int rank,
                                                const unsigned char *terms, int term_stride, f32x4 (&acc)[4][TT]) {
  constexpr int ES = kElementBytes<P>;
  constexpr int CH = kChunk<P>;
  constexpr bool F32 = std::is_same_v<P, F32Payload>;
  constexpr int PER = CH / 4;                       // MFMA tiles per 16-byte run
  constexpr int C = NRT * 16 / CH;                  // B chunks of a row
  constexpr int STEPS = F32 ? C / 4 : C / 2;        // MFMA steps: r columns, or 2 r
  constexpr int FRAGS = F32 ? C / 4 : (C + 3) / 4;  // distinct B operands among them
  const int lane = threadIdx.x & 63;
  const int row16 = lane & 15;
  const int quarter = lane >> 4;
  const bool whole = ld_w % CH == 0;
  u32x4 ws[4][FRAGS];
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    int64_t n = c0 + (m / PER) * 4 * CH + (row16 >> 2) * CH + (m % PER) * 4 + (row16 & 3);
    n = n < n_end ? n : n_end - 1;
    const unsigned char *source = w + n * ld_w * ES;
#pragma unroll
    for (int f = 0; f < FRAGS; ++f) {
      const int chunk = (f * 4 + quarter) % C;
      const int within = rank - chunk * CH;  // its columns that are within the rank
      u32x4 value = {0u, 0u, 0u, 0u};
      if (within >= CH || (whole && within > 0)) {
        value = load16_any(source + chunk * 16);
      } else if (within > 0) {
        value = load_chunk_tail<P, P>(source + chunk * 16, within);
      }
      ws[m][f] = value;
    }
  }
  if (whole && rank % CH != 0) {
    // Columns past the rank may hold anything.
#pragma unroll
    for (int m = 0; m < 4; ++m) {
#pragma unroll
      for (int f = 0; f < FRAGS; ++f) {
        const int within = rank - (f * 4 + quarter) % C * CH;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          if (j >= within) {
            if constexpr (F32) {
              ws[m][f][j] = 0u;
            } else {
              ws[m][f][j / 2] &= j % 2 == 0 ? 0xffff0000u : 0x0000ffffu;
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    u32x4 ts[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      ts[t] = *reinterpret_cast<const u32x4 *>(terms + (t * 16 + row16) * term_stride + (s * 4 + quarter) * 16);
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

// The products at the fewest rank tiles (1, 2, 4 or 8) that hold `rank`.
template <class P, int RT, int TT>
__device__ __forceinline__ void expand_rank_products(const unsigned char *w, int64_t c0, int64_t n_end, int ld_w,
                                                     int rank, const unsigned char *terms, int term_stride,
                                                     f32x4 (&acc)[4][TT]) {
  if constexpr (RT > 1) {
    if (rank <= 8 * RT) {
      return expand_rank_products<P, RT / 2, TT>(w, c0, n_end, ld_w, rank, terms, term_stride, acc);
    }
  }
  expand_products<P, RT, TT>(w, c0, n_end, ld_w, rank, terms, term_stride, acc);
}

template <class P, int RT, int TT, bool ACT>
__device__ __forceinline__ void expand_body(const AdapterExpandArgs &a, int group, int rank, float scale, bool poison,
                                            int rows, const int *list, const unsigned char *terms, int term_stride,
                                            int64_t column_begin, int64_t column_end) {
  constexpr int ES = kElementBytes<P>;
  constexpr int CH = kChunk<P>;
  constexpr bool F32 = std::is_same_v<P, F32Payload>;
  constexpr int CHUNKS = kAdapterExpandColumns / (4 * CH);  // 16-byte runs per lane and row
  constexpr int PER = CH / 4;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int row16 = lane & 15;
  const int quarter = lane >> 4;
  int row[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const int at = t * 16 + row16;
    row[t] = at < rows ? list[at] : -1;
  }
  const unsigned char *w = static_cast<const unsigned char *>(a.w) + static_cast<int64_t>(group) * a.n * a.ld_w * ES;
  const bool gated = ACT && a.act.gated != 0;
  for (int64_t c0 = column_begin + wave * kAdapterExpandColumns; c0 < column_end;
       c0 += kAdapterExpandWaves * kAdapterExpandColumns) {
    u32x4 base[TT][CHUNKS];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
#pragma unroll
      for (int p = 0; p < CHUNKS; ++p) {
        const int64_t n = c0 + p * 4 * CH + quarter * CH;
        base[t][p] = u32x4{0u, 0u, 0u, 0u};
        if (a.base != nullptr && row[t] >= 0 && n < a.n) {
          const unsigned char *source = static_cast<const unsigned char *>(a.base) + (row[t] * a.ld_base + n) * ES;
          base[t][p] = n + CH <= a.n ? load16_any(source) : load_chunk_tail<P, P>(source, a.n - n);
        }
      }
    }
    f32x4 acc[4][TT];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        acc[m][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
    }
    if (rank > 0) {
      expand_rank_products<P, RT, TT>(w, c0, a.n, a.ld_w, rank, terms, term_stride, acc);
    }
    // Lane holds columns 4 (lane / 16) + j of every B tile for row lane % 16.
#pragma unroll
    for (int t = 0; t < TT; ++t) {
#pragma unroll
      for (int p = 0; p < CHUNKS; ++p) {
        const int64_t n = c0 + p * 4 * CH + quarter * CH;
        if (row[t] < 0 || n >= a.n) {
          continue;
        }
        const int count = a.n - n < CH ? static_cast<int>(a.n - n) : CH;
        float value[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          float from_base;
          if constexpr (F32) {
            from_base = __uint_as_float(base[t][p][j]);
          } else {
            from_base = P::widen(j % 2 == 0 ? base[t][p][j / 2] & 0xffffu : base[t][p][j / 2] >> 16);
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
            activated[j] = apply_gated(value[2 * j], value[2 * j + 1], a.act);
          }
          store_values<P>(out + (row[t] * a.ld_out + n / 2) * ES, activated, count / 2);
        } else {
          if constexpr (ACT) {
#pragma unroll
            for (int j = 0; j < CH; ++j) {
              value[j] = apply_function(value[j], a.act);
            }
          }
          store_values<P>(out + (row[t] * a.ld_out + n) * ES, value, count);
        }
      }
    }
  }
}

// t of the tile's rows: the K ranges' sums, in range order, as the operands that expand_body reads
// (columns up to 16 tiles_r; past the rank they are zero).
template <class P>
__device__ __forceinline__ void stage_terms(const AdapterExpandArgs &a, int columns, int rows, const int *list,
                                            unsigned char *terms, int term_stride) {
  constexpr int kBatch = 8;
  const int quads = columns / 4;
  const int64_t plane = a.batch.rows * a.rp;
  for (int index = threadIdx.x; index < rows * quads; index += kAdapterExpandWaves * kWave) {
    const int at = index / quads;
    const int quad = index - at * quads;
    const float *source = a.partials + static_cast<int64_t>(list[at]) * a.rp + 4 * quad;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t first = 0; first < a.ranges; first += kBatch) {
      f32x4 part[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        if (first + j < a.ranges) {
          part[j] = *reinterpret_cast<const f32x4 *>(source + (first + j) * plane);
        }
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        if (first + j < a.ranges) {
          sum += part[j];
        }
      }
    }
    unsigned char *target = terms + at * term_stride;
    if constexpr (std::is_same_v<P, F32Payload>) {
      *reinterpret_cast<f32x4 *>(target + 16 * quad) = sum;
    } else {
      u32x2 high;
      u32x2 low;
      uint32_t h;
      uint32_t l;
      split_pair(sum[0], sum[1], h, l);
      high[0] = h;
      low[0] = l;
      split_pair(sum[2], sum[3], h, l);
      high[1] = h;
      low[1] = l;
      *reinterpret_cast<u32x2 *>(target + 8 * quad) = high;
      *reinterpret_cast<u32x2 *>(target + 2 * columns + 8 * quad) = low;
    }
  }
  __syncthreads();
}

template <class P, int RT, bool ACT>
__global__ __launch_bounds__(kAdapterExpandWaves *kWave) void adapter_expand_kernel(AdapterExpandArgs a) {
  constexpr int kStride = kAdapterTermStride<P, RT>;
  __shared__ int list[kAdapterTileRows];
  __shared__ __attribute__((aligned(16))) unsigned char terms[kAdapterTileRows * kStride];
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * a.columns;
  const int64_t end = begin + a.columns < a.n ? begin + a.columns : a.n;
  for (int64_t slot = blockIdx.y;; slot += gridDim.y) {
    const AdapterTile tile = adapter_tile(a.batch, slot, true, list);
    if (tile.group < 0) {
      return;
    }
    const bool own = tile.group < a.batch.count;
    const bool poison = tile.group > a.batch.count;
    const int rank = own ? adapter_rank(a.ranks, tile.group, a.max_rank) : 0;
    const float scale = own && a.scales != nullptr ? a.scales[tile.group] : 1.0f;
    if (poison && a.batch.head == nullptr && threadIdx.x == 0) {
      raise_fault(a.fault, kFaultAdapterOutOfRange);
    }
    if (rank > 0) {
      int columns = 16;
      while (columns < rank) {
        columns *= 2;
      }
      stage_terms<P>(a, columns, tile.rows, list, terms, kStride);
    }
    if (rank > 0 || poison || !a.in_place) {
      if (tile.rows <= 16) {
        expand_body<P, RT, 1, ACT>(a, tile.group, rank, scale, poison, tile.rows, list, terms, kStride, begin, end);
      } else {
        expand_body<P, RT, 4, ACT>(a, tile.group, rank, scale, poison, tile.rows, list, terms, kStride, begin, end);
      }
    }
    __syncthreads();  // the list and the terms are rewritten
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
  const int total = a.batch.head[2];
  for (int64_t run = blockIdx.y; run < total; run += gridDim.y) {
    const int group = __builtin_amdgcn_readfirstlane(a.batch.outer[4 * run]);
    const int first = __builtin_amdgcn_readfirstlane(a.batch.outer[4 * run + 1]);
    const int end = __builtin_amdgcn_readfirstlane(a.batch.outer[4 * run + 2]);
    const int slot = __builtin_amdgcn_readfirstlane(a.batch.outer[4 * run + 3]);
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
  static const void *expand(int rank_tiles, bool activation);
  static const void *outer(int rank_tiles);
};
extern template struct AdapterKernels<Bf16Payload>;
extern template struct AdapterKernels<F16Payload>;
extern template struct AdapterKernels<F32Payload>;

}  // namespace xp
