// Per-expert counts of a Router's routes, its balance loss and the gradient of its logits on gfx950.
//
//   counts_e = routes of the live rows to expert e,  f_e = counts_e E / (topk T)
//   p_t = softmax(l_t), or sigmoid(l_t) / sum sigmoid(l_t)  (the Router's two score functions)
//   loss = c sum_e f_e (1 / T) sum_t p_te
//   d loss / d l_te = (c / T) p_te (f_e - sum_j f_j p_tj) s_te,  s = 1 (softmax), 1 - sigmoid(l_te)
// over the T live rows; counts are constants of the gradient.  A row whose logits are all -inf has p = 0.
//
// Bound by memory: the loss reads the logits and ids once, the gradient reads the logits and writes
// as much (65536 rows of 128 fp32 logits, eight routes each: the loss 12.5 us, 2.8 TB/s, and 5.5 us for
// the workgroups' sums, the gradient 17 to 18 us, 3.8 TB/s; both launches end in a few microseconds of
// latency that does not shrink with the rows).  A row is held by a 16-, 32- or 64-lane part of a wave, four
// consecutive experts per lane and load, so that a wave takes several narrow rows at once; sums over a row go
// through DPP within 16 lanes.  The loss keeps sum_t p_te of the lane's own experts in registers over all of its
// rows and adds waves, then workgroups, in a fixed order: no floating-point atomics, equal bits
// every time.  Counts are integers, added by LDS atomics.

#include "xp_elements.hpp"
#include "xp_kernels.hpp"

#include <algorithm>

namespace xp {
namespace {

template <int CTRL>
__device__ __forceinline__ float dpp(float value) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(value), CTRL, 0xf, 0xf, true));
}

// Reduction over aligned groups of L lanes; every lane gets the result.
template <int L, class Op>
__device__ __forceinline__ float group_reduce(float value, Op op) {
  value = op(value, dpp<0xB1>(value));   // lane ^ 1
  value = op(value, dpp<0x4E>(value));   // lane ^ 2
  value = op(value, dpp<0x141>(value));  // the other four of eight
  value = op(value, dpp<0x140>(value));  // the other eight of sixteen
  if constexpr (L > 16) {
    value = op(value, __shfl_xor(value, 16, kWave));
  }
  if constexpr (L > 32) {
    value = op(value, __shfl_xor(value, 32, kWave));
  }
  return value;
}
template <int L>
__device__ __forceinline__ float group_max(float value) {
  return group_reduce<L>(value, [](float a, float b) { return fmaxf(a, b); });
}
template <int L>
__device__ __forceinline__ float group_sum(float value) {
  return group_reduce<L>(value, [](float a, float b) { return a + b; });
}

constexpr float kLowest = -__builtin_inff();

// Experts 4 (c L + lane) + j, c < CN, of one row of logits; past the last expert -inf.
template <class T, int L, int CN>
__device__ __forceinline__ void load_logits(const void *logits, int64_t row, int experts, int lane, float (&value)[CN][4]) {
#pragma unroll
  for (int c = 0; c < CN; ++c) {
    const int first = 4 * (c * L + lane);
    const unsigned char *source =
        static_cast<const unsigned char *>(logits) + (row * experts + first) * kElementBytes<T>;
    if (first + 4 <= experts) {
      if constexpr (kElementBytes<T> == 4) {
        const u32x4 words = load16_any(source);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          value[c][j] = __uint_as_float(words[j]);
        }
      } else {
        const u32x2 words = load8_any(source);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          value[c][j] = T::widen(j % 2 == 0 ? words[j / 2] & 0xffffu : words[j / 2] >> 16);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        value[c][j] = first + j < experts ? load_value(source, j, kDtypeOf<T>) : kLowest;
      }
    }
  }
}

// Scores of a row in place of its logits, up to a factor that the row shares and not yet divided by their
// sum, and the sum's inverse (0 for a row whose scores are all zero).  `slope` gets s of the gradient; 1 - sigmoid(l) is sigmoid(-l), which the
// difference from a rounded sigmoid loses from l = 10 on (all of it from 17.4).
template <int L, int CN>
__device__ __forceinline__ float scores(float (&value)[CN][4], bool softmax, float (&slope)[CN][4]) {
  auto largest = [&]() __attribute__((always_inline)) {
    float most = kLowest;
#pragma unroll
    for (int c = 0; c < CN; ++c) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        most = fmaxf(most, value[c][j]);
      }
    }
    most = group_max<L>(most);
    return most == kLowest ? 0.0f : most;
  };
  float sum = 0.0f;
  if (softmax) {
    const float most = largest();
#pragma unroll
    for (int c = 0; c < CN; ++c) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        value[c][j] = expf(value[c][j] - most);
        slope[c][j] = 1.0f;
        sum += value[c][j];
      }
    }
    sum = group_sum<L>(sum);
  } else {
    float score[CN][4];
#pragma unroll
    for (int c = 0; c < CN; ++c) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float small = expf(-fabsf(value[c][j]));
        const float whole = 1.0f / (1.0f + small);
        const float part = small * whole;
        slope[c][j] = value[c][j] > 0.0f ? part : whole;
        score[c][j] = value[c][j] > 0.0f ? whole : part;
        sum += score[c][j];
      }
    }
    sum = group_sum<L>(sum);
    if (sum < 0x1p-40f) {
      // Every logit is far below zero: divided by exp of the largest, scores keep the ratios that sigmoids lose
      // towards the end of the exponents' range.  A row's lanes take the branch together.  (The largest logit of
      // every row in place of this sum took 149 us instead of 114 for 32768 rows of 1000 fp32 logits, both passes.)
      const float most = largest();
      sum = 0.0f;
#pragma unroll
      for (int c = 0; c < CN; ++c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          score[c][j] = expf(value[c][j] - most) * slope[c][j];
          sum += score[c][j];
        }
      }
      sum = group_sum<L>(sum);
    }
#pragma unroll
    for (int c = 0; c < CN; ++c) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        value[c][j] = score[c][j];
      }
    }
  }
  return sum == 0.0f ? 0.0f : 1.0f / sum;
}

__device__ __forceinline__ int64_t live_rows(const int32_t *payload_rows, int64_t rows) {
  if (payload_rows == nullptr) {
    return rows;
  }
  const int64_t live = *payload_rows;
  return live < 0 ? 0 : live < rows ? live : rows;
}

constexpr int kBalanceThreads = 1024;
constexpr int kBalanceWaves = kBalanceThreads / kWave;

// counts and loss from the workgroups' sums: one thread per expert adds them in workgroup order.
__device__ __forceinline__ void finish_balance(const BalanceArgs &a, int64_t live, int count, float share, double *sums) {
  const int tid = threadIdx.x;
  double term = 0.0;
  if (tid < a.experts) {
    a.counts[tid] = count;
    term = static_cast<double>(count) * static_cast<double>(share);
  }
  if (a.loss == nullptr) {
    return;
  }
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) {
    term += __shfl_xor(term, offset, kWave);
  }
  if ((tid & 63) == 0) {
    sums[tid >> 6] = term;
  }
  __syncthreads();
  if (tid == 0) {
    double total = 0.0;
    for (int w = 0; w < kBalanceWaves; ++w) {
      total += sums[w];
    }
    const double rows = static_cast<double>(live);
    *a.loss = live == 0 ? 0.0f
                        : static_cast<float>(static_cast<double>(a.coefficient) * total * a.experts /
                                             (static_cast<double>(a.topk) * rows * rows));
  }
}

template <class T, int L, int CN, int U>
__global__ __launch_bounds__(kBalanceThreads) void moe_balance_kernel(BalanceArgs a) {
  __shared__ int histogram[kMoeMaxExperts];
  __shared__ float shares[kBalanceWaves][kMoeMaxExperts];
  __shared__ double sums[kBalanceWaves];
  const int tid = threadIdx.x;
  const int lane = tid & (L - 1);
  const int experts = a.experts;
  const int64_t live = live_rows(a.payload_rows, a.rows);
  for (int e = tid; e < experts; e += kBalanceThreads) {
    histogram[e] = 0;
  }
  __syncthreads();
  const int64_t routes = live * a.topk;
  for (int64_t route = static_cast<int64_t>(blockIdx.x) * kBalanceThreads + tid; route < routes;
       route += static_cast<int64_t>(gridDim.x) * kBalanceThreads) {
    const int id = a.ids[route];
    if (id >= 0 && id < experts) {
      atomicAdd(&histogram[id], 1);
    }
  }
  float share[CN][4];
#pragma unroll
  for (int c = 0; c < CN; ++c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      share[c][j] = 0.0f;
    }
  }
  if (a.logits != nullptr) {
    constexpr int kParts = kBalanceThreads / L;  // rows per workgroup at a time
    const int64_t stride = static_cast<int64_t>(gridDim.x) * kParts;
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * kParts + tid / L; row0 < live; row0 += U * stride) {
      float value[U][CN][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = row0 + u * stride;
        load_logits<T, L, CN>(a.logits, row < live ? row : row0, experts, lane, value[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (row0 + u * stride < live) {
          float unused[CN][4];
          const float inverse = scores<L, CN>(value[u], a.softmax != 0, unused);
#pragma unroll
          for (int c = 0; c < CN; ++c) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              share[c][j] += inverse == 0.0f ? 0.0f : value[u][c][j] * inverse;
            }
          }
        }
      }
    }
#pragma unroll
    for (int c = 0; c < CN; ++c) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (L <= 16) {
          share[c][j] += __shfl_xor(share[c][j], 16, kWave);
        }
        if constexpr (L <= 32) {
          share[c][j] += __shfl_xor(share[c][j], 32, kWave);
        }
        if ((tid & 63) < L) {
          const int expert = 4 * (c * L + lane) + j;
          if (expert < experts) {
            shares[tid >> 6][expert] = share[c][j];
          }
        }
      }
    }
  }
  __syncthreads();
  int count = 0;
  float total = 0.0f;
  if (tid < experts) {
    count = histogram[tid];
    if (a.logits != nullptr) {
      for (int w = 0; w < kBalanceWaves; ++w) {
        total += shares[w][tid];
      }
    }
  }
  if (gridDim.x == 1) {
    finish_balance(a, live, count, total, sums);
  } else if (tid < experts) {
    a.partial_counts[static_cast<int64_t>(blockIdx.x) * experts + tid] = count;
    a.partial_shares[static_cast<int64_t>(blockIdx.x) * experts + tid] = total;
  }
}

__global__ __launch_bounds__(kBalanceThreads) void moe_balance_finish_kernel(BalanceArgs a) {
  __shared__ double sums[kBalanceWaves];
  __shared__ int counts[kBalanceThreads];
  __shared__ float shares[kBalanceThreads];
  // Few experts: several threads per expert, each over a run of the workgroups' sums.
  const int experts = a.experts;
  int parts = 1;
  while (2 * parts * experts <= kBalanceThreads && 2 * parts <= a.blocks) {
    parts *= 2;
  }
  const int expert = static_cast<int>(threadIdx.x) % experts;
  const int part = static_cast<int>(threadIdx.x) / experts;
  int count = 0;
  float share = 0.0f;
  if (part < parts) {
    const int64_t run = (a.blocks + parts - 1) / parts;
    const int64_t end = (part + 1) * run < a.blocks ? (part + 1) * run : a.blocks;
#pragma unroll 8
    for (int64_t block = part * run; block < end; ++block) {
      count += a.partial_counts[block * experts + expert];
      share += a.partial_shares[block * experts + expert];
    }
  }
  counts[threadIdx.x] = count;
  shares[threadIdx.x] = share;
  __syncthreads();
  count = 0;
  share = 0.0f;
  if (static_cast<int>(threadIdx.x) < experts) {
    for (int p = 0; p < parts; ++p) {
      count += counts[p * experts + threadIdx.x];
      share += shares[p * experts + threadIdx.x];
    }
  }
  finish_balance(a, live_rows(a.payload_rows, a.rows), count, share, sums);
}

template <class T, int L, int CN, int U>
__global__ __launch_bounds__(256) void moe_balance_backward_kernel(BalanceArgs a) {
  const int lane = threadIdx.x & (L - 1);
  const int experts = a.experts;
  const int64_t live = live_rows(a.payload_rows, a.rows);
  float load[CN][4];
  const float whole = live > 0 ? static_cast<float>(experts) / (static_cast<float>(a.topk) * static_cast<float>(live)) : 0.0f;
#pragma unroll
  for (int c = 0; c < CN; ++c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int expert = 4 * (c * L + lane) + j;
      load[c][j] = expert < experts ? static_cast<float>(a.counts[expert]) * whole : 0.0f;
    }
  }
  const float upstream = a.grad_loss != nullptr ? *a.grad_loss : 1.0f;
  const float factor = live > 0 ? a.coefficient * upstream / static_cast<float>(live) : 0.0f;
  constexpr int kParts = 256 / L;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kParts;
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * kParts + threadIdx.x / L; row0 < a.rows; row0 += U * stride) {
    float value[U][CN][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = row0 + u * stride;
      if (row < live) {
        load_logits<T, L, CN>(a.logits, row, experts, lane, value[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = row0 + u * stride;
      if (row >= a.rows) {
        continue;
      }
      if (row < live) {
        float slope[CN][4];
        const float inverse = scores<L, CN>(value[u], a.softmax != 0, slope);
        float mean = 0.0f;
#pragma unroll
        for (int c = 0; c < CN; ++c) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mean += load[c][j] * value[u][c][j];
          }
        }
        mean = group_sum<L>(mean) * inverse;
#pragma unroll
        for (int c = 0; c < CN; ++c) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float grad = factor * (value[u][c][j] * inverse) * slope[c][j] * (load[c][j] - mean);
            value[u][c][j] = inverse == 0.0f ? 0.0f : grad;
          }
        }
      } else {
        // Rows past the live ones take no part in the loss.
#pragma unroll
        for (int c = 0; c < CN; ++c) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            value[u][c][j] = 0.0f;
          }
        }
      }
#pragma unroll
      for (int c = 0; c < CN; ++c) {
        const int first = 4 * (c * L + lane);
        unsigned char *target =
            static_cast<unsigned char *>(a.grad_logits) + (row * experts + first) * kElementBytes<T>;
        if (first + 4 <= experts) {
          if constexpr (kElementBytes<T> == 4) {
            __builtin_memcpy(target, value[u][c], 16);
          } else {
            const u32x2 packed = {T::pack2(value[u][c][0], value[u][c][1]), T::pack2(value[u][c][2], value[u][c][3])};
            __builtin_memcpy(target, &packed, 8);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 3; ++j) {
            if (first + j < experts) {
              store_value(target, j, value[u][c][j], kDtypeOf<T>);
            }
          }
        }
      }
    }
  }
}

// Lanes per row and loads per lane by the expert count.
template <class T>
const void *balance_kernel_for(int experts, bool backward) {
  if (experts <= 64) {
    return backward ? reinterpret_cast<const void *>(&moe_balance_backward_kernel<T, 16, 1, 4>)
                    : reinterpret_cast<const void *>(&moe_balance_kernel<T, 16, 1, 4>);
  }
  if (experts <= 128) {
    return backward ? reinterpret_cast<const void *>(&moe_balance_backward_kernel<T, 32, 1, 4>)
                    : reinterpret_cast<const void *>(&moe_balance_kernel<T, 32, 1, 4>);
  }
  if (experts <= 256) {
    return backward ? reinterpret_cast<const void *>(&moe_balance_backward_kernel<T, 64, 1, 4>)
                    : reinterpret_cast<const void *>(&moe_balance_kernel<T, 64, 1, 4>);
  }
  if (experts <= 512) {
    return backward ? reinterpret_cast<const void *>(&moe_balance_backward_kernel<T, 64, 2, 2>)
                    : reinterpret_cast<const void *>(&moe_balance_kernel<T, 64, 2, 2>);
  }
  return backward ? reinterpret_cast<const void *>(&moe_balance_backward_kernel<T, 64, 4, 1>)
                  : reinterpret_cast<const void *>(&moe_balance_kernel<T, 64, 4, 1>);
}

const void *balance_kernel_for(const BalanceArgs &args, bool backward) {
  return args.dtype == kDtypeF32   ? balance_kernel_for<F32Payload>(args.experts, backward)
         : args.dtype == kDtypeF16 ? balance_kernel_for<F16Payload>(args.experts, backward)
                                   : balance_kernel_for<Bf16Payload>(args.experts, backward);
}

int64_t lanes_per_row(int64_t experts) { return experts <= 64 ? 16 : experts <= 128 ? 32 : 64; }

// Rows that one workgroup takes alone, without a second launch to add the sums.
constexpr int64_t kBalanceOneWorkgroupRows = 256;
// One per CU: 512 read 65536 x 128 fp32 logits and eight ids a row in 11.4 us instead of 12.2, but leave
// twice the sums, which the finishing launch adds in 8.1 us instead of 5.2.
constexpr int64_t kBalanceWorkgroups = 256;
constexpr int64_t kBalanceBackwardWorkgroups = 1024;

}  // namespace

int64_t balance_blocks(int64_t rows, int64_t experts) {
  if (rows <= kBalanceOneWorkgroupRows) {
    return 1;
  }
  const int64_t parts = kBalanceThreads / lanes_per_row(experts);
  return std::min(kBalanceWorkgroups, (rows + parts - 1) / parts);
}

KernelLaunch make_balance(const BalanceArgs &args) {
  KernelLaunch kernel;
  kernel.func = balance_kernel_for(args, false);
  kernel.grid = dim3(static_cast<unsigned>(args.blocks), 1, 1);
  kernel.block = dim3(kBalanceThreads, 1, 1);
  kernel.set_args(args);
  return kernel;
}

KernelLaunch make_balance_finish(const BalanceArgs &args) {
  KernelLaunch kernel;
  if (args.blocks > 1) {
    kernel.func = reinterpret_cast<const void *>(&moe_balance_finish_kernel);
    kernel.block = dim3(kBalanceThreads, 1, 1);
    kernel.set_args(args);
  }
  return kernel;
}

KernelLaunch make_balance_backward(const BalanceArgs &args) {
  KernelLaunch kernel;
  kernel.func = balance_kernel_for(args, true);
  const int64_t parts = 256 / lanes_per_row(args.experts);
  kernel.grid = dim3(static_cast<unsigned>(std::min(kBalanceBackwardWorkgroups, (args.rows + parts - 1) / parts)), 1, 1);
  kernel.block = dim3(256, 1, 1);
  kernel.set_args(args);
  return kernel;
}

}  // namespace xp
