// Routing rows to clusters: the k most probable clusters of each row, how
// often each cluster is chosen, and the loss that keeps them balanced, with
// its gradient.
//
// No reference operator.  For valid rows t of scores z (columns are clusters):
//   l_t = log sum_e e^z_te,  p = e^(z - l),  ids = the k largest z (equal ones
//   by cluster), weights = p at ids, counts_e = rows that chose e,
//   loss = E sum_e f_e P_e,  f_e = counts_e / (k rows),  P_e = sum_t p_te / rows
// and with a_te = g_loss E f_e / rows + (g_w of e, where row t chose it):
//   dz_te = p_te (a_te - sum_j a_tj p_tj + g_l)
// A row whose flag is off, or without a score above -inf, is no valid row: it
// has ids -1, weights 0, l = -inf, and gradients of zero.
//
// A row stays in registers from its one read on: LPR lanes hold U units of 8
// columns each.  Lane i's columns are the same for every row, so the column
// sums of p are accumulated in registers too, and joined once per workgroup;
// workgroups write their sums and counts, which the second kernel adds up in
// order (no floating-point atomics: the same inputs give the same bits).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <mutex>

#include "score_ops.hpp"
#include "st_errors.hpp"

namespace st {
int cu_count();

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxProbes = 64;
constexpr int kMaxClusters = 32768;
constexpr int kFinishColumns = 64;  // clusters per workgroup of the second kernel
constexpr float kLog2e = 1.4426950408889634f;

struct RouteArgs {
  const void* logits;
  int64_t rows, row_stride;
  int clusters, probes;
  const uint8_t* valid;   // null: all
  int64_t* ids;
  float *weights, *lse, *stats;  // stats [rows, 2]: max and sum of exponentials
  float* part_sums;       // [groups, clusters]
  uint32_t* part_counts;  // [groups, clusters]
  uint32_t* part_rows;    // [groups]
  uint32_t* ticket;
};

template <int LPR>
__device__ __forceinline__ float row_max(float x, float* red) {
  if constexpr (LPR == 8) return join8(x, [](float a, float b) { return fmaxf(a, b); });
  x = wave_max(x);
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    const int wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 0) red[wave] = x;
    __syncthreads();
    const int first = wave / W * W;
    x = red[first];
#pragma unroll
    for (int w = 1; w < W; ++w) x = fmaxf(x, red[first + w]);
  }
  return x;
}

template <int LPR>
__device__ __forceinline__ float row_sum(float x, float* red) {
  if constexpr (LPR == 8) return join8(x, [](float a, float b) { return a + b; });
  x = wave_sum(x);
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    const int wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 0) red[wave] = x;
    __syncthreads();
    const int first = wave / W * W;
    x = red[first];
#pragma unroll
    for (int w = 1; w < W; ++w) x += red[first + w];
  }
  return x;
}

// Column of value i of a lane whose first column is `own`.
template <int LPR>
__device__ __forceinline__ int column_of(int own, int i) {
  return own + LPR * 8 * (i >> 3) + (i & 7);
}

// One step of taking the largest value left: the best of the lane group's
// values (value, then lowest column), which its owner marks as taken.
template <int LPR, int U>
__device__ __forceinline__ void take_best(const float v[U * 8], uint32_t& taken, int own, float& value,
                                          uint32_t& column) {
  float best = kMinusInf;
  int at = -1;
#pragma unroll
  for (int i = 0; i < U * 8; ++i) {
    const uint32_t gone = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(taken), i, 1));
    const float x = __uint_as_float((0xFF800000u & gone) | (__float_as_uint(v[i]) & ~gone));
    if (x > best) {
      best = x;
      at = i;
    }
  }
  const uint32_t mine = at < 0 ? ~0u : static_cast<uint32_t>(column_of<LPR>(own, at));
  constexpr int L = LPR < 64 ? LPR : 64;
  if constexpr (L == 8)
    value = join8(best, [](float a, float b) { return fmaxf(a, b); });
  else
    value = wave_max(best);
  uint32_t low = best == value ? mine : ~0u;
#pragma unroll
  for (int o = 1; o < L; o <<= 1) low = min(low, static_cast<uint32_t>(__shfl_xor(static_cast<int>(low), o)));
  if (at >= 0 && mine == low) taken |= 1u << at;
  column = low;  // ~0: nothing left
}

__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// The wave's best k of its values, unordered, as keys in list[0, n); n <= 64.
// The k-th largest of the lanes' maxima bounds the k-th best value from below;
// it is found bit by bit from the top, and few more than k values reach it.
// Where many do (equal values), k steps of taking the best replace that.
template <int LPR, int U>
__device__ __forceinline__ int wave_select(const float v[U * 8], int own, int k, uint64_t* list) {
  const int lane = threadIdx.x % 64;
  float best = kMinusInf;
#pragma unroll
  for (int i = 0; i < U * 8; ++i) best = fmaxf(best, v[i]);
  const uint32_t order = ordered_score(best);
  uint32_t bound = 0;
  for (int b = 31; b >= 0; --b) {
    const uint32_t t = bound | (1u << b);
    const int n = __popcll(__ballot(order >= t));
    if (n >= k) {
      bound = t;
      if (n == k) break;
    }
  }
  bound = max(bound, 0x00800000u);  // above -inf
  const float least = score_from_ordered(bound);
  int n = 0;
#pragma unroll
  for (int i = 0; i < U * 8; ++i) {
    const bool take = v[i] >= least;
    const uint64_t who = __ballot(take);
    if (who != 0) {
      const int at = n + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(who >> 32),
                                                   __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who), 0));
      if (take && at < 64) list[at] = score_key(v[i], column_of<LPR>(own, i));
      n += __popcll(who);
    }
  }
  if (n > 64) {
    n = 0;
    uint32_t taken = 0;
    for (int j = 0; j < k; ++j) {
      float value;
      uint32_t column;
      take_best<LPR, U>(v, taken, own, value, column);  // of the wave's own columns
      if (column == ~0u) break;
      if (lane == 0) list[n] = score_key(value, column);
      ++n;
    }
  }
  return n;
}

template <int DT, int LPR, int U>
__global__ __launch_bounds__(kThreads) void route_kernel(RouteArgs a) {
  constexpr int kRows = kThreads / LPR;             // rows at a time
  constexpr int kWavesPerRow = LPR > 64 ? LPR / 64 : 1;
  extern __shared__ __align__(16) uint8_t lds_raw[];
  uint64_t* lists = reinterpret_cast<uint64_t*>(lds_raw);                 // [kWaves][64]
  uint32_t* hist = reinterpret_cast<uint32_t*>(lists + kWaves * 64);      // [clusters]
  float* sums = reinterpret_cast<float*>(hist + a.clusters);              // [clusters], with kRows > 1
  __shared__ float red_max[kWaves], red_sum[kWaves];
  __shared__ int list_n[kWaves];
  __shared__ uint32_t row_count;
  const int tid = threadIdx.x;
  const int wave = tid / 64, lane = tid % 64;
  const int group = tid / LPR, in_row = tid % LPR;
  const int clusters = a.clusters, k = a.probes;
  for (int e = tid; e < clusters; e += kThreads) hist[e] = 0;
  if (tid == 0) {
    row_count = 0;
    if (blockIdx.x == 0) *a.ticket = 0;  // the second kernel's workgroups count on it
  }
  __syncthreads();

  float acc[U * 8];
#pragma unroll
  for (int i = 0; i < U * 8; ++i) acc[i] = 0.0f;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < a.rows;
       base += static_cast<int64_t>(gridDim.x) * kRows) {
    const int64_t r = base + group;
    const bool mine = r < a.rows;
    const bool on = mine && (a.valid == nullptr || a.valid[r] != 0);
    // The columns are computed where they are used: kept in registers over the
    // loop they would push the scores out.
    int own = in_row * 8;
    asm volatile("" : "+v"(own));
    const char* row = static_cast<const char*>(a.logits) + r * a.row_stride * kScoreBytes<DT>;
    float v[U * 8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int col = column_of<LPR>(own, u * 8);
      if (on && col + 8 <= clusters) {
        unpack8<DT>(load_raw8<DT>(row, col), v + u * 8);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[u * 8 + i] = on && col + i < clusters ? load_score<DT>(row, col + i) : kMinusInf;
      }
    }
    float top = kMinusInf;
#pragma unroll
    for (int i = 0; i < U * 8; ++i) top = fmaxf(top, v[i]);
    top = row_max<LPR>(top, red_max);
    const float m = top == kMinusInf ? 0.0f : top;
    uint64_t* list = lists + wave * 64;
    int n = 0;
    if constexpr (LPR > 8) n = wave_select<LPR, U>(v, own, k, list);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < U * 8; ++i) {
      const float e = __builtin_amdgcn_exp2f((v[i] - m) * kLog2e);
      sum += e;
      if constexpr (LPR > 8) v[i] = e;  // the selection is done with the scores
    }
    sum = row_sum<LPR>(sum, red_sum);
    const bool some = !(top == kMinusInf && sum == 0.0f);
    const float inv = some ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int i = 0; i < U * 8; ++i)
      acc[i] = fmaf(LPR > 8 ? v[i] : __builtin_amdgcn_exp2f((v[i] - m) * kLog2e), inv, acc[i]);
    if (mine && in_row == 0) {
      a.lse[r] = some ? top + logf(sum) : kMinusInf;
      a.stats[2 * r] = top;
      a.stats[2 * r + 1] = sum;
      if (some) atomicAdd(&row_count, 1u);
    }

    if constexpr (LPR == 8) {
      uint32_t kept_column = ~0u, taken = 0;
      float kept = kMinusInf;
      for (int j = 0; j < k; ++j) {
        float value;
        uint32_t column;
        take_best<LPR, U>(v, taken, own, value, column);
        if (in_row == j % 8) {
          kept_column = column;
          kept = value;
        }
        const int at = j / 8 * 8 + in_row;
        if ((j % 8 == 7 || j == k - 1) && mine && at <= j) {
          const bool is = kept_column != ~0u;
          a.ids[r * k + at] = is ? static_cast<int64_t>(kept_column) : -1;
          a.weights[r * k + at] = is ? __builtin_amdgcn_exp2f((kept - m) * kLog2e) * inv : 0.0f;
          if (is) atomicAdd(&hist[kept_column], 1u);
        }
      }
    } else {
      int total = n;
      const uint64_t* from = list;
      if constexpr (kWavesPerRow > 1) {
        if (lane == 0) list_n[wave] = n;
        __syncthreads();
        from = lists + group * kWavesPerRow * 64;
        total = 0;
#pragma unroll
        for (int w = 0; w < kWavesPerRow; ++w) total += list_n[group * kWavesPerRow + w];
      } else {
        wave_fence();
      }
      // each key's place is the number of keys above it; a thread per key of
      // its wave's list
      if (lane < n) {
        const uint64_t key = list[lane];
        int above = 0;
        if constexpr (kWavesPerRow > 1) {
          for (int w = 0; w < kWavesPerRow; ++w) {
            const int nw = list_n[group * kWavesPerRow + w];
            for (int j = 0; j < nw; ++j) above += from[w * 64 + j] > key ? 1 : 0;
          }
        } else {
          for (int j = 0; j < n; ++j) above += from[j] > key ? 1 : 0;
        }
        if (above < k) {
          const uint32_t column = ~static_cast<uint32_t>(key);
          a.ids[r * k + above] = column;
          a.weights[r * k + above] =
              __builtin_amdgcn_exp2f((score_from_ordered(static_cast<uint32_t>(key >> 32)) - m) * kLog2e) * inv;
          atomicAdd(&hist[column], 1u);
        }
      }
      if (mine && in_row < k && in_row >= total) {
        a.ids[r * k + in_row] = -1;
        a.weights[r * k + in_row] = 0.0f;
      }
      if constexpr (kWavesPerRow == 1) wave_fence();
    }
  }

  // the workgroup's column sums, row group by row group
  __syncthreads();
  float* out = a.part_sums + static_cast<int64_t>(blockIdx.x) * clusters;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int i = 0; i < U * 8; ++i) {
      const int col = column_of<LPR>(in_row * 8, i);
      if (col < clusters) out[col] = acc[i];
    }
  } else {
    if constexpr (LPR == 8) {
#pragma unroll
      for (int i = 0; i < U * 8; ++i)
#pragma unroll
        for (int o = 8; o < 64; o <<= 1) acc[i] += __shfl_xor(acc[i], o);
    }
    constexpr int kTurns = LPR > 64 ? kRows : kWaves;
    const int turn = LPR > 64 ? group : wave;
    for (int w = 0; w < kTurns; ++w) {
      if (turn == w && (LPR >= 64 || lane < LPR)) {
#pragma unroll
        for (int i = 0; i < U * 8; ++i) {
          const int col = column_of<LPR>(in_row * 8, i);
          if (col < clusters) sums[col] = w == 0 ? acc[i] : sums[col] + acc[i];
        }
      }
      __syncthreads();
    }
    for (int e = tid; e < clusters; e += kThreads) out[e] = sums[e];
  }
  uint32_t* counts = a.part_counts + static_cast<int64_t>(blockIdx.x) * clusters;
  for (int e = tid; e < clusters; e += kThreads) counts[e] = hist[e];
  if (tid == 0) a.part_rows[blockIdx.x] = row_count;
}

struct FinishArgs {
  const float* part_sums;
  const uint32_t *part_counts, *part_rows;
  int groups, clusters, probes;
  int64_t* counts;
  float* slopes;   // [clusters]: dloss / dp of a row
  float* loss;
  double* part_loss;
  uint32_t* ticket;
};

// Adds up the workgroups' parts: 64 clusters per workgroup, 16 slices of the
// parts each; the last workgroup to end adds up the loss.
__global__ __launch_bounds__(kThreads) void route_finish_kernel(FinishArgs a) {
  __shared__ float sums[kWaves][kFinishColumns];
  __shared__ uint32_t counts[kWaves][kFinishColumns];
  __shared__ uint32_t rows_of[kWaves];
  __shared__ bool last;
  const int tid = threadIdx.x, slice = tid / 64, lane = tid % 64;
  const int e = blockIdx.x * kFinishColumns + lane;
  float sum = 0.0f;
  uint32_t count = 0, rows = 0;
  if (e < a.clusters)
    for (int g = slice; g < a.groups; g += kWaves) {
      sum += a.part_sums[static_cast<int64_t>(g) * a.clusters + e];
      count += a.part_counts[static_cast<int64_t>(g) * a.clusters + e];
    }
  for (int g = tid; g < a.groups; g += kThreads) rows += a.part_rows[g];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) rows += __shfl_xor(rows, o);
  sums[slice][lane] = sum;
  counts[slice][lane] = count;
  if (lane == 0) rows_of[slice] = rows;
  __syncthreads();
  if (slice == 0) {
    double total_rows = 0.0;
    double p = 0.0;
    int64_t n = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      total_rows += rows_of[w];
      p += sums[w][lane];
      n += counts[w][lane];
    }
    const double scale = total_rows > 0.0 ? a.clusters / (total_rows * total_rows * a.probes) : 0.0;
    double part = 0.0;
    if (e < a.clusters) {
      a.counts[e] = n;
      a.slopes[e] = static_cast<float>(scale * static_cast<double>(n));
      part = scale * static_cast<double>(n) * p;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) part += __shfl_xor(part, o);
    if (lane == 0) {
      __hip_atomic_store(&a.part_loss[blockIdx.x], part, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __threadfence();
      last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
      __threadfence();
    }
  }
  __syncthreads();
  if (last && slice == 0) {
    double part = 0.0;
    for (unsigned b = lane; b < gridDim.x; b += 64)
      part += __hip_atomic_load(&a.part_loss[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) part += __shfl_xor(part, o);
    if (lane == 0) *a.loss = static_cast<float>(part);
  }
}

struct RouteBackwardArgs {
  const void* logits;
  int64_t rows, row_stride;
  int clusters, probes;
  const int64_t* ids;
  const float *weights, *stats, *slopes;
  const float *g_weights, *g_lse, *g_loss;  // each may be null: zero
  void* grad;                               // [rows, clusters], contiguous
};

// dz = p (g_loss slope - dot + g_l), then the chosen clusters again with their
// own g_w; dot = sum of g_loss slope p over the row and of g_w p over the chosen.
template <int DT, int LPR, int U>
__global__ __launch_bounds__(kThreads) void route_backward_kernel(RouteBackwardArgs a) {
  constexpr int kRows = kThreads / LPR;
  __shared__ float red_sum[2][kWaves];
  const int tid = threadIdx.x;
  const int group = tid / LPR, in_row = tid % LPR;
  const int clusters = a.clusters, k = a.probes;
  const float g_loss = a.g_loss != nullptr ? *a.g_loss : 0.0f;
  float slope[U * 8];
#pragma unroll
  for (int i = 0; i < U * 8; ++i) {
    const int col = column_of<LPR>(in_row * 8, i);
    slope[i] = col < clusters ? g_loss * a.slopes[col] : 0.0f;
  }
  int turn = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < a.rows;
       base += static_cast<int64_t>(gridDim.x) * kRows, turn ^= 1) {
    const int64_t r = base + group;
    const bool mine = r < a.rows;
    const float top = mine ? a.stats[2 * r] : kMinusInf, sum = mine ? a.stats[2 * r + 1] : 0.0f;
    const bool some = mine && !(top == kMinusInf && sum == 0.0f);
    const float m = top == kMinusInf ? 0.0f : top;
    const float inv = some ? 1.0f / sum : 0.0f;
    const char* row = static_cast<const char*>(a.logits) + r * a.row_stride * kScoreBytes<DT>;
    char* out = static_cast<char*>(a.grad) + r * clusters * kScoreBytes<DT>;
    float v[U * 8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int col = column_of<LPR>(in_row * 8, u * 8);
      if (some && col + 8 <= clusters) {
        unpack8<DT>(load_raw8<DT>(row, col), v + u * 8);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[u * 8 + i] = some && col + i < clusters ? load_score<DT>(row, col + i) : kMinusInf;
      }
    }
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < U * 8; ++i) {
      v[i] = __builtin_amdgcn_exp2f((v[i] - m) * kLog2e) * inv;
      dot = fmaf(slope[i], v[i], dot);
    }
    float own[kMaxProbes / (LPR < kMaxProbes ? LPR : kMaxProbes)];
    constexpr int kOwn = kMaxProbes / (LPR < kMaxProbes ? LPR : kMaxProbes);
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      const int i = in_row + LPR * j;
      own[j] = some && i < k && a.g_weights != nullptr ? a.g_weights[r * k + i] : 0.0f;
      if (some && i < k) dot = fmaf(own[j], a.weights[r * k + i], dot);
    }
    dot = row_sum<LPR>(dot, red_sum[turn]);
    const float shift = (a.g_lse != nullptr && some ? a.g_lse[r] : 0.0f) - dot;
    if (mine) {
#pragma unroll
      for (int i = 0; i < U * 8; ++i) v[i] = some ? v[i] * (slope[i] + shift) : 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int col = column_of<LPR>(in_row * 8, u * 8);
        if (col + 8 <= clusters) {
          store8<DT>(out, col, v + u * 8);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (col + i < clusters) store_score<DT>(out, col + i, v[u * 8 + i]);
        }
      }
    }
    if (a.g_weights != nullptr) {  // the same for every thread
      if constexpr (LPR > 64)
        __syncthreads();
      else
        wave_fence();
      if (some) {
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
          const int i = in_row + LPR * j;
          const int64_t id = i < k ? a.ids[r * k + i] : -1;
          if (id >= 0)
            store_score<DT>(out, id, a.weights[r * k + i] * (g_loss * a.slopes[id] + shift + own[j]));
        }
      }
    }
  }
}

void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw Error(ST_ERR_HIP, cat(what, " launch failed: ", hipGetErrorString(e)));
}

// Calls f with the lanes per row and the units per lane that hold a row.
template <typename F>
void for_shape(int64_t clusters, F f) {
  using std::integral_constant;
#define ST_SHAPE(L, U) return f(integral_constant<int, L>{}, integral_constant<int, U>{})
  if (clusters <= 64) ST_SHAPE(8, 1);
  if (clusters <= 128) ST_SHAPE(8, 2);
  if (clusters <= 256) ST_SHAPE(8, 4);
  if (clusters <= 512) ST_SHAPE(64, 1);
  if (clusters <= 1024) ST_SHAPE(64, 2);
  if (clusters <= 2048) ST_SHAPE(64, 4);
  if (clusters <= 4096) ST_SHAPE(256, 2);
  if (clusters <= 8192) ST_SHAPE(256, 4);
  if (clusters <= 16384) ST_SHAPE(1024, 2);
  ST_SHAPE(1024, 4);
#undef ST_SHAPE
}

int rows_at_once(int64_t clusters) {
  int n = 0;
  for_shape(clusters, [&](auto lpr, auto) { n = kThreads / lpr(); });
  return n;
}

int group_count(int64_t rows, int64_t clusters) {
  const int64_t n = rows_at_once(clusters);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((rows + n - 1) / n, 2 * cu_count())));
}

size_t route_lds(int64_t clusters) {
  return kWaves * 64 * 8 + clusters * 4 * (rows_at_once(clusters) > 1 ? 2 : 1);
}

int64_t finish_groups(int64_t clusters) { return (clusters + kFinishColumns - 1) / kFinishColumns; }

template <int DT>
void launch_route(const RouteArgs& a, int groups, hipStream_t s) {
  for_shape(a.clusters, [&](auto lpr, auto units) {
    auto kernel = route_kernel<DT, lpr(), units()>;
    const size_t lds = route_lds(a.clusters);
    if (lds > 48 * 1024) {
      static std::once_flag once;
      std::call_once(once, [&] {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, 159 * 1024);
        if (e != hipSuccess) throw Error(ST_ERR_HIP, cat("hipFuncSetAttribute failed: ", hipGetErrorString(e)));
      });
    }
    hipLaunchKernelGGL(kernel, dim3(groups), dim3(kThreads), lds, s, a);
    check_launch("route_kernel");
  });
}

template <int DT>
void launch_route_backward(const RouteBackwardArgs& a, hipStream_t s) {
  for_shape(a.clusters, [&](auto lpr, auto units) {
    const int64_t n = kThreads / lpr();
    const int64_t grid = std::min<int64_t>((a.rows + n - 1) / n, 4 * cu_count());
    hipLaunchKernelGGL((route_backward_kernel<DT, lpr(), units()>), dim3(static_cast<unsigned>(grid)), dim3(kThreads),
                       0, s, a);
    check_launch("route_backward_kernel");
  });
}

void check_route(int score_type, int64_t rows, int64_t clusters, int64_t row_stride, int64_t probes) {
  ST_CHECK(score_type == ST_SCORE_F32 || score_type == ST_SCORE_F16 || score_type == ST_SCORE_BF16,
           "scores must be float32, float16 or bfloat16");
  ST_CHECK(rows >= 0 && row_stride >= 0, "negative sizes");
  ST_CHECK(clusters >= 1 && clusters <= kMaxClusters, "clusters must be in [1, ", kMaxClusters, "], got ", clusters);
  ST_CHECK(probes >= 1 && probes <= kMaxProbes, "probes must be in [1, ", kMaxProbes, "], got ", probes);
}

}  // namespace
}  // namespace st

extern "C" int64_t st_cluster_route_workspace_bytes(int64_t rows, int64_t clusters) {
  using namespace st;
  if (rows < 0 || clusters < 1 || clusters > kMaxClusters) return 0;
  const int64_t groups = group_count(rows, clusters);
  return 8 * finish_groups(clusters) + groups * (8 * clusters + 4) + 64;
}

extern "C" int st_cluster_route(const void* logits, int score_type, int64_t rows, int64_t clusters,
                                int64_t row_stride, int64_t probes, const uint8_t* valid, void* workspace,
                                int64_t* cluster_ids, float* weights, float* lse, int64_t* counts, float* loss,
                                float* stats, float* slopes, void* stream) {
  using namespace st;
  return guarded([&] {
    check_route(score_type, rows, clusters, row_stride, probes);
    ST_CHECK(workspace && counts && loss && slopes, "null device pointer");
    ST_CHECK(rows == 0 || (logits && cluster_ids && weights && lse && stats), "null device pointer");
    const int groups = group_count(rows, clusters);
    FinishArgs f{};
    f.part_loss = static_cast<double*>(workspace);
    float* sums = reinterpret_cast<float*>(f.part_loss + finish_groups(clusters));
    uint32_t* part_counts = reinterpret_cast<uint32_t*>(sums + static_cast<int64_t>(groups) * clusters);
    uint32_t* part_rows = part_counts + static_cast<int64_t>(groups) * clusters;
    RouteArgs a{};
    a.logits = logits;
    a.rows = rows;
    a.row_stride = row_stride;
    a.clusters = static_cast<int>(clusters);
    a.probes = static_cast<int>(probes);
    a.valid = valid;
    a.ids = cluster_ids;
    a.weights = weights;
    a.lse = lse;
    a.stats = stats;
    a.part_sums = sums;
    a.part_counts = part_counts;
    a.part_rows = part_rows;
    a.ticket = part_rows + groups;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (score_type == ST_SCORE_F32)
      launch_route<ST_SCORE_F32>(a, groups, s);
    else if (score_type == ST_SCORE_F16)
      launch_route<ST_SCORE_F16>(a, groups, s);
    else
      launch_route<ST_SCORE_BF16>(a, groups, s);
    f.part_sums = sums;
    f.part_counts = part_counts;
    f.part_rows = part_rows;
    f.groups = groups;
    f.clusters = a.clusters;
    f.probes = a.probes;
    f.counts = counts;
    f.slopes = slopes;
    f.loss = loss;
    f.ticket = a.ticket;
    hipLaunchKernelGGL(route_finish_kernel, dim3(static_cast<unsigned>(finish_groups(clusters))), dim3(kThreads), 0, s, f);
    check_launch("route_finish_kernel");
  });
}

extern "C" int st_cluster_route_backward(const void* logits, int score_type, int64_t rows, int64_t clusters,
                                         int64_t row_stride, int64_t probes, const int64_t* cluster_ids,
                                         const float* weights, const float* stats, const float* slopes,
                                         const float* grad_weights, const float* grad_lse, const float* grad_loss,
                                         void* grad_logits, void* stream) {
  using namespace st;
  return guarded([&] {
    check_route(score_type, rows, clusters, row_stride, probes);
    if (rows == 0) return;
    ST_CHECK(logits && cluster_ids && weights && stats && slopes && grad_logits, "null device pointer");
    RouteBackwardArgs a{};
    a.logits = logits;
    a.rows = rows;
    a.row_stride = row_stride;
    a.clusters = static_cast<int>(clusters);
    a.probes = static_cast<int>(probes);
    a.ids = cluster_ids;
    a.weights = weights;
    a.stats = stats;
    a.slopes = slopes;
    a.g_weights = grad_weights;
    a.g_lse = grad_lse;
    a.g_loss = grad_loss;
    a.grad = grad_logits;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (score_type == ST_SCORE_F32)
      launch_route_backward<ST_SCORE_F32>(a, s);
    else if (score_type == ST_SCORE_F16)
      launch_route_backward<ST_SCORE_F16>(a, s);
    else
      launch_route_backward<ST_SCORE_BF16>(a, s);
  });
}
