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

constexpr int kMaxProbes = 64;
constexpr int kMaxClusters = 32768;
constexpr int kFinishThreads = 1024;
constexpr int kFinishColumns = 16;  // clusters per workgroup of the second kernel
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kRowList = 512, kWaveList = 128;  // candidates of a row of several waves, of one

// Threads of a workgroup, four waves a SIMD: rows of one wave or less take two
// workgroups a CU (five or six waves a SIMD measured the same or slower: 65,536
// x 64 18.6 and 17.1 us against 16.8); rows of more waves want few workgroups,
// whose sums are written.
template <int LPR>
constexpr int kThreads = LPR > 64 ? 1024 : 512;

struct RouteArgs {
  const void* logits;
  int64_t rows, row_stride;
  int clusters, probes;
  const uint8_t* valid;   // null: all
  int64_t* ids;
  float *weights, *lse, *stats;  // stats [rows, 2]: max and sum of exponentials (reference)
  float* part_sums;       // [groups, clusters]
  uint32_t* part_counts;  // [groups, clusters]
  uint32_t* part_rows;    // [groups]
  uint32_t* ticket;
  // the results over all rows, written here when there is one workgroup
  int64_t* counts;
  float *slopes, *loss;
};

// A row's exponentials are 2^(z c - ref), c = log2 e and ref = m c rounded, or,
// of rows whose maximum m is wide, 2^((z - m) c).  The rounding is half an ulp
// of m c at most, 1/16 for those that are not; from 2^31 on it could pass the
// exponents of 32 bits.
__device__ __forceinline__ bool is_wide(float m) { return !(fabsf(m) < 0x1p20f); }

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

// The values of lane ^ T.
template <int T>
__device__ __forceinline__ float lane_xor(float x) {
  if constexpr (T == 1) return dpp_move<0xB1>(x);                  // quad_perm [1, 0, 3, 2]
  if constexpr (T == 2) return dpp_move<0x4E>(x);                  // quad_perm [2, 3, 0, 1]
  if constexpr (T == 4) return dpp_move<0x141>(dpp_move<0x1B>(x));  // ^ 3, then row_half_mirror: ^ 7
  return dpp_move<0x128>(x);                                       // row_ror:8
}

// The values of lane ^ T, T 16 or 32.
template <int T>
__device__ __forceinline__ float wave_swap(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto pair = T == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false)
                            : __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(threadIdx.x % 64 & T ? pair[0] : pair[1]);
}

// One step of sorting values over lanes, largest first: sequences of S lanes,
// partners T apart.  LAST: the last sequences, all in one direction.
template <int S, int T, bool LAST>
__device__ __forceinline__ float sort_step(float x) {
  const int lane = threadIdx.x % 64;
  float a = x, b;
  if constexpr (T >= 16) {
    const uint32_t u = __float_as_uint(x);
    const auto pair = T == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false)
                              : __builtin_amdgcn_permlane32_swap(u, u, false, false);
    a = __uint_as_float(pair[0]);
    b = __uint_as_float(pair[1]);
  } else {
    b = lane_xor<T>(x);
  }
  return ((lane & T) == 0) == (LAST || (lane & S) == 0) ? fmaxf(a, b) : fminf(a, b);
}

template <int S, int T, bool LAST = S == 64>
__device__ __forceinline__ float sort_merge(float x) {
  x = sort_step<S, T, LAST>(x);
  if constexpr (T > 1) x = sort_merge<S, T / 2, LAST>(x);
  return x;
}

// A bound that at least k of the wave's values reach, the lowest finite one if
// fewer are above -inf; `top` becomes the largest.  The k-th largest of 16, 32
// or 64 groups' maxima, at least twice k if there are as many, by up to 21
// compare-exchange steps without a branch (bisecting the bits of a value takes
// as many vector instructions but waits for the scalar unit after each).
__device__ __forceinline__ float wave_bound(float& top, int k) {
  float x = top;
  if (k <= 16) x = fmaxf(x, wave_swap<32>(x));
  if (k <= 8) x = fmaxf(x, wave_swap<16>(x));
  x = sort_merge<2, 1>(x);
  x = sort_merge<4, 2>(x);
  x = sort_merge<8, 4>(x);
  if (k <= 8) {
    x = sort_merge<16, 8, true>(x);
  } else {
    x = sort_merge<16, 8>(x);
    if (k <= 16) {
      x = sort_merge<32, 16, true>(x);
    } else {
      x = sort_merge<32, 16>(x);
      x = sort_merge<64, 32>(x);
    }
  }
  const int bits = __float_as_int(x);
  top = __int_as_float(__builtin_amdgcn_readlane(bits, 0));
  return fmaxf(__int_as_float(__builtin_amdgcn_readlane(bits, k - 1)), -3.4028234663852886e38f);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// The largest of a lane's values.
template <int N>
__device__ __forceinline__ float lane_max(const float v[N]) {
  float top = max3(v[0], v[1], v[2]);
#pragma unroll
  for (int i = 3; i + 1 < N; i += 2) top = max3(top, v[i], v[i + 1]);
  return N % 2 == 0 ? fmaxf(top, v[N - 1]) : top;
}

// A candidate as it is kept until it is ranked, and its key.
__device__ __forceinline__ uint64_t candidate(float value, int column) {
  return (static_cast<uint64_t>(__float_as_uint(value)) << 32) | static_cast<uint32_t>(column);
}
__device__ __forceinline__ uint64_t key_of(uint64_t c) {
  return score_key(__uint_as_float(static_cast<uint32_t>(c >> 32)), static_cast<uint32_t>(c));
}

// Puts the wave's values that reach `least` into list[n, size) as candidates,
// one register at a time; returns n and their number, which may pass the size.
template <int LPR, int U>
__device__ __forceinline__ int append(const float v[U * 8], float least, int own, uint64_t* list, int n, int size) {
#pragma unroll
  for (int i = 0; i < U * 8; ++i) {
    const bool take = v[i] >= least;
    const uint64_t who = __ballot(take);
    if (who != 0) {
      const int at = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(who >> 32),
                                               __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who), n));
      if (take && at < size) list[at] = candidate(v[i], column_of<LPR>(own, i));
      n += __popcll(who);
    }
  }
  return n;
}

// The wave's best k by k steps of taking the best, for rows whose bound more
// values reach than there is room for: equal scores, or high ones side by side
// in few lanes.
template <int LPR, int U>
__device__ __forceinline__ int append_in_steps(const float v[U * 8], int own, int k, uint64_t* list) {
  uint32_t taken = 0;
  for (int j = 0; j < k; ++j) {
    float value;
    uint32_t column;
    take_best<LPR, U>(v, taken, own, value, column);  // of the wave's own columns
    if (column == ~0u) return j;
    if (threadIdx.x % 64 == 0) list[j] = candidate(value, static_cast<int>(column));
  }
  return k;
}

// The sum over a workgroup, in the first thread, in a fixed order.
template <int T>
__device__ __forceinline__ double sum_workgroup(double x, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = x;
  __syncthreads();
  x = threadIdx.x < T / 64 ? red[threadIdx.x] : 0.0;
  if (threadIdx.x < 64) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) x += __shfl_xor(x, o);  // at most 16 waves
  }
  return x;
}

// dloss / dp of a row is this times the cluster's count.
__device__ __forceinline__ double loss_scale(int clusters, int probes, double rows) {
  return rows > 0.0 ? clusters / (rows * rows * probes) : 0.0;
}

// The k-th largest of the lanes' maxima (of a row of one wave; of 64 groups of
// lanes of a row of more, which meet in LDS) bounds the k-th best score from
// below; few more than k scores reach it, and each one's place is the number of
// keys above it.  Exponentials are 2^(z c - ref), ref the rounded m c, one
// multiply-add each; p = e / sum e does not depend on ref, and lse takes it
// back as it is.  The next row's scores are loaded before a row is worked on.
//
// What bounds it: vector instructions.  A row of 1,024 scores in one wave takes
// some 400 of them (a third for the exponentials and sums, the rest for the
// selection), more than its 2 KB take to arrive; a row of several waves waits at
// three barriers besides.  Measured with the second kernel: 65,536 x 1,024
// bfloat16, 8 probes 72 us (46 us without a selection, 37 us for the reads
// alone); 16,001 x 5,000 float32, 24 probes 134 us; 65,536 x 64 bfloat16, 2
// probes 17 us; 8 x 2,500 float32, 16 probes 14.5 us in one workgroup.
template <int DT, int LPR, int U>
__global__ __launch_bounds__(kThreads<LPR>, 4) void route_kernel(RouteArgs a) {
  constexpr int T = kThreads<LPR>;
  constexpr int kWaves = T / 64;
  constexpr int kRows = T / LPR;  // rows at a time
  constexpr int kWavesPerRow = LPR > 64 ? LPR / 64 : 1;
  constexpr int kList = LPR > 64 ? kRowList : kWaveList;  // keys of a row
  // Whether registers are left for the next row's scores: once a register is
  // spilled, its reload waits for them too (16,001 x 5,000 float32: 162 us with
  // them, 134 us without).
  constexpr bool kAhead = U < (LPR == 64 && DT != ST_SCORE_F32 ? 4 : 3);
  extern __shared__ __align__(16) uint8_t lds_raw[];
  uint64_t* lists = reinterpret_cast<uint64_t*>(lds_raw);  // [kRows or kWaves][kList]
  uint32_t* hist = reinterpret_cast<uint32_t*>(lists + (LPR > 64 ? kRows : kWaves) * kList);  // [clusters]
  float* sums = reinterpret_cast<float*>(hist + (a.clusters + 7) / 8 * 8);  // likewise, with kRows > 1
  __shared__ float maxima[LPR > 64 ? kRows * 64 : 1];
  __shared__ float part_sum[kWaves], row_bound[kRows], row_top[kRows];
  __shared__ uint32_t list_n[2][kRows];
  __shared__ uint32_t row_count;
  __shared__ double red[kWaves];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
  const int group = LPR >= 64 ? wave / kWavesPerRow : tid / LPR, in_row = tid % LPR;
  [[maybe_unused]] const int first = group * kWavesPerRow;  // the row's first wave
  const int clusters = a.clusters, k = a.probes;
  for (int e = tid; e < clusters; e += T) hist[e] = 0;
  if (tid < kRows) list_n[0][tid] = list_n[1][tid] = 0;
  if (tid == 0) {
    row_count = 0;
    if (blockIdx.x == 0) *a.ticket = 0;  // the second kernel's workgroups count on it
  }

  // Scores of row r, -inf where there are none, and its flag, which nothing
  // waits for here.
  auto load = [&](int64_t r, Raw8<DT> raw[U], uint32_t& flag) {
    const bool on = r < a.rows;
    flag = 1;
    if (on && a.valid != nullptr) flag = a.valid[r];
    const char* row = static_cast<const char*>(a.logits) + r * a.row_stride * kScoreBytes<DT>;
    int own = in_row * 8;
    // The columns are computed where they are used: kept in registers over the
    // loop they would push the scores out.
    asm volatile("" : "+v"(own));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int col = column_of<LPR>(own, u * 8);
      constexpr uint32_t kNone = DT == ST_SCORE_F32 ? 0xFF800000u : DT == ST_SCORE_F16 ? 0xFC00FC00u : 0xFF80FF80u;
      Raw8<DT> x;
#pragma unroll
      for (auto& w : x.w) w = u32x4{kNone, kNone, kNone, kNone};
      if (on && col + 8 <= clusters) {
        x = load_raw8<DT>(row, col);
      } else if (on && col < clusters) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (col + i >= clusters) continue;
          if constexpr (DT == ST_SCORE_F32) {
            x.w[i / 4][i % 4] = reinterpret_cast<const uint32_t*>(row)[col + i];
          } else {
            const uint32_t h = reinterpret_cast<const uint16_t*>(row)[col + i], old = x.w[0][i / 2];
            x.w[0][i / 2] = (i & 1) ? (old & 0xFFFFu) | (h << 16) : (old & 0xFFFF0000u) | h;
          }
        }
      }
      raw[u] = x;
    }
  };

  const int64_t stride = static_cast<int64_t>(gridDim.x) * kRows;
  float acc[U * 8];
#pragma unroll
  for (int i = 0; i < U * 8; ++i) acc[i] = 0.0f;
  Raw8<DT> next[U];
  uint32_t next_flag = 1;
  if constexpr (kAhead) load(static_cast<int64_t>(blockIdx.x) * kRows + group, next, next_flag);
  __syncthreads();

  int turn_of_lists = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < a.rows; base += stride) {
    const int64_t r = base + group;
    const bool mine = r < a.rows;
    int own = in_row * 8;
    asm volatile("" : "+v"(own));
    float v[U * 8];
    auto take = [&] {
      const bool off = next_flag == 0;
#pragma unroll
      for (int u = 0; u < U; ++u) unpack8<DT>(next[u], v + u * 8);
      if (off) {
#pragma unroll
        for (int i = 0; i < U * 8; ++i) v[i] = kMinusInf;
      }
    };
    if constexpr (!kAhead) load(r, next, next_flag);
    take();
    if constexpr (kAhead) load(r + stride, next, next_flag);

    // the row's maximum, and the keys that may be among its best k
    float top = fmaxf(lane_max<U * 8>(v), kMinusInf);  // never NaN: the sorting steps would double its neighbour
    uint64_t* list = lists + (LPR > 64 ? group : wave) * kList;
    uint32_t* const count = &list_n[turn_of_lists][group];
    int n = 0;
    if constexpr (LPR == 8) {
      top = join8(top, [](float x, float y) { return fmaxf(x, y); });
    } else if constexpr (LPR == 64) {
      const float least = wave_bound(top, k);
      n = append<LPR, U>(v, least, own, list, 0, kList);
      if (n > kList) n = append_in_steps<LPR, U>(v, own, k, list);
    } else {
      // 64 groups of lanes
      float most = fmaxf(top, dpp_move<0xB1>(top));
      most = fmaxf(most, dpp_move<0x4E>(most));
      if constexpr (LPR == 1024) {
        most = fmaxf(most, dpp_move<0x141>(most));
        most = fmaxf(most, dpp_move<0x140>(most));
      }
      if (in_row % (LPR / 64) == 0) maxima[group * 64 + in_row / (LPR / 64)] = most;
      __syncthreads();
      // one wave finds the bound, in each row group on another SIMD
      if (wave == first + group % 4) {
        top = maxima[group * 64 + lane];
        const float least = wave_bound(top, k);
        if (lane == 0) {
          row_bound[group] = least;
          row_top[group] = top;
        }
      }
      __syncthreads();
      const float least = row_bound[group];
      top = row_top[group];
      // this wave's scores that reach it go to the row's list
      int here = 0;
#pragma unroll
      for (int i = 0; i < U * 8; ++i) here += __popcll(__ballot(v[i] >= least));
      if (here != 0) {
        int at = 0;
        if (lane == 0) at = static_cast<int>(atomicAdd(count, static_cast<uint32_t>(here)));
        append<LPR, U>(v, least, own, list, __builtin_amdgcn_readfirstlane(at), kList);
      }
    }

    // exponentials and their sum
    const float m = top == kMinusInf ? 0.0f : top;
    const bool wide = is_wide(m);
    const float ref = wide ? 0.0f : m * kLog2e;
    auto exponential = [&](float z) {
      return __builtin_amdgcn_exp2f(wide ? (z - m) * kLog2e : fmaf(z, kLog2e, -ref));
    };
    float sum = 0.0f;
    if (!wide) {
#pragma unroll
      for (int i = 0; i < U * 8; ++i) {
        const float e = __builtin_amdgcn_exp2f(fmaf(v[i], kLog2e, -ref));
        sum += e;
        if constexpr (LPR > 8) v[i] = e;  // the selection is done with the scores
      }
    } else {
#pragma unroll
      for (int i = 0; i < U * 8; ++i) {
        const float e = __builtin_amdgcn_exp2f((v[i] - m) * kLog2e);
        sum += e;
        if constexpr (LPR > 8) v[i] = e;
      }
    }
    if constexpr (LPR == 8)
      sum = join8(sum, [](float x, float y) { return x + y; });
    else
      sum = wave_sum(sum);
    if constexpr (kWavesPerRow > 1) {
      if (lane == 0) part_sum[wave] = sum;
      if (tid < kRows) list_n[turn_of_lists ^ 1][tid] = 0;
      __syncthreads();
      sum = part_sum[first];
#pragma unroll
      for (int w = 1; w < kWavesPerRow; ++w) sum += part_sum[first + w];
      // A row with more candidates than its list holds is read again, and its
      // waves' own best k, found in steps, make the list; all row groups of the
      // workgroup go through the barriers.
      bool full = false;
#pragma unroll
      for (int g = 0; g < kRows; ++g) full |= list_n[turn_of_lists][g] > kList;
      n = static_cast<int>(*count);
      if (full) {
        const bool again = n > kList;
        __syncthreads();
        if (again && tid % LPR == 0) *count = 0;
        __syncthreads();
        // one wave after the other, so that k keys a wave are room enough: the
        // list keeps the best k after each
        for (int w = 0; w < kWavesPerRow; ++w) {
          if (again && wave == first + w) {
            float z[U * 8];
            Raw8<DT> raw[U];
            uint32_t flag;
            load(r, raw, flag);
#pragma unroll
            for (int u = 0; u < U; ++u) unpack8<DT>(raw[u], z + u * 8);
            const int had = static_cast<int>(*count);
            const int got = append_in_steps<LPR, U>(z, own, k, list + had);
            wave_fence();
            // of had + got keys, at most 2 k, the best k
            uint64_t keep[2];
            int place[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int at = lane + 64 * i;
              keep[i] = at < had + got ? list[at] : 0;
              place[i] = 0;
              for (int j = 0; j < had + got; ++j) place[i] += key_of(list[j]) > key_of(keep[i]) ? 1 : 0;
            }
            wave_fence();
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (lane + 64 * i < had + got && place[i] < k) list[place[i]] = keep[i];
            if (lane == 0) *count = min(had + got, k);
          }
          __syncthreads();
        }
        n = static_cast<int>(*count);
      }
      turn_of_lists ^= 1;
    } else if constexpr (LPR == 64) {
      wave_fence();
    }
    const bool some = !(top == kMinusInf && sum == 0.0f);
    const float inv = some ? __builtin_amdgcn_rcpf(sum) : 0.0f;  // sum is 2^(-1/16) or more
#pragma unroll
    for (int i = 0; i < U * 8; ++i) acc[i] = fmaf(LPR > 8 ? v[i] : exponential(v[i]), inv, acc[i]);
    if (mine && in_row == 0) {
      const float log2_sum = __builtin_amdgcn_logf(sum);
      a.lse[r] = !some ? kMinusInf : wide ? fmaf(log2_sum, kLn2, top) : (ref + log2_sum) * kLn2;
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
          a.weights[r * k + at] = is ? exponential(kept) * inv : 0.0f;
          if (is) atomicAdd(&hist[kept_column], 1u);
        }
      }
    } else {
      // Each lane ranks a candidate (of the row's first ones, by its first
      // waves): its place is the number of keys above its own.
      for (int from = LPR > 64 ? in_row - lane : 0; from < max(n, k); from += LPR) {
        const int at = from + lane;
        const uint64_t own_candidate = at < n ? list[at] : 0;
        const uint64_t key = key_of(own_candidate);
        int above = 0;
        if (LPR == 64 && n <= 64) {
          const uint32_t lo = static_cast<uint32_t>(key), hi = static_cast<uint32_t>(key >> 32);
          for (int j = 0; j < n; ++j) {
            const uint32_t other_hi = __builtin_amdgcn_readlane(hi, j), other_lo = __builtin_amdgcn_readlane(lo, j);
            above += ((static_cast<uint64_t>(other_hi) << 32) | other_lo) > key ? 1 : 0;
          }
        } else {
          for (int j = 0; j < n; ++j) above += key_of(list[j]) > key ? 1 : 0;
        }
        if (at < n && above < k) {
          const uint32_t column = static_cast<uint32_t>(own_candidate);
          a.ids[r * k + above] = column;
          a.weights[r * k + above] = exponential(__uint_as_float(static_cast<uint32_t>(own_candidate >> 32))) * inv;
          atomicAdd(&hist[column], 1u);
        }
        if (mine && at < k && at >= n) {
          a.ids[r * k + at] = -1;
          a.weights[r * k + at] = 0.0f;
        }
      }
      if constexpr (LPR == 64) wave_fence();
    }
  }

  // The workgroup's column sums, row group by row group; `each` takes every
  // column's.
  __syncthreads();
  auto over_columns = [&](auto each) {
    if constexpr (kRows == 1) {
#pragma unroll
      for (int i = 0; i < U * 8; ++i) {
        const int col = column_of<LPR>(in_row * 8, i);
        if (col < clusters) each(col, acc[i]);
      }
    } else {
      for (int e = tid; e < clusters; e += T) each(e, sums[e]);
    }
  };
  if constexpr (kRows > 1) {
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
        for (int u = 0; u < U; ++u) {
          const int col = column_of<LPR>(in_row * 8, u * 8);
          if (col >= clusters) continue;
          float* at = sums + col;  // whole units: there is room for eight past the last
          float old[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) old[i] = w == 0 ? 0.0f : at[i];
#pragma unroll
          for (int i = 0; i < 8; ++i) at[i] = old[i] + acc[u * 8 + i];
        }
      }
      __syncthreads();
    }
  }
  if (gridDim.x == 1) {
    const double scale = loss_scale(clusters, k, row_count);
    double loss = 0.0;
    over_columns([&](int e, float p) {
      const uint32_t n = hist[e];
      a.counts[e] = n;
      a.slopes[e] = static_cast<float>(scale * n);
      loss += scale * n * p;
    });
    loss = sum_workgroup<T>(loss, red);
    if (tid == 0) *a.loss = static_cast<float>(loss);
  } else {
    float* out = a.part_sums + static_cast<int64_t>(blockIdx.x) * clusters;
    uint32_t* counts = a.part_counts + static_cast<int64_t>(blockIdx.x) * clusters;
    over_columns([&](int e, float p) { out[e] = p; });
    for (int e = tid; e < clusters; e += T) counts[e] = hist[e];
    if (tid == 0) a.part_rows[blockIdx.x] = row_count;
  }
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

// Adds up the workgroups' parts: 16 clusters per workgroup, 64 slices of the
// parts each; the last workgroup to end adds up the loss.  Latency bounds it: 9
// us for 512 parts of 1,024 clusters (4 MB), 19 us for 256 of 5,000 (10 MB), 28
// us for 256 of 8,000 (16 MB), read in pieces of 64 bytes.
__global__ __launch_bounds__(kFinishThreads) void route_finish_kernel(FinishArgs a) {
  constexpr int kSlices = kFinishThreads / kFinishColumns;
  __shared__ double sums[kSlices][kFinishColumns];
  __shared__ uint32_t counts[kSlices][kFinishColumns];
  __shared__ double red[kFinishThreads / 64];
  __shared__ uint32_t all_rows;
  __shared__ bool last;
  const int tid = threadIdx.x, slice = tid / kFinishColumns, column = tid % kFinishColumns;
  const int e = blockIdx.x * kFinishColumns + column;
  double sum = 0.0;
  uint32_t count = 0, rows = 0;
  if (e < a.clusters) {
#pragma unroll 8
    for (int g = slice; g < a.groups; g += kSlices) {
      sum += a.part_sums[static_cast<int64_t>(g) * a.clusters + e];
      count += a.part_counts[static_cast<int64_t>(g) * a.clusters + e];
    }
  }
  for (int g = tid; g < a.groups; g += kFinishThreads) rows += a.part_rows[g];
  if (tid == 0) all_rows = 0;
  sums[slice][column] = sum;
  counts[slice][column] = count;
  __syncthreads();
  if (rows != 0) atomicAdd(&all_rows, rows);
  __syncthreads();
  const double scale = loss_scale(a.clusters, a.probes, all_rows);
  double part = 0.0;
  if (slice == 0 && e < a.clusters) {
    double p = 0.0;
    int64_t n = 0;
#pragma unroll 8
    for (int w = 0; w < kSlices; ++w) {
      p += sums[w][column];
      n += counts[w][column];
    }
    a.counts[e] = n;
    a.slopes[e] = static_cast<float>(scale * static_cast<double>(n));
    part = scale * static_cast<double>(n) * p;
  }
  if (tid < 64) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) part += __shfl_xor(part, o);
    if (tid == 0) {
      __hip_atomic_store(&a.part_loss[blockIdx.x], part, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __threadfence();
      last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
      __threadfence();
    }
  }
  __syncthreads();
  if (!last) return;
  double loss = 0.0;
  for (unsigned b = tid; b < gridDim.x; b += kFinishThreads)
    loss += __hip_atomic_load(&a.part_loss[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  loss = sum_workgroup<kFinishThreads>(loss, red);
  if (tid == 0) *a.loss = static_cast<float>(loss);
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
// own g_w; dot = sum of g_loss slope p over the row and of g_w p over the
// chosen.  A row's scores and what belongs to it are loaded while the one
// before is worked on; HBM bounds it: 65,536 x 1,024 bfloat16 59 us (4.6 TB/s),
// 16,001 x 5,000 float32 121 us (5.3 TB/s).
template <int DT, int LPR, int U>
__global__ __launch_bounds__(kThreads<LPR>) void route_backward_kernel(RouteBackwardArgs a) {
  constexpr int kRows = kThreads<LPR> / LPR;
  constexpr int kOwn = LPR < kMaxProbes ? kMaxProbes / LPR : 1;  // chosen clusters of a lane
  __shared__ float red_sum[2][kThreads<LPR> / 64];
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

  struct Row {
    Raw8<DT> raw[U];
    float top, sum, g_lse;
    int id[kOwn];
    float weight[kOwn], g[kOwn];
  };
  // Rows past the last are read as the last; -inf past the last column.
  auto load = [&](int64_t row, Row& x) {
    const int64_t r = min(row, a.rows - 1);
    const char* at = static_cast<const char*>(a.logits) + r * a.row_stride * kScoreBytes<DT>;
    int own = in_row * 8;
    asm volatile("" : "+v"(own));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int col = column_of<LPR>(own, u * 8);
      constexpr uint32_t kNone = DT == ST_SCORE_F32 ? 0xFF800000u : DT == ST_SCORE_F16 ? 0xFC00FC00u : 0xFF80FF80u;
      Raw8<DT> w;
#pragma unroll
      for (auto& e : w.w) e = u32x4{kNone, kNone, kNone, kNone};
      if (col + 8 <= clusters) {
        w = load_raw8<DT>(at, col);
      } else if (col < clusters) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (col + i >= clusters) continue;
          if constexpr (DT == ST_SCORE_F32) {
            w.w[i / 4][i % 4] = reinterpret_cast<const uint32_t*>(at)[col + i];
          } else {
            const uint32_t h = reinterpret_cast<const uint16_t*>(at)[col + i], old = w.w[0][i / 2];
            w.w[0][i / 2] = (i & 1) ? (old & 0xFFFFu) | (h << 16) : (old & 0xFFFF0000u) | h;
          }
        }
      }
      x.raw[u] = w;
    }
    x.top = a.stats[2 * r];
    x.sum = a.stats[2 * r + 1];
    x.g_lse = a.g_lse != nullptr ? a.g_lse[r] : 0.0f;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      const int i = in_row + LPR * j;
      const bool is = i < k;
      x.id[j] = is ? static_cast<int>(a.ids[r * k + i]) : -1;
      x.weight[j] = is ? a.weights[r * k + i] : 0.0f;
      x.g[j] = is && a.g_weights != nullptr ? a.g_weights[r * k + i] : 0.0f;
    }
  };

  const int64_t stride = static_cast<int64_t>(gridDim.x) * kRows;
  Row next;
  load(static_cast<int64_t>(blockIdx.x) * kRows + group, next);
  int turn = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < a.rows; base += stride, turn ^= 1) {
    const int64_t r = base + group;
    const bool mine = r < a.rows;
    float v[U * 8];
#pragma unroll
    for (int u = 0; u < U; ++u) unpack8<DT>(next.raw[u], v + u * 8);
    const float top = next.top, sum = next.sum, g_lse = next.g_lse;
    int id[kOwn];
    float weight[kOwn], own[kOwn], slope_there[kOwn];
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      id[j] = next.id[j];
      weight[j] = next.weight[j];
      own[j] = id[j] >= 0 ? next.g[j] : 0.0f;
      slope_there[j] = a.slopes[max(id[j], 0)];
    }
    load(r + stride, next);
    const bool some = !(top == kMinusInf && sum == 0.0f);
    const float m = top == kMinusInf ? 0.0f : top;
    // Exponentials are relative to m here, the sum is to the rounded m c: 2^rest
    // between them.  (Put back where the sum is stored, the forward kernel took
    // 129 us instead of 111 for 65,536 x 200 with 32 probes.)
    const float rest = is_wide(m) ? 0.0f : fmaf(m, kLog2e, -(m * kLog2e));
    const float inv = some ? __builtin_amdgcn_exp2f(rest) / sum : 0.0f;
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < U * 8; ++i) {
      v[i] = __builtin_amdgcn_exp2f((v[i] - m) * kLog2e);
      dot = fmaf(slope[i], v[i], dot);
    }
    dot *= inv;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) dot = fmaf(own[j], weight[j], dot);
    dot = row_sum<LPR>(dot, red_sum[turn]);
    const float shift = g_lse - dot;
    char* out = static_cast<char*>(a.grad) + r * clusters * kScoreBytes<DT>;
    if (mine) {
#pragma unroll
      for (int i = 0; i < U * 8; ++i) v[i] = some ? v[i] * inv * (slope[i] + shift) : 0.0f;
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
      if (mine) {
#pragma unroll
        for (int j = 0; j < kOwn; ++j)
          if (id[j] >= 0) store_score<DT>(out, id[j], weight[j] * (g_loss * slope_there[j] + shift + own[j]));
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
  if (clusters <= 1536) ST_SHAPE(64, 3);
  if (clusters <= 2048) ST_SHAPE(64, 4);
  if (clusters <= 4096) ST_SHAPE(256, 2);
  if (clusters <= 6144) ST_SHAPE(256, 3);
  if (clusters <= 8192) ST_SHAPE(256, 4);
  if (clusters <= 16384) ST_SHAPE(1024, 2);
  ST_SHAPE(1024, 4);
#undef ST_SHAPE
}

struct RouteShape {
  int rows;      // at once, in a workgroup
  int per_cu;    // workgroups
  size_t lds;
};

RouteShape route_shape(int64_t clusters) {
  RouteShape s{};
  for_shape(clusters, [&](auto lpr, auto units) {
    constexpr int T = kThreads<lpr()>;
    s.rows = T / lpr();
    s.per_cu = 1024 / T;
    s.lds = (lpr() > 64 ? s.rows * kRowList : T / 64 * kWaveList) * 8 + (clusters + 7) / 8 * 8 * 4 * (s.rows > 1 ? 2 : 1);
  });
  return s;
}

// One workgroup ends the work itself: for few rows that takes less than a
// second launch does.
int group_count(int64_t rows, int64_t clusters) {
  const RouteShape s = route_shape(clusters);
  if (rows <= 2 * s.rows) return 1;
  return static_cast<int>(std::min<int64_t>((rows + s.rows - 1) / s.rows, s.per_cu * cu_count()));
}

int64_t finish_groups(int64_t clusters) { return (clusters + kFinishColumns - 1) / kFinishColumns; }

template <int DT>
void launch_route(const RouteArgs& a, int groups, hipStream_t s) {
  for_shape(a.clusters, [&](auto lpr, auto units) {
    auto kernel = route_kernel<DT, lpr(), units()>;
    const size_t lds = route_shape(a.clusters).lds;
    if (lds > 48 * 1024) {
      static std::once_flag once;
      std::call_once(once, [&] {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, 140 * 1024);
        if (e != hipSuccess) throw Error(ST_ERR_HIP, cat("hipFuncSetAttribute failed: ", hipGetErrorString(e)));
      });
    }
    hipLaunchKernelGGL(kernel, dim3(groups), dim3(kThreads<lpr()>), lds, s, a);
    check_launch("route_kernel");
  });
}

template <int DT>
void launch_route_backward(const RouteBackwardArgs& a, hipStream_t s) {
  for_shape(a.clusters, [&](auto lpr, auto units) {
    const int64_t n = kThreads<lpr()> / lpr();
    const int64_t grid = std::min<int64_t>((a.rows + n - 1) / n, (lpr() > 64 ? 1 : 2) * cu_count());
    hipLaunchKernelGGL((route_backward_kernel<DT, lpr(), units()>), dim3(static_cast<unsigned>(grid)),
                       dim3(kThreads<lpr()>), 0, s, a);
    check_launch("route_backward_kernel");
  });
}

void check_route(int score_type, int64_t rows, int64_t clusters, int64_t row_stride, int64_t probes) {
  ST_CHECK(score_type == ST_SCORE_F32 || score_type == ST_SCORE_F16 || score_type == ST_SCORE_BF16,
           "scores must be float32, float16 or bfloat16");
  ST_CHECK(rows >= 0 && rows < (1ll << 31) && row_stride >= 0, "sizes must not be negative, rows below 2^31; got ", rows);
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
    a.counts = counts;
    a.slopes = slopes;
    a.loss = loss;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (score_type == ST_SCORE_F32)
      launch_route<ST_SCORE_F32>(a, groups, s);
    else if (score_type == ST_SCORE_F16)
      launch_route<ST_SCORE_F16>(a, groups, s);
    else
      launch_route<ST_SCORE_BF16>(a, groups, s);
    if (groups == 1) return;
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
    hipLaunchKernelGGL(route_finish_kernel, dim3(static_cast<unsigned>(finish_groups(clusters))),
                       dim3(kFinishThreads), 0, s, f);
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
