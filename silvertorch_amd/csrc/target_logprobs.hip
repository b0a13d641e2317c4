// Log-probabilities of given documents, with the distribution's entropy and
// its best alternatives, and their gradient.
//
// No reference operator.  For a row of scores z at temperature T, over the
// columns its filter lets pass (the packed search output: document d at bit
// 63 - d % 64 of word d / 64) and whose score is above -inf:
//   l = log sum_j e^(z_j / T),  log p_j = z_j / T - l
//   outputs: log p of the row's target, H = -sum_j p_j log p_j, l, and the k
//            columns of largest z (equal ones by column) with their log p.
//   dL/dz_j = 1/T [ g_t (d_jt - p_j) + sum_i g_i (d_{j,id_i} - p_j)
//                   - g_H p_j (log p_j + H) + g_l p_j ]
// Excluded columns are neither summed nor ranked, whatever they hold, and get
// a gradient of zero.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "score_ops.hpp"
#include "st_errors.hpp"

namespace st {
int cu_count();

namespace {

constexpr int kUnit = 8;              // columns a thread takes at once
constexpr int kMaxAlternatives = 128;
constexpr int kMaxChunks = 256;       // parts of a row
constexpr int kRoundUnits = 256;      // units examined for candidates at a time
constexpr int kCandidates = kRoundUnits * kUnit + 256;
constexpr int kJoinThreads = 256;
constexpr int kBackwardThreads = 256;
constexpr int kBackwardUnits = 4;     // units per thread
constexpr unsigned kMaxGrid = 1u << 22;

struct LogprobsArgs {
  const void* logits;
  int64_t rows, columns, row_stride;  // stride in elements
  const int64_t* targets;
  const uint64_t* mask;               // null: every column passes
  int64_t mask_stride;                // words; 0: one row for all
  int topk;
  float c, inv_t;                     // log2(e) / T, 1 / T
  int chunks;
  int64_t chunk_columns;              // a multiple of kUnit
  SoftStats* part_stats;              // [rows, chunks], with chunks > 1
  uint64_t* part_keys;                // [rows, chunks, topk], descending
  float *logprobs, *entropy, *lse, *top_logprobs;
  int64_t* top_ids;
  float* stats;                       // [rows, 2] or null: m and s, what the gradient needs
};

// Scores of an 8-column unit with the excluded ones at -inf: bit 7 - i of
// `pass` lets score i through.
__device__ __forceinline__ void exclude8(float v[8], uint32_t pass) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t keep = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(pass), 7 - i, 1));
    v[i] = __uint_as_float((__float_as_uint(v[i]) & keep) | (0xFF800000u & ~keep));
  }
}

// The filter's byte for columns [8 u, 8 u + 8): words are little-endian and
// documents go from the top bit down, so bytes run backwards within a word.
__device__ __forceinline__ uint32_t pass_byte(const uint64_t* mask, int64_t u) {
  return reinterpret_cast<const uint8_t*>(mask)[u ^ 7];
}

// Scores of the unit at `col`, of which `n` (1..8) exist.
template <int DT, bool MASKED>
__device__ __forceinline__ void load_unit(const void* row, const uint64_t* mask, int64_t col, int n, float v[8]) {
  if (n >= kUnit) {
    unpack8<DT>(load_raw8<DT>(row, col), v);
  } else {
#pragma unroll
    for (int i = 0; i < kUnit; ++i) v[i] = i < n ? load_score<DT>(row, col + i) : kMinusInf;
  }
  if constexpr (MASKED) exclude8(v, pass_byte(mask, col / kUnit));
}

// Adds a unit's scores to a thread's statistics; true when they hold a new
// maximum.
__device__ __forceinline__ bool take_unit(SoftStats& a, const float v[8], float c) {
  float top = fmaxf(fmaxf(v[0], v[1]), v[2]);
  top = fmaxf(fmaxf(top, v[3]), v[4]);
  top = fmaxf(fmaxf(top, v[5]), fmaxf(v[6], v[7]));
  const bool higher = top > a.m;
  if (higher) a = soft_rebase(a, top, c);
  const float m = a.m == kMinusInf ? 0.0f : a.m;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = v[i] - m;
    const float e = __builtin_amdgcn_exp2f(d * c);
    a.s += e;
    a.t = fmaf(e, fmaxf(d, -1e30f), a.t);  // an excluded score's d is -inf and its e 0
  }
  return higher;
}

struct SelectLds {
  uint64_t keys[kCandidates];
  uint64_t top[kMaxAlternatives];
  uint64_t threshold;
  uint32_t count, segments;
  uint16_t segment[1024];
};

// Writes the k largest of keys[0, n) to top, largest first and 0 past the
// last; every thread of the workgroup calls it.  A key's place is the number
// of keys above it.
template <int T>
__device__ __forceinline__ void rank_keys(SelectLds& l, uint32_t n, int k) {
  const int tid = threadIdx.x;
  if (tid < k) l.top[tid] = 0;
  if (tid == 0) l.keys[n] = 0;
  __syncthreads();
  for (uint32_t i = tid; i < n; i += T) {
    const uint64_t key = l.keys[i];
    uint32_t above = 0;
    for (uint32_t j = 0; j < n; j += 2) {
      above += l.keys[j] > key ? 1u : 0u;
      above += l.keys[j + 1] > key ? 1u : 0u;
    }
    if (above < static_cast<uint32_t>(k)) l.top[above] = key;
  }
  __syncthreads();
}

// After a round of pushes: when another round might not fit, keeps the best k
// so far and raises the threshold to the last of them.
template <int T>
__device__ __forceinline__ void make_room(SelectLds& l, int k) {
  const uint32_t n = l.count;
  __syncthreads();  // every thread has read the count before the next round's pushes
  if (n <= kCandidates - 1 - kRoundUnits * kUnit) return;
  rank_keys<T>(l, n, k);
  const int tid = threadIdx.x;
  if (tid < k) l.keys[tid] = l.top[tid];
  if (tid == 0) {
    l.count = k;  // more than k keys were there
    l.threshold = l.top[k - 1];
  }
  __syncthreads();
}

// The k best keys of the workgroup's units, to l.top.  Thread t has read units
// t, t + T, ... and knows its largest score and the first unit that holds it.
// The k-th largest of disjoint groups' maxima bounds the k-th best score from
// below, so only threads whose maximum reaches it hold candidates, and their
// units are read again: about k threads of T, whose scores are in the caches.
// Rounds of 256 units keep the candidates' list bounded whatever the scores.
template <int DT, bool MASKED, int T>
__device__ void select_top(SelectLds& l, const void* row, const uint64_t* mask, int64_t first, int64_t columns,
                           float top, uint32_t top_unit, int k) {
  const int tid = threadIdx.x;
  const uint32_t units = static_cast<uint32_t>((columns + kUnit - 1) / kUnit);
  // The lowest key that a score of this value has in this unit.
  const uint64_t mine =
      top > kMinusInf ? score_key(top, static_cast<uint32_t>(first) + top_unit * kUnit + (kUnit - 1)) : 0;
  // Twice as many groups as alternatives leave few candidates more than k.
  const int groups = k <= 32 ? 64 : 256;
  l.keys[tid] = mine;
  if (tid == 0) {
    l.threshold = 0;
    l.count = 0;
    l.segments = 0;
  }
  __syncthreads();
  uint64_t group = 0;
  if (tid < groups)
    for (int j = tid; j < T; j += groups) group = l.keys[j] > group ? l.keys[j] : group;
  __syncthreads();
  if (tid < groups) l.keys[tid] = group;
  __syncthreads();
  if (tid < groups && group != 0) {
    int above = 0;
    for (int j = 0; j < groups; j += 2) {
      above += l.keys[j] > group ? 1 : 0;
      above += l.keys[j + 1] > group ? 1 : 0;
    }
    if (above == k - 1) l.threshold = group;
  }
  __syncthreads();
  const uint64_t bound = l.threshold;
  if (mine != 0 && mine >= bound) l.segment[atomicAdd(&l.segments, 1u)] = static_cast<uint16_t>(tid);
  __syncthreads();
  const uint32_t per = (units + T - 1) / T;
  const uint32_t pairs = l.segments * per;
  for (uint32_t base = 0; base < pairs; base += kRoundUnits) {
    const uint32_t p = base + tid;
    if (tid < kRoundUnits && p < pairs) {
      const uint32_t u = l.segment[p / per] + T * (p % per);
      if (u < units) {
        const int64_t col = first + static_cast<int64_t>(u) * kUnit;
        const int64_t left = first + columns - col;
        float v[8];
        load_unit<DT, MASKED>(row, mask, col, left < kUnit ? static_cast<int>(left) : kUnit, v);
        const uint64_t least = l.threshold;
#pragma unroll
        for (int i = 0; i < kUnit; ++i) {
          const uint64_t key = score_key(v[i], static_cast<uint32_t>(col) + i);
          if (v[i] > kMinusInf && key >= least) l.keys[atomicAdd(&l.count, 1u)] = key;
        }
      }
    }
    __syncthreads();
    make_room<T>(l, k);
  }
  rank_keys<T>(l, l.count, k);
}

// The row's outputs from its statistics, by one thread.
template <int DT>
__device__ void finish_row(const LogprobsArgs& a, int64_t row, const SoftStats& st) {
  const bool none = st.m == kMinusInf && st.s == 0.0f;
  const float log_s = logf(st.s);
  a.lse[row] = none ? kMinusInf : fmaf(st.m, a.inv_t, log_s);
  const float h = log_s - st.t / st.s * a.inv_t;
  a.entropy[row] = none || h < 0.0f ? 0.0f : h;  // NaN stays
  if (a.stats != nullptr) {
    a.stats[2 * row] = st.m;
    a.stats[2 * row + 1] = st.s;
  }
  const int64_t target = a.targets[row];
  float lp = kMinusInf;
  if (target == -1) {
    lp = 0.0f;
  } else if (!none && target >= 0 && target < a.columns) {
    const bool pass =
        a.mask == nullptr || ((a.mask[row * a.mask_stride + (target >> 6)] >> (63 - (target & 63))) & 1) != 0;
    const float z = load_score<DT>(static_cast<const char*>(a.logits) + row * a.row_stride * kScoreBytes<DT>, target);
    if (pass && z != kMinusInf) lp = fmaf(z - st.m, a.inv_t, -log_s);
  }
  a.logprobs[row] = lp;
}

// Alternative i of the row from its key, by one thread each.
__device__ __forceinline__ void finish_alternative(const LogprobsArgs& a, int64_t row, int i, uint64_t key,
                                                   const SoftStats& st) {
  const int64_t at = row * a.topk + i;
  a.top_ids[at] = key == 0 ? -1 : static_cast<int64_t>(~static_cast<uint32_t>(key));
  a.top_logprobs[at] =
      key == 0 ? kMinusInf : fmaf(score_from_ordered(static_cast<uint32_t>(key >> 32)) - st.m, a.inv_t, -logf(st.s));
}

// The workgroup's statistics, in every thread.
template <int T>
__device__ __forceinline__ SoftStats join_workgroup(SoftStats st, float c) {
  __shared__ SoftStats waves[T / 64];
  st = soft_wave_join<64>(st, c);
  if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = st;
  __syncthreads();
  st = waves[0];
#pragma unroll
  for (int w = 1; w < T / 64; ++w) st = soft_join(st, waves[w], c);
  __syncthreads();
  return st;
}

// One workgroup per row, or per part of a row.
template <int DT, bool MASKED, int T>
__global__ __launch_bounds__(T, 8) void logprobs_kernel(LogprobsArgs a) {
  extern __shared__ __align__(16) uint8_t lds_raw[];
  SelectLds& l = *reinterpret_cast<SelectLds*>(lds_raw);
  const int tid = threadIdx.x;
  const int64_t items = a.rows * a.chunks;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t r = item / a.chunks;
    const int64_t first = (item - r * a.chunks) * a.chunk_columns;
    const int64_t columns = min(a.chunk_columns, a.columns - first);
    const char* row = static_cast<const char*>(a.logits) + r * a.row_stride * kScoreBytes<DT>;
    const uint64_t* mask = MASKED ? a.mask + r * a.mask_stride : nullptr;
    const uint32_t full = static_cast<uint32_t>(columns / kUnit);
    SoftStats st = soft_none();
    uint32_t top_unit = 0;
    constexpr int kAhead = DT == ST_SCORE_F32 ? 2 : 4;  // 64 bytes a thread in flight
    uint32_t u = tid;
    for (; u + (kAhead - 1) * T < full; u += kAhead * T) {
      Raw8<DT> raw[kAhead];
      uint32_t pass[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int64_t col = first + static_cast<int64_t>(u + i * T) * kUnit;
        raw[i] = load_raw8<DT>(row, col);
        if constexpr (MASKED) pass[i] = pass_byte(mask, col / kUnit);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        float v[8];
        unpack8<DT>(raw[i], v);
        if constexpr (MASKED) exclude8(v, pass[i]);
        if (take_unit(st, v, a.c)) top_unit = u + i * T;
      }
    }
    const uint32_t units = static_cast<uint32_t>((columns + kUnit - 1) / kUnit);
    for (; u < units; u += T) {
      const int64_t col = first + static_cast<int64_t>(u) * kUnit;
      float v[8];
      load_unit<DT, MASKED>(row, mask, col, u < full ? kUnit : static_cast<int>(columns % kUnit), v);
      if (take_unit(st, v, a.c)) top_unit = u;
    }
    if (a.topk > 0)
      select_top<DT, MASKED, T>(l, row, mask, first, columns, st.m, top_unit, a.topk);
    st = join_workgroup<T>(st, a.c);
    if (a.chunks > 1) {
      if (tid == 0) a.part_stats[item] = st;
      if (tid < a.topk) a.part_keys[item * a.topk + tid] = l.top[tid];
    } else {
      if (tid == 0) finish_row<DT>(a, r, st);
      if (tid < a.topk) finish_alternative(a, r, tid, l.top[tid], st);
    }
    __syncthreads();
  }
}

// Joins a row's parts: one workgroup per row.  The parts' lists are in order,
// so their j-th entries bound the k-th best key from below: with j = ceil(2k /
// parts), ceil(k / j) lists have at least k keys at or above the
// ceil(k / j)-th largest of them.
template <int DT>
__global__ __launch_bounds__(kJoinThreads) void logprobs_join_kernel(LogprobsArgs a) {
  extern __shared__ __align__(16) uint8_t lds_raw[];
  SelectLds& l = *reinterpret_cast<SelectLds*>(lds_raw);
  const int tid = threadIdx.x;
  const int k = a.topk;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const uint64_t* lists = a.part_keys + r * a.chunks * k;
    if (k > 0) {
      const int depth = min(k, (2 * k + a.chunks - 1) / a.chunks);
      const int need = (k + depth - 1) / depth;  // <= chunks
      uint64_t mine = tid < a.chunks ? lists[static_cast<int64_t>(tid) * k + depth - 1] : 0;
      l.keys[tid] = mine;
      if (tid == 0) {
        l.threshold = 0;
        l.count = 0;
      }
      __syncthreads();
      if (mine != 0) {
        int above = 0;
        for (int j = 0; j < a.chunks; ++j) above += l.keys[j] > mine ? 1 : 0;
        if (above == need - 1) l.threshold = mine;
      }
      __syncthreads();
      const int64_t entries = static_cast<int64_t>(a.chunks) * k;
      for (int64_t base = 0; base < entries; base += kRoundUnits * kUnit) {
        const uint64_t least = l.threshold;
#pragma unroll
        for (int i = 0; i < kRoundUnits * kUnit / kJoinThreads; ++i) {
          const int64_t e = base + i * kJoinThreads + tid;
          const uint64_t key = e < entries ? lists[e] : 0;
          if (key != 0 && key >= least) l.keys[atomicAdd(&l.count, 1u)] = key;
        }
        __syncthreads();
        make_room<kJoinThreads>(l, k);
      }
      rank_keys<kJoinThreads>(l, l.count, k);
    }
    SoftStats st = tid < a.chunks ? a.part_stats[r * a.chunks + tid] : soft_none();
    st = join_workgroup<kJoinThreads>(st, a.c);
    if (tid == 0) finish_row<DT>(a, r, st);
    if (tid < k) finish_alternative(a, r, tid, l.top[tid], st);
    __syncthreads();
  }
}

struct BackwardArgs {
  const void* logits;
  int64_t rows, columns, row_stride;
  const int64_t* targets;
  const uint64_t* mask;
  int64_t mask_stride;
  int topk;
  float c, inv_t;
  const float* stats;
  const int64_t* top_ids;
  const float *g_logprobs, *g_entropy, *g_lse, *g_top;  // each may be null: zero
  void* grad;                                           // [rows, columns], contiguous
  int64_t chunks;                                       // parts of a row
};

__device__ __forceinline__ bool passes(const BackwardArgs& a, int64_t row, int64_t col) {
  return a.mask == nullptr || ((a.mask[row * a.mask_stride + (col >> 6)] >> (63 - (col & 63))) & 1) != 0;
}

// With e = e^((z-m)/T), p = e/s and log p + H = (z-m)/T + (H - log s):
// dL/dz = e (k0 + k1 (z-m)) outside the target and the alternatives.
template <int DT, bool MASKED>
__global__ __launch_bounds__(kBackwardThreads, 8) void logprobs_backward_kernel(BackwardArgs a, const float* entropy) {
  constexpr int kColumns = kBackwardThreads * kBackwardUnits * kUnit;
  const int tid = threadIdx.x;
  const int64_t items = a.rows * a.chunks;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t r = item / a.chunks;
    const int64_t first = (item - r * a.chunks) * kColumns;
    const int64_t end = min(first + kColumns, a.columns);
    const char* row = static_cast<const char*>(a.logits) + r * a.row_stride * kScoreBytes<DT>;
    char* out = static_cast<char*>(a.grad) + r * a.columns * kScoreBytes<DT>;
    const uint64_t* mask = MASKED ? a.mask + r * a.mask_stride : nullptr;

    // the row's factors (uniform over the workgroup)
    const float m = a.stats[2 * r], s = a.stats[2 * r + 1];
    const bool none = m == kMinusInf && s == 0.0f;
    const int64_t target = a.targets[r];
    float g_target = 0.0f;
    if (a.g_logprobs != nullptr && target >= 0 && target < a.columns && passes(a, r, target) &&
        load_score<DT>(row, target) != kMinusInf)
      g_target = a.g_logprobs[r];
    float whole = g_target;
    if (a.g_top != nullptr)
      for (int i = 0; i < a.topk; ++i)
        if (a.top_ids[r * a.topk + i] >= 0) whole += a.g_top[r * a.topk + i];
    if (a.g_lse != nullptr) whole -= a.g_lse[r];
    const float inv_s = 1.0f / s;
    float k0 = -whole, k1 = 0.0f;
    if (a.g_entropy != nullptr) {
      const float g = a.g_entropy[r];
      k0 -= g * (entropy[r] - logf(s));
      k1 = -g * a.inv_t;
    }
    // e is taken 2^24 times as large, so that none is flushed to zero whose
    // product with large factors (1 / T among them) is in the type's range
    k0 *= inv_s * a.inv_t * 0x1p-24f;
    k1 *= inv_s * a.inv_t * 0x1p-24f;
    if (none) k0 = k1 = 0.0f;
    const float low = none ? 0.0f : m;
    auto slope = [&](float z) {
      const float d = fmaxf(z - low, -1e18f);  // -inf: e is 0
      return __builtin_amdgcn_exp2f(fmaf(d, a.c, 24.0f)) * fmaf(d, k1, k0);
    };

    const int64_t units = (end - first + kUnit - 1) / kUnit;
    if (units == kBackwardThreads * kBackwardUnits && end - first == kColumns) {
      Raw8<DT> raw[kBackwardUnits];
      uint32_t pass[kBackwardUnits];
#pragma unroll
      for (int i = 0; i < kBackwardUnits; ++i) {
        const int64_t col = first + static_cast<int64_t>(i * kBackwardThreads + tid) * kUnit;
        raw[i] = load_raw8<DT>(row, col);
        if constexpr (MASKED) pass[i] = pass_byte(mask, col / kUnit);
      }
#pragma unroll
      for (int i = 0; i < kBackwardUnits; ++i) {
        const int64_t col = first + static_cast<int64_t>(i * kBackwardThreads + tid) * kUnit;
        float v[8];
        unpack8<DT>(raw[i], v);
#pragma unroll
        for (int j = 0; j < kUnit; ++j) {
          v[j] = slope(v[j]);
          if constexpr (MASKED) v[j] = (pass[i] >> (7 - j)) & 1 ? v[j] : 0.0f;
        }
        store8<DT>(out, col, v);
      }
    } else {
      for (int64_t u = tid; u < units; u += kBackwardThreads) {
        const int64_t col = first + u * kUnit;
        const int n = static_cast<int>(min(static_cast<int64_t>(kUnit), end - col));
        const uint32_t pass = MASKED ? pass_byte(mask, col / kUnit) : 0xFFu;
        if (n == kUnit) {
          float v[8];
          unpack8<DT>(load_raw8<DT>(row, col), v);
#pragma unroll
          for (int j = 0; j < kUnit; ++j) v[j] = (pass >> (7 - j)) & 1 ? slope(v[j]) : 0.0f;
          store8<DT>(out, col, v);
        } else {
          for (int j = 0; j < n; ++j)
            store_score<DT>(out, col + j, (pass >> (7 - j)) & 1 ? slope(load_score<DT>(row, col + j)) : 0.0f);
        }
      }
    }

    // The target's and the alternatives' own terms: their elements are written
    // again, whole, by one thread each (ids are distinct; a target among the
    // alternatives is theirs).
    __syncthreads();
    if (!none) {
      for (int i = tid; i < a.topk; i += kBackwardThreads) {
        const int64_t id = a.top_ids[r * a.topk + i];
        if (id < first || id >= end) continue;
        const float g = (a.g_top != nullptr ? a.g_top[r * a.topk + i] : 0.0f) + (id == target ? g_target : 0.0f);
        store_score<DT>(out, id, fmaf(g, a.inv_t, slope(load_score<DT>(row, id))));
      }
      if (tid == kBackwardThreads - 1 && g_target != 0.0f && target >= first && target < end) {
        bool listed = false;
        for (int i = 0; i < a.topk; ++i) listed |= a.top_ids[r * a.topk + i] == target;
        if (!listed) store_score<DT>(out, target, fmaf(g_target, a.inv_t, slope(load_score<DT>(row, target))));
      }
    }
    __syncthreads();
  }
}

void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw Error(ST_ERR_HIP, cat(what, " launch failed: ", hipGetErrorString(e)));
}

// Parts of a row: enough workgroups of 1,024 threads for two on every CU, each
// with at least 8,192 columns (a unit per thread).
int row_chunks(int64_t rows, int64_t columns) {
  const int64_t want = (2 * cu_count() + rows - 1) / std::max<int64_t>(rows, 1);
  const int64_t most = (columns + 8191) / 8192;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, most, kMaxChunks})));
}

// Workgroups of 256 threads, eight on a CU, once rows fill them.
bool small_groups(int64_t rows) { return rows >= 8 * cu_count(); }

unsigned grid_of(int64_t items) { return static_cast<unsigned>(std::min<int64_t>(items, kMaxGrid)); }

template <int DT, bool MASKED>
void launch_forward(const LogprobsArgs& a, hipStream_t s) {
  const size_t lds = a.topk > 0 ? sizeof(SelectLds) : 0;
  const unsigned grid = grid_of(a.rows * a.chunks);
  if (a.chunks == 1 && small_groups(a.rows))
    hipLaunchKernelGGL((logprobs_kernel<DT, MASKED, 256>), dim3(grid), dim3(256), lds, s, a);
  else
    hipLaunchKernelGGL((logprobs_kernel<DT, MASKED, 1024>), dim3(grid), dim3(1024), lds, s, a);
  check_launch("logprobs_kernel");
  if (a.chunks > 1) {
    hipLaunchKernelGGL((logprobs_join_kernel<DT>), dim3(grid_of(a.rows)), dim3(kJoinThreads), lds, s, a);
    check_launch("logprobs_join_kernel");
  }
}

template <int DT>
void launch_backward(const BackwardArgs& a, const float* entropy, hipStream_t s) {
  const unsigned grid = grid_of(a.rows * a.chunks);
  if (a.mask != nullptr)
    hipLaunchKernelGGL((logprobs_backward_kernel<DT, true>), dim3(grid), dim3(kBackwardThreads), 0, s, a, entropy);
  else
    hipLaunchKernelGGL((logprobs_backward_kernel<DT, false>), dim3(grid), dim3(kBackwardThreads), 0, s, a, entropy);
  check_launch("logprobs_backward_kernel");
}

void check_logprobs(const void* logits, int dtype, int64_t rows, int64_t columns, int64_t row_stride,
                    const int64_t* targets, const int64_t* mask, int64_t mask_stride, int64_t mask_words, int64_t topk,
                    double temperature) {
  ST_CHECK(dtype == ST_SCORE_F32 || dtype == ST_SCORE_F16 || dtype == ST_SCORE_BF16,
           "scores must be float32, float16 or bfloat16");
  ST_CHECK(rows >= 0 && columns >= 0 && columns < (1ll << 31), "rows and columns must not be negative, columns below 2^31; got ",
           rows, " x ", columns);
  ST_CHECK(row_stride >= 0 && mask_stride >= 0, "negative strides");
  ST_CHECK(topk >= 0 && topk <= kMaxAlternatives, "topk must be in [0, ", kMaxAlternatives, "], got ", topk);
  ST_CHECK(std::isfinite(temperature) && temperature >= 1e-6 && temperature <= 1e6,
           "temperature must be in [1e-6, 1e6], got ", temperature);
  ST_CHECK(mask == nullptr || mask_words * 64 >= columns, "the mask's ", mask_words, " words a row hold fewer than ",
           columns, " documents");
  if (rows == 0) return;
  ST_CHECK(targets != nullptr && (columns == 0 || logits != nullptr), "null device pointer");
}

}  // namespace
}  // namespace st

extern "C" int64_t st_target_logprobs_workspace_bytes(int64_t rows, int64_t columns, int64_t topk) {
  using namespace st;
  if (rows <= 0 || columns <= 0 || topk < 0 || topk > kMaxAlternatives) return 0;
  const int64_t chunks = row_chunks(rows, columns);
  if (chunks == 1) return 0;
  return rows * chunks * (static_cast<int64_t>(sizeof(SoftStats)) + 8 * topk) + 16;
}

extern "C" int st_target_logprobs(const void* logits, int score_type, int64_t rows, int64_t columns,
                                  int64_t row_stride, const int64_t* targets, const int64_t* mask,
                                  int64_t mask_stride, int64_t mask_words, int64_t topk, double temperature,
                                  void* workspace, float* logprobs, float* entropy, float* lse, int64_t* top_ids,
                                  float* top_logprobs, float* stats, void* stream) {
  using namespace st;
  return guarded([&] {
    check_logprobs(logits, score_type, rows, columns, row_stride, targets, mask, mask_stride, mask_words, topk,
                   temperature);
    if (rows == 0) return;
    ST_CHECK(logprobs && entropy && lse && (topk == 0 || (top_ids && top_logprobs)), "null device pointer");
    LogprobsArgs a{};
    a.logits = logits;
    a.rows = rows;
    a.columns = columns;
    a.row_stride = row_stride;
    a.targets = targets;
    a.mask = reinterpret_cast<const uint64_t*>(mask);
    a.mask_stride = mask_stride;
    a.topk = static_cast<int>(topk);
    a.c = static_cast<float>(1.4426950408889634 / temperature);
    a.inv_t = static_cast<float>(1.0 / temperature);
    a.chunks = row_chunks(rows, columns);
    a.chunk_columns = ((columns + a.chunks - 1) / a.chunks + kUnit - 1) / kUnit * kUnit;
    if (a.chunks > 1) {
      ST_CHECK(workspace != nullptr, "null workspace");
      a.part_keys = static_cast<uint64_t*>(workspace);
      a.part_stats = reinterpret_cast<SoftStats*>(a.part_keys + rows * a.chunks * topk);
    }
    a.logprobs = logprobs;
    a.entropy = entropy;
    a.lse = lse;
    a.top_ids = top_ids;
    a.top_logprobs = top_logprobs;
    a.stats = stats;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool masked = mask != nullptr;
    if (score_type == ST_SCORE_F32)
      masked ? launch_forward<ST_SCORE_F32, true>(a, s) : launch_forward<ST_SCORE_F32, false>(a, s);
    else if (score_type == ST_SCORE_F16)
      masked ? launch_forward<ST_SCORE_F16, true>(a, s) : launch_forward<ST_SCORE_F16, false>(a, s);
    else
      masked ? launch_forward<ST_SCORE_BF16, true>(a, s) : launch_forward<ST_SCORE_BF16, false>(a, s);
  });
}

extern "C" int st_target_logprobs_backward(const void* logits, int score_type, int64_t rows, int64_t columns,
                                           int64_t row_stride, const int64_t* targets, const int64_t* mask,
                                           int64_t mask_stride, int64_t mask_words, int64_t topk, double temperature,
                                           const float* entropy, const float* stats, const int64_t* top_ids,
                                           const float* grad_logprobs, const float* grad_entropy,
                                           const float* grad_lse, const float* grad_top_logprobs, void* grad_logits,
                                           void* stream) {
  using namespace st;
  return guarded([&] {
    check_logprobs(logits, score_type, rows, columns, row_stride, targets, mask, mask_stride, mask_words, topk,
                   temperature);
    if (rows == 0 || columns == 0) return;
    ST_CHECK(entropy && stats && grad_logits && (topk == 0 || top_ids), "null device pointer");
    BackwardArgs a{};
    a.logits = logits;
    a.rows = rows;
    a.columns = columns;
    a.row_stride = row_stride;
    a.targets = targets;
    a.mask = reinterpret_cast<const uint64_t*>(mask);
    a.mask_stride = mask_stride;
    a.topk = static_cast<int>(topk);
    a.c = static_cast<float>(1.4426950408889634 / temperature);
    a.inv_t = static_cast<float>(1.0 / temperature);
    a.stats = stats;
    a.top_ids = top_ids;
    a.g_logprobs = grad_logprobs;
    a.g_entropy = grad_entropy;
    a.g_lse = grad_lse;
    a.g_top = topk > 0 ? grad_top_logprobs : nullptr;
    a.grad = grad_logits;
    constexpr int64_t kColumns = kBackwardThreads * kBackwardUnits * kUnit;
    a.chunks = (columns + kColumns - 1) / kColumns;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (score_type == ST_SCORE_F32)
      launch_backward<ST_SCORE_F32>(a, entropy, s);
    else if (score_type == ST_SCORE_F16)
      launch_backward<ST_SCORE_F16>(a, entropy, s);
    else
      launch_backward<ST_SCORE_BF16>(a, entropy, s);
  });
}
