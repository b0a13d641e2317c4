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
#include <type_traits>

#include "score_ops.hpp"
#include "st_errors.hpp"

namespace st {
int cu_count();

namespace {

constexpr int kUnit = 8;              // columns a thread takes at once
constexpr int kMaxAlternatives = 128;
constexpr int kMaxChunks = 256;       // parts of a row
constexpr int kRoundUnits = 256;      // units examined for candidates at a time
constexpr int kCandidates = kRoundUnits * kUnit + 192;
constexpr int kJoinThreads = 512;
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
  float limit;                        // fast_limit(c)
  int chunks;
  int64_t chunk_columns;              // a multiple of kUnit
  SoftStats* part_stats;              // [rows, chunks], with chunks > 1
  uint64_t* part_keys;                // [rows, chunks, topk], descending
  float *logprobs, *entropy, *lse, *top_logprobs;
  int64_t* top_ids;
  float* stats;                       // [rows, 2] or null: m and s, what the gradient needs
};

// Scores of an 8-column unit with the excluded ones at `fill`: bit 7 - i of
// `pass` lets score i through.
__device__ __forceinline__ void exclude8(float v[8], uint32_t pass, float fill) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t keep = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(pass), 7 - i, 1));
    v[i] = __uint_as_float((__float_as_uint(v[i]) & keep) | (__float_as_uint(fill) & ~keep));
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
  if constexpr (MASKED) exclude8(v, pass_byte(mask, col / kUnit), kMinusInf);
}

// A thread's running statistics.  In the loop they are kept relative to k =
// round(m c) instead of m c: then e^((z-m)/T) is 2^(z c - k), one multiply-add
// and the exponential, and t adds up e (z c - k).  What the rounding of k moved
// is put back once at the end (rest = m c - k is exact).  rest is half an ulp
// of m c at most, and past 2^31 2^rest may not be a finite number: maxima
// outside (-limit, limit], where rest is 64 at most, are kept relative to m
// itself.  A rest that large costs no accuracy: the scores' own spacing is more
// than it, so that only those equal to m count.  (Limits as low as 2^26 took a
// second look at units with scores of -1e9: 2,000 x 30,000 bfloat16, half of
// them so, 27.2 against 24.8 us.)
struct Running {
  SoftStats a;      // a.m: the maximum itself, -inf before any
  float least, k;   // max(m, -limit) and its k
};

float fast_limit(float c) { return 0x1.Fp30f / c; }

__device__ __forceinline__ bool is_fast(float m, float limit) { return m > -limit && m <= limit; }

__device__ __forceinline__ Running running_none(float c, float limit) { return {soft_none(), -limit, -limit * c}; }

// To the reference m (t in units of z) and back.
__device__ __forceinline__ SoftStats settled(const Running& r, float c, float limit) {
  if (!is_fast(r.a.m, limit)) return r.a;
  const float rest = fmaf(r.a.m, c, -r.k);
  const float back = __builtin_amdgcn_exp2f(-rest);
  return {r.a.m, r.a.s * back, (r.a.t - rest * r.a.s) * back / c};
}

__device__ __forceinline__ Running running_of(const SoftStats& a, float c, float limit) {
  Running r{a, fmaxf(a.m, -limit), 0.0f};
  r.k = r.least * c;
  if (is_fast(a.m, limit)) {
    const float rest = fmaf(a.m, c, -r.k), on = __builtin_amdgcn_exp2f(rest);
    r.a.s = a.s * on;
    r.a.t = (a.t * c + rest * a.s) * on;
  }
  return r;
}

// Adds eight scores of any size, -inf for none, to statistics relative to m.
__device__ __forceinline__ SoftStats take_any(SoftStats a, const float v[8], float top, float c) {
  if (top > a.m) a = soft_rebase(a, top, c);
  const float m = a.m == kMinusInf ? 0.0f : a.m;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = v[i] - m;
    const float e = __builtin_amdgcn_exp2f(d * c);
    a.s += e;
    a.t = fmaf(e, fmaxf(d, -1e30f), a.t);  // -inf: e is 0
  }
  return a;
}

__device__ __forceinline__ float max8(const float v[8]) {
  const float a = fmaxf(fmaxf(v[0], v[1]), v[2]), b = fmaxf(fmaxf(v[3], v[4]), v[5]);
  return fmaxf(fmaxf(a, b), fmaxf(v[6], v[7]));
}

__device__ __forceinline__ float min8(const float v[8]) {
  const float a = fminf(fminf(v[0], v[1]), v[2]), b = fminf(fminf(v[3], v[4]), v[5]);
  return fminf(fminf(a, b), fminf(v[6], v[7]));
}

// Adds a unit's scores, those that `pass` excludes (MASKED) left out, to a
// thread's statistics; true when they hold a new maximum.
template <bool MASKED>
__device__ __forceinline__ bool take_unit(Running& r, float v[8], uint32_t pass, float c, float limit) {
  const float fill = -2.0f * limit;  // stands in an excluded column: 2^(fill c - k) is 0
  const float low = min8(v);
  if constexpr (MASKED) exclude8(v, pass, fill);
  float top = max8(v);
  if (__any(!(low > -limit) || fmaxf(top, r.least) > limit)) {
    if constexpr (MASKED) {
      exclude8(v, pass, kMinusInf);
      top = max8(v);
    }
    // Maxima that are not ordinary take the general way; -inf and very low
    // scores beside ordinary ones count as excluded ones do (their e is 0).
    const bool general = fmaxf(top, r.a.m) > limit || (top > kMinusInf && top <= -limit && !(r.a.m > -limit));
    if (__any(general)) {
      const float before = r.a.m;
      r = running_of(take_any(settled(r, c, limit), v, top, c), c, limit);
      return r.a.m > before;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] < fill ? fill : v[i];
  }
  const bool higher = top > r.least;
  if (higher) {
    if (r.a.m > -limit) {
      const float k = top * c;
      const float d = r.k - k, scale = __builtin_amdgcn_exp2f(d);
      r.a.t = scale == 0.0f ? 0.0f : (r.a.t + r.a.s * d) * scale;
      r.a.s *= scale;
      r.a.m = r.least = top;
      r.k = k;
    } else {  // nothing yet, or lower maxima, kept relative to themselves
      r = running_of(soft_rebase(r.a, top, c), c, limit);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = fmaf(v[i], c, -r.k);
    const float e = __builtin_amdgcn_exp2f(d);
    r.a.s += e;
    r.a.t = fmaf(e, d, r.a.t);
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

// Writes the k largest of keys[0, n) to top (zeroed before); every thread of
// the workgroup calls it, after a barrier that follows the last key.  A key's
// place is the number of keys above it, counted by four lanes.
template <int T>
__device__ __forceinline__ void rank_keys(SelectLds& l, uint32_t n, int k) {
  const uint32_t part = threadIdx.x % 4;
  for (uint32_t i = threadIdx.x / 4; i < n; i += T / 4) {
    const uint64_t key = l.keys[i];
    int above = 0;
#pragma unroll 8
    for (uint32_t j = part; j < n; j += 4) above += l.keys[j] > key ? 1 : 0;
    above += __builtin_amdgcn_update_dpp(0, above, 0xB1, 0xF, 0xF, false);  // the quad's sum
    above += __builtin_amdgcn_update_dpp(0, above, 0x4E, 0xF, 0xF, false);
    if (part == 0 && above < k) l.top[above] = key;
  }
  __syncthreads();
}

// A bound that exactly k of the wave's 64 N distinct keys reach (0 if fewer
// are above 0), found bit by bit from the top: first the scores' half, then,
// where more scores are equal than may count, the columns'.
template <int N>
__device__ __forceinline__ uint64_t wave_kth(const uint64_t key[N], int k) {
  auto search = [&](auto part, int want, auto takes_part) {
    uint32_t bound = 0;
    for (int b = 31; b >= 0; --b) {
      const uint32_t t = bound | (1u << b);
      int n = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) n += __popcll(__ballot(takes_part(i) && part(i) >= t));
      if (n >= want) bound = t;
      if (n == want) break;
    }
    return bound;
  };
  const uint32_t high = search([&](int i) { return static_cast<uint32_t>(key[i] >> 32); }, k, [](int) { return true; });
  int above = 0, reach = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t h = static_cast<uint32_t>(key[i] >> 32);
    above += __popcll(__ballot(h > high));
    reach += __popcll(__ballot(h >= high));
  }
  uint32_t low = 0;
  if (reach > k && high != 0)
    low = search([&](int i) { return static_cast<uint32_t>(key[i]); }, k - above,
                 [&](int i) { return static_cast<uint32_t>(key[i] >> 32) == high; });
  return (static_cast<uint64_t>(high) << 32) | low;
}

__device__ __forceinline__ void push_key(SelectLds& l, uint64_t key) {
  const uint32_t at = atomicAdd(&l.count, 1u);
  if (at < kCandidates) l.keys[at] = key;
}

// After a round of pushes: when another round might not fit, keeps the best k
// so far and raises the threshold to the last of them.
template <int T>
__device__ __forceinline__ void make_room(SelectLds& l, int k) {
  const uint32_t n = l.count;
  __syncthreads();  // every thread has read the count before the next round's pushes
  if (n <= kCandidates - kRoundUnits * kUnit) return;
  rank_keys<T>(l, n, k);
  const int tid = threadIdx.x;
  if (tid < k) {  // more than k keys were there
    const uint64_t key = l.top[tid];
    l.keys[tid] = key;
    l.top[tid] = 0;
    if (tid == k - 1) l.threshold = key;
  }
  if (tid == 0) l.count = k;
  __syncthreads();
}

// The k best keys of the workgroup's units, to l.top.  Thread t has read units
// t, t + T, ... and knows its largest score and the first unit that holds it.
// The k-th largest of disjoint groups' maxima bounds the k-th best score from
// below, so only threads whose maximum reaches it hold candidates, and their
// units are read again: few more than k threads of T, whose scores are in the
// caches.  That is done in one go; should more scores reach the bound than
// there is room for, again in rounds of 256 units that keep the best k so far.
// `ready` runs before the first barrier.
template <int DT, bool MASKED, int T, typename F>
__device__ void select_top(SelectLds& l, const void* row, const uint64_t* mask, int64_t first, int64_t columns,
                           float top, uint32_t top_unit, int k, F ready) {
  const int tid = threadIdx.x;
  const uint32_t units = static_cast<uint32_t>((columns + kUnit - 1) / kUnit);
  // The lowest key that a score of this value has in this unit.
  const uint64_t mine =
      top > kMinusInf ? score_key(top, static_cast<uint32_t>(first) + top_unit * kUnit + (kUnit - 1)) : 0;
  l.keys[tid] = mine;
  if (tid < kMaxAlternatives) l.top[tid] = 0;
  if (tid == 0) {
    l.threshold = 0;
    l.count = 0;
    l.segments = 0;
  }
  ready();
  __syncthreads();
  // One wave finds the bound; twice as many groups as alternatives leave few
  // candidates more than k.
  auto bound_of = [&](auto groups) {
    constexpr int N = groups();
    uint64_t group[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      group[i] = 0;
#pragma unroll
      for (int j = 64 * i; j < T; j += 64 * N) group[i] = l.keys[j + tid] > group[i] ? l.keys[j + tid] : group[i];
    }
    const uint64_t bound = wave_kth<N>(group, k);
    if (tid == 0) l.threshold = bound;
  };
  if (tid < 64) {
    if (k <= 32)
      bound_of(std::integral_constant<int, 1>{});
    else
      bound_of(std::integral_constant<int, 4>{});
  }
  __syncthreads();
  const uint64_t bound = l.threshold;
  const uint32_t per = (units + T - 1) / T;
  auto push_unit = [&](uint32_t u, uint64_t least) {
    const int64_t col = first + static_cast<int64_t>(u) * kUnit;
    const int64_t left = first + columns - col;
    float v[8];
    load_unit<DT, MASKED>(row, mask, col, left < kUnit ? static_cast<int>(left) : kUnit, v);
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
      const uint64_t key = score_key(v[i], static_cast<uint32_t>(col) + i);
      if (v[i] > kMinusInf && key >= least) push_key(l, key);
    }
  };
  if (per == 1) {  // each thread has its own unit
    if (mine != 0 && mine >= bound) push_unit(tid, bound);
  } else {
    if (mine != 0 && mine >= bound) l.segment[atomicAdd(&l.segments, 1u)] = static_cast<uint16_t>(tid);
    __syncthreads();
    const uint32_t pairs = l.segments * per;
    for (uint32_t p = tid; p < pairs; p += T) {
      const uint32_t u = l.segment[p / per] + T * (p % per);
      if (u < units) push_unit(u, bound);
    }
  }
  __syncthreads();
  uint32_t n = l.count;
  if (n > kCandidates) {
    __syncthreads();
    if (per == 1) {  // nobody has listed the threads yet
      if (mine != 0 && mine >= bound) l.segment[atomicAdd(&l.segments, 1u)] = static_cast<uint16_t>(tid);
    }
    if (tid == 0) l.count = 0;
    __syncthreads();
    const uint32_t pairs = l.segments * per;
    for (uint32_t base = 0; base < pairs; base += kRoundUnits) {
      const uint32_t p = base + tid;
      if (tid < kRoundUnits && p < pairs) {
        const uint32_t u = l.segment[p / per] + T * (p % per);
        if (u < units) push_unit(u, l.threshold);
      }
      __syncthreads();
      make_room<T>(l, k);
    }
    n = l.count;
  }
  rank_keys<T>(l, n, k);
}

// The row's target: its score, or -inf where it is excluded.  The id is read
// before the row's scores, the score after them, so that neither is waited for.
struct Target {
  float z;
  bool none;  // -1: no target
};

template <int DT>
__device__ __forceinline__ Target find_target(const LogprobsArgs& a, int64_t row, int64_t target) {
  Target t{kMinusInf, target == -1};
  if (target >= 0 && target < a.columns &&
      (a.mask == nullptr || ((a.mask[row * a.mask_stride + (target >> 6)] >> (63 - (target & 63))) & 1) != 0))
    t.z = load_score<DT>(static_cast<const char*>(a.logits) + row * a.row_stride * kScoreBytes<DT>, target);
  return t;
}

// The row's outputs from its statistics, by one thread.
__device__ void finish_row(const LogprobsArgs& a, int64_t row, const Target& target, const SoftStats& st) {
  const bool none = st.m == kMinusInf && st.s == 0.0f;
  const float log_s = logf(st.s);
  a.lse[row] = none ? kMinusInf : fmaf(st.m, a.inv_t, log_s);
  const float h = log_s - st.t / st.s * a.inv_t;
  a.entropy[row] = none || h < 0.0f ? 0.0f : h;  // NaN stays
  if (a.stats != nullptr) {
    a.stats[2 * row] = st.m;
    a.stats[2 * row + 1] = st.s;
  }
  float lp = target.none ? 0.0f : kMinusInf;
  if (!none && target.z != kMinusInf) lp = fmaf(target.z - st.m, a.inv_t, -log_s);
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

// The workgroup's statistics: each wave leaves its own, and after a barrier
// any thread can join them.
template <int T>
struct WorkgroupStats {
  SoftStats waves[T / 64];
  __device__ __forceinline__ void put(SoftStats st, float c) {
    st = soft_wave_join(st, c);
    if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = st;
  }
  __device__ __forceinline__ SoftStats get(float c) const {
    const int w = threadIdx.x % 64;
    return soft_wave_join(w < T / 64 ? waves[w] : soft_none(), c);
  }
};

// One workgroup per row, or per part of a row (row_chunks, row_threads).
//
// What bounds it: the one read of the scores.  Statistics take a multiply-add,
// an exponential and two sums a score, in registers, rescaled when a thread's
// maximum rises (settled, take_unit); joins go over lanes and LDS once a row.
// The alternatives cost a second read of about k threads' units (select_top).
//
// Measured: 4,096 x 100,000 bfloat16 147 us (5.6 TB/s); 512 x 100,000 bfloat16,
// 20 alternatives 27 us (3.7 TB/s: two workgroups a CU end together, and the
// selection's latency shows); 16 x 2.5M float32 filtered, 100 alternatives 56 us
// with the join (42 us without alternatives); 1 x 100,000 float32 filtered, 10
// alternatives 13 us (two launches; 7.5 us without alternatives).
template <int DT, bool MASKED, int T>
__global__ __launch_bounds__(T, T == 256 ? 4 : 8) void logprobs_kernel(LogprobsArgs a) {
  extern __shared__ __align__(16) uint8_t lds_raw[];
  SelectLds& l = *reinterpret_cast<SelectLds*>(lds_raw);
  __shared__ WorkgroupStats<T> joined;
  const int tid = threadIdx.x;
  const int64_t items = a.rows * a.chunks;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t r = item / a.chunks;
    const int64_t first = (item - r * a.chunks) * a.chunk_columns;
    const int64_t columns = min(a.chunk_columns, a.columns - first);
    const char* row = static_cast<const char*>(a.logits) + r * a.row_stride * kScoreBytes<DT>;
    const uint64_t* mask = MASKED ? a.mask + r * a.mask_stride : nullptr;
    const uint32_t full = static_cast<uint32_t>(columns / kUnit);
    const int64_t target_id = tid == 0 && a.chunks == 1 ? a.targets[r] : -1;
    Running run = running_none(a.c, a.limit);
    uint32_t top_unit = 0;
    // units a thread has in flight: 64 bytes, half that beside the filter's registers
    constexpr int kAhead = (DT == ST_SCORE_F32 ? 2 : 4) / (MASKED ? 2 : 1);
    uint32_t u = tid;
    for (; u + (kAhead - 1) * T < full; u += kAhead * T) {
      Raw8<DT> raw[kAhead];
      uint32_t pass[kAhead] = {};
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
        if (take_unit<MASKED>(run, v, pass[i], a.c, a.limit)) top_unit = u + i * T;
      }
    }
    const uint32_t units = static_cast<uint32_t>((columns + kUnit - 1) / kUnit);
    for (; u < units; u += T) {
      const int64_t col = first + static_cast<int64_t>(u) * kUnit;
      float v[8];
      load_unit<DT, false>(row, mask, col, u < full ? kUnit : static_cast<int>(columns % kUnit), v);
      uint32_t pass = 0xFFu;
      if constexpr (MASKED) pass = pass_byte(mask, col / kUnit);
      if (take_unit<MASKED>(run, v, pass, a.c, a.limit)) top_unit = u;
    }
    SoftStats st = settled(run, a.c, a.limit);
    const Target target = find_target<DT>(a, r, target_id);  // one thread's
    if (a.topk > 0) {
      select_top<DT, MASKED, T>(l, row, mask, first, columns, st.m, top_unit, a.topk, [&] { joined.put(st, a.c); });
    } else {
      joined.put(st, a.c);
      __syncthreads();
    }
    st = joined.get(a.c);
    if (a.chunks > 1) {
      if (tid == 0) a.part_stats[item] = st;
      if (tid < a.topk) a.part_keys[item * a.topk + tid] = l.top[tid];
    } else {
      if (tid == 0) finish_row(a, r, target, st);
      if (tid < a.topk) finish_alternative(a, r, tid, l.top[tid], st);
    }
    __syncthreads();
  }
}

// Joins a row's parts: one workgroup per row.  The parts' lists are in order,
// so their j-th entries bound the k-th best key from below: with j = ceil(2k /
// parts), ceil(k / j) lists have at least k keys at or above the
// ceil(k / j)-th largest of them.  Everything is read at the start, the first
// kRoundUnits * kUnit entries into registers.  Up to a few thousand entries the
// kernel is one latency after another (4-12 us), of which the launch is the
// largest; 25,600 (one row of 4M, 100 alternatives) take 26 us.
template <int DT>
__global__ __launch_bounds__(kJoinThreads) void logprobs_join_kernel(LogprobsArgs a) {
  extern __shared__ __align__(16) uint8_t lds_raw[];
  SelectLds& l = *reinterpret_cast<SelectLds*>(lds_raw);
  __shared__ WorkgroupStats<kJoinThreads> joined;
  constexpr int kEach = kRoundUnits * kUnit / kJoinThreads;
  const int tid = threadIdx.x;
  const int k = a.topk;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const uint64_t* lists = a.part_keys + r * a.chunks * k;
    const int64_t entries = static_cast<int64_t>(a.chunks) * k;
    const int depth = k > 0 ? min(k, (2 * k + a.chunks - 1) / a.chunks) : 0;
    SoftStats st = tid < a.chunks ? a.part_stats[r * a.chunks + tid] : soft_none();
    uint64_t head[kMaxChunks / 64] = {};  // of the first wave
    if (k > 0 && tid < 64) {
#pragma unroll
      for (int i = 0; i < kMaxChunks / 64; ++i) {
        const int chunk = tid + 64 * i;
        if (chunk < a.chunks) head[i] = lists[static_cast<int64_t>(chunk) * k + depth - 1];
      }
    }
    uint64_t key[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int64_t e = i * kJoinThreads + tid;
      key[i] = e < entries ? lists[e] : 0;
    }
    const Target target = find_target<DT>(a, r, tid == 0 ? a.targets[r] : -1);
    joined.put(st, a.c);
    if (k > 0) {
      const int need = (k + depth - 1) / depth;  // <= chunks
      if (tid < kMaxAlternatives) l.top[tid] = 0;
      if (tid < 64) {
        const uint64_t bound = wave_kth<kMaxChunks / 64>(head, need);
        if (tid == 0) {
          l.threshold = bound;
          l.count = 0;
        }
      }
      __syncthreads();
      for (int64_t base = 0; base < entries; base += kRoundUnits * kUnit) {
        const uint64_t least = l.threshold;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          if (base > 0) {
            const int64_t e = base + i * kJoinThreads + tid;
            key[i] = e < entries ? lists[e] : 0;
          }
          if (key[i] != 0 && key[i] >= least) push_key(l, key[i]);
        }
        __syncthreads();
        make_room<kJoinThreads>(l, k);
      }
      rank_keys<kJoinThreads>(l, l.count, k);
    } else {
      __syncthreads();
    }
    st = joined.get(a.c);
    if (tid == 0) finish_row(a, r, target, st);
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
// dL/dz = e (k0 + k1 (z-m)) outside the target and the alternatives.  Scores are
// read once and gradients written once; parts of 8,192 columns a workgroup keep
// the row's factors in registers.  HBM bounds it: 4,096 x 100,000 bfloat16 280
// us (5.9 TB/s), 1,000 x 33,333 float32 filtered 48 us (5.6 TB/s).
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

// Parts of a row.  One workgroup reads up to 64K columns sooner than a second
// launch joins parts (one row of 40,000 with 10 alternatives: 10.3 us whole,
// 12.6 us in parts; of 100,000: 12.3 and 12.1; 256 rows of 50,000: 10.1 and
// 15.9).  Longer rows: two workgroups of 1,024 threads for every CU, each with
// at least 8,192 columns, a unit per thread (100,000 columns, 1 row: 12.1 us
// against 14.0 with 32,768).
int row_chunks(int64_t rows, int64_t columns) {
  if (columns <= 65536) return 1;
  const int64_t want = (2 * cu_count() + rows - 1) / std::max<int64_t>(rows, 1);
  const int64_t most = (columns + 8191) / 8192;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, most, kMaxChunks})));
}

// Threads of a row's workgroup: as few as let the rows fill every CU's 2,048.
int row_threads(int64_t rows, int chunks) {
  if (chunks > 1 || rows <= 2 * cu_count()) return 1024;
  return rows <= 4 * cu_count() ? 512 : 256;
}

unsigned grid_of(int64_t items) { return static_cast<unsigned>(std::min<int64_t>(items, kMaxGrid)); }

template <int DT, bool MASKED>
void launch_forward(const LogprobsArgs& a, hipStream_t s) {
  const size_t lds = a.topk > 0 ? sizeof(SelectLds) : 0;
  const unsigned grid = grid_of(a.rows * a.chunks);
  const int threads = row_threads(a.rows, a.chunks);
  if (threads == 256)
    hipLaunchKernelGGL((logprobs_kernel<DT, MASKED, 256>), dim3(grid), dim3(256), lds, s, a);
  else if (threads == 512)
    hipLaunchKernelGGL((logprobs_kernel<DT, MASKED, 512>), dim3(grid), dim3(512), lds, s, a);
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
    a.limit = fast_limit(a.c);
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
