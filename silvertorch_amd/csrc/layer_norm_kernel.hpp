// Layer norm: y = n w + b with n = (h - mean h) r, r = 1 / sqrt(var h + eps),
// of each row h; h = x, or h = residual + dropout(x) rounded to the residual's
// type and returned too.  Backward, with g = gy w:
//   gh = r (g - mean g - n mean(g n)) + (the sum's own gradient),
//   gw = sum_rows gy n,  gb = sum_rows gy,
// gx = gh, or what dropout leaves of it.  Statistics and sums are 32-bit.
// No reference operator.
//
// A row lies in registers from its one read on, 8 columns a lane and step: the
// mean first, then what its rounding left and the squares of what is apart from
// it, so that rows far from 0 lose no digits: n is (h - mean) - rest times r in both
// directions.  HBM bounds them: 100 million bfloat16 elements take 78 to 85 us forward
// and 119 to 127 us backward in rows of 64 to 16,384 columns.  Longer: lengths that
// are no multiple of 8, 83 to 95 and 122 to 139, with 160 backward at 5,001 and 5,003;
// rows of 16 and 24, 97 and 104, 138 and 141; past 16,384 columns 97 to 144 and 212 to
// 263 (all without a warm cache).
#pragma once

#include <hip/hip_runtime.h>

#include "code_ops.hpp"
#include "dropout_bits.hpp"
#include "score_ops.hpp"

namespace st {

constexpr int64_t kMaxNormColumns = 32768;
constexpr int kNormStats = ST_NORM_STATS;  // the mean, what its rounding left, r

struct NormArgs {
  const void *x, *residual, *weight, *bias;  // residual, weight and bias may be null
  void *y, *sum;                             // y: codes, where the result is 8-bit; sum: null without residual
  float* scales;                             // of the codes
  float* stats;                              // null, or kNormStats of each row
  int64_t rows, x_stride, residual_stride;
  int dim, code_columns;
  int weight_type;
  int normalise;  // 0: the codes of x itself
  float eps;
  DropoutArgs dropout;
};

struct NormBackwardArgs {
  const void *gy, *gsum, *h, *weight;  // gsum and weight may be null
  void *gx, *gh;                       // null: not wanted (gh: the residual's gradient)
  const float* stats;
  float* partial;  // [workgroups, 2, dim]: gw, then gb; null: not wanted
  int64_t rows, h_stride;
  int dim, weight_type;
  float inverse_dim;
  DropoutArgs dropout;
};

// Lanes of a row and steps of 8 columns a lane: the first that holds a row.  Two or
// three steps: what a row costs besides its columns is shared by more of them, and a
// wave has more rows under way (500,000 x 200 bfloat16 in one step 116 and 145 us
// forward and backward, in two 84 and 123).
struct NormLayout {
  int lanes, steps;
};
constexpr NormLayout kNormLayouts[] = {{1, 1},   {1, 2},   {1, 3},   {2, 2},   {2, 3},   {4, 2},   {4, 3},  {8, 2},
                                       {8, 3},   {16, 2},  {16, 3},  {32, 2},  {32, 3},  {64, 2},  {64, 3}, {128, 2},
                                       {128, 3}, {256, 2}, {256, 3}, {512, 2}, {512, 3}, {1024, 2}, {1024, 3}, {1024, 4}};
// Where codes are the result, instructions bound it, a good part of them the same
// for any number of columns a lane has: 24,414 x 4,096 bfloat16 with 256 lanes 72 us,
// with 128 63.  Lengths just past a power of two leave lanes idle: 11,111 x 9,000 119
// us, 12,207 x 8,192 61.
constexpr NormLayout kCodeLayouts[] = {{2, 1},  {4, 1},  {8, 1},   {16, 1},  {16, 2}, {16, 4},
                                       {32, 4}, {64, 4}, {128, 4}, {256, 4}, {512, 4}, {1024, 4}};
constexpr int kNormLayoutCount = sizeof(kNormLayouts) / sizeof(kNormLayouts[0]);
constexpr int kCodeLayoutCount = sizeof(kCodeLayouts) / sizeof(kCodeLayouts[0]);

constexpr int norm_layout(int64_t dim, const NormLayout* layouts = kNormLayouts) {
  int i = 0;
  while (layouts[i].lanes * layouts[i].steps * 8 < dim) ++i;
  return i;
}
constexpr int norm_threads(int lanes) { return lanes <= 64 ? 256 : lanes; }
constexpr int norm_rows(int lanes) { return lanes <= 64 ? 256 / lanes : 1; }

// Waves a SIMD that the backward kernel's registers leave room for (its launch
// bounds hold them to it).
constexpr int norm_backward_waves(int lanes, int steps) {
  return lanes == 1024 || steps == 1 ? 4 : lanes <= 256 && steps == 2 ? 3 : 2;
}

struct NormShape {
  const void* kernel;
  int threads, rows;  // of a workgroup
  int per_cu;         // workgroups that a CU holds at once
};

template <typename K>
NormShape norm_shape(K* kernel, int threads, int rows) {
  int n = 0;
  const hipError_t e = hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0);
  return {reinterpret_cast<const void*>(kernel), threads, rows, e == hipSuccess && n > 0 ? n : 1};
}

// The kernels for `dim` columns, by the type of x (one translation unit each).
template <int DT>
NormShape norm_forward(int dim, bool wide_sum, bool codes);
template <int DT>
const void* norm_backward(int dim, bool wide_sum);
template <int DT>
const void* norm_columns(bool wide_sum);

// Whether the backward kernel leaves the weight's and the bias's gradients to
// norm_columns_kernel.
constexpr bool norm_columns_apart(int64_t dim) {
  const NormLayout l = kNormLayouts[norm_layout(dim)];
  return l.lanes * l.steps > 2048;
}

#ifdef ST_NORM_TYPE
namespace {

// Columns [col, col + 8) of a row as they are stored; 0 past its end.  LAST: where
// the row ends inside, its last eight for `settle`, one load; put together one by one,
// those of 16-bit types had to be waited for before their row was due (20,000 x 5,004
// bfloat16 112 and 216 us forward and backward, so 79 and 126).
template <int DT, bool LAST = false>
__device__ __forceinline__ Raw8<DT> load_raw_columns(const void* row, int col, int dim) {
  Raw8<DT> r{};
  if constexpr (LAST) {
    if (col < dim) r = load_raw8<DT>(row, min(col, dim - 8));
    return r;
  }
  if (col + 8 <= dim) return load_raw8<DT>(row, col);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (col + i >= dim) continue;
    if constexpr (DT == ST_SCORE_F32)
      r.w[i / 4][i % 4] = static_cast<const uint32_t*>(row)[col + i];
    else
      r.w[0][i / 2] |= static_cast<uint32_t>(static_cast<const uint16_t*>(row)[col + i]) << (16 * (i & 1));
  }
  return r;
}

// What load_raw_columns gave, in its place.
template <int DT, bool LAST>
__device__ __forceinline__ void settle(Raw8<DT>& r, int col, int dim) {
  if constexpr (!LAST) return;
  if (col <= dim - 8) return;
  const int shift = -dim & 7;
  u32x4& w = r.w[0];
  if (shift & 4) w = u32x4{w[2], w[3], 0, 0};
  if (shift & 2) w = u32x4{w[1], w[2], w[3], 0};
  if (shift & 1)
    w = u32x4{__builtin_amdgcn_alignbit(w[1], w[0], 16), __builtin_amdgcn_alignbit(w[2], w[1], 16),
              __builtin_amdgcn_alignbit(w[3], w[2], 16), w[3] >> 16};
}

// Whether rows of type DT are loaded so by L lanes in S steps: where they have eight
// columns (layouts of more than 16), and registers have room for it (not float32's;
// of 1,024 lanes bfloat16's in three steps, 4,999 x 20,001 155 and 267 us, so 144 and
// 263, but in two or four they spill, 6,103 x 16,384 backward 121 us, so 165, and
// float16's in three, 5,000 x 20,000 215 us, so 335).
template <int DT, int L, int S>
constexpr bool kLast = DT != ST_SCORE_F32 && L * S > 2 && (L != 1024 || (S == 3 && DT == ST_SCORE_BF16));

template <int DT>
__device__ __forceinline__ void load_columns(const void* row, int col, int dim, float v[8]) {
  unpack8<DT>(load_raw_columns<DT>(row, col, dim), v);
}

__device__ __forceinline__ void load_columns_typed(const void* row, int col, int dim, int type, float v[8]) {
  if (type == ST_SCORE_F32)
    load_columns<ST_SCORE_F32>(row, col, dim, v);
  else if (type == ST_SCORE_F16)
    load_columns<ST_SCORE_F16>(row, col, dim, v);
  else
    load_columns<ST_SCORE_BF16>(row, col, dim, v);
}

typedef uint32_t u32x2_by2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32_by2 __attribute__((aligned(2)));

template <int DT, bool LAST = false>
__device__ __forceinline__ void store_columns(void* row, int col, int dim, const float v[8]) {
  if (col + 8 <= dim) {
    store8<DT>(row, col, v);
  } else if constexpr (!LAST) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < dim) store_score<DT>(row, col + i, v[i]);
  } else if (col < dim) {
    // four, two and one of the last columns
    const int left = dim & 7;
    const auto pick = [](bool b, float x, float y) { return b ? x : y; };  // by value: an array indexed goes to memory
    uint16_t* to = static_cast<uint16_t*>(row) + col;
    if (left & 4) *reinterpret_cast<u32x2_by2*>(to) = u32x2_by2{score_bits2<DT>(v[0], v[1]), score_bits2<DT>(v[2], v[3])};
    if (left & 2) *reinterpret_cast<u32_by2*>(to + (left & 4)) = score_bits2<DT>(pick(left & 4, v[4], v[0]), pick(left & 4, v[5], v[1]));
    if (left & 1)
      store_score<DT>(to, left & 6, pick(left & 4, pick(left & 2, v[6], v[4]), pick(left & 2, v[2], v[0])));
  }
}

// f over the L lanes of a row (of a wave: L <= 64), in each of them, in a fixed
// order.
template <int L, typename F>
__device__ __forceinline__ float join_lanes(float x, F f) {
  if constexpr (L >= 2) x = f(x, dpp_move<0xB1>(x));    // quad_perm [1, 0, 3, 2]
  if constexpr (L >= 4) x = f(x, dpp_move<0x4E>(x));    // quad_perm [2, 3, 0, 1]
  if constexpr (L >= 8) x = f(x, dpp_move<0x141>(x));   // row_half_mirror
  if constexpr (L >= 16) x = f(x, dpp_move<0x140>(x));  // row_mirror
  if constexpr (L >= 32) {
    const int i = __float_as_int(x);
    const float r0 = __int_as_float(__builtin_amdgcn_readlane(i, 0)), r1 = __int_as_float(__builtin_amdgcn_readlane(i, 16));
    const float r2 = __int_as_float(__builtin_amdgcn_readlane(i, 32)), r3 = __int_as_float(__builtin_amdgcn_readlane(i, 48));
    if constexpr (L == 32)
      x = threadIdx.x & 32 ? f(r2, r3) : f(r0, r1);
    else
      x = f(f(r0, r1), f(r2, r3));
  }
  return x;
}

// f over the L lanes of a row, N numbers of it at once.  Rows of a whole
// workgroup go through `room` (a place of its own for each of the calls that no
// barrier parts).
template <int L, int N, typename F>
__device__ __forceinline__ void join_row(float (&x)[N], float* room, F f) {
#pragma unroll
  for (int n = 0; n < N; ++n) x[n] = join_lanes<(L < 64 ? L : 64)>(x[n], f);
  if constexpr (L > 64) {
    constexpr int kWaves = L / 64;
    if (threadIdx.x % 64 == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) room[n * kWaves + threadIdx.x / 64] = x[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float t = room[n * kWaves];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) t = f(t, room[n * kWaves + w]);
      x[n] = t;
    }
  }
}

constexpr auto kAdd = [](float a, float b) { return a + b; };
constexpr auto kMost = [](float a, float b) { return fmaxf(a, b); };

// HT: the type of h.  CODES: the result goes to 8 bits with a scale for each
// row, from its 32-bit values.
template <int DT, int HT, int L, int S, bool CODES>
__global__ __launch_bounds__(norm_threads(L)) void norm_kernel(NormArgs a) {
  constexpr int kRows = norm_rows(L);
  // Weights stay in registers from row to row where there is room for them.
  constexpr bool kHold = L * S <= 2048 && (CODES || S <= 3);
  __shared__ float room[L > 64 ? 4 * (L / 64) : 1];
  const int lane = threadIdx.x % L, wave_lane = __builtin_amdgcn_readfirstlane(lane);  // of the wave's first
  const DropoutKey key = a.dropout.state ? dropout_key(a.dropout.state) : DropoutKey{};
  if (a.dropout.used && blockIdx.x == 0 && threadIdx.x < 2) a.dropout.used[threadIdx.x] = a.dropout.state[threadIdx.x];

  float w[kHold ? S : 1][8], b[kHold ? S : 1][8];
  auto load_weights = [&](const void* weight, const void* bias, int s, float (&ws)[8], float (&bs)[8]) {
    const int col = (s * L + lane) * 8;
    if (weight)
      load_columns_typed(weight, col, a.dim, a.weight_type, ws);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) ws[i] = 1.0f;
    if (bias)
      load_columns_typed(bias, col, a.dim, a.weight_type, bs);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) bs[i] = 0.0f;
  };
  if constexpr (kHold) {
#pragma unroll
    for (int s = 0; s < S; ++s) load_weights(a.weight, a.bias, s, w[s], b[s]);
  }

  // A wave's rows go through the loop together; what a lane of a row past the
  // last computes is not stored.  The next row is on its way while one is worked on,
  // where there are registers for it (3,051 x 32,768 114 us without, 100 with).
  constexpr bool kNext = L * S <= 2048 || (HT != ST_SCORE_F32 && !CODES);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / (L < 64 ? 64 : L) * (L < 64 ? 64 / L : 1);
  const int within = L < 64 ? threadIdx.x % 64 / L : 0;
  Raw8<DT> next_x[S];
  Raw8<HT> next_residual[S];
  auto fetch = [&](int64_t base) {
    if (base >= a.rows) return;
    const int64_t row = min(base + within, a.rows - 1);
    const char* x = static_cast<const char*>(a.x) + row * a.x_stride * kScoreBytes<DT>;
#pragma unroll
    for (int s = 0; s < S; ++s) next_x[s] = load_raw_columns<DT, kLast<DT, L, S>>(x, (s * L + lane) * 8, a.dim);
    if constexpr (!CODES) {
      if (a.residual) {
        const char* residual = static_cast<const char*>(a.residual) + row * a.residual_stride * kScoreBytes<HT>;
#pragma unroll
        for (int s = 0; s < S; ++s) next_residual[s] = load_raw_columns<HT, kLast<HT, L, S>>(residual, (s * L + lane) * 8, a.dim);
      }
    }
  };
  if constexpr (kNext) fetch(first);
  for (int64_t base = first; base < a.rows; base += step) {
    const int64_t at = base + within;
    const bool live = at < a.rows;
    const int64_t row = live ? at : a.rows - 1;
    if constexpr (!kNext) fetch(base);
    char* sum = static_cast<char*>(a.sum) + row * a.dim * kScoreBytes<HT>;
    // Whether all lanes of this wave have eight columns of the row in step s.
    auto whole = [&](int s) { return (s * L + (L > 64 ? wave_lane + 64 : L)) * 8 <= a.dim; };
    float h[S][8];
    // h of step s
    auto values = [&](int s, float (&v)[8]) {
      const int col = (s * L + lane) * 8;
      if (!whole(s)) settle<DT, kLast<DT, L, S>>(next_x[s], col, a.dim);
      unpack8<DT>(next_x[s], v);
      if constexpr (!CODES) {
        if (!a.residual) return;
        if (!whole(s)) settle<HT, kLast<HT, L, S>>(next_residual[s], col, a.dim);
        float more[8];
        unpack8<HT>(next_residual[s], more);
        uint32_t keeps = 0xFF;
        if (a.dropout.state) keeps = dropout_keeps(key, static_cast<uint64_t>(row) * a.dim + col, a.dropout.dropped);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          // the norm is of the sum as it is returned
          v[i] = score_of_bits<HT>(score_bits<HT>(dropout_add(more[i], v[i], (keeps >> i) & 1, a.dropout.times)));
        }
        if (live) store_columns<HT, kLast<HT, L, S>>(sum, col, a.dim, v);
      }
    };
    const void *weight = a.weight, *bias = a.bias;
    if constexpr (!kHold) asm volatile("" : "+s"(weight), "+s"(bias));  // else the compiler holds them after all, and spills

    float mean = 0.0f, rest = 0.0f, r = 1.0f;
    float total[1] = {0.0f};
#pragma unroll
    for (int s = 0; s < S; ++s) {
      values(s, h[s]);
      if (!CODES || a.normalise)
#pragma unroll
        for (int i = 0; i < 8; ++i) total[0] += h[s][i];
    }
    if constexpr (kNext) fetch(base + step);
    if (!CODES || a.normalise) {
      join_row<L>(total, room, kAdd);
      mean = __fdiv_rn(total[0], static_cast<float>(a.dim));
      // the squares about the rounded mean, and what its rounding left
      float left[2] = {};
#pragma unroll
      for (int s = 0; s < S; ++s) {
#pragma unroll
        for (int i = 0; i < 8; ++i) h[s][i] -= mean;
        if (!whole(s))
#pragma unroll
          for (int i = 0; i < 8; ++i) h[s][i] = (s * L + lane) * 8 + i < a.dim ? h[s][i] : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          left[0] = fmaf(h[s][i], h[s][i], left[0]);
          left[1] += h[s][i];
        }
      }
      join_row<L>(left, room + (L > 64 ? L / 64 : 0), kAdd);
      // Divided, where float32's sums are not exact, so that rows of one value leave
      // just what all their columns are off by; those of 16 bits are, up to 8,192
      // columns, and the product takes ten instructions less (codes of 1,000,000 x 100
      // bfloat16 105 -> 99 us).
      rest = HT == ST_SCORE_F32 ? __fdiv_rn(left[1], static_cast<float>(a.dim)) : left[1] * (1.0f / static_cast<float>(a.dim));
      // a maximum with 0 would turn NaN into it
      float squares = fmaf(-rest, left[1], left[0]);
      squares = squares < 0.0f ? 0.0f : squares;
      r = __fdiv_rn(1.0f, __fsqrt_rn(fmaf(squares, 1.0f / static_cast<float>(a.dim), a.eps)));
      if (a.stats && live && lane == 0) {
        a.stats[kNormStats * row] = mean;
        a.stats[kNormStats * row + 1] = rest;
        a.stats[kNormStats * row + 2] = r;
      }
    }
    // the result's values of step s
    auto result = [&](int s, float (&v)[8]) {
      if (CODES && !a.normalise) return;
      if constexpr (!kHold) load_weights(weight, bias, s, w[0], b[0]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = fmaf(v[i], r, -rest * r);
        v[i] = fmaf(n, w[kHold ? s : 0][i], b[kHold ? s : 0][i]);
      }
    };
    if constexpr (!CODES) {
      char* y = static_cast<char*>(a.y) + row * a.dim * kScoreBytes<DT>;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        result(s, h[s]);
        if (live) store_columns<DT, kLast<DT, L, S>>(y, (s * L + lane) * 8, a.dim, h[s]);
      }
    } else {
      float most[1] = {0.0f};
#pragma unroll
      for (int s = 0; s < S; ++s) {
        result(s, h[s]);
        if (!whole(s))
#pragma unroll
          for (int i = 0; i < 8; ++i) h[s][i] = (s * L + lane) * 8 + i < a.dim ? h[s][i] : 0.0f;
        most[0] = most_of8(most[0], h[s]);
      }
      most[0] = most_or_infinity(most[0]);
      join_row<L>(most, room + (L > 64 ? 3 * (L / 64) : 0), kMost);
      const CodeScale c = code_scale(most[0]);
      if (live && lane == 0) a.scales[row] = c.scale;
      int8_t* codes = static_cast<int8_t*>(a.y) + row * a.code_columns;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int col = (s * L + lane) * 8;
        if (live && col < a.code_columns) *reinterpret_cast<uint64_t*>(codes + col) = codes8(h[s], c);
      }
      // without the norm's barriers the next row's maximum could overtake
      if constexpr (L > 64)
        if (!a.normalise) __syncthreads();
    }
  }
}

// Lanes own the same columns in every row, so the weight's and the bias's
// gradients are sums in registers, joined once a workgroup and then, in a fixed
// order, by norm_finish_kernel: no atomics, the same bits every time.  The longest
// rows leave no registers for them (spilled, they took 3,051 x 32,768 to 640 us):
// norm_columns_kernel reads everything once more.
template <int DT, int HT, int L, int S>
__global__ __launch_bounds__(norm_threads(L), norm_backward_waves(L, S)) void norm_backward_kernel(NormBackwardArgs a) {
  constexpr int kRows = norm_rows(L);
  constexpr bool kHold = S <= 3, kSums = L * S <= 2048, kNext = L * S <= 1024;
  __shared__ float room[L > 64 ? 4 * (L / 64) : 1];
  __shared__ float joined[L <= 64 ? 256 * 8 : 1];
  const int lane = threadIdx.x % L, wave_lane = __builtin_amdgcn_readfirstlane(lane);  // of the wave's first
  const DropoutKey key = a.dropout.state ? dropout_key(a.dropout.state) : DropoutKey{};

  float w[kHold ? S : 1][8], gw[kSums ? S : 1][8], gb[kSums ? S : 1][8];
  auto load_weights = [&](const void* weight, int s, float (&ws)[8]) {
    if (weight)
      load_columns_typed(weight, (s * L + lane) * 8, a.dim, a.weight_type, ws);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) ws[i] = 1.0f;
  };
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if constexpr (kHold) load_weights(a.weight, s, w[s]);
#pragma unroll
    for (int i = 0; i < 8; ++i) gw[kSums ? s : 0][i] = gb[kSums ? s : 0][i] = 0.0f;
  }

  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / (L < 64 ? 64 : L) * (L < 64 ? 64 / L : 1);
  const int within = L < 64 ? threadIdx.x % 64 / L : 0;
  // The next row is on its way while one is worked on, where there are registers for
  // it.
  Raw8<DT> next_g[S];
  Raw8<HT> next_h[S];
  auto fetch = [&](int64_t base) {
    if (base >= a.rows) return;
    const int64_t row = min(base + within, a.rows - 1);
    const char* gy = static_cast<const char*>(a.gy) + row * a.dim * kScoreBytes<DT>;
    const char* hs = static_cast<const char*>(a.h) + row * a.h_stride * kScoreBytes<HT>;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      next_g[s] = load_raw_columns<DT, kLast<DT, L, S>>(gy, (s * L + lane) * 8, a.dim);
      next_h[s] = load_raw_columns<HT, kLast<HT, L, S>>(hs, (s * L + lane) * 8, a.dim);
    }
  };
  // as in norm_kernel
  auto whole = [&](int s) { return (s * L + (L > 64 ? wave_lane + 64 : L)) * 8 <= a.dim; };
  int turn = 0;
  if constexpr (kNext) fetch(first);
  for (int64_t base = first; base < a.rows; base += step, turn ^= 1) {
    const int64_t at = base + within;
    const bool live = at < a.rows;
    const int64_t row = live ? at : a.rows - 1;
    const float mean = a.stats[kNormStats * row], rest = a.stats[kNormStats * row + 1], r = a.stats[kNormStats * row + 2];
    if constexpr (!kNext) fetch(base);
    float g[S][8], n[S][8];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (!whole(s)) {
        settle<DT, kLast<DT, L, S>>(next_g[s], (s * L + lane) * 8, a.dim);
        settle<HT, kLast<HT, L, S>>(next_h[s], (s * L + lane) * 8, a.dim);
      }
      unpack8<DT>(next_g[s], g[s]);
      unpack8<HT>(next_h[s], n[s]);
    }
    if constexpr (kNext) fetch(base + step);
    const void* weight = a.weight;
    if constexpr (!kHold) asm volatile("" : "+s"(weight));  // as in norm_kernel
    float sums[2] = {0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if constexpr (!kHold) load_weights(weight, s, w[0]);
#pragma unroll
      for (int i = 0; i < 8; ++i) n[s][i] = ((n[s][i] - mean) - rest) * r;
      if (!whole(s))
#pragma unroll
        for (int i = 0; i < 8; ++i) n[s][i] = (s * L + lane) * 8 + i < a.dim ? n[s][i] : 0.0f;
      if (kSums && live) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          gw[kSums ? s : 0][i] = fmaf(g[s][i], n[s][i], gw[kSums ? s : 0][i]);
          gb[kSums ? s : 0][i] += g[s][i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        g[s][i] *= w[kHold ? s : 0][i];
        sums[0] += g[s][i];
        sums[1] = fmaf(g[s][i], n[s][i], sums[1]);
      }
    }
    if (!a.gx && !a.gh) continue;
    join_row<L>(sums, room + (L > 64 ? turn * 2 * (L / 64) : 0), kAdd);
    const float mean_g = sums[0] * a.inverse_dim, mean_gn = sums[1] * a.inverse_dim;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int col = (s * L + lane) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) g[s][i] = fmaf(n[s][i], -mean_gn * r, fmaf(g[s][i], r, -mean_g * r));
      if (a.gsum) {
        float more[8];
        load_columns<HT>(static_cast<const char*>(a.gsum) + row * a.dim * kScoreBytes<HT>, col, a.dim, more);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[s][i] += more[i];
      }
      if (a.gh && live) store_columns<HT, kLast<HT, L, S>>(static_cast<char*>(a.gh) + row * a.dim * kScoreBytes<HT>, col, a.dim, g[s]);
      if (a.gx) {
        if (a.dropout.state) {
          const uint32_t keeps = dropout_keeps(key, static_cast<uint64_t>(row) * a.dim + col, a.dropout.dropped);
#pragma unroll
          for (int i = 0; i < 8; ++i) g[s][i] = (keeps >> i) & 1 ? g[s][i] * a.dropout.times : 0.0f;
        }
        if (live) store_columns<DT, kLast<DT, L, S>>(static_cast<char*>(a.gx) + row * a.dim * kScoreBytes<DT>, col, a.dim, g[s]);
      }
    }
  }

  if (!kSums || !a.partial) return;
  float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.dim;
  if constexpr (L > 64) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      store_columns<ST_SCORE_F32>(out, (s * L + lane) * 8, a.dim, gw[kSums ? s : 0]);
      store_columns<ST_SCORE_F32>(out + a.dim, (s * L + lane) * 8, a.dim, gb[kSums ? s : 0]);
    }
  } else {
    // the workgroup's rows, a step and a gradient at a time
    auto join = [&](const float (&v)[8], int s, float* to) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) joined[threadIdx.x / L * L * 8 + i * L + lane] = v[i];
      __syncthreads();
      for (int c = threadIdx.x; c < L * 8; c += 256) {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < kRows; ++k) t += joined[k * L * 8 + c];
        const int col = (s * L + c % L) * 8 + c / L;
        if (col < a.dim) to[col] = t;
      }
    };
#pragma unroll
    for (int s = 0; s < S; ++s) {
      join(gw[kSums ? s : 0], s, out);
      join(gb[kSums ? s : 0], s, out + a.dim);
    }
  }
}

// The weight's and the bias's gradients alone: a workgroup has 2,048 columns of
// every gridDim.y-th row.
template <int DT, int HT>
__global__ __launch_bounds__(256) void norm_columns_kernel(NormBackwardArgs a) {
  const int col = (blockIdx.x * 256 + threadIdx.x) * 8;
  if (col >= a.dim) return;
  float gw[8] = {}, gb[8] = {};
#pragma unroll 2
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    float g[8], h[8];
    load_columns<DT>(static_cast<const char*>(a.gy) + row * a.dim * kScoreBytes<DT>, col, a.dim, g);
    load_columns<HT>(static_cast<const char*>(a.h) + row * a.h_stride * kScoreBytes<HT>, col, a.dim, h);
    const float mean = a.stats[kNormStats * row], rest = a.stats[kNormStats * row + 1], r = a.stats[kNormStats * row + 2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      gw[i] = fmaf(g[i], ((h[i] - mean) - rest) * r, gw[i]);
      gb[i] += g[i];
    }
  }
  float* out = a.partial + static_cast<int64_t>(blockIdx.y) * 2 * a.dim;
  store_columns<ST_SCORE_F32>(out, col, a.dim, gw);
  store_columns<ST_SCORE_F32>(out + a.dim, col, a.dim, gb);
}

template <int DT, int HT, int L, int S, bool CODES>
NormShape forward_shape() {
  static const NormShape shape = norm_shape(norm_kernel<DT, HT, L, S, CODES>, norm_threads(L), norm_rows(L));
  return shape;
}

template <int DT, int HT, bool CODES, int I = 0>
NormShape forward_for(int layout) {
  constexpr const NormLayout* layouts = CODES ? kCodeLayouts : kNormLayouts;
  if constexpr (I < (CODES ? kCodeLayoutCount : kNormLayoutCount)) {
    if (layout == I) return forward_shape<DT, HT, layouts[I].lanes, layouts[I].steps, CODES>();
    return forward_for<DT, HT, CODES, I + 1>(layout);
  }
  return {};
}

template <int DT, int HT, int I = 0>
const void* backward_for(int layout) {
  if constexpr (I < kNormLayoutCount) {
    if (layout == I)
      return reinterpret_cast<const void*>(&norm_backward_kernel<DT, HT, kNormLayouts[I].lanes, kNormLayouts[I].steps>);
    return backward_for<DT, HT, I + 1>(layout);
  }
  return nullptr;
}

}  // namespace

template <>
NormShape norm_forward<ST_NORM_TYPE>(int dim, bool wide_sum, bool codes) {
  if (codes) return forward_for<ST_NORM_TYPE, ST_NORM_TYPE, true>(norm_layout(dim, kCodeLayouts));
  const int layout = norm_layout(dim);
  if (wide_sum) return forward_for<ST_NORM_TYPE, ST_SCORE_F32, false>(layout);
  return forward_for<ST_NORM_TYPE, ST_NORM_TYPE, false>(layout);
}

template <>
const void* norm_backward<ST_NORM_TYPE>(int dim, bool wide_sum) {
  const int layout = norm_layout(dim);
  if (wide_sum) return backward_for<ST_NORM_TYPE, ST_SCORE_F32>(layout);
  return backward_for<ST_NORM_TYPE, ST_NORM_TYPE>(layout);
}

template <>
const void* norm_columns<ST_NORM_TYPE>(bool wide_sum) {
  if (wide_sum) return reinterpret_cast<const void*>(&norm_columns_kernel<ST_NORM_TYPE, ST_SCORE_F32>);
  return reinterpret_cast<const void*>(&norm_columns_kernel<ST_NORM_TYPE, ST_NORM_TYPE>);
}
#endif

}  // namespace st
