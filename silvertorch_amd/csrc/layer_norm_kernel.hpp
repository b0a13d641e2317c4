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
// it, so that rows far from 0 lose no digits.  Rows of up
// to 512 columns take 8 to 64 lanes of a wave, longer ones a wave, then a
// workgroup, with the fewest steps (S) that hold them.  HBM bounds both
// directions.
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
NormShape norm_backward(int dim, bool wide_sum);

#ifdef ST_NORM_TYPE
namespace {

__device__ __forceinline__ float load_typed(const void* p, int64_t i, int type) {
  if (type == ST_SCORE_F32) return load_score<ST_SCORE_F32>(p, i);
  if (type == ST_SCORE_F16) return load_score<ST_SCORE_F16>(p, i);
  return load_score<ST_SCORE_BF16>(p, i);
}

// Columns [col, col + 8) of a row; 0 past its end.
template <int DT>
__device__ __forceinline__ void load_columns(const void* row, int col, int dim, float v[8]) {
  if (col + 8 <= dim) {
    unpack8<DT>(load_raw8<DT>(row, col), v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < dim ? load_score<DT>(row, col + i) : 0.0f;
  }
}

__device__ __forceinline__ void load_columns_typed(const void* row, int col, int dim, int type, float v[8]) {
  if (type == ST_SCORE_F32)
    load_columns<ST_SCORE_F32>(row, col, dim, v);
  else if (type == ST_SCORE_F16)
    load_columns<ST_SCORE_F16>(row, col, dim, v);
  else
    load_columns<ST_SCORE_BF16>(row, col, dim, v);
}

template <int DT>
__device__ __forceinline__ void store_columns(void* row, int col, int dim, const float v[8]) {
  if (col + 8 <= dim) {
    store8<DT>(row, col, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < dim) store_score<DT>(row, col + i, v[i]);
  }
}

// f over the L lanes of a row (of a wave: L <= 64), in each of them, in a fixed
// order.
template <int L, typename F>
__device__ __forceinline__ float join_lanes(float x, F f) {
  x = join8(x, f);
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

constexpr int norm_threads(int lanes) { return lanes <= 256 ? 256 : lanes; }

// HT: the type of h.  CODES: the result goes to 8 bits with a scale for each
// row, from its 32-bit values.
template <int DT, int HT, int L, int S, bool CODES>
__global__ __launch_bounds__(norm_threads(L)) void norm_kernel(NormArgs a) {
  constexpr int kRows = L <= 64 ? norm_threads(L) / L : 1;
  // Weights stay in registers from row to row where there is room for them.
  constexpr bool kHold = S <= 2;
  __shared__ float room[L > 64 ? 4 * (L / 64) : 1];
  const int lane = threadIdx.x % L;
  const DropoutKey key = a.dropout.state ? dropout_key(a.dropout.state) : DropoutKey{};
  if (a.dropout.used && blockIdx.x == 0 && threadIdx.x < 2) a.dropout.used[threadIdx.x] = a.dropout.state[threadIdx.x];

  float w[kHold ? S : 1][8], b[kHold ? S : 1][8];
  auto load_weights = [&](int s, float (&ws)[8], float (&bs)[8]) {
    const int col = (s * L + lane) * 8;
    if (a.weight)
      load_columns_typed(a.weight, col, a.dim, a.weight_type, ws);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) ws[i] = 1.0f;
    if (a.bias)
      load_columns_typed(a.bias, col, a.dim, a.weight_type, bs);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) bs[i] = 0.0f;
  };
  if constexpr (kHold) {
#pragma unroll
    for (int s = 0; s < S; ++s) load_weights(s, w[s], b[s]);
  }

  // A wave's rows go through the loop together; what a lane of a row past the
  // last computes is not stored.
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / (L < 64 ? 64 : L) * (L < 64 ? 64 / L : 1);
  for (int64_t base = first; base < a.rows; base += static_cast<int64_t>(gridDim.x) * kRows) {
    const int64_t at = base + (L < 64 ? threadIdx.x % 64 / L : 0);
    const bool live = at < a.rows;
    const int64_t row = live ? at : a.rows - 1;
    const char* x = static_cast<const char*>(a.x) + row * a.x_stride * kScoreBytes<DT>;
    float h[S][8];
#pragma unroll
    for (int s = 0; s < S; ++s) load_columns<DT>(x, (s * L + lane) * 8, a.dim, h[s]);
    if constexpr (!CODES) {
      if (a.residual) {
        const char* residual = static_cast<const char*>(a.residual) + row * a.residual_stride * kScoreBytes<HT>;
        char* sum = static_cast<char*>(a.sum) + row * a.dim * kScoreBytes<HT>;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const int col = (s * L + lane) * 8;
          float more[8];
          load_columns<HT>(residual, col, a.dim, more);
          uint32_t keeps = 0xFF;
          if (a.dropout.state)
            keeps = dropout_keeps(key, static_cast<uint64_t>(row) * a.dim + col, a.dropout.dropped);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float kept = (keeps >> i) & 1 ? __fmul_rn(h[s][i], a.dropout.times) : 0.0f;
            // the norm is of the sum as it is returned
            h[s][i] = score_of_bits<HT>(score_bits<HT>(__fadd_rn(more[i], kept)));
          }
          if (live) store_columns<HT>(sum, col, a.dim, h[s]);
        }
      }
    }

    if (!CODES || a.normalise) {
      float total[1] = {0.0f};
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) total[0] += h[s][i];
      join_row<L>(total, room, kAdd);
      const float mean = __fdiv_rn(total[0], static_cast<float>(a.dim));
      // what the mean's rounding left, and the squares about the rounded one
      float left[2] = {0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int col = (s * L + lane) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          h[s][i] = col + i < a.dim ? h[s][i] - mean : 0.0f;
          left[0] += h[s][i];
          left[1] = fmaf(h[s][i], h[s][i], left[1]);
        }
      }
      join_row<L>(left, room + (L > 64 ? L / 64 : 0), kAdd);
      const float rest = __fdiv_rn(left[0], static_cast<float>(a.dim));
      // a maximum with 0 would turn NaN into it
      float squares = fmaf(-rest, left[0], left[1]);
      squares = squares < 0.0f ? 0.0f : squares;
      const float r = __fdiv_rn(1.0f, __fsqrt_rn(fmaf(squares, 1.0f / static_cast<float>(a.dim), a.eps)));
      if (a.stats && live && lane == 0) {
        a.stats[kNormStats * row] = mean;
        a.stats[kNormStats * row + 1] = rest;
        a.stats[kNormStats * row + 2] = r;
      }
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if constexpr (!kHold) load_weights(s, w[0], b[0]);
        const int hold = kHold ? s : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[s][i] = fmaf((h[s][i] - rest) * r, w[hold][i], b[hold][i]);
      }
    }

    if constexpr (!CODES) {
      char* y = static_cast<char*>(a.y) + row * a.dim * kScoreBytes<DT>;
      if (live)
#pragma unroll
        for (int s = 0; s < S; ++s) store_columns<DT>(y, (s * L + lane) * 8, a.dim, h[s]);
    } else {
      float most[1] = {0.0f};
      float odd = 0.0f;  // NaN if there is one, or an infinity, in the row
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int col = (s * L + lane) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (col + i >= a.dim) h[s][i] = 0.0f;
          most[0] = fmaxf(most[0], fabsf(h[s][i]));
          odd = fmaf(h[s][i], 0.0f, odd);
        }
      }
      if (odd != odd) most[0] = __builtin_inff();
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
// order, by norm_finish_kernel: no atomics, the same bits every time.
template <int DT, int HT, int L, int S>
__global__ __launch_bounds__(norm_threads(L)) void norm_backward_kernel(NormBackwardArgs a) {
  constexpr int kRows = L <= 64 ? norm_threads(L) / L : 1;
  constexpr bool kHold = S <= 2;
  __shared__ float room[L > 64 ? 4 * (L / 64) : 1];
  __shared__ float joined[L <= 64 ? 256 * 8 : 1];
  const int lane = threadIdx.x % L;
  const DropoutKey key = a.dropout.state ? dropout_key(a.dropout.state) : DropoutKey{};

  float w[kHold ? S : 1][8], gw[S][8], gb[S][8];
  auto load_weights = [&](int s, float (&ws)[8]) {
    if (a.weight)
      load_columns_typed(a.weight, (s * L + lane) * 8, a.dim, a.weight_type, ws);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) ws[i] = 1.0f;
  };
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if constexpr (kHold) load_weights(s, w[s]);
#pragma unroll
    for (int i = 0; i < 8; ++i) gw[s][i] = gb[s][i] = 0.0f;
  }

  const int64_t first = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / (L < 64 ? 64 : L) * (L < 64 ? 64 / L : 1);
  int turn = 0;
  for (int64_t base = first; base < a.rows; base += static_cast<int64_t>(gridDim.x) * kRows, turn ^= 1) {
    const int64_t at = base + (L < 64 ? threadIdx.x % 64 / L : 0);
    const bool live = at < a.rows;
    const int64_t row = live ? at : a.rows - 1;
    const char* gy = static_cast<const char*>(a.gy) + row * a.dim * kScoreBytes<DT>;
    const char* hs = static_cast<const char*>(a.h) + row * a.h_stride * kScoreBytes<HT>;
    const float mean = a.stats[kNormStats * row], rest = a.stats[kNormStats * row + 1], r = a.stats[kNormStats * row + 2];
    float g[S][8], n[S][8];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int col = (s * L + lane) * 8;
      load_columns<DT>(gy, col, a.dim, g[s]);
      load_columns<HT>(hs, col, a.dim, n[s]);
    }
    float sums[2] = {0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int col = (s * L + lane) * 8;
      if constexpr (!kHold) load_weights(s, w[0]);
      const int hold = kHold ? s : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        n[s][i] = col + i < a.dim ? ((n[s][i] - mean) - rest) * r : 0.0f;
        if (live) {
          gw[s][i] = fmaf(g[s][i], n[s][i], gw[s][i]);
          gb[s][i] += g[s][i];
        }
        g[s][i] *= w[hold][i];
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
      for (int i = 0; i < 8; ++i) g[s][i] = r * ((g[s][i] - mean_g) - n[s][i] * mean_gn);
      if (a.gsum) {
        float more[8];
        load_columns<HT>(static_cast<const char*>(a.gsum) + row * a.dim * kScoreBytes<HT>, col, a.dim, more);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[s][i] += more[i];
      }
      if (a.gh && live) store_columns<HT>(static_cast<char*>(a.gh) + row * a.dim * kScoreBytes<HT>, col, a.dim, g[s]);
      if (a.gx) {
        if (a.dropout.state) {
          const uint32_t keeps = dropout_keeps(key, static_cast<uint64_t>(row) * a.dim + col, a.dropout.dropped);
#pragma unroll
          for (int i = 0; i < 8; ++i) g[s][i] = (keeps >> i) & 1 ? g[s][i] * a.dropout.times : 0.0f;
        }
        if (live) store_columns<DT>(static_cast<char*>(a.gx) + row * a.dim * kScoreBytes<DT>, col, a.dim, g[s]);
      }
    }
  }

  if (!a.partial) return;
  float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.dim;
  if constexpr (L > 64) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      store_columns<ST_SCORE_F32>(out, (s * L + lane) * 8, a.dim, gw[s]);
      store_columns<ST_SCORE_F32>(out + a.dim, (s * L + lane) * 8, a.dim, gb[s]);
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
      join(gw[s], s, out);
      join(gb[s], s, out + a.dim);
    }
  }
}

template <int DT, int HT, int L, int S, bool CODES>
NormShape forward_shape() {
  static const NormShape shape = norm_shape(norm_kernel<DT, HT, L, S, CODES>, norm_threads(L), L <= 64 ? norm_threads(L) / L : 1);
  return shape;
}

template <int DT, int HT, bool CODES>
NormShape forward_for(int dim) {
  if (dim <= 64) return forward_shape<DT, HT, 8, 1, CODES>();
  if (dim <= 128) return forward_shape<DT, HT, 16, 1, CODES>();
  if (dim <= 256) return forward_shape<DT, HT, 32, 1, CODES>();
  if (dim <= 512) return forward_shape<DT, HT, 64, 1, CODES>();
  if (dim <= 1024) return forward_shape<DT, HT, 64, 2, CODES>();
  if (dim <= 2048) return forward_shape<DT, HT, 256, 1, CODES>();
  if (dim <= 4096) return forward_shape<DT, HT, 256, 2, CODES>();
  if (dim <= 8192) return forward_shape<DT, HT, 1024, 1, CODES>();
  if (dim <= 16384) return forward_shape<DT, HT, 1024, 2, CODES>();
  return forward_shape<DT, HT, 1024, 4, CODES>();
}

template <int DT, int HT, int L, int S>
NormShape backward_shape() {
  static const NormShape shape = norm_shape(norm_backward_kernel<DT, HT, L, S>, norm_threads(L), L <= 64 ? norm_threads(L) / L : 1);
  return shape;
}

template <int DT, int HT>
NormShape backward_for(int dim) {
  if (dim <= 64) return backward_shape<DT, HT, 8, 1>();
  if (dim <= 128) return backward_shape<DT, HT, 16, 1>();
  if (dim <= 256) return backward_shape<DT, HT, 32, 1>();
  if (dim <= 512) return backward_shape<DT, HT, 64, 1>();
  if (dim <= 1024) return backward_shape<DT, HT, 64, 2>();
  if (dim <= 2048) return backward_shape<DT, HT, 256, 1>();
  if (dim <= 4096) return backward_shape<DT, HT, 256, 2>();
  if (dim <= 8192) return backward_shape<DT, HT, 1024, 1>();
  if (dim <= 16384) return backward_shape<DT, HT, 1024, 2>();
  return backward_shape<DT, HT, 1024, 4>();
}

}  // namespace

template <>
NormShape norm_forward<ST_NORM_TYPE>(int dim, bool wide_sum, bool codes) {
  if (codes) return forward_for<ST_NORM_TYPE, ST_NORM_TYPE, true>(dim);
  if (wide_sum) return forward_for<ST_NORM_TYPE, ST_SCORE_F32, false>(dim);
  return forward_for<ST_NORM_TYPE, ST_NORM_TYPE, false>(dim);
}

template <>
NormShape norm_backward<ST_NORM_TYPE>(int dim, bool wide_sum) {
  if (wide_sum) return backward_for<ST_NORM_TYPE, ST_SCORE_F32>(dim);
  return backward_for<ST_NORM_TYPE, ST_NORM_TYPE>(dim);
}
#endif

}  // namespace st
