// Products of a table held in 8 bits with vectors held in 8 bits, and both's
// making.  No reference operator.
//
//   y[m, n] = x_scale[m] scale[n] sum_k x[m, k] code[n, k] + bias[n]
// The sum is exact (32-bit integers); each row of the table (a document, an
// output channel) and each vector (a query, a token) has one scale.  Rows are
// whole blocks of 16 columns; vectors that come as floats are taken to 8 bits
// on the way (code_ops.hpp), zeros past their last column.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <mutex>

#include "code_ops.hpp"
#include "layer_norm_kernel.hpp"
#include "score_ops.hpp"
#include "st_errors.hpp"

namespace st {
int cu_count();
void launch_codes(const void* x, int x_type, int64_t rows, int64_t dim, int64_t x_stride, int8_t* codes, int64_t columns,
                  float* scales, hipStream_t s);

namespace {

constexpr int64_t kMaxColumns = (1 << 17) - 16;  // 2^14 a product: sums stay below 2^31
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kFusedBytes = 32 * 1024;  // of LDS for vectors that the product itself takes to 8 bits

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

struct MatmulArgs {
  const int8_t* codes;
  const float* scales;
  const float* bias;  // or null
  const void* x;      // codes [tokens, columns], or what they are made of
  const float* x_scales;
  void* y;
  int64_t rows, tokens, x_stride;
  int dim, columns;
  int x_type, y_type;
};

__device__ __forceinline__ void store_typed(void* y, int64_t at, float v, int type) {
  if (type == ST_SCORE_F32)
    store_score<ST_SCORE_F32>(y, at, v);
  else if (type == ST_SCORE_F16)
    store_score<ST_SCORE_F16>(y, at, v);
  else
    store_score<ST_SCORE_BF16>(y, at, v);
}

template <int DT>
__device__ __forceinline__ void load_eight(const void* row, int col, int dim, float v[8]) {
  if (col + 8 <= dim) {
    unpack8<DT>(load_raw8<DT>(row, col), v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < dim ? load_score<DT>(row, col + i) : 0.0f;
  }
}

// One vector to 8 bits by one wave: codes to LDS in the order of the matrix
// instruction's operand (1 KB for 64 columns of 16 vectors: 256 bytes for each
// 16 columns), zeros up to `padded`; returns the scale.
template <int DT>
__device__ __forceinline__ float codes_to_lds(const void* row, int dim, int padded, uint8_t* to, int step_bytes) {
  const int lane = threadIdx.x % 64;
  float most = 0.0f, odd = 0.0f, v[8];
  for (int col = lane * 8; col < dim; col += 512) {
    load_eight<DT>(row, col, dim, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      most = fmaxf(most, fabsf(v[i]));
      odd = fmaf(v[i], 0.0f, odd);
    }
  }
  const CodeScale c = code_scale(wave_max(odd != odd ? __builtin_inff() : most));
  for (int col = lane * 8; col < padded; col += 512) {
    load_eight<DT>(row, col, dim, v);
    *reinterpret_cast<uint64_t*>(to + (col >> 6) * step_bytes + ((col >> 4) & 3) * 256 + (col & 15)) = codes8(v, c);
  }
  return c.scale;
}

// Few vectors: HBM bounds it, the table's bytes or the results'.  The table goes
// from memory to registers, 16 rows x 64 columns an instruction, vectors (16 T at
// a time) beside it.  R blocks of 16 rows a wave, J steps of 64 columns at a
// time; SPLIT waves share a row's columns.
template <int T, int R, int J, bool SPLIT, bool FUSED>
__global__ __launch_bounds__(kThreads) void few_kernel(MatmulArgs a) {
  extern __shared__ uint8_t lds[];
  __shared__ float fused_scales[FUSED ? 16 * T : 1];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, q = lane / 16, c = lane % 16;
  const int64_t token0 = static_cast<int64_t>(blockIdx.y) * (16 * T);
  const int tokens = static_cast<int>(min(a.tokens - token0, static_cast<int64_t>(16 * T)));
  const int steps = (a.columns + 64 * J - 1) / (64 * J);  // of J times 64 columns
  constexpr int kStepBytes = T * 1024;                    // of LDS, for 64 columns

  if constexpr (FUSED) {
    for (int m = wave; m < tokens; m += kWaves) {
      uint8_t* to = lds + (m / 16) * 1024 + (m % 16) * 16;
      const int64_t row = (token0 + m) * a.x_stride;
      float scale;
      if (a.x_type == ST_SCORE_F32)
        scale = codes_to_lds<ST_SCORE_F32>(static_cast<const float*>(a.x) + row, a.dim, steps * J * 64, to, kStepBytes);
      else if (a.x_type == ST_SCORE_F16)
        scale = codes_to_lds<ST_SCORE_F16>(static_cast<const uint16_t*>(a.x) + row, a.dim, steps * J * 64, to, kStepBytes);
      else
        scale = codes_to_lds<ST_SCORE_BF16>(static_cast<const uint16_t*>(a.x) + row, a.dim, steps * J * 64, to, kStepBytes);
      if (lane == 0) fused_scales[m] = scale;
    }
    __syncthreads();
  }

  struct Step {
    i32x4 w[R][J], x[FUSED ? 1 : T][FUSED ? 1 : J];
  };
  const int64_t tiles = (a.rows + 16 * R - 1) / (16 * R);
  const int64_t tile_step = static_cast<int64_t>(gridDim.x) * (SPLIT ? 1 : kWaves);
  int64_t tile = SPLIT ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * kWaves + wave;
  const int first_step = SPLIT ? wave : 0;
  constexpr int kStepStep = SPLIT ? kWaves : 1;

  auto load = [&](int64_t at, int step, Step& s) {
    const int64_t row0 = at * (16 * R);
    const int8_t* table = a.codes + row0 * a.columns;
    const int last = static_cast<int>(min(a.rows - row0, static_cast<int64_t>(16 * R))) - 1;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int k = (step * J + j) * 64 + q * 16;
      const bool in = k < a.columns;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        // rows past the last and columns past theirs read others; the former's
        // results are not stored, the latter meet zeros of x
        const int64_t offset = static_cast<int64_t>(min(16 * r + c, last)) * a.columns + (in ? k : 0);
        s.w[r][j] = *reinterpret_cast<const i32x4*>(table + offset);
      }
      if constexpr (!FUSED) {
#pragma unroll
        for (int t = 0; t < T; ++t) {
          const int64_t m = token0 + min(16 * t + c, tokens - 1);
          i32x4 v = *reinterpret_cast<const i32x4*>(static_cast<const int8_t*>(a.x) + m * a.columns + (in ? k : 0));
          if (!in) v = i32x4{0, 0, 0, 0};
          s.x[t][j] = v;
        }
      }
    }
  };

  i32x4 acc[T][R];
  auto clear = [&] {
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int r = 0; r < R; ++r) acc[t][r] = i32x4{0, 0, 0, 0};
  };
  auto compute = [&](int step, const Step& s) {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int t = 0; t < T; ++t) {
        i32x4 x;
        if constexpr (FUSED)
          x = *reinterpret_cast<const i32x4*>(lds + (step * J + j) * kStepBytes + t * 1024 + lane * 16);
        else
          x = s.x[t][j];
#pragma unroll
        for (int r = 0; r < R; ++r) acc[t][r] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, s.w[r][j], acc[t][r], 0, 0, 0);
      }
  };
  auto x_scale = [&](int m) { return FUSED ? fused_scales[m] : a.x_scales[token0 + m]; };
  auto put = [&](int m, int64_t n, int sum, float scale, float bias) {
    store_typed(a.y, (token0 + m) * a.rows + n, fmaf(static_cast<float>(sum) * x_scale(m), scale, bias), a.y_type);
  };

  if (tile >= tiles) return;
  Step next;
  load(tile, min(first_step, steps - 1), next);
  for (; tile < tiles; tile += tile_step) {
    clear();
    for (int step = first_step; step < steps; step += kStepStep) {
      const Step now = next;
      const bool more = step + kStepStep < steps;
      // past the end: this step again, not used
      const int64_t to = more || tile + tile_step >= tiles ? tile : tile + tile_step;
      load(to, more ? step + kStepStep : min(first_step, steps - 1), next);
      compute(step, now);
    }
    const int64_t row0 = tile * (16 * R);
    if constexpr (SPLIT) {
      static_assert(R == 1 && kWaves == 4, "");
      i32x4* sums = reinterpret_cast<i32x4*>(lds + (FUSED ? steps * J * kStepBytes : 0));
#pragma unroll
      for (int t = 0; t < T; ++t) sums[(wave * T + t) * 64 + lane] = acc[t][0];
      __syncthreads();
      // element i of each lane by wave i
      const int64_t n = row0 + c;
#pragma unroll
      for (int t = 0; t < T; ++t) {
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += reinterpret_cast<const int*>(sums)[((w * T + t) * 64 + lane) * 4 + wave];
        const int m = 16 * t + 4 * q + wave;
        if (m < tokens && n < a.rows) put(m, n, sum, a.scales[n], a.bias ? a.bias[n] : 0.0f);
      }
      __syncthreads();
    } else {
      static_assert(R == 4, "");
      const int64_t n = row0 + lane;
      const bool live = n < a.rows;
      const float scale = live ? a.scales[n] : 0.0f, bias = live && a.bias ? a.bias[n] : 0.0f;
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (16 * t + i >= tokens) continue;
          // one vector's results of 64 rows side by side
          const u32x4 v = transpose4(u32x4{static_cast<uint32_t>(acc[t][0][i]), static_cast<uint32_t>(acc[t][1][i]),
                                           static_cast<uint32_t>(acc[t][2][i]), static_cast<uint32_t>(acc[t][3][i])});
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int m = 16 * t + 4 * j + i;
            if (m < tokens && live) put(m, n, static_cast<int>(v[j]), scale, bias);
          }
        }
    }
  }
}

template <int T, bool FUSED>
void launch_few(const MatmulArgs& a, hipStream_t s) {
  const int64_t passes = (a.tokens + 16 * T - 1) / (16 * T);
  const bool split = a.columns >= 1024 && (a.rows + 63) / 64 < 8 * cu_count();
  const int64_t groups = split ? (a.rows + 15) / 16 : (a.rows + 64 * kWaves - 1) / (64 * kWaves);
  const int64_t grid = std::min<int64_t>(groups, 4 * cu_count());
  const int padded = split ? (a.columns + 255) / 256 * 256 : (a.columns + 63) / 64 * 64;
  const size_t fused = FUSED ? static_cast<size_t>(padded) * 16 * T : 0;
  for (int64_t at = 0; at < passes; at += 32768) {
    MatmulArgs part = a;
    const int64_t first = at * 16 * T;
    part.tokens = std::min<int64_t>(a.tokens - first, static_cast<int64_t>(32768) * 16 * T);
    const int x_bytes = a.x_type == ST_CODE_I8 ? 1 : a.x_type == ST_SCORE_F32 ? 4 : 2;
    const int y_bytes = a.y_type == ST_SCORE_F32 ? 4 : 2;
    part.x = static_cast<const char*>(a.x) + first * a.x_stride * x_bytes;
    if (a.x_scales) part.x_scales = a.x_scales + first;
    part.y = static_cast<char*>(a.y) + first * a.rows * y_bytes;
    const dim3 blocks(static_cast<unsigned>(grid), static_cast<unsigned>((part.tokens + 16 * T - 1) / (16 * T)));
    if (split)
      hipLaunchKernelGGL((few_kernel<T, 1, 4, true, FUSED>), blocks, dim3(kThreads), fused + T * kThreads * 16, s, part);
    else
      hipLaunchKernelGGL((few_kernel<T, 4, 1, false, FUSED>), blocks, dim3(kThreads), fused, s, part);
  }
}

// Many vectors: the matrix units bound it, and the power they may draw: 16x16x64
// blocks run at 4,840 TOP/s on zeros and 4,070 on random codes (registers alone),
// 32x32x32 ones at 3,290 and 2,600.  A workgroup of NT x NR waves takes tiles of
// NT WT vectors x NR WR rows, each wave its part of them, with the sums in registers.
//
// Columns go in parts of 128 (whole cache lines), two steps of 64 each, a step in
// groups of one block of vectors by all of rows.  While a group's products run, the
// vectors of the group `kAhead` on, or the rows of the next step, go from LDS to
// registers.  Two buffers in LDS; one barrier a part, where its last vectors are in
// registers: from there on the next part is read, and the one after it goes from
// memory straight to LDS.  The stream of parts does not end with a tile: the next
// tile's first two are under way while a tile's results are stored.
//
// In LDS a row is 8 chunks of 16 bytes, chunk c at place c ^ f(row): the 16 lanes
// that read or write at once (two rows, whose addresses differ by half of the 64
// banks, or one chunk of 16 rows) meet all banks.
template <int YT, int WT, int WR, int NT, int NR>
__global__ __launch_bounds__(64 * NT * NR, WT* WR < 64 * 128 ? 2 : 1) void many_kernel(MatmulArgs a) {
  constexpr int BT = WT / 16, BR = WR / 16;                           // blocks of a wave
  constexpr int kAhead = BT >= 8 ? 3 : 2;                             // groups between a block's read and its use
  constexpr int kTokens = NT * WT, kRows = NR * WR;                   // of the workgroup
  constexpr int kAtOnce = 8 * NT * NR;                                // rows that its waves bring with one load each
  constexpr int LT = kTokens / kAtOnce, LR = kRows / kAtOnce, kMoves = LT + LR;
  constexpr int kX = kTokens * 128, kW = kRows * 128;  // bytes of a buffer
  constexpr int kGroups = 2 * BT, kTurn = kGroups - kAhead;  // the group ahead of which the barrier is
  static_assert(kAtOnce % 16 == 0 && BT % 4 == 0, "");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int q = lane / 16, in_block = lane % 16;
  const int parts = (a.columns + 127) / 128;

  // Tiles in an order that shares the last-level caches: an eighth of them to
  // each of the 8 dies (workgroups go round them), there 8 tiles of vectors by
  // one of rows after another.
  const int64_t tiles_t = (a.tokens + kTokens - 1) / kTokens, tiles_r = (a.rows + kRows - 1) / kRows;
  const int64_t all = tiles_t * tiles_r;
  struct Tile {
    int64_t token0, row0;
  };
  auto tile_of = [&](int64_t id) {
    const int64_t each = all / 8, more = all % 8, die = id % 8;
    id = die * each + min(die, more) + id / 8;
    const int64_t in_group = 8 * tiles_r, group = id / in_group, within = id - group * in_group;
    const int64_t height = min(static_cast<int64_t>(8), tiles_t - group * 8);
    return Tile{(group * 8 + within % height) * kTokens, within / height * kRows};
  };

  // What a wave brings: 8 rows a load, lane l the chunk that belongs at place l % 8
  // of row kAtOnce i + 8 wave + l / 8 (f of rows 16 apart is the same).  Rows past the
  // last read it again; their sums are not stored.
  const auto place = [](int row) { return (row >> 1) & 7; };
  const int first_row = wave * 8 + lane / 8, chunk = (lane % 8) ^ place(first_row);
  // Columns past the last are read at the part's start, and of the vectors zeros put
  // in their places once they are there (`settle`).
  const int past = (parts - 1) * 128 + chunk * 16 >= a.columns ? chunk * 16 : 0;
  int64_t bring_id = blockIdx.x;  // the tile and the part that are brought next, and its buffer
  int bring_part = 0, bring_buffer = 0;
  const int8_t *x, *w;
  uint32_t from[kMoves];
  auto aim = [&] {
    const Tile tile = tile_of(bring_id);
    x = static_cast<const int8_t*>(a.x) + tile.token0 * a.columns;
    w = a.codes + tile.row0 * a.columns;
    const int last_token = static_cast<int>(min(a.tokens - tile.token0, static_cast<int64_t>(kTokens))) - 1;
    const int last_row = static_cast<int>(min(a.rows - tile.row0, static_cast<int64_t>(kRows))) - 1;
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      const int row = i < LT ? min(kAtOnce * i + first_row, last_token) : min(kAtOnce * (i - LT) + first_row, last_row);
      from[i] = static_cast<uint32_t>(row) * a.columns + chunk * 16;
    }
  };
  auto place_of = [&](int buffer, int i) {
    return lds + (i < LT ? buffer * kX + i * kAtOnce * 128 : 2 * kX + buffer * kW + (i - LT) * kAtOnce * 128) + wave * 1024;
  };
  auto bring = [&](int i) {
    const int8_t* base = (i < LT ? x : w) + static_cast<int64_t>(bring_part) * 128;
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void*)(base + (from[i] - (bring_part == parts - 1 ? past : 0))),
        (__attribute__((address_space(3))) void*)place_of(bring_buffer, i), 16, 0, 0);
  };
  auto brought = [&] {
    bring_buffer ^= 1;
    if (++bring_part < parts) return;
    bring_part = 0;
    bring_id += gridDim.x;
    if (bring_id < all) aim();
  };
  // Waits for what this wave brought, and for its reads of LDS.
  auto settle = [&](int part, int buffer) {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0)
    if (part == parts - 1 && past != 0) {
#pragma unroll
      for (int i = 0; i < LT; ++i) *reinterpret_cast<i32x4*>(place_of(buffer, i) + lane * 16) = i32x4{0, 0, 0, 0};
    }
  };
  auto barrier = [] {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };

  // Operands: block t of the vectors, into a ring of four; block r of the rows, into
  // the step's set.
  const int x_row = (wave / NR) * WT + in_block, w_row = (wave % NR) * WR + in_block;
  i32x4 fx[4], fw[2][BR];
  auto read_x = [&](int buffer, int step, int t) {
    fx[t & 3] = *reinterpret_cast<const i32x4*>(lds + buffer * kX + x_row * 128 + (((step * 4 + q) ^ place(x_row)) * 16) + t * 2048);
  };
  auto read_w = [&](int buffer, int step, int r) {
    fw[step][r] = *reinterpret_cast<const i32x4*>(lds + 2 * kX + buffer * kW + w_row * 128 + (((step * 4 + q) ^ place(w_row)) * 16) + r * 2048);
  };

  i32x4 acc[BT][BR];
  auto clear = [&] {
#pragma unroll
    for (int t = 0; t < BT; ++t)
#pragma unroll
      for (int r = 0; r < BR; ++r) acc[t][r] = i32x4{0, 0, 0, 0};
  };

  // Results by way of LDS, each wave in a part of its own: 16 vectors x WR rows of
  // sums, chunk c of 4 at place c ^ vector, so that a store writes whole lines of a
  // result's row (16 bytes here and there, straight from the sums: 620 us for 16,384 x
  // 4,096 x 8,192 where this took 509).
  constexpr int kEach = YT == ST_SCORE_F32 ? 4 : 8;  // results a lane stores at once, 16 bytes
  constexpr int kLanes = WR / kEach;                 // of a vector's
  i32x4* sums = reinterpret_cast<i32x4*>(lds + 2 * (kX + kW)) + wave * 4 * WR;
  auto store = [&](const Tile& tile) {
    const int64_t n = tile.row0 + (wave % NR) * WR + lane % kLanes * kEach;
    const int count = static_cast<int>(max(static_cast<int64_t>(0), min(a.rows - n, static_cast<int64_t>(kEach))));
    float scale[kEach], bias[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      scale[i] = i < count ? a.scales[n + i] : 0.0f;
      bias[i] = a.bias && i < count ? a.bias[n + i] : 0.0f;
    }
    constexpr int kStores = 16 * kLanes / 64;  // of a block of vectors
    float x_scales[BT][kStores];
#pragma unroll
    for (int t = 0; t < BT; ++t)
#pragma unroll
      for (int g = 0; g < kStores; ++g)
        x_scales[t][g] = a.x_scales[min(tile.token0 + (wave / NR) * WT + t * 16 + g * (64 / kLanes) + lane / kLanes, a.tokens - 1)];
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): no load is left for the loop to wait for
#pragma unroll
    for (int t = 0; t < BT; ++t) {
#pragma unroll
      for (int r = 0; r < BR; ++r) sums[in_block * (WR / 4) + ((r * 4 + q) ^ in_block)] = acc[t][r];
      // LDS serves a wave in order; only the compiler must keep it
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
#pragma unroll
      for (int g = 0; g < kStores; ++g) {
        const int in = g * (64 / kLanes) + lane / kLanes;
        const int64_t m = tile.token0 + (wave / NR) * WT + t * 16 + in;
        if (m >= a.tokens || count == 0) continue;
        const float x_scale = x_scales[t][g];
        float v[8];
#pragma unroll
        for (int c = 0; c < kEach / 4; ++c) {
          const i32x4 sum = sums[in * (WR / 4) + ((lane % kLanes * (kEach / 4) + c) ^ in)];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[4 * c + i] = fmaf(static_cast<float>(sum[i]) * x_scale, scale[4 * c + i], bias[4 * c + i]);
        }
        const int64_t at = m * a.rows + n;
        if (count == kEach) {
          if constexpr (YT == ST_SCORE_F32) {
            *reinterpret_cast<u32x4_by4*>(static_cast<float*>(a.y) + at) =
                u32x4_by4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
          } else {
            store8<YT>(a.y, at, v);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kEach; ++i)
            if (i < count) store_score<YT>(a.y, at + i, v[i]);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    }
  };

  aim();
#pragma unroll
  for (int i = 0; i < kMoves; ++i) bring(i);
  brought();
  settle(0, 0);
  barrier();
  if (bring_id < all) {
#pragma unroll
    for (int i = 0; i < kMoves; ++i) bring(i);
    brought();
  }
#pragma unroll
  for (int r = 0; r < BR; ++r) read_w(0, 0, r);
#pragma unroll
  for (int t = 0; t < kAhead; ++t) read_x(0, 0, t);
  clear();
  int64_t id = blockIdx.x;
  int part = 0, buffer = 0;
#pragma unroll 1
  while (true) {
    const int next_part = part + 1 < parts ? part + 1 : 0;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int step = g / BT, t = g % BT;
      if (g == kTurn) {
        settle(next_part, buffer ^ 1);
        barrier();
      }
      // reads: the block kAhead groups on; the next step's rows
      if (g < kTurn)
        read_x(buffer, (g + kAhead) / BT, (g + kAhead) % BT);
      else
        read_x(buffer ^ 1, 0, g - kTurn);
      if (step == 0) {
#pragma unroll
        for (int r = t * BR / BT; r < (t + 1) * BR / BT; ++r) read_w(buffer, 1, r);
      } else if (g == kTurn) {
#pragma unroll
        for (int r = 0; r < BR; ++r) read_w(buffer ^ 1, 0, r);
      }
#pragma unroll
      for (int r = 0; r < BR; ++r)
        acc[t][r] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[step][r], fx[t & 3], acc[t][r], 0, 0, 0);
      // the part after the next, into this one's buffer
      if (g >= kTurn && bring_id < all) {
#pragma unroll
        for (int i = (g - kTurn) * kMoves / kAhead; i < (g - kTurn + 1) * kMoves / kAhead; ++i) bring(i);
        if (g == kGroups - 1) brought();
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    buffer ^= 1;
    part = next_part;
    if (part != 0) continue;
    store(tile_of(id));
    id += gridDim.x;
    if (id >= all) break;
    clear();
  }
}

template <int YT, int WT, int WR, int NT, int NR>
void launch_many_as(const MatmulArgs& a, hipStream_t s) {
  constexpr int kLds = 2 * (NT * WT + NR * WR) * 128 + NT * NR * 64 * WR;
  const auto kernel = many_kernel<YT, WT, WR, NT, NR>;
  static std::once_flag once;
  std::call_once(once, [&] {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e != hipSuccess) throw Error(ST_ERR_HIP, cat("hipFuncSetAttribute failed: ", hipGetErrorString(e)));
  });
  const int64_t tiles = ((a.tokens + NT * WT - 1) / (NT * WT)) * ((a.rows + NR * WR - 1) / (NR * WR));
  const int64_t grid = std::min<int64_t>(tiles, cu_count() * (160 * 1024 / kLds));
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(64 * NT * NR), kLds, s, a);
}

template <int WT, int WR, int NT, int NR>
void launch_many(const MatmulArgs& a, hipStream_t s) {
  if (a.y_type == ST_SCORE_F32)
    launch_many_as<ST_SCORE_F32, WT, WR, NT, NR>(a, s);
  else if (a.y_type == ST_SCORE_F16)
    launch_many_as<ST_SCORE_F16, WT, WR, NT, NR>(a, s);
  else
    launch_many_as<ST_SCORE_BF16, WT, WR, NT, NR>(a, s);
}

// Whether the product takes the vectors to 8 bits itself: each workgroup does it
// again, so they have to be few; a launch of its own (about 4 us) does it
// otherwise.
bool is_fused(int x_type, int64_t tokens, int64_t columns) {
  return x_type != ST_CODE_I8 && tokens <= 16 && (columns + 255) / 256 * 256 * 16 <= kFusedBytes;
}

void check_codes(int64_t rows, int64_t columns) {
  ST_CHECK(rows >= 0, "negative number of rows");
  ST_CHECK(columns >= 16 && columns % 16 == 0 && columns <= kMaxColumns,
           "rows of codes are whole blocks of 16 columns, at most ", kMaxColumns, ", got ", columns);
}

void check_type(int type, const char* what) {
  ST_CHECK(type == ST_SCORE_F32 || type == ST_SCORE_F16 || type == ST_SCORE_BF16, what,
           " must be float32, float16 or bfloat16");
}

void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw Error(ST_ERR_HIP, cat(what, " launch failed: ", hipGetErrorString(e)));
}

// Vectors of more columns than the norm's kernels hold: a workgroup each, which
// reads them twice.
template <int DT>
__global__ __launch_bounds__(1024) void long_codes_kernel(const void* x, int64_t x_stride, int dim, int columns, int8_t* codes,
                                                          float* scales) {
  __shared__ float room[16];
  const char* row = static_cast<const char*>(x) + blockIdx.x * x_stride * kScoreBytes<DT>;
  float most = 0.0f, odd = 0.0f, v[8];
  for (int col = threadIdx.x * 8; col < dim; col += 8192) {
    load_eight<DT>(row, col, dim, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      most = fmaxf(most, fabsf(v[i]));
      odd = fmaf(v[i], 0.0f, odd);
    }
  }
  most = wave_max(odd != odd ? __builtin_inff() : most);
  if (threadIdx.x % 64 == 0) room[threadIdx.x / 64] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 16; ++w) most = fmaxf(most, room[w]);
  const CodeScale c = code_scale(most);
  if (threadIdx.x == 0) scales[blockIdx.x] = c.scale;
  for (int col = threadIdx.x * 8; col < columns; col += 8192) {
    load_eight<DT>(row, col, dim, v);
    *reinterpret_cast<uint64_t*>(codes + static_cast<int64_t>(blockIdx.x) * columns + col) = codes8(v, c);
  }
}

void quantize(const void* x, int x_type, int64_t rows, int64_t dim, int64_t x_stride, int8_t* codes, float* scales,
              hipStream_t s) {
  const int64_t columns = (dim + 15) / 16 * 16;
  if (dim <= kMaxNormColumns) {
    launch_codes(x, x_type, rows, dim, x_stride, codes, columns, scales, s);
    return;
  }
  const int64_t most = 1 << 21;  // rows a launch: 2^31 threads
  for (int64_t at = 0; at < rows; at += most) {
    const dim3 grid(static_cast<unsigned>(std::min(most, rows - at)));
    const char* from = static_cast<const char*>(x) + at * x_stride * (x_type == ST_SCORE_F32 ? 4 : 2);
    int8_t* to = codes + at * columns;
    const int d = static_cast<int>(dim), c = static_cast<int>(columns);
    if (x_type == ST_SCORE_F32)
      hipLaunchKernelGGL((long_codes_kernel<ST_SCORE_F32>), grid, dim3(1024), 0, s, from, x_stride, d, c, to, scales + at);
    else if (x_type == ST_SCORE_F16)
      hipLaunchKernelGGL((long_codes_kernel<ST_SCORE_F16>), grid, dim3(1024), 0, s, from, x_stride, d, c, to, scales + at);
    else
      hipLaunchKernelGGL((long_codes_kernel<ST_SCORE_BF16>), grid, dim3(1024), 0, s, from, x_stride, d, c, to, scales + at);
    check_launch("long_codes_kernel");
  }
}

int64_t codes_bytes(int64_t tokens, int64_t columns) { return (tokens * columns + 255) / 256 * 256; }

}  // namespace
}  // namespace st

extern "C" int64_t st_int8_columns(int64_t dim) { return (dim + 15) / 16 * 16; }

extern "C" int st_int8_quantize(const void* x, int x_type, int64_t rows, int64_t dim, int64_t x_stride, int8_t* codes,
                                float* scales, void* stream) {
  using namespace st;
  return guarded([&] {
    check_type(x_type, "x");
    ST_CHECK(dim >= 1, "a row has at least one column, got ", dim);
    check_codes(rows, st_int8_columns(dim));
    if (rows == 0) return;
    ST_CHECK(x && codes && scales, "null device pointer");
    ST_CHECK(reinterpret_cast<uintptr_t>(codes) % 16 == 0, "codes must be 16-byte aligned");
    quantize(x, x_type, rows, dim, x_stride, codes, scales, static_cast<hipStream_t>(stream));
  });
}

extern "C" int64_t st_int8_matmul_workspace_bytes(int x_type, int64_t tokens, int64_t columns) {
  using namespace st;
  if (x_type == ST_CODE_I8 || tokens <= 0 || columns <= 0 || is_fused(x_type, tokens, columns)) return 0;
  return codes_bytes(tokens, columns) + tokens * static_cast<int64_t>(sizeof(float));
}

extern "C" int st_int8_matmul(const int8_t* codes, const float* scales, int64_t rows, int64_t columns, const void* x,
                              int x_type, const float* x_scales, int64_t tokens, int64_t dim, int64_t x_stride,
                              const float* bias, void* y, int y_type, void* workspace, void* stream) {
  using namespace st;
  return guarded([&] {
    if (x_type != ST_CODE_I8) check_type(x_type, "x");
    check_type(y_type, "the result");
    check_codes(rows, columns);
    ST_CHECK(tokens >= 0, "negative number of vectors");
    ST_CHECK(dim >= 1 && st_int8_columns(dim) == columns, "the table's rows have ", columns, " columns, vectors of ", dim,
             " take ", st_int8_columns(dim));
    ST_CHECK(x_type != ST_CODE_I8 || (dim == columns && x_stride == columns), "vectors of codes are whole rows side by side");
    if (rows == 0 || tokens == 0) return;
    ST_CHECK(codes && scales && x && y, "null device pointer");
    ST_CHECK(reinterpret_cast<uintptr_t>(codes) % 16 == 0, "the table must be 16-byte aligned");
    ST_CHECK(x_type != ST_CODE_I8 || (x_scales && reinterpret_cast<uintptr_t>(x) % 16 == 0),
             "vectors of codes come with scales and must be 16-byte aligned");
    hipStream_t s = static_cast<hipStream_t>(stream);
    MatmulArgs a{codes, scales, bias, x, x_scales, y, rows, tokens, x_stride, static_cast<int>(dim), static_cast<int>(columns),
                 x_type, y_type};
    if (is_fused(x_type, tokens, columns)) {
      launch_few<1, true>(a, s);
      check_launch("few_kernel");
      return;
    }
    if (x_type != ST_CODE_I8) {
      ST_CHECK(workspace, "null device pointer");
      int8_t* made = static_cast<int8_t*>(workspace);
      float* made_scales = reinterpret_cast<float*>(made + codes_bytes(tokens, columns));
      quantize(x, x_type, tokens, dim, x_stride, made, made_scales, s);
      a.x = made;
      a.x_scales = made_scales;
      a.x_type = ST_CODE_I8;
      a.x_stride = columns;
      a.dim = static_cast<int>(columns);
    }
    if (tokens > 64 && columns >= 256) {
      if (((tokens + 255) / 256) * ((rows + 255) / 256) >= cu_count() / 2)
        launch_many<128, 64, 2, 4>(a, s);
      else
        launch_many<64, 64, 2, 2>(a, s);
      check_launch("many_kernel");
      return;
    }
    if (tokens <= 16)
      launch_few<1, false>(a, s);
    else if (tokens <= 32)
      launch_few<2, false>(a, s);
    else
      launch_few<4, false>(a, s);
    check_launch("few_kernel");
  });
}
