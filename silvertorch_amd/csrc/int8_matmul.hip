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
constexpr int kFewTokens = 4, kFewColumns = 2048;  // of few_kernel
constexpr int64_t kFewBytes = 32 << 20;              // of its table

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

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
__device__ __forceinline__ float codes_to_lds(const void* row, int dim, int padded, uint8_t* to) {
  const int lane = threadIdx.x % 64;
  float most = 0.0f, v[8];
  for (int col = lane * 8; col < dim; col += 512) {
    load_eight<DT>(row, col, dim, v);
    most = most_of8(most, v);
  }
  const CodeScale c = code_scale(wave_max(most_or_infinity(most)));
  for (int col = lane * 8; col < padded; col += 512) {
    load_eight<DT>(row, col, dim, v);
    *reinterpret_cast<uint64_t*>(to + (col >> 6) * 1024 + ((col >> 4) & 3) * 256 + (col & 15)) = codes8(v, c);
  }
  return c.scale;
}

// One to four vectors of floats against a table of a few megabytes, where a launch
// counts: every workgroup takes the vectors to 8 bits itself, into LDS, while its
// first rows are on their way.  R blocks of 16 rows a wave, J steps of 64 columns at a
// time, straight from memory to registers; with SPLIT four waves share a row's
// columns.
template <int R, int J, bool SPLIT>
__global__ __launch_bounds__(kThreads) void few_kernel(MatmulArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ float x_scales[kFewTokens];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, q = lane / 16, c = lane % 16;
  const int tokens = static_cast<int>(a.tokens);
  const int steps = (a.columns + 64 * J - 1) / (64 * J);  // of J times 64 columns

  const int64_t tiles = (a.rows + 16 * R - 1) / (16 * R);
  const int64_t tile_step = static_cast<int64_t>(gridDim.x) * (SPLIT ? 1 : kWaves);
  int64_t tile = SPLIT ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * kWaves + wave;
  const int first_step = SPLIT ? wave : 0;
  constexpr int kStepStep = SPLIT ? kWaves : 1;
  struct Step {
    i32x4 w[R][J];
  };
  auto load = [&](int64_t at, int step, Step& s) {
    at = min(at, tiles - 1);
    const int64_t row0 = at * (16 * R);
    const int8_t* table = a.codes + row0 * a.columns;
    const int last = static_cast<int>(min(a.rows - row0, static_cast<int64_t>(16 * R))) - 1;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int k = (step * J + j) * 64 + q * 16;
#pragma unroll
      for (int r = 0; r < R; ++r)
        // rows past the last and columns past theirs read others; the former's
        // results are not stored, the latter meet zeros of x
        s.w[r][j] = *reinterpret_cast<const i32x4*>(table + static_cast<int64_t>(min(16 * r + c, last)) * a.columns + (k < a.columns ? k : 0));
    }
  };
  Step next;
  load(tile, min(first_step, steps - 1), next);

  if (wave < tokens) {
    const int64_t row = wave * a.x_stride;
    float scale;
    if (a.x_type == ST_SCORE_F32)
      scale = codes_to_lds<ST_SCORE_F32>(static_cast<const float*>(a.x) + row, a.dim, steps * J * 64, lds + wave * 16);
    else if (a.x_type == ST_SCORE_F16)
      scale = codes_to_lds<ST_SCORE_F16>(static_cast<const uint16_t*>(a.x) + row, a.dim, steps * J * 64, lds + wave * 16);
    else
      scale = codes_to_lds<ST_SCORE_BF16>(static_cast<const uint16_t*>(a.x) + row, a.dim, steps * J * 64, lds + wave * 16);
    if (lane == 0) x_scales[wave] = scale;
  }
  __syncthreads();

  auto put = [&](int m, int64_t n, int sum) {
    store_typed(a.y, m * a.rows + n, fmaf(static_cast<float>(sum) * x_scales[m], a.scales[n], a.bias ? a.bias[n] : 0.0f), a.y_type);
  };
  for (; tile < tiles; tile += tile_step) {
    i32x4 acc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = i32x4{0, 0, 0, 0};
    for (int step = first_step; step < steps; step += kStepStep) {
      const Step now = next;
      const bool more = step + kStepStep < steps;
      load(more ? tile : tile + tile_step, more ? step + kStepStep : min(first_step, steps - 1), next);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        // vectors past the last hold whatever LDS does; their sums are not stored
        const i32x4 x = *reinterpret_cast<const i32x4*>(lds + (step * J + j) * 1024 + lane * 16);
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, now.w[r][j], acc[r], 0, 0, 0);
      }
    }
    // vector m's sums lie in element m of the first 16 lanes
    const int64_t row0 = tile * (16 * R);
    if constexpr (SPLIT) {
      static_assert(R == 1 && kWaves == kFewTokens, "");
      int* sums = reinterpret_cast<int*>(lds + steps * J * 1024);
      if (q == 0) *reinterpret_cast<i32x4*>(sums + (wave * 16 + c) * 4) = acc[0];
      __syncthreads();
      // vector `wave` by wave `wave`
      if (q == 0 && wave < tokens && row0 + c < a.rows) {
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += sums[(w * 16 + c) * 4 + wave];
        put(wave, row0 + c, sum);
      }
      __syncthreads();
    } else {
      static_assert(R == 4, "");
      const int64_t n = row0 + lane;
#pragma unroll
      for (int i = 0; i < kFewTokens; ++i) {
        if (i >= tokens) break;
        // 64 rows side by side
        const u32x4 v = transpose4(u32x4{static_cast<uint32_t>(acc[0][i]), static_cast<uint32_t>(acc[1][i]),
                                         static_cast<uint32_t>(acc[2][i]), static_cast<uint32_t>(acc[3][i])});
        if (n < a.rows) put(i, n, static_cast<int>(v[0]));
      }
    }
  }
}

// Too few rows for as many waves as hide a load's latency: four share a row.
bool few_split(const MatmulArgs& a) { return a.columns >= 1024 && (a.rows + 63) / 64 < 8 * cu_count(); }

void launch_few(const MatmulArgs& a, hipStream_t s) {
  const bool split = few_split(a);
  const int64_t groups = split ? (a.rows + 15) / 16 : (a.rows + 64 * kWaves - 1) / (64 * kWaves);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(groups, 4 * cu_count())));
  const size_t padded = split ? (a.columns + 255) / 256 * 256 : (a.columns + 63) / 64 * 64;
  if (split)
    hipLaunchKernelGGL((few_kernel<1, 4, true>), grid, dim3(kThreads), padded * 16 + kWaves * 256, s, a);
  else
    hipLaunchKernelGGL((few_kernel<4, 1, false>), grid, dim3(kThreads), padded * 16, s, a);
}

// Many vectors: the matrix units bound it, 0.56 of whose cycles issue a product, and
// the power they draw (16,384 x 4,096 x 8,192: 472 us at 1.8 to 2.0 GHz, 400 on zeros,
// where the clock stays at 2.4, in as many cycles).  From registers alone 16x16x64
// blocks run at 4,840 TOP/s on zeros and 4,070 on random codes, 32x32x32
// ones at 3,290 and 2,600.  A workgroup of NT x NR waves takes tiles of
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
  static_assert(kAtOnce % 16 == 0 && kGroups % 4 == 0 && kGroups > kAhead, "");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int q = lane / 16, in_block = lane % 16;
  const int parts = (a.columns + 127) / 128;

  // Tiles in an order that shares the last-level caches: an eighth of them to
  // each of the 8 dies (workgroups go round them), there 8 tiles of vectors by
  // one of rows after another.
  const uint32_t tiles_t = static_cast<uint32_t>((a.tokens + kTokens - 1) / kTokens);
  const uint32_t tiles_r = static_cast<uint32_t>((a.rows + kRows - 1) / kRows), all = tiles_t * tiles_r;
  struct Tile {
    int64_t token0, row0;
  };
  auto tile_of = [&](uint32_t id) {
    const uint32_t die = id % 8;
    id = die * (all / 8) + min(die, all % 8) + id / 8;
    const uint32_t group = id / (8 * tiles_r), within = id - group * (8 * tiles_r);
    const uint32_t height = min(8u, tiles_t - group * 8), column = within / height;
    return Tile{static_cast<int64_t>(group * 8 + (within - column * height)) * kTokens, static_cast<int64_t>(column) * kRows};
  };

  // What a wave brings: 8 rows a load, lane l the chunk that belongs at place l % 8
  // of row kAtOnce i + 8 wave + l / 8 (f of rows 16 apart is the same).  Rows past the
  // last read it again; their sums are not stored.
  const auto place = [](int row) { return (row >> 1) & 7; };
  const int first_row = wave * 8 + lane / 8, chunk = (lane % 8) ^ place(first_row);
  // Columns past the last are read at the part's start, and of the vectors zeros put
  // in their places once they are there (`settle`).
  const int past = (parts - 1) * 128 + chunk * 16 >= a.columns ? chunk * 16 : 0;
  uint32_t bring_id = blockIdx.x;  // the tile and the part that are brought next, and its buffer
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
  // Waits for what this wave brought, and for its reads of LDS; not for `stored`
  // stores that it issued since.
  auto settle = [&](int part, int buffer, int stored) {
    constexpr int kFull = BT * (16 * (WR / (YT == ST_SCORE_F32 ? 4 : 8)) / 64);
    if (stored == 0)
      __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0)
    else if (stored == 1)
      __builtin_amdgcn_s_waitcnt(0x0071);
    else
      __builtin_amdgcn_s_waitcnt(0x0070 | (kFull & 15) | ((kFull & 0x30) << 10));
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
    fx[(step * BT + t) & 3] = *reinterpret_cast<const i32x4*>(lds + buffer * kX + x_row * 128 + (((step * 4 + q) ^ place(x_row)) * 16) + t * 2048);
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
  // sums times the vectors' scales, chunk c of 4 at place c ^ vector, so that a store
  // writes whole lines of a result's row (16 bytes here and there, straight from the
  // sums: 620 us for 16,384 x 4,096 x 8,192 where this took 509).
  constexpr int kEach = YT == ST_SCORE_F32 ? 4 : 8;  // results a lane stores at once, 16 bytes
  constexpr int kLanes = WR / kEach;                 // of a vector's
  constexpr int kStores = 16 * kLanes / 64;          // of a block of vectors
  f32x4* sums = reinterpret_cast<f32x4*>(lds + 2 * (kX + kW)) + wave * 4 * WR;
  float scale[kEach], bias[kEach], x_scale[BT];
  Tile now;
  int64_t n;
  int count;
  // What a tile's results need, a part ahead: a load after the next parts' would
  // have to wait for them.
  auto prepare = [&](uint32_t id) {
    now = tile_of(id);
    const int here = (wave % NR) * WR + lane % kLanes * kEach;
    n = now.row0 + here;
    count = max(0, min(static_cast<int>(min(a.rows - now.row0, static_cast<int64_t>(kRows))) - here, kEach));
    const float* scales = a.scales + now.row0;
    const float* biases = (a.bias ? a.bias : a.scales) + now.row0;
    if (count == kEach) {
#pragma unroll
      for (int i = 0; i < kEach; i += 4) {
        const u32x4_by4 s = *reinterpret_cast<const u32x4_by4*>(scales + here + i), b = *reinterpret_cast<const u32x4_by4*>(biases + here + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          scale[i + e] = __uint_as_float(s[e]);
          bias[i + e] = __uint_as_float(b[e]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        scale[i] = i < count ? scales[here + i] : 0.0f;
        bias[i] = i < count ? biases[here + i] : 0.0f;
      }
    }
    const float* x_scales = a.x_scales + now.token0;
    const int last_token = static_cast<int>(min(a.tokens - now.token0, static_cast<int64_t>(kTokens))) - 1;
#pragma unroll
    for (int t = 0; t < BT; ++t) x_scale[t] = x_scales[min((wave / NR) * WT + t * 16 + in_block, last_token)];
  };
  // Returns how many stores this wave has certainly issued, none or all of a full
  // tile's or one.
  auto store = [&] {
#pragma unroll
    for (int i = 0; i < kEach; ++i) bias[i] = a.bias ? bias[i] : 0.0f;
    const int64_t m0 = now.token0 + (wave / NR) * WT;
    const int tokens = static_cast<int>(max(static_cast<int64_t>(0), min(a.tokens - m0, static_cast<int64_t>(WT))));
#pragma unroll
    for (int t = 0; t < BT; ++t) {
      if (t * 16 >= tokens) break;
#pragma unroll
      for (int r = 0; r < BR; ++r) {
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(acc[t][r][i]) * x_scale[t];
        sums[in_block * (WR / 4) + ((r * 4 + q) ^ (in_block & (WR / 4 - 1)))] = v;
      }
      // LDS serves a wave in order; only the compiler must keep to it
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
#pragma unroll
      for (int g = 0; g < kStores; ++g) {
        const int in = g * (64 / kLanes) + lane / kLanes;
        if (t * 16 + in >= tokens || count == 0) continue;
        float v[8];
#pragma unroll
        for (int c = 0; c < kEach / 4; ++c) {
          const f32x4 sum = sums[in * (WR / 4) + ((lane % kLanes * (kEach / 4) + c) ^ (in & (WR / 4 - 1)))];
#pragma unroll
          for (int i = 0; i < 4; ++i) v[4 * c + i] = fmaf(sum[i], scale[4 * c + i], bias[4 * c + i]);
        }
        const int64_t at = (m0 + t * 16 + in) * a.rows + n;
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
    if (now.row0 + (wave % NR) * WR + WR > a.rows || tokens == 0) return 0;
    return tokens == WT ? BT * kStores : 1;
  };

  aim();
#pragma unroll
  for (int i = 0; i < kMoves; ++i) bring(i);
  brought();
  settle(0, 0, 0);
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
  uint32_t id = blockIdx.x;
  int part = 0, buffer = 0, stored = 0;
#pragma unroll 1
  while (true) {
    const int next_part = part + 1 < parts ? part + 1 : 0;
    if (next_part == 0) prepare(id);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int step = g / BT, t = g % BT;
      if (g == kTurn) {
        settle(next_part, buffer ^ 1, stored);
        stored = 0;
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
        acc[t][r] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[step][r], fx[g & 3], acc[t][r], 0, 0, 0);
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
    stored = store();
    id += gridDim.x;
    if (id >= all) break;
    clear();
  }
}

// Parts of a wave in long_kernel: what 160 KB hold of eight waves'.
constexpr int long_depth(int blocks) { return blocks == 1 ? 3 : 2; }

// Few results of long rows, where tiles of all columns would leave most of the
// chip idle: a workgroup takes 16 TB vectors x 32 rows, and its eight waves take
// turns with the parts of 128 columns, each by itself, `kDepth` parts in LDS or on
// the way to it; no barrier but the one before their sums are added.
template <int YT, int TB>
__global__ __launch_bounds__(512) void long_kernel(MatmulArgs a) {
  constexpr int kSplit = 8, kRows = 32;
  constexpr int LT = 2 * TB, kMoves = LT + kRows / 8;  // loads of 8 rows
  constexpr int kBuffer = kMoves * 1024, kDepth = long_depth(TB);
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int q = lane / 16, in_block = lane % 16;
  const int64_t token0 = static_cast<int64_t>(blockIdx.y) * (16 * TB), row0 = static_cast<int64_t>(blockIdx.x) * kRows;
  const int8_t* x = static_cast<const int8_t*>(a.x) + token0 * a.columns;
  const int8_t* w = a.codes + row0 * a.columns;
  const int last_token = static_cast<int>(min(a.tokens - token0, static_cast<int64_t>(16 * TB))) - 1;
  const int last_row = static_cast<int>(min(a.rows - row0, static_cast<int64_t>(kRows))) - 1;
  const int parts = (a.columns + 127) / 128;

  // rows and chunks as in many_kernel
  const auto place = [](int row) { return (row >> 1) & 7; };
  uint8_t* own = lds + wave * kDepth * kBuffer;
  uint32_t from[kMoves];
  int chunk[2];  // of even and odd loads: rows 8 apart are at other places
#pragma unroll
  for (int i = 0; i < 2; ++i) chunk[i] = (lane % 8) ^ place(8 * i + lane / 8);
#pragma unroll
  for (int i = 0; i < kMoves; ++i) {
    const int row = i < LT ? min(8 * i + lane / 8, last_token) : min(8 * (i - LT) + lane / 8, last_row);
    from[i] = static_cast<uint32_t>(row) * a.columns + chunk[i & 1] * 16;
  }
  auto past = [&](int part, int i) { return part * 128 + chunk[i & 1] * 16 >= a.columns; };
  auto bring = [&](int part, int buffer) {
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      const int8_t* base = (i < LT ? x : w) + static_cast<int64_t>(part) * 128;
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(base + (from[i] - (past(part, i) ? chunk[i & 1] * 16 : 0))),
          (__attribute__((address_space(3))) void*)(own + buffer * kBuffer + i * 1024), 16, 0, 0);
    }
  };

  i32x4 acc[TB][2];
#pragma unroll
  for (int t = 0; t < TB; ++t)
#pragma unroll
    for (int r = 0; r < 2; ++r) acc[t][r] = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int d = 0; d < kDepth - 1; ++d)
    if (wave + d * kSplit < parts) bring(wave + d * kSplit, d);
  int buffer = 0;
#pragma unroll 1
  for (int part = wave; part < parts; part += kSplit, buffer = buffer + 1 < kDepth ? buffer + 1 : 0) {
    if (part + (kDepth - 1) * kSplit < parts) {
      bring(part + (kDepth - 1) * kSplit, buffer > 0 ? buffer - 1 : kDepth - 1);
      constexpr int kLater = (kDepth - 1) * kMoves;  // loads issued after this part's
      __builtin_amdgcn_s_waitcnt(0x0f70 | (kLater & 15) | ((kLater & 0x30) << 10));
    } else {
      __builtin_amdgcn_s_waitcnt(0x0f70);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    uint8_t* here = own + buffer * kBuffer;
    if (part == parts - 1 && a.columns % 128 != 0) {
#pragma unroll
      for (int i = 0; i < LT; ++i)
        if (past(part, i)) *reinterpret_cast<i32x4*>(here + i * 1024 + lane * 16) = i32x4{0, 0, 0, 0};
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    }
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      i32x4 fx[TB], fw[2];
      const int at = in_block * 128 + (((step * 4 + q) ^ place(in_block)) * 16);
#pragma unroll
      for (int r = 0; r < 2; ++r) fw[r] = *reinterpret_cast<const i32x4*>(here + (LT + 2 * r) * 1024 + at);
#pragma unroll
      for (int t = 0; t < TB; ++t) fx[t] = *reinterpret_cast<const i32x4*>(here + 2 * t * 1024 + at);
#pragma unroll
      for (int t = 0; t < TB; ++t)
#pragma unroll
        for (int r = 0; r < 2; ++r) acc[t][r] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[r], fx[t], acc[t][r], 0, 0, 0);
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the buffer is free for the next loads
  }

  // The waves' sums: block (t, r) of wave v at 256 numbers from (v TB + t) 2 + r on.
  __syncthreads();
  i32x4* sums = reinterpret_cast<i32x4*>(lds);
#pragma unroll
  for (int t = 0; t < TB; ++t)
#pragma unroll
    for (int r = 0; r < 2; ++r) sums[((wave * TB + t) * 2 + r) * 64 + lane] = acc[t][r];
  __syncthreads();
  const int64_t n = row0 + threadIdx.x % 32;
  if (n >= a.rows) return;
  const float scale = a.scales[n], bias = a.bias ? a.bias[n] : 0.0f;
#pragma unroll
  for (int t = 0; t < TB; ++t) {
    const int64_t m = token0 + t * 16 + threadIdx.x / 32;
    if (m >= a.tokens) break;
    const int r = threadIdx.x % 32 / 16, of = threadIdx.x % 16;
    int sum = 0;
#pragma unroll
    for (int v = 0; v < kSplit; ++v)
      sum += reinterpret_cast<const int*>(sums)[(((v * TB + t) * 2 + r) * 64 + of / 4 * 16 + threadIdx.x / 32) * 4 + of % 4];
    store_score<YT>(a.y, m * a.rows + n, fmaf(static_cast<float>(sum) * a.x_scales[m], scale, bias));
  }
}

template <int YT, int TB>
void launch_long_as(const MatmulArgs& a, hipStream_t s) {
  constexpr int kLds = 8 * long_depth(TB) * (2 * TB + 4) * 1024;
  const auto kernel = long_kernel<YT, TB>;
  static std::once_flag once;
  std::call_once(once, [&] {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e != hipSuccess) throw Error(ST_ERR_HIP, cat("hipFuncSetAttribute failed: ", hipGetErrorString(e)));
  });
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((a.rows + 31) / 32), static_cast<unsigned>((a.tokens + 16 * TB - 1) / (16 * TB))),
                     dim3(512), kLds, s, a);
}

template <int TB>
void launch_long(const MatmulArgs& a, hipStream_t s) {
  if (a.y_type == ST_SCORE_F32)
    launch_long_as<ST_SCORE_F32, TB>(a, s);
  else if (a.y_type == ST_SCORE_F16)
    launch_long_as<ST_SCORE_F16, TB>(a, s);
  else
    launch_long_as<ST_SCORE_BF16, TB>(a, s);
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
  ST_CHECK(tiles < (1ll << 31), "the product has too many results");
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

// Whether the product takes the vectors to 8 bits itself (few_kernel) where a launch
// of its own does otherwise.  Four vectors: 8,192 x 2,048 6.5 us and 20,000 x 512 7.1
// us, 8 us with that launch (4 us); but 500,000 x 128, 64 MB, 17.6 us as well, and one
// vector x 4,096 x 4,096 8.9 us against 7.3.
bool is_fused(int x_type, int64_t tokens, int64_t rows, int64_t columns) {
  return x_type != ST_CODE_I8 && tokens <= kFewTokens && columns <= kFewColumns && rows <= kFewBytes / columns;
}

// The kernel for codes on both sides.
//
// Few results of long rows go to long_kernel: 64 x 4,096 x 8,192 12.1 us (20.9 in
// tiles of 32 x 128), 40 x 1,024 x 8,192 5.6 (6.4), 16 x 512 x 8,192 4.0 (4.1); but 96 x
// 8,192 x 8,192 47 (36.5), 32 x 512 x 16,384 5.8 (4.6).
//
// Else the tile whose rounds over the chip take least: `full` with as many
// workgroups as it holds, `first` for less than one a CU and nothing before, `last` for
// that after full rounds (two a CU of three: `two`), in hundredths of a round of
// 256 x 256.  In tiles of 256 x 256, 128 x 128, 64 x 128 and 32 x 128: 200 x 128 x 500,000
// 56, 65, 79 and 91 us; 64 x 2,048 x 50,000 29, 20.5, 18 and 26; 4,097 x 4,096 x 4,096 100,
// 85, 107 and 130; 2,048 x 4,096 x 4,096 53, 40, 48 and 66; 300 x 4,096 x 4,096 47, 22, 17
// and 20; 512 x 512 x 4,096 12.3, 7.0, 5.7 and 5.7; one vector x 128 x 20,000,000 868,
// 669, 632 and 573.
void launch_codes_product(const MatmulArgs& a, hipStream_t s) {
  const int64_t cus = cu_count();
  auto tiles = [&](int64_t tokens, int64_t rows) { return ((a.tokens + tokens - 1) / tokens) * ((a.rows + rows - 1) / rows); };
  const int64_t groups = tiles(32, 32);
  if ((groups <= cus && a.columns >= 256) || (groups <= 2 * cus && a.columns >= 1024)) {
    if (a.tokens <= 16)
      launch_long<1>(a, s);
    else
      launch_long<2>(a, s);
    return;
  }
  auto cost = [&](int64_t count, int per_cu, int full, int first, int last, int two) {
    const int64_t rounds = count / (per_cu * cus), rest = count % (per_cu * cus);
    return rounds * full + (rest == 0 ? 0 : rest > 2 * cus ? full : rest > cus ? two : rounds == 0 ? first : last);
  };
  const int64_t of_256 = cost(tiles(256, 256), 1, 100, 100, 100, 100), of_128 = cost(tiles(128, 128), 2, 70, 50, 30, 70);
  const int64_t of_64 = cost(tiles(64, 128), 2, 46, 35, 33, 46), of_32 = cost(tiles(32, 128), 3, 48, 28, 28, 42);
  const int64_t least = std::min(std::min(of_256, of_128), std::min(of_64, of_32));
  if (of_256 == least)
    launch_many<128, 64, 2, 4>(a, s);
  else if (of_128 == least)
    launch_many<64, 64, 2, 2>(a, s);
  else if (of_64 == least)
    launch_many<64, 32, 1, 4>(a, s);
  else
    launch_many<32, 32, 1, 4>(a, s);
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
// reads them twice (3,000 x 40,000 bfloat16 86 us).
template <int DT>
__global__ __launch_bounds__(1024) void long_codes_kernel(const void* x, int64_t x_stride, int dim, int columns, int8_t* codes,
                                                          float* scales) {
  __shared__ float room[16];
  const char* row = static_cast<const char*>(x) + blockIdx.x * x_stride * kScoreBytes<DT>;
  float most = 0.0f, v[8];
  for (int col = threadIdx.x * 8; col < dim; col += 8192) {
    load_eight<DT>(row, col, dim, v);
    most = most_of8(most, v);
  }
  most = wave_max(most_or_infinity(most));
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

extern "C" int64_t st_int8_matmul_workspace_bytes(int x_type, int64_t tokens, int64_t rows, int64_t columns) {
  using namespace st;
  if (x_type == ST_CODE_I8 || tokens <= 0 || rows <= 0 || columns <= 0 || is_fused(x_type, tokens, rows, columns)) return 0;
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
    if (is_fused(x_type, tokens, rows, columns)) {
      launch_few(a, s);
      check_launch("few_kernel");
      return;
    }
    if (x_type != ST_CODE_I8) {
      ST_CHECK(workspace, "null device pointer");
      ST_CHECK(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "the workspace must be 16-byte aligned");
      int8_t* made = static_cast<int8_t*>(workspace);
      float* made_scales = reinterpret_cast<float*>(made + codes_bytes(tokens, columns));
      quantize(x, x_type, tokens, dim, x_stride, made, made_scales, s);
      a.x = made;
      a.x_scales = made_scales;
    }
    launch_codes_product(a, s);
    check_launch("int8_matmul's kernel");
  });
}
