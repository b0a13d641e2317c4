// Matrix-vector products with a table held in 4 bits, and the table's making.
//
// No reference operator.  A table row n has ceil(D / 32) * 16 bytes: column 2j
// in the low half of byte j, column 2j + 1 in the high half.  Each group of
// `group` columns (a multiple of 32; the last may be short) has a scale and,
// with `zeros`, a zero point (else 8):
//   y[b, n] = sum_g scale[n, g] sum_{d in g} (q[n, d] - zero[n, g]) x[b, d]
// What a row's last block of 32 holds past column D is not used.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "score_ops.hpp"
#include "st_errors.hpp"

namespace st {
int cu_count();

namespace {

constexpr int kBlock = 32;  // columns of 16 bytes
constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTileColumns = 64;         // vectors' parts a pass takes
constexpr int kVectorLds = 64 * 1024;       // the vectors' share of LDS, in phases
constexpr int kWholeVectorLds = 128 * 1024;  // or, if they fit at once
constexpr int kMostLds = 160 * 1024 - 512;   // with room for largest[]

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct MatvecArgs {
  const uint8_t* packed;
  const void* scales;
  const uint8_t* zeros;  // null: 8
  const void* x;
  void* y;
  int64_t rows, queries;
  int dim, groups, row_bytes;
  int blocks;            // of 32 columns
  int group_blocks;      // a group's
  uint32_t group_magic;  // block / group_blocks = block * magic >> 32
  int parts;             // float16 parts a vector's element is split into
  int queries_at_once;
  int phase_blocks;      // blocks whose vectors are in LDS at once, a multiple of 16
  int split;             // waves that share a row's columns
  int scale_type, x_type, y_type;
};

__device__ __forceinline__ float load_any(const void* p, int64_t i, int type) {
  if (type == ST_SCORE_F32) return load_score<ST_SCORE_F32>(p, i);
  if (type == ST_SCORE_F16) return load_score<ST_SCORE_F16>(p, i);
  return load_score<ST_SCORE_BF16>(p, i);
}

__device__ __forceinline__ void store_any(void* p, int64_t i, float v, int type) {
  if (type == ST_SCORE_F32)
    store_score<ST_SCORE_F32>(p, i, v);
  else if (type == ST_SCORE_F16)
    store_score<ST_SCORE_F16>(p, i, v);
  else
    store_score<ST_SCORE_BF16>(p, i, v);
}

// Lane groups of 16 and registers transposed: register i of lane group g
// becomes register g of lane group i.
__device__ __forceinline__ u32x4 transpose4(u32x4 d) {
  auto s02 = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false);
  auto s13 = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
  auto s01 = __builtin_amdgcn_permlane16_swap(s02[0], s13[0], false, false);
  auto s23 = __builtin_amdgcn_permlane16_swap(s02[1], s13[1], false, false);
  return u32x4{s01[0], s01[1], s23[0], s23[1]};
}

// Register i: the value of lane group i, in all four groups.
__device__ __forceinline__ u32x4 broadcast4(uint32_t v) {
  auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  auto a = __builtin_amdgcn_permlane16_swap(h[0], h[0], false, false);
  auto b = __builtin_amdgcn_permlane16_swap(h[1], h[1], false, false);
  return u32x4{a[0], a[1], b[0], b[1]};
}

__device__ __forceinline__ half2_t as_half2(uint32_t u) {
  half2_t h;
  __builtin_memcpy(&h, &u, 4);
  return h;
}

// Eight codes less their zero point, exact in float16, in the order 0 4 1 5 2 6
// 3 7.  A code put into the low bits of 1024.0 reads 1024 + q, one four bits
// further up 1024 + 16 q.  low = -(1024 + zero), high = -(64 + zero).
// `base` is 0x64006400 in a vector register: with the mask in a scalar one, and
// and or are one instruction.
__device__ __forceinline__ half8_t codes_of(uint32_t w, uint32_t base, half2_t low, half2_t high) {
  const half2_t sixteenth = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
  const uint32_t v = w >> 8;
  const half2_t a = as_half2((w & 0x000F000Fu) | base) + low;
  const half2_t b = __builtin_elementwise_fma(as_half2((w & 0x00F000F0u) | base), sixteenth, high);
  const half2_t c = as_half2((v & 0x000F000Fu) | base) + low;
  const half2_t d = __builtin_elementwise_fma(as_half2((v & 0x00F000F0u) | base), sixteenth, high);
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The power of two that brings a vector's largest finite element into [2^14,
// 2^15), as an exponent.
__device__ __forceinline__ int shift_of(float largest) {
  if (largest == 0.0f) return 0;
  int e;
  frexpf(largest, &e);
  return min(15 - e, 126);
}

// 2^e for e in [-126, 127]
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Part `part` of an element (x 2^shift): its float16, or what that leaves out
// times 2^11.
__device__ __forceinline__ _Float16 part_of(float x, int part) {
  const _Float16 h = static_cast<_Float16>(x);
  if (part == 0) return h;
  const float left = x - static_cast<float>(h);
  return static_cast<_Float16>(__builtin_isfinite(left) ? left * 2048.0f : 0.0f);
}

// A step's weights of one wave: T tiles of 16 rows by J times 128 columns.
// Lane l reads row l % 16, 16 bytes at block 4 j + l / 16.
template <int T, int J>
struct Step {
  u32x4 w[T][J];
  uint32_t scale[T][J];  // as stored
  uint32_t zero[T][J];
};

// Products on the matrix cores: a wave takes 16 table rows as the columns of a
// 16x16x32 product and up to 16 vectors' parts (C tiles of them) as its rows.
// Vectors are held in LDS as float16, scaled by a power of two that brings the
// largest element to 2^14 or more (undone at the end).  float16's 11 bits and
// its spacing of 2^-24 near zero hold bfloat16 elements exactly down to 2^-31 of
// the largest, to 2^-39 of it below.  float32 ones go in two parts, the second
// 2^11 times as large: what the first leaves out has up to 13 bits with its
// sign, of which float16 holds all but the last of some, so that an element
// keeps 2^-23 of itself (down to 2^-27 of the largest, 2^-50 of it below); the
// rounding of a product in 32 bits is 2^-24.  A third part would hold the last
// bit, for 4 vectors a tile instead of 8.  The parts lie in the order that the
// codes come in.  Codes less zero points are exact in float16; each block of 32
// columns (COARSE: each group, of whole 128 columns) is summed by the matrix
// core in 32 bits and added to the row's sum times its scale in 32 bits.
//
// What bounds it: HBM.  A CU gets some 11 bytes a cycle, 22 codes; unpacking
// takes 9 vector instructions for 8 codes and one matrix instruction 512, so
// both keep up.  Four blocks are read per row (16 rows x 64 bytes a load: a
// row's 16 bytes alone would leave it scattered) and lane groups exchange
// registers (transpose4), which also spreads the scales and zero points (one of
// each per lane and load) over the lanes.  A step is 4 KB: T = 4 tiles of rows
// that are at most 256 columns long, else J = 4 loads along a row, whose columns
// `split` waves share until every CU has work (their sums meet in LDS).  The
// next step's loads are in flight while one is computed.
// SPREAD 4: up to four columns are spread over the product's rows so that a
// lane finds its own in element 0 alone.  STREAMED: past the caches.
//
// Measured: 20M x 128, groups of 128, one vector 244 us (5.7 TB/s; a large copy
// moves 5.1); 2.5M x 128, groups of 32 with zero points, 16 vectors to float32
// 86 us (350 MB, nearly half of it results: 4.05 TB/s); 8,192 x 8,192, one
// vector 14 us (34.6 MB: a launch, the vector's way to LDS and two steps of each
// wave); 100,000 x 64 6.4 us.
template <bool COARSE, bool WIDE, bool ZEROS, int T, int J, int C, int SPREAD, bool STREAMED>
__global__ __launch_bounds__(kThreads, 2) void matvec_kernel(MatvecArgs a) {
  extern __shared__ __align__(16) uint8_t lds_raw[];
  __shared__ uint32_t largest[kMaxTileColumns];
  u32x4* xs = reinterpret_cast<u32x4*>(lds_raw);  // [block][l / 16][column]
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, row16 = lane % 16, quarter = lane / 16;
  const int64_t first_query = static_cast<int64_t>(blockIdx.y) * a.queries_at_once;
  const int queries = static_cast<int>(min(static_cast<int64_t>(a.queries_at_once), a.queries - first_query));
  const int columns = queries * a.parts;
  const int steps4 = (a.blocks + 3) / 4;  // of 128 columns
  const int phases = (a.blocks + a.phase_blocks - 1) / a.phase_blocks;

  float* sums = reinterpret_cast<float*>(xs + static_cast<int64_t>(min(a.phase_blocks, steps4 * 4)) * 4 * columns);

  // Eight elements of vector q from column d on, 0 past the last.
  auto load_x = [&](int q, int d, float v[8]) {
    const int64_t at = (first_query + q) * a.dim + d;
    if (d + 8 <= a.dim) {
      if (a.x_type == ST_SCORE_F32)
        unpack8<ST_SCORE_F32>(load_raw8<ST_SCORE_F32>(a.x, at), v);
      else if (a.x_type == ST_SCORE_F16)
        unpack8<ST_SCORE_F16>(load_raw8<ST_SCORE_F16>(a.x, at), v);
      else
        unpack8<ST_SCORE_BF16>(load_raw8<ST_SCORE_BF16>(a.x, at), v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = d + i < a.dim ? load_any(a.x, at + i, a.x_type) : 0.0f;
    }
  };

  auto top_of = [](const float v[8]) {
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float x = fabsf(v[k]);
      top = x < __builtin_inff() ? fmaxf(top, x) : top;
    }
    return top;
  };
  // Puts unit i (eight elements of a vector, vectors fastest) of a phase into
  // LDS as its parts.
  auto put = [&](int i, int q, const float v[8]) {
    const float scale = a.x_type == ST_SCORE_F16 ? 1.0f : power_of_two(shift_of(__uint_as_float(largest[q])));
    for (int part = 0; part < a.parts; ++part) {
      half8_t h;
#pragma unroll
      for (int k = 0; k < 8; ++k) h[k] = part_of(v[(k >> 1) + 4 * (k & 1)] * scale, part);
      u32x4 raw;
      __builtin_memcpy(&raw, &h, 16);
      xs[i * a.parts + part] = raw;
    }
  };
  auto fill = [&](int phase) {
    const int first = phase * a.phase_blocks;
    const int count = min(a.phase_blocks, steps4 * 4 - first) * 4 * queries;
    for (int i = tid; i < count; i += kThreads) {
      const int at = i / queries, q = i - at * queries;
      float v[8];
      load_x(q, first * kBlock + at * 8, v);
      put(i, q, v);
    }
  };
  // Each vector's largest finite element goes to largest[] (floats that are
  // not negative are in the order of their bits), and, where one phase takes
  // them all, the vectors to LDS: from registers, if they fit.
  auto prepare = [&] {
    constexpr int kHeld = 4;
    const int units = steps4 * 16 * queries;
    const bool held = phases == 1 && units <= kHeld * kThreads;
    const bool scaled = a.x_type != ST_SCORE_F16;
    float v[kHeld][8];
    if (scaled) {
      if (tid < queries) largest[tid] = 0;
      __syncthreads();
    }
    if (held) {
#pragma unroll
      for (int h = 0; h < kHeld; ++h) {
        const int i = tid + h * kThreads, at = i / queries;
        if (i < units) load_x(i - at * queries, at * 8, v[h]);
      }
    }
    if (scaled) {
      if (held && queries == 1) {
        float top = 0.0f;
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
          if (tid + h * kThreads < units) top = fmaxf(top, top_of(v[h]));
        top = wave_max(top);
        if (lane == 0) atomicMax(&largest[0], __float_as_uint(top));
      } else if (held) {
#pragma unroll
        for (int h = 0; h < kHeld; ++h) {
          const int i = tid + h * kThreads;
          if (i < units) atomicMax(&largest[i % queries], __float_as_uint(top_of(v[h])));
        }
      } else {
        for (int i = tid; i < units; i += kThreads) {
          const int at = i / queries, q = i - at * queries;
          float w[8];
          load_x(q, at * 8, w);
          atomicMax(&largest[q], __float_as_uint(top_of(w)));
        }
      }
      __syncthreads();
    }
    if (held) {
#pragma unroll
      for (int h = 0; h < kHeld; ++h) {
        const int i = tid + h * kThreads;
        if (i < units) put(i, i % queries, v[h]);
      }
    } else if (phases == 1) {
      fill(0);
    }
    __syncthreads();
  };

  const int row_waves = kWaves / a.split;
  const int mine = wave / a.split, turn = wave % a.split;
  const int64_t rows_at_once = static_cast<int64_t>(row_waves) * T * 16;
  uint32_t base1024 = 0x64006400u;
  asm volatile("" : "+v"(base1024));
  const half2_t low8 = as_half2(0xE408E408u), high8 = as_half2(0xD480D480u);  // -(1024 + 8), -(64 + 8)

  // Addresses are a scalar base and a 32-bit offset per lane.  Rows and blocks
  // past the last are read as the last, so that every load is issued on every
  // path: a load behind a branch would make the compiler wait for all of them.
  auto load = [&](int64_t base, int step, Step<T, J>& s) {
    const int64_t from = min(base, a.rows - 1);
    const uint32_t last = static_cast<uint32_t>(min(a.rows - 1 - from, static_cast<int64_t>(T * 16)));
    const uint8_t* packed = a.packed + from * a.row_bytes;
    const int64_t scale0 = from * a.groups;
    const uint8_t* scales = static_cast<const uint8_t*>(a.scales) + scale0 * (WIDE ? 4 : 2);
    const uint8_t* zeros = a.zeros + scale0;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const uint32_t row = min(static_cast<uint32_t>(t * 16 + row16), last);
      const uint32_t bytes = __umul24(row, a.row_bytes), groups = __umul24(row, a.groups);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const uint32_t block = min((step * J + j) * 4 + quarter, a.blocks - 1);
        const u32x4* w = reinterpret_cast<const u32x4*>(packed + (bytes + block * 16));
        s.w[t][j] = STREAMED ? __builtin_nontemporal_load(w) : *w;
        const uint32_t of = COARSE ? min((step * J + j) * 4, a.blocks - 1) : block;
        const uint32_t at = groups + (a.group_blocks == 1 ? of : __umulhi(of, a.group_magic));
        s.scale[t][j] = WIDE ? *reinterpret_cast<const uint32_t*>(scales + at * 4)
                             : *reinterpret_cast<const uint16_t*>(scales + at * 2);
        if constexpr (ZEROS) s.zero[t][j] = zeros[at];
      }
    }
  };

  auto scale_of = [&](uint32_t raw) {
    if constexpr (WIDE) return __uint_as_float(raw);
    return a.scale_type == ST_SCORE_F16 ? score_of_bits<ST_SCORE_F16>(raw) : score_of_bits<ST_SCORE_BF16>(raw);
  };

  f32x4 acc[T][C];
  auto compute = [&](int step, int first_block, const Step<T, J>& s) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int block0 = (step * J + j) * 4;
      if (block0 >= a.blocks) break;
      f32x4 part[T][C];
      u32x4 w[T], zero[T], scale[T];
#pragma unroll
      for (int t = 0; t < T; ++t) {
        w[t] = transpose4(s.w[t][j]);
        if constexpr (!COARSE) {
          scale[t] = broadcast4(__float_as_uint(scale_of(s.scale[t][j])));
          if constexpr (ZEROS) zero[t] = broadcast4(s.zero[t][j] * 0x00010001u);
        }
#pragma unroll
        for (int c = 0; c < C; ++c) part[t][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int block = block0 + i;
        if (block >= a.blocks) break;
        half8_t x[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const int column = min(c * 16 + row16 / SPREAD, columns - 1);
          const u32x4 raw = xs[((block - first_block) * 4 + quarter) * columns + column];
          __builtin_memcpy(&x[c], &raw, 16);
        }
#pragma unroll
        for (int t = 0; t < T; ++t) {
          half2_t low = low8, high = high8;
          if constexpr (ZEROS) {
            const uint32_t z = COARSE ? s.zero[t][j] * 0x00010001u : zero[t][i];
            low = as_half2(z | 0xE400E400u);
            high = low + half2_t{static_cast<_Float16>(960.0f), static_cast<_Float16>(960.0f)};
          }
          const half8_t q = codes_of(w[t][i], base1024, low, high);
#pragma unroll
          for (int c = 0; c < C; ++c) {
            if constexpr (COARSE) {
              part[t][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[c], q, part[t][c], 0, 0, 0);
            } else {
              const f32x4 p = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[c], q, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
              for (int e = 0; e < 4; e += SPREAD)
                acc[t][c][e] = fmaf(__uint_as_float(scale[t][i]), p[e], acc[t][c][e]);
            }
          }
        }
      }
      if constexpr (COARSE) {
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 4; e += SPREAD) acc[t][c][e] = fmaf(scale_of(s.scale[t][j]), part[t][c][e], acc[t][c][e]);
      }
    }
  };

  // The wave's steps in order: row groups, phases, steps of 4 J blocks.  The
  // next step's weights are loaded before a step is computed (the first ones
  // before the vectors are in LDS).
  struct Place {
    int64_t base0;
    int phase, step;
  };
  const int64_t stride = static_cast<int64_t>(gridDim.x) * rows_at_once;
  auto first_step = [&](int phase) { return phase * (a.phase_blocks / (4 * J)) + turn; };
  auto end_step = [&](int phase) {
    return (min((phase + 1) * a.phase_blocks, a.blocks) + 4 * J - 1) / (4 * J);
  };
  auto settle = [&](Place& p) {  // the first step at or after p
    while (p.base0 < a.rows && p.step >= end_step(p.phase)) {
      if (++p.phase == phases) {
        p.phase = 0;
        p.base0 += stride;
      }
      p.step = first_step(p.phase);
    }
  };
  const int64_t tile0 = static_cast<int64_t>(mine) * T * 16;
  Step<T, J> next;
  Place ahead{static_cast<int64_t>(blockIdx.x) * rows_at_once, 0, first_step(0)};
  settle(ahead);
  load(ahead.base0 + tile0, ahead.step, next);

  prepare();
  // what undoes the scaling of the vectors whose sums this lane holds
  float unscale[C][4];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < 4; e += SPREAD) {
      const int q = min((c * 16 + (quarter * 4 + e) / SPREAD) / a.parts, queries - 1);
      unscale[c][e] = a.x_type == ST_SCORE_F16 ? 1.0f : power_of_two(-shift_of(__uint_as_float(largest[q])));
    }

  // y of the wave's tiles from its sums
  const bool y_wide = a.y_type == ST_SCORE_F32;
  char* const y = static_cast<char*>(a.y) + first_query * a.rows * (y_wide ? 4 : 2);
  auto put_y = [&](char* at, float v) {
    if (y_wide && STREAMED)
      __builtin_nontemporal_store(v, reinterpret_cast<float*>(at));
    else if (y_wide)
      *reinterpret_cast<float*>(at) = v;
    else
      *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(
          a.y_type == ST_SCORE_F16 ? score_bits<ST_SCORE_F16>(v) : score_bits<ST_SCORE_BF16>(v));
  };
  auto store = [&](int64_t base) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int e = 0; e < 4; e += SPREAD) {
        float v[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
          v[t] = acc[t][c][e];
          if constexpr (SPREAD == 1)
            if (a.parts == 2) v[t] = fmaf(acc[t][c][(e + 1) % 4], 1.0f / 2048.0f, v[t]);
          v[t] *= unscale[c][e];
        }
        if constexpr (T == 4) {
          // Lane groups and tiles exchanged, a wave stores 64 adjacent results
          // of one vector.
          const u32x4 w = transpose4(u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                                           __float_as_uint(v[3])});
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int column = c * 16 + (i * 4 + e) / SPREAD;
            const int q = a.parts == 2 ? column >> 1 : column;
            if ((a.parts == 2 && (column & 1)) || q >= queries) continue;
            if (base + lane < a.rows) put_y(y + (q * a.rows + base + lane) * (y_wide ? 4 : 2), __uint_as_float(w[i]));
          }
        } else {
          const int column = c * 16 + (quarter * 4 + e) / SPREAD;
          const int q = a.parts == 2 ? column >> 1 : column;
          const bool mine_ = (a.parts == 1 || (column & 1) == 0) && q < queries;
          char* at = y + (q * a.rows + base + row16) * (y_wide ? 4 : 2);
#pragma unroll
          for (int t = 0; t < T; ++t)
            if (mine_ && base + t * 16 + row16 < a.rows) put_y(at + t * 16 * (y_wide ? 4 : 2), v[t]);
        }
      }
    }
  };

  for (int64_t base0 = static_cast<int64_t>(blockIdx.x) * rows_at_once; base0 < a.rows; base0 += stride) {
    const int64_t base = base0 + tile0;
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int c = 0; c < C; ++c) acc[t][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int phase = 0; phase < phases; ++phase) {
      if (phases > 1) {
        __syncthreads();
        fill(phase);
        __syncthreads();
      }
      for (int step = first_step(phase); step < end_step(phase); step += a.split) {
        const Step<T, J> now = next;
        ahead.step += a.split;
        settle(ahead);
        load(ahead.base0 + tile0, ahead.step, next);
        compute(step, phase * a.phase_blocks, now);
      }
    }
    if (a.split == 1) {
      store(base);
    } else {
      // the sums of the waves that share the rows, added in order by the first
      constexpr int kEach = T * C * 4;
      float* own = sums + wave * 64 * kEach;
      if (turn > 0) {
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) own[((t * C + c) * 4 + e) * 64 + lane] = acc[t][c][e];
      }
      __syncthreads();
      if (turn == 0) {
        for (int w = 1; w < a.split; ++w)
#pragma unroll
          for (int t = 0; t < T; ++t)
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[t][c][e] += own[w * 64 * kEach + ((t * C + c) * 4 + e) * 64 + lane];
        store(base);
      }
      __syncthreads();
    }
  }
}

struct QuantizeArgs {
  const void* weight;
  uint8_t* packed;
  void* scales;
  uint8_t* zeros;
  int64_t rows, dim, group, groups, row_bytes;
  int symmetric;
};

// A wave per row and group, run once over a table.  Instructions per group bound
// it, not bytes: bfloat16 and float32 take the same time, 2.5M x 128 2.9 ms in
// groups of 32 and 0.9 ms in groups of 128 (a copy's rate would take 0.16 ms for
// the former's bytes in bfloat16); half of the lanes read a group of 32, a
// quarter of them pack it.
//
// Symmetric: scale = max |w| / 7 rounded to the weights' type, code = w / scale
// to the nearest even, kept in [-8, 7], plus 8.
// Else lo = min(w, 0), hi = max(w, 0): scale = (hi - lo) / 15, zero = -lo /
// scale, code = w / scale + zero, each to the nearest even and kept in
// [0, 15]; a difference past float32's range is taken as hi / 15 - lo / 15.  A
// group of zeros has scale 0; one with a value that is not finite has scale NaN,
// so that its products say so.
template <int DT>
__global__ __launch_bounds__(256) void quantize_kernel(QuantizeArgs a) {
  const int lane = threadIdx.x % 64;
  const int64_t items = a.rows * a.groups;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 64; item < items;
       item += static_cast<int64_t>(gridDim.x) * 4) {
    const int64_t n = item / a.groups, g = item - n * a.groups;
    const int64_t first = g * a.group, end = min(first + a.group, a.dim);
    const char* row = static_cast<const char*>(a.weight) + n * a.dim * kScoreBytes<DT>;
    float lo = 0.0f, hi = 0.0f;
    bool finite = true;
    for (int64_t d = first + lane; d < end; d += 64) {
      const float w = load_score<DT>(row, d);
      finite &= __builtin_isfinite(w);
      lo = fminf(lo, w);
      hi = fmaxf(hi, w);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      lo = fminf(lo, __shfl_xor(lo, o));
      hi = fmaxf(hi, __shfl_xor(hi, o));
    }
    finite = __all(finite);
    float scale;
    if (a.symmetric) {
      scale = __fdiv_rn(fmaxf(-lo, hi), 7.0f);
    } else {
      scale = __fdiv_rn(hi - lo, 15.0f);
      if (scale == __builtin_inff()) scale = __fdiv_rn(hi, 15.0f) - __fdiv_rn(lo, 15.0f);
    }
    if (!finite) scale = __builtin_nanf("");
    scale = score_of_bits<DT>(score_bits<DT>(scale));
    const bool any = scale > 0.0f;
    float zero = 8.0f;
    if (!a.symmetric) zero = any ? fminf(fmaxf(rintf(__fdiv_rn(-lo, scale)), 0.0f), 15.0f) : 0.0f;
    if (lane == 0) {
      store_score<DT>(a.scales, item, scale);
      a.zeros[item] = static_cast<uint8_t>(zero);
    }
    // whole blocks of 32 columns, the codes past the last column 0
    const int64_t bytes_end = min((first + a.group) / 2, a.row_bytes);
    for (int64_t j = first / 2 + lane; j < bytes_end; j += 64) {
      uint32_t byte = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t d = 2 * j + h;
        if (d >= end) continue;
        const float q = any ? rintf(__fdiv_rn(load_score<DT>(row, d), scale)) + zero : zero;
        byte |= static_cast<uint32_t>(fminf(fmaxf(q, 0.0f), 15.0f)) << (4 * h);
      }
      a.packed[n * a.row_bytes + j] = static_cast<uint8_t>(byte);
    }
  }
}

void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw Error(ST_ERR_HIP, cat(what, " launch failed: ", hipGetErrorString(e)));
}

template <bool COARSE, bool WIDE, bool ZEROS, int T, int J, int C, int SPREAD, bool STREAMED = false>
void launch_shape(const MatvecArgs& a, int columns, hipStream_t s) {
  const int64_t rows_at_once = static_cast<int64_t>(kWaves / a.split) * T * 16;
  const int64_t passes = (a.queries + a.queries_at_once - 1) / a.queries_at_once;
  const int lds_blocks = std::min(a.phase_blocks, (a.blocks + 3) / 4 * 4);
  size_t lds = static_cast<size_t>(lds_blocks) * 64 * columns;
  if (a.split > 1) lds += sizeof(float) * kWaves * 64 * T * C * 4;
  const auto kernel = matvec_kernel<COARSE, WIDE, ZEROS, T, J, C, SPREAD, STREAMED>;
  if (lds > 48 * 1024) {
    static std::once_flag once;
    std::call_once(once, [&] {
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds);
      if (e != hipSuccess) throw Error(ST_ERR_HIP, cat("hipFuncSetAttribute failed: ", hipGetErrorString(e)));
    });
  }
  // as many workgroups as a CU holds, by registers and LDS
  static const int by_registers = [&] {
    int n = 0;
    const hipError_t e = hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kThreads, 0);
    return e == hipSuccess && n > 0 ? n : 1;
  }();
  const int64_t per_cu = std::max<int64_t>(1, std::min<int64_t>(by_registers, 160 * 1024 / (lds + 512)));
  const int64_t grid = std::min<int64_t>((a.rows + rows_at_once - 1) / rows_at_once, per_cu * cu_count());
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid), static_cast<unsigned>(passes)),
                     dim3(kThreads), lds, s, a);
}

template <bool COARSE, bool WIDE, bool ZEROS, int T, int J>
void launch_columns(const MatvecArgs& a, int columns, hipStream_t s) {
  // One vector against a table that the last-level cache (256 MB) cannot hold
  // for the next call is read, and the results are stored, past the caches:
  // 20M x 128 243 us, 266 us through them.  A smaller table is found there again
  // (1M x 256: 44 us; past the caches 50 us), and several vectors' results, rows
  // of any length apart, need them to put lines together (2.5M x 128, 16
  // vectors: 87 us; past them 103 us).
  if (a.queries == 1 && a.parts == 1 && a.rows * a.row_bytes > (256ll << 20))
    launch_shape<COARSE, WIDE, ZEROS, T, J, 1, 4, true>(a, columns, s);
  else if (columns <= 4 && a.parts == 1)
    launch_shape<COARSE, WIDE, ZEROS, T, J, 1, 4>(a, columns, s);
  else if (columns <= 16)
    launch_shape<COARSE, WIDE, ZEROS, T, J, 1, 1>(a, columns, s);
  else if (columns <= 32)
    launch_shape<COARSE, WIDE, ZEROS, T, J, 2, 1>(a, columns, s);
  else
    launch_shape<COARSE, WIDE, ZEROS, T == 4 ? 2 : T, T == 4 ? 2 : J, 4, 1>(a, columns, s);
}

void launch_matvec(MatvecArgs& a, hipStream_t s) {
  a.parts = a.x_type == ST_SCORE_F32 ? 2 : 1;
  a.queries_at_once = static_cast<int>(std::min<int64_t>(a.queries, kMaxTileColumns / a.parts));
  const bool is_long = a.blocks > 8;
  a.split = 1;
  if (is_long)
    while (a.split < kWaves && (a.rows + 15) / 16 * a.split < 8 * cu_count()) a.split *= 2;
  const int whole = (a.blocks + 15) / 16 * 16;
  auto phase_of = [&](int columns) { return std::max(16, kVectorLds / (64 * columns) / 16 * 16); };
  // Where four or eight waves share a row but a phase of many vectors has fewer
  // steps than that, some would have none: 16 parts a pass then (64 vectors x
  // 8,192 columns: 500 rows 160 -> 41 us, 8,192 rows 211 -> 145 us; 64 x 1,100,
  // 3,000 rows 30 -> 21 us).  With two waves a row, or one, the whole pass and
  // 16 parts a pass measured both ways, and neither the rows nor the columns
  // tell them apart: 760 and 874 us (64 vectors, 100,000 x 8,192), 78 and 96 us
  // (64, 60,000 x 1,500), 48 and 55 us (32 float32, 30,000 x 1,300), 56 and 59
  // us (20, 20,000 x 4,000), but 179 and 128 us (64, 20,000 x 4,000), 312 and
  // 242 us (64, 200,000 x 2,000), 247 and 207 us (40, 200,000 x 2,000).  They
  // read the table once.
  const int most = a.queries_at_once * a.parts;
  if (a.split >= 4 && whole * 64 * most > kWholeVectorLds && a.split > phase_of(most) / 16)
    a.queries_at_once = std::min(a.queries_at_once, 16 / a.parts);
  const int columns = a.queries_at_once * a.parts;
  // block / group_blocks: the reciprocal rounded up is exact while block *
  // group_blocks stays below 2^32 (blocks are at most 2^16); 1 has none
  a.group_magic = a.group_blocks == 1 ? 0 : static_cast<uint32_t>((0x100000000ull + a.group_blocks - 1) / a.group_blocks);
  const bool coarse = a.group_blocks % 4 == 0;
  // All of the vectors at once, if there is room for them beside the sums of
  // the waves that share rows (T = 1; launch_shape).
  const int tiles = columns <= 16 ? 1 : columns <= 32 ? 2 : 4;
  const int sums = a.split > 1 ? static_cast<int>(sizeof(float)) * kWaves * 64 * tiles * 4 : 0;
  a.phase_blocks = whole * 64 * columns <= std::min(kWholeVectorLds, kMostLds - sums)
                       ? whole
                       : phase_of(columns);
  auto launch = [&](auto coarse_, auto wide_, auto zeros_) {
    if (is_long)
      launch_columns<coarse_(), wide_(), zeros_(), 1, 4>(a, columns, s);
    else
      launch_columns<coarse_(), wide_(), zeros_(), 4, 1>(a, columns, s);
  };
  auto with = [](bool b, auto f) { b ? f(std::true_type{}) : f(std::false_type{}); };
  with(coarse, [&](auto c) {
    with(a.scale_type == ST_SCORE_F32, [&](auto w) { with(a.zeros != nullptr, [&](auto z) { launch(c, w, z); }); });
  });
}

// Any group size of check_table is in range: one past the columns makes one group.
int64_t groups_of(int64_t dim, int64_t group_size) { return (dim - 1) / group_size + 1; }

void check_type(int type, const char* what) {
  ST_CHECK(type == ST_SCORE_F32 || type == ST_SCORE_F16 || type == ST_SCORE_BF16, what,
           " must be float32, float16 or bfloat16");
}

void check_table(int64_t rows, int64_t dim, int64_t group) {
  ST_CHECK(rows >= 0 && dim >= 1, "a table has at least one column, got ", rows, " x ", dim);
  ST_CHECK(dim <= (1ll << 21), "columns must be at most 2^21, got ", dim);
  ST_CHECK(group >= kBlock && group % kBlock == 0, "group_size must be a positive multiple of ", kBlock, ", got ", group);
}

}  // namespace
}  // namespace st

extern "C" int st_int4_quantize(const void* weight, int weight_type, int64_t rows, int64_t dim, int64_t group_size,
                                int symmetric, uint8_t* packed, void* scales, uint8_t* zeros, void* stream) {
  using namespace st;
  return guarded([&] {
    check_type(weight_type, "weight");
    check_table(rows, dim, group_size);
    if (rows == 0) return;
    ST_CHECK(weight && packed && scales && zeros, "null device pointer");
    QuantizeArgs a{weight, packed, scales, zeros, rows, dim, group_size, groups_of(dim, group_size),
                   (dim + kBlock - 1) / kBlock * (kBlock / 2), symmetric};
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((rows * a.groups + 3) / 4, 64ll * cu_count()));
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (weight_type == ST_SCORE_F32)
      hipLaunchKernelGGL((quantize_kernel<ST_SCORE_F32>), dim3(grid), dim3(256), 0, s, a);
    else if (weight_type == ST_SCORE_F16)
      hipLaunchKernelGGL((quantize_kernel<ST_SCORE_F16>), dim3(grid), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((quantize_kernel<ST_SCORE_BF16>), dim3(grid), dim3(256), 0, s, a);
    check_launch("quantize_kernel");
  });
}

extern "C" int st_int4_matvec(const uint8_t* packed, const void* scales, int scale_type, const uint8_t* zeros,
                              const void* x, int x_type, int64_t queries, int64_t rows, int64_t dim,
                              int64_t group_size, void* y, int y_type, void* stream) {
  using namespace st;
  return guarded([&] {
    check_type(scale_type, "scales");
    check_type(x_type, "x");
    check_type(y_type, "the result");
    check_table(rows, dim, group_size);
    ST_CHECK(queries >= 0 && queries <= 65536, "vectors must be between 0 and 65536, got ", queries);
    if (rows == 0 || queries == 0) return;
    ST_CHECK(packed && scales && x && y, "null device pointer");
    ST_CHECK(reinterpret_cast<uintptr_t>(packed) % 16 == 0, "the packed table must be 16-byte aligned");
    MatvecArgs a{};
    a.packed = packed;
    a.scales = scales;
    a.zeros = zeros;
    a.x = x;
    a.y = y;
    a.rows = rows;
    a.queries = queries;
    a.dim = static_cast<int>(dim);
    a.groups = static_cast<int>(groups_of(dim, group_size));
    a.blocks = static_cast<int>((dim + kBlock - 1) / kBlock);
    a.row_bytes = a.blocks * (kBlock / 2);
    a.group_blocks = static_cast<int>(std::min<int64_t>(group_size / kBlock, a.blocks));
    a.scale_type = scale_type;
    a.x_type = x_type;
    a.y_type = y_type;
    launch_matvec(a, static_cast<hipStream_t>(stream));
    check_launch("matvec_kernel");
  });
}
