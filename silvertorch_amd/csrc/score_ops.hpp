// Device helpers shared by the kernels that read rows of scores (float32,
// float16 or bfloat16): unaligned 8-element loads and stores, order-preserving
// integer keys, and softmax statistics that can be joined.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/silvertorch_hip.h"

namespace st {

// ST_SCORE_F32, ST_SCORE_F16, ST_SCORE_BF16
template <int DT>
constexpr int kScoreBytes = DT == ST_SCORE_F32 ? 4 : 2;

// Rows start at any multiple of the element size (odd row lengths), so the
// vector types carry the element's alignment; gfx950 loads and stores 16 bytes
// at such addresses with one instruction.
typedef uint32_t u32x4_by4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_by2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float bf16_bits_to_float(uint32_t b) { return __uint_as_float(b << 16); }

// Eight consecutive scores as they are stored.
template <int DT>
struct Raw8 {
  u32x4 w[DT == ST_SCORE_F32 ? 2 : 1];
};

// columns [col, col + 8) of a row of scores
template <int DT>
__device__ __forceinline__ Raw8<DT> load_raw8(const void* row, int64_t col) {
  Raw8<DT> r;
  if constexpr (DT == ST_SCORE_F32) {
    const u32x4_by4* p = reinterpret_cast<const u32x4_by4*>(static_cast<const float*>(row) + col);
    r.w[0] = p[0];
    r.w[1] = p[1];
  } else {
    r.w[0] = *reinterpret_cast<const u32x4_by2*>(static_cast<const uint16_t*>(row) + col);
  }
  return r;
}

template <int DT>
__device__ __forceinline__ float score_of_bits(uint32_t bits) {
  if constexpr (DT == ST_SCORE_F32) {
    return __uint_as_float(bits);
  } else if constexpr (DT == ST_SCORE_F16) {
    const uint16_t h = static_cast<uint16_t>(bits);
    _Float16 f;
    __builtin_memcpy(&f, &h, 2);
    return static_cast<float>(f);
  } else {
    return bf16_bits_to_float(bits);
  }
}

template <int DT>
__device__ __forceinline__ void unpack8(const Raw8<DT>& r, float v[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (DT == ST_SCORE_F32) {
      v[i] = __uint_as_float(r.w[i / 4][i % 4]);
    } else if constexpr (DT == ST_SCORE_F16) {
      v[i] = score_of_bits<DT>((i & 1) ? r.w[0][i / 2] >> 16 : r.w[0][i / 2] & 0xFFFFu);
    } else {
      v[i] = __uint_as_float((i & 1) ? r.w[0][i / 2] & 0xFFFF0000u : r.w[0][i / 2] << 16);
    }
  }
}

template <int DT>
__device__ __forceinline__ float load_score(const void* row, int64_t col) {
  if constexpr (DT == ST_SCORE_F32) return static_cast<const float*>(row)[col];
  return score_of_bits<DT>(static_cast<const uint16_t*>(row)[col]);
}

// `f` rounded once to the score type (nearest even).
template <int DT>
__device__ __forceinline__ uint32_t score_bits(float f) {
  if constexpr (DT == ST_SCORE_F32) {
    return __float_as_uint(f);
  } else if constexpr (DT == ST_SCORE_F16) {
    const _Float16 h = static_cast<_Float16>(f);
    uint16_t u;
    __builtin_memcpy(&u, &h, 2);
    return u;
  } else {
    const __bf16 h = static_cast<__bf16>(f);
    uint16_t u;
    __builtin_memcpy(&u, &h, 2);
    return u;
  }
}

template <int DT>
__device__ __forceinline__ void store_score(void* row, int64_t col, float f) {
  if constexpr (DT == ST_SCORE_F32)
    static_cast<float*>(row)[col] = f;
  else
    static_cast<uint16_t*>(row)[col] = static_cast<uint16_t>(score_bits<DT>(f));
}

template <int DT>
__device__ __forceinline__ void store8(void* row, int64_t col, const float v[8]) {
  if constexpr (DT == ST_SCORE_F32) {
    u32x4_by4* p = reinterpret_cast<u32x4_by4*>(static_cast<float*>(row) + col);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4_by4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[4 * h + i]);
      p[h] = w;
    }
  } else {
    u32x4_by2 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = score_bits<DT>(v[2 * i]) | (score_bits<DT>(v[2 * i + 1]) << 16);
    *reinterpret_cast<u32x4_by2*>(static_cast<uint16_t*>(row) + col) = w;
  }
}

// Monotone map of floats to unsigned ints (larger float, larger int; -0 and +0
// alike).  No float but a NaN maps to 0.
__device__ __forceinline__ uint32_t ordered_score(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}

__device__ __forceinline__ float score_from_ordered(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}

// Descending order of keys: larger scores first, equal ones by column.  Key 0
// sorts below every real one.
__device__ __forceinline__ uint64_t score_key(float f, uint32_t column) {
  return (static_cast<uint64_t>(ordered_score(f)) << 32) | static_cast<uint32_t>(~column);
}

constexpr float kMinusInf = -__builtin_inff();

// Softmax statistics of some scores z at inverse temperature 1/T, with
// c = log2(e)/T: m = max z, s = sum e^((z-m)/T), t = sum e^((z-m)/T) (z-m).
// No scores: m = -inf, s = t = 0.  A NaN among them, or +inf, makes s NaN.
struct SoftStats {
  float m, s, t;
};

__device__ __forceinline__ SoftStats soft_none() { return {kMinusInf, 0.0f, 0.0f}; }

// The statistics with the maximum moved up to `to` (to >= a.m).
__device__ __forceinline__ SoftStats soft_rebase(SoftStats a, float to, float c) {
  if (a.m == to || a.m == kMinusInf) return {to, a.s, a.t};
  const float d = a.m - to;  // -inf when `to` is +inf: the scores below it count nothing
  const float scale = __builtin_amdgcn_exp2f(d * c);
  if (scale == 0.0f) return {to, a.s * 0.0f, a.s * 0.0f};
  return {to, a.s * scale, (a.t + a.s * d) * scale};
}

// A float moved between lanes by DPP; lanes outside the row mask keep theirs.
template <int CONTROL, int ROWS = 0xF>
__device__ __forceinline__ float dpp_move(float x) {
  const int i = __float_as_int(x);
  return __int_as_float(__builtin_amdgcn_update_dpp(i, i, CONTROL, ROWS, 0xF, false));
}

// f over the aligned groups of 8 lanes, in every lane of the group.
template <typename F>
__device__ __forceinline__ float join8(float x, F f) {
  x = f(x, dpp_move<0xB1>(x));   // quad_perm [1, 0, 3, 2]
  x = f(x, dpp_move<0x4E>(x));   // quad_perm [2, 3, 0, 1]
  return f(x, dpp_move<0x141>(x));  // row_half_mirror
}

// The maximum over the wave.
__device__ __forceinline__ float wave_max(float x) {
  x = join8(x, [](float a, float b) { return fmaxf(a, b); });
  x = fmaxf(x, dpp_move<0x140>(x));       // row_mirror
  x = fmaxf(x, dpp_move<0x142, 0xA>(x));  // row_bcast:15 into rows 1 and 3
  x = fmaxf(x, dpp_move<0x143, 0xC>(x));  // row_bcast:31 into rows 2 and 3
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// The sum over the wave, in a fixed order.
__device__ __forceinline__ float wave_sum(float x) {
  x = join8(x, [](float a, float b) { return a + b; });
  x += dpp_move<0x140>(x);
  const int i = __float_as_int(x);
  const float r0 = __int_as_float(__builtin_amdgcn_readlane(i, 0)), r1 = __int_as_float(__builtin_amdgcn_readlane(i, 16));
  const float r2 = __int_as_float(__builtin_amdgcn_readlane(i, 32)), r3 = __int_as_float(__builtin_amdgcn_readlane(i, 48));
  return (r0 + r1) + (r2 + r3);
}

// The statistics of all lanes' scores, in every lane.
__device__ __forceinline__ SoftStats soft_wave_join(SoftStats a, float c) {
  a = soft_rebase(a, wave_max(a.m), c);
  return {a.m, wave_sum(a.s), wave_sum(a.t)};
}

}  // namespace st
