// Rows in 8 bits: scale = max |x| / 127, code = x times (127 times (1 / max |x|)) to
// the nearest even, every step rounded to 32 bits; a code is in [-127, 127].
// One multiplication a code, where a division by the scale would take ten
// instructions.  A row whose largest magnitude is below 2^-119 (the quotient would
// pass 32 bits) is held as zeros, scale 0; one with a value that is not finite
// has codes 0 and scale NaN, so that its products say so.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace st {

struct CodeScale {
  float scale, times;
};

// max(most, |v|), NaN if there is one: one instruction for two values.
__device__ __forceinline__ float most_of8(float most, const float v[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) most = __builtin_elementwise_maximum(most, fabsf(v[i]));
  return most;
}

// Infinity for NaN, which the maximum over lanes would pass by.
__device__ __forceinline__ float most_or_infinity(float most) { return most < __builtin_inff() ? most : __builtin_inff(); }

// `most`: max |x|, infinite where a value is not finite.
__device__ __forceinline__ CodeScale code_scale(float most) {
  if (most == __builtin_inff()) return {__builtin_nanf(""), 0.0f};
  if (most < 0x1p-119f) return {0.0f, 0.0f};
  return {__fdiv_rn(most, 127.0f), __fmul_rn(127.0f, __fdiv_rn(1.0f, most))};
}

// Eight codes.  A number below 2^22 plus 1.5 times 2^23 has it, rounded to the
// nearest even, in its low bits.
__device__ __forceinline__ uint64_t codes8(const float v[8], CodeScale c) {
#pragma clang fp contract(off)  // the product is rounded by itself
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(v[4 * h + i] * c.times + 12582912.0f);
    const uint32_t low = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), high = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    // times 0: whatever v holds is not converted (0 times infinity is none)
    w[h] = c.times == 0.0f ? 0 : low | high;
  }
  return w[0] | (static_cast<uint64_t>(w[1]) << 32);
}

}  // namespace st
