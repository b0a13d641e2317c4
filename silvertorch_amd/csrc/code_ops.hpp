// Rows in 8 bits: scale = max |x| / 127, code = x times (127 / max |x|) to the
// nearest even, both quotients rounded to 32 bits; a code is in [-127, 127].
// One multiplication a code, where a division by the scale would take ten
// instructions.  A row whose largest magnitude is below 2^-119 (127 / it would
// pass 32 bits) is held as zeros, scale 0; one with a value that is not finite
// has codes 0 and scale NaN, so that its products say so.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace st {

struct CodeScale {
  float scale, times;
};

// `most`: max |x|, infinite where a value is not finite.
__device__ __forceinline__ CodeScale code_scale(float most) {
  if (most == __builtin_inff()) return {__builtin_nanf(""), 0.0f};
  if (most < 0x1p-119f) return {0.0f, 0.0f};
  return {__fdiv_rn(most, 127.0f), __fdiv_rn(127.0f, most)};
}

__device__ __forceinline__ int code_of(float x, CodeScale c) {
  // times 0: whatever x holds is not converted (0 times infinity is none)
  return c.times == 0.0f ? 0 : static_cast<int>(__builtin_rintf(__fmul_rn(x, c.times)));
}

__device__ __forceinline__ uint64_t codes8(const float v[8], CodeScale c) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    w[h] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[h] |= (static_cast<uint32_t>(code_of(v[4 * h + i], c)) & 0xFFu) << (8 * i);
  }
  return w[0] | (static_cast<uint64_t>(w[1]) << 32);
}

}  // namespace st
