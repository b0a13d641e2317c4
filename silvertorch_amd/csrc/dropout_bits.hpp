// Dropout's random numbers: Philox4x32-10, the counter-based generator of
// Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3"
// (2011).  Element e of a call takes half word e % 8 of the block whose counter
// is (e / 8, offset) and whose key is the seed; halves go from the low one of
// word 0 to the high one of word 3.  An element stays if its half is at least
// `dropped`, p in units of 2^-16.
//
// Half words, not words: a block is 20 products of 32 x 32 bits, a quarter of
// the vector units' rate each, and with a word an element they, not the bytes,
// would bound bfloat16.  p is off by 2^-17 at most for it (0.1 is 6,554 of 65,536,
// 6e-5 of itself too much); kept elements are multiplied with 2^16 / (2^16 - dropped),
// so the expectation is exact.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace st {

constexpr int kDropoutOne = 1 << 16;  // dropped of p = 1

struct DropoutArgs {
  const int64_t* state;  // seed, offset; null: nothing is dropped
  int64_t* used;         // null, or where a forward call leaves the state that it used
  int dropped;           // in [0, 2^16]
  float times;           // what stays is multiplied with
};

// Checks p; `state` and `used` are passed on (dropout.hip).
DropoutArgs dropout_args(double p, const int64_t* state, int64_t* used);

struct DropoutKey {
  uint32_t key[2], offset[2];
};

__device__ __forceinline__ DropoutKey dropout_key(const int64_t* state) {
  const uint64_t seed = static_cast<uint64_t>(state[0]), offset = static_cast<uint64_t>(state[1]);
  return {{static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32)},
          {static_cast<uint32_t>(offset), static_cast<uint32_t>(offset >> 32)}};
}

// The words of one block of eight elements.
__device__ __forceinline__ void dropout_words(const DropoutKey& k, uint64_t block, uint32_t w[4]) {
  uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32), c2 = k.offset[0], c3 = k.offset[1];
  uint32_t k0 = k.key[0], k1 = k.key[1];
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0;
  w[1] = c1;
  w[2] = c2;
  w[3] = c3;
}

// Bit i: whether element first + i stays, i = 0..7.  Two blocks where `first`
// is no multiple of 8.
__device__ __forceinline__ uint32_t dropout_keeps(const DropoutKey& k, uint64_t first, uint32_t dropped) {
  uint32_t w[4], keeps = 0;
  dropout_words(k, first >> 3, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) keeps |= ((i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu) >= dropped ? 1u : 0u) << i;
  const uint32_t skip = static_cast<uint32_t>(first) & 7;
  if (skip != 0) {
    dropout_words(k, (first >> 3) + 1, w);
    uint32_t more = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) more |= ((i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu) >= dropped ? 1u : 0u) << i;
    keeps = (keeps | (more << 8)) >> skip;
  }
  return keeps;
}

// residual + what is left of x, the product rounded by itself.
__device__ __forceinline__ float dropout_add(float residual, float x, bool keep, float times) {
#pragma clang fp contract(off)
  const float kept = keep ? x * times : 0.0f;
  return residual + kept;
}

}  // namespace st
