// The order in which values are kept: largest first, among equal ones the lowest index (globals.js:66-74).
#pragma once
#include <stdint.h>

namespace wgpt {

// Order-preserving bits of a value; -0 and +0 are equal, as in the reference's sort.
__device__ __forceinline__ uint32_t value_key(float v) {
  uint32_t u = __float_as_uint(v);
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// The value's key in the high word, ~index in the low word: a larger key comes earlier.
__device__ __forceinline__ unsigned long long sample_key(float v, int idx) {
  return ((unsigned long long)value_key(v) << 32) | (unsigned long long)(0xFFFFFFFFu - (uint32_t)idx);
}

__device__ __forceinline__ int sample_key_index(unsigned long long c) {
  return (int)(0xFFFFFFFFu - (uint32_t)(c & 0xFFFFFFFFull));
}

__device__ __forceinline__ float sample_key_value(unsigned long long c) {
  const uint32_t k = (uint32_t)(c >> 32);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

}  // namespace wgpt
