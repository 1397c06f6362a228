// What the kernels of the paged cache share: page arithmetic and the scales' exponents.
#pragma once
#include <cuda_runtime.h>

namespace st {

constexpr int kMinExponent = -60, kMaxExponent = 60;      // of a page's scale

// Page sizes are powers of two from 16 to 256; -1 for others.
inline int page_shift(int page_size) {
  for (int s = 4; s <= 8; ++s)
    if (page_size == 1 << s) return s;
  return -1;
}

// Blocks that `tokens` take, at most the table's width.
__device__ __forceinline__ int blocks_of(long long tokens, int shift, int width) {
  const long long n = (tokens + (1 << shift) - 1) >> shift;
  return n < width ? static_cast<int>(n) : width;
}

// 2^e for a normal exponent.
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }

// The exponent of a scale that is a power of two, kept to the range whatever lies in memory.
__device__ __forceinline__ int scale_exponent(float s) {
  const int e = static_cast<int>((__float_as_uint(s) >> 23) & 255) - 127;
  return e < kMinExponent ? kMinExponent : e > kMaxExponent ? kMaxExponent : e;
}

// The least e with m <= 448 * 2^e = 1.75 * 2^(e + 8), in range; m is finite and not negative.
__device__ __forceinline__ int page_exponent(float m) {
  const unsigned u = __float_as_uint(m);
  const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffff) > 0x600000);      // subnormal m: far below the range
  return e < kMinExponent ? kMinExponent : e > kMaxExponent ? kMaxExponent : e;
}

}  // namespace st
