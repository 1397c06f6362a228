// Weights of four bits: the layout that the kernels share.
//
// A matrix [rows, cols] is cut into tiles of 16 rows by 64 columns.  Tile (u, c) takes 512 bytes, 16 for each lane of a warp: word s (columns 16 s to
// 16 s + 15) of lane 4 g + t holds, in its nibbles e and e + 4, the codes of columns k and k + 1 of row g (e = 0: k = 2 t; e = 2: k = 2 t + 8) and of row
// g + 8 (e = 1, 3).  That is the order in which a warp's matrix instruction takes a 16 x 16 operand, and in which tensor memory is written from
// registers, so one 16-byte load per lane is an operand of four steps and nothing is exchanged between lanes.  Tiles of one u follow one another.
// Scales: [u][group][16] bf16, those of rows g and g + 8 next to one another.  What lies behind the last row or column is code 8 (zero).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include "../common/ptx.cuh"

namespace st4 {

constexpr int kTileRows = 16, kTileCols = 64, kTileBytes = 512;

template <typename T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float(float x) { return x; }
template <> __device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float(float x) { return x; }
template <> __device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

__device__ __forceinline__ float bf16_bits(uint32_t low16) { return __uint_as_float(low16 << 16); }

__device__ __forceinline__ float activate(float v, int act) {      // 0 none, 1 relu (NaN stays), 2 gelu
  return act == 1 ? fmaxf(v, 0.0f) + (v != v ? v : 0.0f) : act == 2 ? st::gelu_tanh(v) : v;
}

// (word & mask) | bits in one instruction
__device__ __forceinline__ uint32_t pick(uint32_t word, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(word), "r"(mask), "r"(bits));
  return d;
}

// Nibbles e and e + 4 of a word as two numbers of -8 to 7 units, exactly (the published method of mixed-precision kernels): the nibble is put into the low bits of 128 (bf16) or 1024 (fp16) units, where a unit is 1, and
// 136 or 1032 of them are subtracted.  A unit is 1 in fp16 and 2^-10 in bf16: the products with a group of 128 inputs then sum up to no more than the largest of them, so that no
// finite bf16 overflows before the scale is known.  They stay whole multiples of 2^-143, which fp32 holds.
template <typename T> constexpr float kUnits = 1.0f;      // in 1
template <> constexpr float kUnits<__nv_bfloat16> = 1024.0f;
template <typename T> __device__ __forceinline__ uint32_t codes_to_pair(uint32_t word, int e);
template <> __device__ __forceinline__ uint32_t codes_to_pair<__nv_bfloat16>(uint32_t word, int e) {
  const uint32_t v = pick(word >> (4 * e), 0x000F000Fu, 0x3E003E00u);
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), __float2bfloat162_rn(136.0f / kUnits<__nv_bfloat16>));
  return *reinterpret_cast<const uint32_t*>(&d);
}
template <> __device__ __forceinline__ uint32_t codes_to_pair<__half>(uint32_t word, int e) {
  const uint32_t v = pick(word >> (4 * e), 0x000F000Fu, 0x64006400u);
  const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&v), __half2(__float2half_rn(1032.0f), __float2half_rn(1032.0f)));
  return *reinterpret_cast<const uint32_t*>(&d);
}

// Two codes times their scale in a type, exactly.  bf16 in one step: 64 + code, whose unit is bit 1, times s less 72 s, both of which bf16 holds.  fp16 does not
// hold 72 s of large scales: the code first.
template <typename T> struct Scale;
template <> struct Scale<__nv_bfloat16> {
  __nv_bfloat162 s, less;
  __device__ __forceinline__ void set(uint32_t low16) {
    const uint32_t both = __byte_perm(low16, 0, 0x1010);
    s = *reinterpret_cast<const __nv_bfloat162*>(&both);
    less = __hmul2(s, __float2bfloat162_rn(-72.0f));
  }
  __device__ __forceinline__ uint32_t pair(uint32_t word, int e) const {
    const uint32_t v = pick(e == 0 ? word << 1 : word >> (4 * e - 1), 0x001E001Eu, 0x42804280u);
    const __nv_bfloat162 d = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&v), s, less);
    return *reinterpret_cast<const uint32_t*>(&d);
  }
};
template <> struct Scale<__half> {
  __half2 s;
  __device__ __forceinline__ void set(uint32_t low16) { s = __float2half2_rn(bf16_bits(low16 & 0xFFFFu)); }
  __device__ __forceinline__ uint32_t pair(uint32_t word, int e) const {
    const uint32_t v = codes_to_pair<__half>(word, e);
    const __half2 d = __hmul2(*reinterpret_cast<const __half2*>(&v), s);
    return *reinterpret_cast<const uint32_t*>(&d);
  }
};
}  // namespace st4
