// Quantising weights to four bits by groups, and reading them back.
//
//   m = the element of a row's group of largest magnitude (the negative one of two),  s = -m / 8 rounded to 4 significant bits, 2^-20 <= |s| <= 1.875 * 2^12
//   q = w / s rounded to the nearest (ties to even), clamped to -8..7
//
// Four significant bits of the scale and four of the code make q s a number of 8: exact in bf16 and in fp16 (whose smallest unit, 2^-24, and largest number,
// 65504, bound the scale), so that every product with these weights multiplies the same numbers.  For normal weights in groups of 64 that
// costs 0.4% of the error that scales of full precision leave (0.0953 and 0.0949 of the weights' size).  The sign of s puts the extremum on -8, which symmetric codes of
// -7..7 leave unused (0.108).  A group with a NaN or an infinity has a scale that is NaN.
//
// A warp takes 16 rows by 128 columns, which holds whole groups of every size: its loads are all in flight together, extrema are joined by
// shuffles, and 1 KB of shared memory turns the codes from rows to the order of int4.cuh.
// Measured: 8192 x 8192 in bf16 43 to 44 us quantised, 3.9 TB/s of the 6.6 that a copy reaches: instructions bound it (the ALU pipe busy 76%); 30 to 31 us read back, 5.6 TB/s.  In fp16 41
// and 30, in fp32 83 and 52 us (3.7 and 5.8 TB/s).
#include "../common/host.h"
#include "../common/chain.cuh"
#include "int4.cuh"
#include <type_traits>

namespace {
using namespace st4;
using st::chain_begin;

constexpr int kWarps = 2;      // few: small matrices on as many SMs as they fill
constexpr int kCols = 128;      // of a warp's block
constexpr float kLeast = 9.5367431640625e-07f, kLargest = 7680.0f;      // 2^-20, 1.875 * 2^12

struct WeightsParams {
  long long stride;      // of the matrix's rows, in elements
  int rows, cols, groups, chunks, blocks;      // groups of a row; tiles and 128-column blocks beside one another
};

// The scale from the group's least and largest element, either of which is NaN where one of the group is.
__device__ __forceinline__ float scale_of(float low, float high) {
  const bool pos = high > -low;      // the extremum is positive: the scale negative
  uint32_t u = __float_as_uint(fmaxf(high, -low) * 0.125f);
  u = (u + 0x7FFFFu + ((u >> 20) & 1u)) & ~0xFFFFFu;      // 3 of 23 bits behind the leading one
  const float s = fminf(fmaxf(__uint_as_float(u), kLeast), kLargest);
  return !(isfinite(low) && isfinite(high)) ? __uint_as_float(0x7FC00000u) : pos ? -s : s;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// 16 bytes or, of fp32, 32: 8 elements of a row.
template <typename T> __device__ __forceinline__ void extremes(const Vec<T, 8>& v, float& low, float& high);
template <> __device__ __forceinline__ void extremes(const Vec<float, 8>& v, float& low, float& high) {
  low = high = v.v[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) low = min_nan(low, v.v[e]), high = max_nan(high, v.v[e]);
}
template <> __device__ __forceinline__ void extremes(const Vec<__nv_bfloat16, 8>& v, float& low, float& high) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&v);
  const __nv_bfloat162 a = __hmin2_nan(__hmin2_nan(p[0], p[1]), __hmin2_nan(p[2], p[3])), b = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3]));
  low = min_nan(__low2float(a), __high2float(a)), high = max_nan(__low2float(b), __high2float(b));
}
template <> __device__ __forceinline__ void extremes(const Vec<__half, 8>& v, float& low, float& high) {
  const __half2* p = reinterpret_cast<const __half2*>(&v);
  const __half2 a = __hmin2_nan(__hmin2_nan(p[0], p[1]), __hmin2_nan(p[2], p[3])), b = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3]));
  low = min_nan(__low2float(a), __high2float(a)), high = max_nan(__low2float(b), __high2float(b));
}

// 8 codes plus 8, four bits each: w / s to the nearest, ties to even, within -8..7.
// w * (1 / s), of an approximate reciprocal, may lie up to 2^-19 beside the quotient.  A quotient of a 16-bit w that is no tie is at least 2^-16 from one (w is at most 11 bits, s 4):
// rounded to multiples of 2^-17 first, ties are ties again and nothing else changes sides.  For fp32 the remainder, which fmaf gives exactly, says on which side of
// the border w is.
template <typename T>
__device__ __forceinline__ uint32_t codes_of(const Vec<T, 8>& v, float s) {
  const float inv = st::rcp_approx(s);
  uint32_t packed = 0;
  if constexpr (sizeof(T) == 2) {
    const bool within = fabsf(s) < kLargest;      // nothing lies below -8.5 steps, which is -8, unless the scale was bounded
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      float2 t = st::mul2(make_float2(to_float(v.v[e]), to_float(v.v[e + 1])), st::splat2(inv));
      if (!within) t = make_float2(fmaxf(t.x, -8.0f), fmaxf(t.y, -8.0f));                 // and NaN: -8, which the scale covers
      t = make_float2(fminf(t.x, 7.0f), fminf(t.y, 7.0f));
      t = st::add2(st::add2(t, st::splat2(96.0f)), st::splat2(-96.0f));
      t = st::add2(t, st::splat2(12582912.0f + 8.0f));                                    // 1.5 2^23: whole numbers in the low bits
      packed += (__float_as_uint(t.x) << (4 * e)) + (__float_as_uint(t.y) << (4 * e + 4));
    }
    uint32_t more = 0;      // 0x4B400000 of each
#pragma unroll
    for (int e = 0; e < 8; ++e) more += 0x4B400000u << (4 * e);
    return packed - more;
  } else {
    const float half = 0.5f * fabsf(s);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float w = v.v[e];
      float q = rintf(w * inv);
      const float r = fmaf(-q, s, w), a = fabsf(r);
      if (a > half || (a == half && (static_cast<int>(q) & 1))) q += (r < 0.0f) == (s < 0.0f) ? 1.0f : -1.0f;
      packed |= static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(q, -8.0f), 7.0f)) + 8) << (4 * e);
    }
    return packed;
  }
}

// Lane l of a warp holds columns 8 (l % 16) to 8 (l % 16) + 7 of rows 2 i + l / 16.
template <typename T, int GROUP, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32) quantize_kernel(const T* w, uint8_t* codes, __nv_bfloat16* scales, const WeightsParams p) {
  __shared__ uint32_t word[kWarps][16][17];      // 8 codes of a row; 17: rows on banks of their own
  chain_begin(w, codes, scales);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long b = static_cast<long long>(blockIdx.x) * kWarps + warp;
  const int u = static_cast<int>(b / p.blocks), j = static_cast<int>(b - static_cast<long long>(u) * p.blocks);
  if (u * kTileRows >= p.rows) return;
  const int c0 = j * kCols + (lane & 15) * 8, r0 = u * kTileRows + (lane >> 4);
  Vec<T, 8> v[8];
  const T* at = w + r0 * p.stride + c0;
  if (WIDE && (u + 1) * kTileRows <= p.rows && (j + 1) * kCols <= p.cols) {
#pragma unroll
    for (int i = 0; i < 8; ++i, at += 2 * p.stride)
#pragma unroll
      for (int h = 0; h < static_cast<int>(sizeof(T)) / 2; ++h) reinterpret_cast<uint4*>(&v[i])[h] = reinterpret_cast<const uint4*>(at)[h];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i, at += 2 * p.stride)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i].v[e] = r0 + 2 * i < p.rows && c0 + e < p.cols ? at[e] : from_float<T>(0.0f);
  }
  __nv_bfloat16* to = scales + (static_cast<long long>(u) * p.groups + c0 / GROUP) * 16 + (lane >> 4) * 2;
  const bool first = c0 % GROUP == 0 && c0 / GROUP < p.groups;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float low, high;
    extremes(v[i], low, high);
#pragma unroll
    for (int o = 1; o < GROUP / 8; o <<= 1) {
      low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, o));
      high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    const float s = scale_of(low, high);
    word[warp][2 * i + (lane >> 4)][lane & 15] = codes_of(v[i], s);
    if (first) to[(i & 3) * 4 + (i >> 2)] = __float2bfloat16_rn(s);      // row 2 i + l / 16: place 2 (row % 8) + row / 8
  }
  __syncwarp();
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (2 * j + c >= p.chunks) break;
    uint32_t out[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {      // byte t of 8 codes: columns 2 t and 2 t + 1 of them; of the 4 bytes the low nibbles, then the high ones
      const uint8_t* from = reinterpret_cast<const uint8_t*>(&word[warp][g][8 * c + 2 * s]) + t;
      const uint32_t four = __byte_perm(__byte_perm(from[0], from[8 * 17 * 4], 0x0040), __byte_perm(from[4], from[8 * 17 * 4 + 4], 0x0040), 0x5410);
      const uint32_t low = four & 0x0F0F0F0Fu, high = four >> 4 & 0x0F0F0F0Fu;
      out[s] = __byte_perm(low | low >> 4, high | high >> 4, 0x6420);
    }
    *reinterpret_cast<uint4*>(codes + (static_cast<long long>(u) * p.chunks + 2 * j + c) * kTileBytes + lane * 16) = make_uint4(out[0], out[1], out[2], out[3]);
  }
}

// The pairs of numbers that a lane's words hold go to shared memory as rows, from where they leave 16 bytes a lane.
template <typename T, int GROUP, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32) dequantize_kernel(const uint8_t* codes, const __nv_bfloat16* scales, T* w, const WeightsParams p) {
  using E = typename std::conditional<std::is_same<T, __half>::value, __half, __nv_bfloat16>::type;      // fp32 from bf16, which holds them all
  __shared__ __align__(16) uint32_t pair[kWarps][16][68];      // 64 pairs of a row; 68: rows on banks of their own
  chain_begin(codes, scales, w);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long b = static_cast<long long>(blockIdx.x) * kWarps + warp;
  const int u = static_cast<int>(b / p.blocks), j = static_cast<int>(b - static_cast<long long>(u) * p.blocks);
  if (u * kTileRows >= p.rows) return;
  uint4 in[2];
  uint32_t both[128 / GROUP];      // scales of rows g and g + 8
  const uint32_t* from = reinterpret_cast<const uint32_t*>(scales + (static_cast<long long>(u) * p.groups + j * (128 / GROUP)) * 16) + g;
#pragma unroll
  for (int c = 0; c < 2; ++c)
    if (2 * j + c < p.chunks) in[c] = *reinterpret_cast<const uint4*>(codes + (static_cast<long long>(u) * p.chunks + 2 * j + c) * kTileBytes + lane * 16);
#pragma unroll
  for (int i = 0; i < 128 / GROUP; ++i)
    if (j * (128 / GROUP) + i < p.groups) both[i] = from[i * 8];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (2 * j + c >= p.chunks) break;
    const uint32_t word[4] = {in[c].x, in[c].y, in[c].z, in[c].w};
    Scale<E> low, high;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      constexpr int kSteps = GROUP >= 64 ? 4 : 2;      // of 16 columns in a group
      if (s % kSteps == 0) low.set(both[(c * 64 + s * 16) / GROUP]), high.set(both[(c * 64 + s * 16) / GROUP] >> 16);
      uint32_t* to = &pair[warp][g][c * 32 + s * 8 + t];
      to[0] = low.pair(word[s], 0), to[4] = low.pair(word[s], 2);
      to[8 * 68] = high.pair(word[s], 1), to[8 * 68 + 4] = high.pair(word[s], 3);
    }
  }
  __syncwarp();
  const int c0 = j * kCols + (lane & 15) * 8;
  if (c0 >= p.cols) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = 2 * i + (lane >> 4), r = u * kTileRows + row;
    if (r >= p.rows) break;
    const uint4 eight = *reinterpret_cast<const uint4*>(&pair[warp][row][(lane & 15) * 4]);
    T* at = w + r * p.stride + c0;
    if constexpr (sizeof(T) == 2) {
      if (WIDE && c0 + 8 <= p.cols) {
        *reinterpret_cast<uint4*>(at) = eight;
        continue;
      }
    }
    const Vec<E, 8> v = *reinterpret_cast<const Vec<E, 8>*>(&eight);
    if constexpr (sizeof(T) == 4) {
      if (WIDE && c0 + 8 <= p.cols) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          reinterpret_cast<float4*>(at)[h] = make_float4(to_float(v.v[4 * h]), to_float(v.v[4 * h + 1]), to_float(v.v[4 * h + 2]), to_float(v.v[4 * h + 3]));
        continue;
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c0 + k < p.cols) at[k] = from_float<T>(to_float(v.v[k]));
  }
}

int plan(WeightsParams& p, unsigned& grid, int group, const void* codes, const void* scales) {
  if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) & 15) return st::fail(ST_ERR_INVALID, "int4: codes and scales must lie on 16-byte boundaries");
  if (p.rows < 1 || p.cols < 1 || p.rows > 1 << 30 || p.cols > 1 << 30 || (group != 32 && group != 64 && group != 128)) return st::fail(ST_ERR_INVALID, "int4: sizes out of range");
  p.groups = (p.cols + group - 1) / group;
  p.chunks = (p.cols + kTileCols - 1) / kTileCols;
  p.blocks = (p.cols + kCols - 1) / kCols;
  const long long n = (static_cast<long long>((p.rows + kTileRows - 1) / kTileRows) * p.blocks + kWarps - 1) / kWarps;
  if (n > 2147483647LL) return st::fail(ST_ERR_TOO_LARGE, "int4: matrix too large");
  grid = static_cast<unsigned>(n);
  return ST_OK;
}

template <typename T, int GROUP>
int quantize(const void* w, uint8_t* codes, __nv_bfloat16* scales, const WeightsParams& p, unsigned grid, cudaStream_t stream) {
  const bool wide = (reinterpret_cast<uintptr_t>(w) & 15) == 0 && p.stride * sizeof(T) % 16 == 0;
  const cudaError_t e = st::chained(wide ? quantize_kernel<T, GROUP, true> : quantize_kernel<T, GROUP, false>, dim3(grid), dim3(kWarps * 32), 0, stream)(
      static_cast<const T*>(w), codes, scales, p);
  return e == cudaSuccess ? ST_OK : st::fail_cuda(e, "int4 quantize");
}
template <typename T>
int quantize(const void* w, uint8_t* codes, __nv_bfloat16* scales, const WeightsParams& p, unsigned grid, int group, cudaStream_t stream) {
  if (group == 32) return quantize<T, 32>(w, codes, scales, p, grid, stream);
  if (group == 64) return quantize<T, 64>(w, codes, scales, p, grid, stream);
  return quantize<T, 128>(w, codes, scales, p, grid, stream);
}

template <typename T, int GROUP>
int dequantize(const uint8_t* codes, const __nv_bfloat16* scales, void* w, const WeightsParams& p, unsigned grid, cudaStream_t stream) {
  const bool wide = (reinterpret_cast<uintptr_t>(w) & 15) == 0 && p.stride * sizeof(T) % 16 == 0;
  const cudaError_t e = st::chained(wide ? dequantize_kernel<T, GROUP, true> : dequantize_kernel<T, GROUP, false>, dim3(grid), dim3(kWarps * 32), 0, stream)(
      codes, scales, static_cast<T*>(w), p);
  return e == cudaSuccess ? ST_OK : st::fail_cuda(e, "int4 dequantize");
}
template <typename T>
int dequantize(const uint8_t* codes, const __nv_bfloat16* scales, void* w, const WeightsParams& p, unsigned grid, int group, cudaStream_t stream) {
  if (group == 32) return dequantize<T, 32>(codes, scales, w, p, grid, stream);
  if (group == 64) return dequantize<T, 64>(codes, scales, w, p, grid, stream);
  return dequantize<T, 128>(codes, scales, w, p, grid, stream);
}
}  // namespace

struct StInt4WeightsArgs {
  void* w;
  void* codes;
  void* scales;
  long long stride;
  int rows, cols, group, type;
};

// w [rows, cols] (type 0 bf16, 1 fp16, 2 fp32; rows `stride` elements apart, columns contiguous) to codes and scales in the layout of int4.cuh; group: 32, 64 or 128.
ST_API int st_int4_quantize(const StInt4WeightsArgs* a, void* stream_v) {
  WeightsParams p{a->stride, a->rows, a->cols, 0, 0, 0};
  unsigned grid;
  if (const int e = plan(p, grid, a->group, a->codes, a->scales)) return e;
  uint8_t* c = static_cast<uint8_t*>(a->codes);
  __nv_bfloat16* s = static_cast<__nv_bfloat16*>(a->scales);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  switch (a->type) {
    case 0: return quantize<__nv_bfloat16>(a->w, c, s, p, grid, a->group, stream);
    case 1: return quantize<__half>(a->w, c, s, p, grid, a->group, stream);
    case 2: return quantize<float>(a->w, c, s, p, grid, a->group, stream);
  }
  return st::fail(ST_ERR_INVALID, "int4: unknown type");
}

// The weights that codes and scales stand for, into w.
ST_API int st_int4_dequantize(const StInt4WeightsArgs* a, void* stream_v) {
  WeightsParams p{a->stride, a->rows, a->cols, 0, 0, 0};
  unsigned grid;
  if (const int e = plan(p, grid, a->group, a->codes, a->scales)) return e;
  const uint8_t* c = static_cast<const uint8_t*>(a->codes);
  const __nv_bfloat16* s = static_cast<const __nv_bfloat16*>(a->scales);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  switch (a->type) {
    case 0: return dequantize<__nv_bfloat16>(c, s, a->w, p, grid, a->group, stream);
    case 1: return dequantize<__half>(c, s, a->w, p, grid, a->group, stream);
    case 2: return dequantize<float>(c, s, a->w, p, grid, a->group, stream);
  }
  return st::fail(ST_ERR_INVALID, "int4: unknown type");
}
