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
// Bound by memory.  A warp takes 16 rows by 128 columns, which holds whole groups of every size: its loads are all in flight together, extrema are joined by
// shuffles, and 1 KB of shared memory turns the codes from rows to the order of int4.cuh.
#include "../common/host.h"
#include "../common/chain.cuh"
#include "int4.cuh"

namespace {
using namespace st4;
using st::chain_begin;

constexpr int kWarps = 4;
constexpr int kCols = 128;      // of a warp's block
constexpr float kLeast = 9.5367431640625e-07f, kLargest = 7680.0f;      // 2^-20, 1.875 * 2^12

struct WeightsParams {
  long long stride;      // of the matrix's rows, in elements
  int rows, cols, groups, chunks, blocks;      // groups of a row; tiles and 128-column blocks beside one another
};

// The scale from the group's least and largest element.
__device__ __forceinline__ float scale_of(float low, float high, bool finite) {
  const bool pos = high > -low;      // the extremum is positive: the scale negative
  uint32_t u = __float_as_uint(fmaxf(high, -low) * 0.125f);
  u = (u + 0x7FFFFu + ((u >> 20) & 1u)) & ~0xFFFFFu;      // 3 of 23 bits behind the leading one
  const float s = fminf(fmaxf(__uint_as_float(u), kLeast), kLargest);
  return !finite ? __uint_as_float(0x7FC00000u) : pos ? -s : s;
}

// w / s to the nearest, ties to even.  w * (1 / s) may fall on the wrong side of a border; the remainder, which fmaf gives exactly, says so.
__device__ __forceinline__ int code_of(float w, float s, float inv, float half) {
  float q = rintf(w * inv);
  const float r = fmaf(-q, s, w);
  const float a = fabsf(r);
  if (a > half || (a == half && (static_cast<int>(q) & 1))) q += (r < 0.0f) == (s < 0.0f) ? 1.0f : -1.0f;
  return static_cast<int>(fminf(fmaxf(q, -8.0f), 7.0f));      // NaN: -8, which the scale covers
}

// Lane l of a warp holds columns 8 (l % 16) to 8 (l % 16) + 7 of rows 2 i + l / 16.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32) quantize_kernel(const T* w, uint8_t* codes, __nv_bfloat16* scales, const WeightsParams p, const int group) {
  __shared__ uint32_t word[kWarps][16][17];      // 8 codes of a row; 17: rows on banks of their own
  chain_begin(w, codes, scales);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long b = static_cast<long long>(blockIdx.x) * kWarps + warp;
  const int u = static_cast<int>(b / p.blocks), j = static_cast<int>(b - static_cast<long long>(u) * p.blocks);
  if (u * kTileRows >= p.rows) return;
  const int c0 = j * kCols + (lane & 15) * 8, r0 = u * kTileRows + (lane >> 4);
  Vec<T, 8> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 2 * i;
    const T* at = w + r * p.stride + c0;
    if (WIDE && r < p.rows && c0 + 8 <= p.cols) {
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(&v[i]) = *reinterpret_cast<const uint4*>(at);
      } else {
        reinterpret_cast<uint4*>(&v[i])[0] = reinterpret_cast<const uint4*>(at)[0];
        reinterpret_cast<uint4*>(&v[i])[1] = reinterpret_cast<const uint4*>(at)[1];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i].v[e] = r < p.rows && c0 + e < p.cols ? at[e] : from_float<T>(0.0f);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float low = to_float(v[i].v[0]), high = low;
    bool finite = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = to_float(v[i].v[e]);
      low = fminf(low, x);
      high = fmaxf(high, x);
      finite = finite && isfinite(x);
    }
    for (int o = 1; o < group / 8; o <<= 1) {
      low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
      high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
      finite = __shfl_xor_sync(0xffffffffu, finite, o) && finite;
    }
    const float s = scale_of(low, high, finite), inv = 1.0f / s, half = 0.5f * fabsf(s);
    uint32_t packed = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) packed |= static_cast<uint32_t>(code_of(to_float(v[i].v[e]), s, inv, half) + 8) << (4 * e);
    const int row = 2 * i + (lane >> 4);
    word[warp][row][lane & 15] = packed;
    const int at = c0 / group;
    if (c0 % group == 0 && at < p.groups)
      scales[(static_cast<long long>(u) * p.groups + at) * 16 + 2 * (row & 7) + (row >> 3)] = __float2bfloat16_rn(s);
  }
  __syncwarp();
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (2 * j + c >= p.chunks) break;
    uint32_t out[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      out[s] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {      // byte t of 8 codes: columns 2 t and 2 t + 1 of them
        const uint32_t pair = word[warp][g + 8 * (e & 1)][8 * c + 2 * s + (e >> 1)] >> (8 * t);
        out[s] |= (pair & 15u) << (4 * e) | ((pair >> 4) & 15u) << (4 * e + 16);
      }
    }
    *reinterpret_cast<uint4*>(codes + (static_cast<long long>(u) * p.chunks + 2 * j + c) * kTileBytes + lane * 16) = make_uint4(out[0], out[1], out[2], out[3]);
  }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32) dequantize_kernel(const uint8_t* codes, const __nv_bfloat16* scales, T* w, const WeightsParams p, const int group) {
  __shared__ uint4 word[kWarps][2][4][8];      // [tile][word][g]: those of lanes 4 g to 4 g + 3 together
  chain_begin(codes, scales, w);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long b = static_cast<long long>(blockIdx.x) * kWarps + warp;
  const int u = static_cast<int>(b / p.blocks), j = static_cast<int>(b - static_cast<long long>(u) * p.blocks);
  if (u * kTileRows >= p.rows) return;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (2 * j + c >= p.chunks) break;
    const uint4 in = *reinterpret_cast<const uint4*>(codes + (static_cast<long long>(u) * p.chunks + 2 * j + c) * kTileBytes + lane * 16);
    const uint32_t part[4] = {in.x, in.y, in.z, in.w};
#pragma unroll
    for (int s = 0; s < 4; ++s) reinterpret_cast<uint32_t*>(word[warp][c][s])[lane] = part[s];
  }
  __syncwarp();
  const int c0 = j * kCols + (lane & 15) * 8;
  if (c0 >= p.cols) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = 2 * i + (lane >> 4), r = u * kTileRows + row;
    if (r >= p.rows) break;
    const uint4 in = word[warp][(lane >> 3) & 1][(lane & 7) >> 1][row & 7];
    const uint32_t part[4] = {in.x, in.y, in.z, in.w};
    const float s = __bfloat162float(scales[(static_cast<long long>(u) * p.groups + c0 / group) * 16 + 2 * (row & 7) + (row >> 3)]);
    const int e = 2 * (lane & 1) + (row >> 3);
    Vec<T, 8> v;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      v.v[2 * t] = from_float<T>(static_cast<float>(static_cast<int>((part[t] >> (4 * e)) & 15u) - 8) * s);
      v.v[2 * t + 1] = from_float<T>(static_cast<float>(static_cast<int>((part[t] >> (4 * e + 16)) & 15u) - 8) * s);
    }
    T* at = w + r * p.stride + c0;
    if (WIDE && c0 + 8 <= p.cols) {
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(&v);
      } else {
        reinterpret_cast<uint4*>(at)[0] = reinterpret_cast<const uint4*>(&v)[0];
        reinterpret_cast<uint4*>(at)[1] = reinterpret_cast<const uint4*>(&v)[1];
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c0 + k < p.cols) at[k] = v.v[k];
    }
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

template <typename T>
int quantize(const void* w, uint8_t* codes, __nv_bfloat16* scales, const WeightsParams& p, unsigned grid, int group, cudaStream_t stream) {
  const bool wide = (reinterpret_cast<uintptr_t>(w) & 15) == 0 && p.stride * sizeof(T) % 16 == 0;
  const cudaError_t e = st::chained(wide ? quantize_kernel<T, true> : quantize_kernel<T, false>, dim3(grid), dim3(kWarps * 32), 0, stream)(
      static_cast<const T*>(w), codes, scales, p, group);
  return e == cudaSuccess ? ST_OK : st::fail_cuda(e, "int4 quantize");
}

template <typename T>
int dequantize(const uint8_t* codes, const __nv_bfloat16* scales, void* w, const WeightsParams& p, unsigned grid, int group, cudaStream_t stream) {
  const bool wide = (reinterpret_cast<uintptr_t>(w) & 15) == 0 && p.stride * sizeof(T) % 16 == 0;
  const cudaError_t e = st::chained(wide ? dequantize_kernel<T, true> : dequantize_kernel<T, false>, dim3(grid), dim3(kWarps * 32), 0, stream)(
      codes, scales, static_cast<T*>(w), p, group);
  return e == cudaSuccess ? ST_OK : st::fail_cuda(e, "int4 dequantize");
}
}  // namespace

// w [rows, cols] (type 0 bf16, 1 fp16, 2 fp32; rows `stride` elements apart, columns contiguous) to codes and scales in the layout of int4.cuh; group: 32, 64 or 128.
ST_API int st_int4_quantize(const void* w, void* codes, void* scales, int rows, int cols, long long stride, int group, int type, void* stream_v) {
  WeightsParams p{stride, rows, cols, 0, 0, 0};
  unsigned grid;
  if (const int e = plan(p, grid, group, codes, scales)) return e;
  uint8_t* c = static_cast<uint8_t*>(codes);
  __nv_bfloat16* s = static_cast<__nv_bfloat16*>(scales);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  switch (type) {
    case 0: return quantize<__nv_bfloat16>(w, c, s, p, grid, group, stream);
    case 1: return quantize<__half>(w, c, s, p, grid, group, stream);
    case 2: return quantize<float>(w, c, s, p, grid, group, stream);
  }
  return st::fail(ST_ERR_INVALID, "int4: unknown type");
}

// The weights that codes and scales stand for, into w.
ST_API int st_int4_dequantize(const void* codes, const void* scales, void* w, int rows, int cols, long long stride, int group, int type, void* stream_v) {
  WeightsParams p{stride, rows, cols, 0, 0, 0};
  unsigned grid;
  if (const int e = plan(p, grid, group, codes, scales)) return e;
  const uint8_t* c = static_cast<const uint8_t*>(codes);
  const __nv_bfloat16* s = static_cast<const __nv_bfloat16*>(scales);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  switch (type) {
    case 0: return dequantize<__nv_bfloat16>(c, s, w, p, grid, group, stream);
    case 1: return dequantize<__half>(c, s, w, p, grid, group, stream);
    case 2: return dequantize<float>(c, s, w, p, grid, group, stream);
  }
  return st::fail(ST_ERR_INVALID, "int4: unknown type");
}
