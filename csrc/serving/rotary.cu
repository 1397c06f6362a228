// Rotary positions for queries and keys at any positions: half or interleaved pairs, a part of the head, any frequencies.
//
//   y_a = m (x_a cos t - s x_b sin t),  y_b = m (x_b cos t + s x_a sin t),  t = position * freq[j],  s = 1 or, for the gradient, -1
//
// for the pairs (a, b) = (j, R/2 + j) or, interleaved, (2j, 2j + 1), j < R/2; elements from R on are copied.
// Bound by memory: every element is read and written once, 3 operations on it.  The angles are no table, which would cap the
// positions and be read from far away: a block forms those of its tokens once, in turns and fp64 (position * freq / 2 pi keeps 2^-35 of a
// turn at position 2^17, where fp32 keeps 2^-7), takes the sine and cosine of the fraction of a turn in fp32, adds what fp32 does not hold of the fraction
// to first order (its square is below 2^-46), and keeps them in shared memory for all heads of the token.
// Measured: 16384 rows of 16 + 16 heads of 128 in bf16, forward and backward, 92 us, 5.8 TB/s of the 6.5 that a copy reaches.  A step of 64 rows is a launch.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "../common/host.h"
#include "../common/chain.cuh"

namespace {
using st::chain_begin;

constexpr int kThreads = 256;
constexpr int kMaxTokens = 8;      // of a block
constexpr int kMaxAngles = 48 * 1024 / sizeof(float2);      // of a block

struct RotaryParams {
  long long q_row, q_head, k_row, k_head, qo_row, qo_head, ko_row, ko_head;
  long long tokens;
  int heads, kv_heads, half, dim, units, tokens_per_block;
  float magnitude, sign;
};

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

// A unit is F pairs: two vectors of F elements.  F = 16 bytes of elements, or 1 where sizes or strides do not allow that, which takes 3.4 times as long
// (16384 rows of 16 + 16 heads of 128 in bf16, one direction: all of the head 48 us, 120 or 116 elements of it, whose halves are no multiple of 8, 162).
template <typename T, int F, bool INTER, typename POS>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const T* q, const T* k, T* qo, T* ko, const POS* __restrict__ positions,
                                                          const double* __restrict__ freq, const RotaryParams p) {
  extern __shared__ float2 turn[];      // [tokens of the block][half]: (cos, sin), both times the magnitude
  chain_begin(q, k, positions, freq);
  const long long t0 = static_cast<long long>(blockIdx.x) * p.tokens_per_block;
  const int nt = static_cast<int>(min(static_cast<long long>(p.tokens_per_block), p.tokens - t0));
  for (int i = threadIdx.x; i < nt * p.half; i += kThreads) {
    const int t = i / p.half, j = i - t * p.half;
    const double turns = static_cast<double>(positions[t0 + t]) * freq[j] * 0.15915494309189533577;      // 1 / 2 pi
    const double halves = 2.0 * (turns - rint(turns));
    const float main = static_cast<float>(halves), rest = static_cast<float>(halves - main) * 3.14159265f;      // |rest| <= pi 2^-25
    float s, c;
    sincospif(main, &s, &c);
    turn[i] = make_float2(fmaf(-s, rest, c) * p.magnitude, fmaf(c, rest, s) * p.magnitude * p.sign);
  }
  __syncthreads();
  const int heads = p.heads + p.kv_heads, per_token = heads * p.units, rotated = p.half / F;
  for (int i = threadIdx.x; i < nt * per_token; i += kThreads) {
    const int t = i / per_token, r = i - t * per_token, h = r / p.units, u = r - h * p.units;
    const long long token = t0 + t;
    const T* src;
    T* dst;
    if (h < p.heads) {
      src = q + token * p.q_row + h * p.q_head;
      dst = qo + token * p.qo_row + h * p.qo_head;
    } else {
      src = k + token * p.k_row + (h - p.heads) * p.k_head;
      dst = ko + token * p.ko_row + (h - p.heads) * p.ko_head;
    }
    using V = Vec<T, F>;
    if (u >= rotated) {      // behind the rotated part; the last element of an odd rest stands alone (only where F is 1)
      const int d = 2 * p.half + (u - rotated) * 2 * F;
      *reinterpret_cast<V*>(dst + d) = *reinterpret_cast<const V*>(src + d);
      if (d + F < p.dim) *reinterpret_cast<V*>(dst + d + F) = *reinterpret_cast<const V*>(src + d + F);
      continue;
    }
    const int j = u * F, first = INTER ? 2 * j : j, second = INTER ? 2 * j + F : p.half + j;
    const V x = *reinterpret_cast<const V*>(src + first), y = *reinterpret_cast<const V*>(src + second);
    V ox, oy;
#pragma unroll
    for (int e = 0; e < F; ++e) {
      const float2 cs = turn[t * p.half + j + e];
      // interleaved: the 2F elements of both vectors in order are the pairs
      const float a = to_float(INTER ? (2 * e < F ? x.v[(2 * e) % F] : y.v[(2 * e) % F]) : x.v[e]);
      const float b = to_float(INTER ? (2 * e + 1 < F ? x.v[(2 * e + 1) % F] : y.v[(2 * e + 1) % F]) : y.v[e]);
      const T oa = from_float<T>(a * cs.x - b * cs.y), ob = from_float<T>(b * cs.x + a * cs.y);
      if constexpr (INTER) {
        (2 * e < F ? ox : oy).v[(2 * e) % F] = oa;
        (2 * e + 1 < F ? ox : oy).v[(2 * e + 1) % F] = ob;
      } else {
        ox.v[e] = oa;
        oy.v[e] = ob;
      }
    }
    *reinterpret_cast<V*>(dst + first) = ox;
    *reinterpret_cast<V*>(dst + second) = oy;
  }
}

template <typename T, int F, bool INTER, typename POS>
int launch(const void* q, const void* k, void* qo, void* ko, const void* positions, const double* freq, RotaryParams p, bool in_place, cudaStream_t stream) {
  p.units = p.half / F + (in_place ? 0 : (p.dim - 2 * p.half + 2 * F - 1) / (2 * F));
  // enough tokens to a block for two units per thread, while that leaves two blocks per SM and their angles need no opting in
  const int per_token = (p.heads + p.kv_heads) * p.units;
  int n = 1;
  while (n < kMaxTokens && n * per_token < 2 * kThreads && 2 * n * p.half <= kMaxAngles && p.tokens / (2 * n) >= 2 * st::sm_count()) n *= 2;
  p.tokens_per_block = n;
  const long long blocks = (p.tokens + n - 1) / n;
  if (blocks > 2147483647LL) return st::fail(ST_ERR_TOO_LARGE, "rotary: too many tokens");
  const size_t smem = static_cast<size_t>(n) * p.half * sizeof(float2);
  const cudaError_t e = st::chained(rotary_kernel<T, F, INTER, POS>, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), smem, stream)(
      static_cast<const T*>(q), static_cast<const T*>(k), static_cast<T*>(qo), static_cast<T*>(ko), static_cast<const POS*>(positions), freq, p);
  if (e != cudaSuccess) return st::fail_cuda(e, "rotary");
  return ST_OK;
}

template <typename T>
int dispatch(const void* q, const void* k, void* qo, void* ko, const void* positions, int pos64, const double* freq, const RotaryParams& p, bool inter, bool in_place,
             cudaStream_t stream) {
  constexpr int F = 16 / sizeof(T);
  const long long all = p.q_row | p.q_head | p.k_row | p.k_head | p.qo_row | p.qo_head | p.ko_row | p.ko_head;
  const uintptr_t at = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(qo) | reinterpret_cast<uintptr_t>(ko);
  const bool wide = p.half % F == 0 && p.dim % (2 * F) == 0 && all % F == 0 && (at & 15) == 0;
#define ST_ROTARY(FF, II) \
  (pos64 ? launch<T, FF, II, long long>(q, k, qo, ko, positions, freq, p, in_place, stream) : launch<T, FF, II, int>(q, k, qo, ko, positions, freq, p, in_place, stream))
  if (wide) return inter ? ST_ROTARY(F, true) : ST_ROTARY(F, false);
  return inter ? ST_ROTARY(1, true) : ST_ROTARY(1, false);
#undef ST_ROTARY
}
}  // namespace

// Rotates q [tokens, heads, dim] into qo and, unless kv_heads is 0, k [tokens, kv_heads, dim] into ko (dim contiguous, any row and head
// strides, in elements; qo == q and ko == k with the same strides: in place).  freq: fp64 [half].  type: 0 bf16, 1 fp16, 2 fp32.
ST_API int st_rotary(const void* q, const void* k, void* qo, void* ko, const void* positions, int pos64, const double* freq, long long tokens, int heads, int kv_heads,
                     int dim, int half, long long q_row, long long q_head, long long k_row, long long k_head, long long qo_row, long long qo_head,
                     long long ko_row, long long ko_head, int interleaved, float magnitude, int backward, int type, void* stream_v) {
  if (tokens < 0 || heads < 1 || kv_heads < 0 || dim < 2 || half < 1 || 2 * half > dim || half > 2048)
    return st::fail(ST_ERR_INVALID, "rotary: sizes out of range");
  if (tokens == 0) return ST_OK;
  const RotaryParams p{q_row, q_head, k_row, k_head, qo_row, qo_head, ko_row, ko_head, tokens, heads, kv_heads, half, dim, 0, 1, magnitude, backward ? -1.0f : 1.0f};
  const bool in_place = q == qo && k == ko;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  switch (type) {
    case 0: return dispatch<__nv_bfloat16>(q, k, qo, ko, positions, pos64, freq, p, interleaved != 0, in_place, stream);
    case 1: return dispatch<__half>(q, k, qo, ko, positions, pos64, freq, p, interleaved != 0, in_place, stream);
    case 2: return dispatch<float>(q, k, qo, ko, positions, pos64, freq, p, interleaved != 0, in_place, stream);
  }
  return st::fail(ST_ERR_INVALID, "rotary: unknown type");
}
