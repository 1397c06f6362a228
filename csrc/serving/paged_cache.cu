// A key / value cache of pages of 8-bit codes: block tables and slot maps from request lengths, storing tokens, reading them back.
//
// Codes are e4m3, [pages, kv_heads, page, dim]; a page and head has one scale, a power of two: 2^e with the least e for which
// the largest finite magnitude of the page is at most 448 * 2^e, kept to -60..60.  With a power of two the product code * scale is exact (in bf16
// too), the code has e4m3's four significant bits whatever e is, and where a later token raises e the page's older codes only change
// if they become subnormal.  Magnitudes above 448 * 2^e (infinities) are stored as that largest value, NaN as NaN.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "paged.cuh"

namespace {
using st::chain_begin;

// ---- block tables and slot maps -------------------------------------------------------------------------------------------------
// Integer work on a few KB where a step decodes, on 12 bytes per row where prompts are admitted; launch latency bounds the
// first, stores the second.  Every block forms the prefix sums over all sequences in its own shared memory (8 bytes per
// sequence, from L2), so that none waits for another and one launch does it; then each takes its share of the rows and of the new pages.
constexpr int kPlanThreads = 512;
constexpr int kMaxSequences = 8192;

// Exclusive prefix sums of (tokens added, pages needed) of all sequences into shared memory, totals at [B].
__device__ void plan_scan(const int* __restrict__ lengths, const int* __restrict__ added, int B, int width, int shift, int* tok, int* blk) {
  __shared__ int2 warp_total[kPlanThreads / 32];
  __shared__ int2 carry;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) carry = make_int2(0, 0);
  __syncthreads();
  for (int base = 0; base < B; base += kPlanThreads) {
    const int b = base + threadIdx.x;
    int x = 0, y = 0;
    if (b < B) {
      const int have = max(lengths[b], 0);
      x = max(added[b], 0);
      y = st::blocks_of(have + static_cast<long long>(x), shift, width) - st::blocks_of(have, shift, width);
    }
    int sx = x, sy = y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int ux = __shfl_up_sync(0xffffffffu, sx, o), uy = __shfl_up_sync(0xffffffffu, sy, o);
      if (lane >= o) sx += ux, sy += uy;
    }
    if (lane == 31) warp_total[warp] = make_int2(sx, sy);
    __syncthreads();
    int2 before = carry;
    for (int w = 0; w < warp; ++w) before.x += warp_total[w].x, before.y += warp_total[w].y;
    if (b < B) tok[b] = before.x + sx - x, blk[b] = before.y + sy - y;
    __syncthreads();
    if (threadIdx.x == kPlanThreads - 1) carry = make_int2(before.x + sx, before.y + sy);
    __syncthreads();
  }
  if (threadIdx.x == 0) tok[B] = carry.x, blk[B] = carry.y;
  __syncthreads();
}

// The last b with first[b] <= i; sequences with nothing share their successor's entry and are passed over.
__device__ __forceinline__ int owner(const int* first, int B, int i) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const int* __restrict__ lengths, const int* __restrict__ added, int* table, long long table_row, int width,
                                                            const int* __restrict__ free_list, const int* __restrict__ free_count, int free_size, int shift, int B, long long rows,
                                                            int* starts, int* positions, long long* slots, int* lengths_after, int* free_after) {
  extern __shared__ int sums[];
  chain_begin(lengths, added, free_list, free_count);
  int *tok = sums, *blk = sums + B + 1;
  plan_scan(lengths, added, B, width, shift, tok, blk);
  const int total = tok[B], fresh = blk[B], count = min(*free_count, free_size), P = 1 << shift;
  const int first = blockIdx.x * kPlanThreads + threadIdx.x, stride = gridDim.x * kPlanThreads;
  for (int b = first; b <= B; b += stride) {
    starts[b] = tok[b];
    if (b < B) lengths_after[b] = max(lengths[b], 0) + max(added[b], 0);
  }
  if (first == 0) *free_after = count - fresh;
  // new pages, from the end of the list in the order of sequences and blocks; none left: -1
  for (int i = first; i < fresh; i += stride) {
    const int b = owner(blk, B, i), nth = count - 1 - i;
    table[b * table_row + st::blocks_of(max(lengths[b], 0), shift, width) + i - blk[b]] = nth >= 0 ? free_list[nth] : -1;
  }
  // four rows a thread: one search, then a walk
  for (long long r0 = 4LL * first; r0 < rows; r0 += 4LL * stride) {
    int pos[4];
    long long slot[4];
    int b = r0 < total ? owner(tok, B, static_cast<int>(r0)) : B, have = 0, held = 0, at = -1, page = -1;
    if (b < B) have = max(lengths[b], 0), held = st::blocks_of(have, shift, width);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long r = r0 + j;
      pos[j] = 0, slot[j] = -1;
      if (r >= total) continue;
      while (r >= tok[b + 1]) {
        ++b, at = -1;
        have = max(lengths[b], 0), held = st::blocks_of(have, shift, width);
      }
      pos[j] = have + static_cast<int>(r - tok[b]);
      const int block = pos[j] >> shift;
      if (block >= width) continue;
      if (block != at) {
        at = block;
        const int nth = count - 1 - (blk[b] + block - held);
        page = block < held ? table[b * table_row + block] : nth >= 0 ? free_list[nth] : -1;
      }
      if (page >= 0) slot[j] = (static_cast<long long>(page) << shift) + (pos[j] & (P - 1));
    }
    if (r0 + 4 <= rows) {
      *reinterpret_cast<int4*>(positions + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<longlong2*>(slots + r0) = make_longlong2(slot[0], slot[1]);
      *reinterpret_cast<longlong2*>(slots + r0 + 2) = make_longlong2(slot[2], slot[3]);
    } else {
      for (int j = 0; r0 + j < rows; ++j) positions[r0 + j] = pos[j], slots[r0 + j] = slot[j];
    }
  }
}

// Pages of finished sequences back to the end of the list, in the order of sequences and blocks.  One block: a warp counts a
// sequence's pages at a time, the counts are summed, and the warps write.
__global__ void __launch_bounds__(kPlanThreads) release_kernel(int* lengths, const unsigned char* __restrict__ done, int* table, long long table_row, int width, int* free_list,
                                                               int* free_count, int free_size, int shift, int B, unsigned* err) {
  extern __shared__ int sums[];
  chain_begin(done);
  __shared__ int carry;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int b = warp; b < B; b += kPlanThreads / 32) {
    int n = 0;
    if (done[b])
      for (int i = lane, e = st::blocks_of(max(lengths[b], 0), shift, width); i < e; i += 32) n += table[b * table_row + i] >= 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) sums[b] = n;
  }
  __syncthreads();
  if (warp == 0) {      // exclusive prefix sums in place, 32 at a time
    int before = max(*free_count, 0);
    for (int base = 0; base < B; base += 32) {
      const int x = base + lane < B ? sums[base + lane] : 0;
      int s = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
      }
      if (base + lane < B) sums[base + lane] = before + s - x;
      before += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) carry = before;
  }
  __syncthreads();
  for (int b = warp; b < B; b += kPlanThreads / 32) {
    if (!done[b]) continue;
    int at = sums[b];
    for (int i0 = 0, e = st::blocks_of(max(lengths[b], 0), shift, width); i0 < e; i0 += 32) {
      const int page = i0 + lane < e ? table[b * table_row + i0 + lane] : -1;
      const unsigned some = __ballot_sync(0xffffffffu, page >= 0);
      if (page >= 0) {
        const int to = at + __popc(some & ((1u << lane) - 1));
        if (to < free_size) free_list[to] = page;      // more pages than the list has room for were never taken from it
        else st::report_error(err, st::ERR_BOUNDS, 0x7001);
      }
      at += __popc(some);
      if (i0 + lane < e) table[b * table_row + i0 + lane] = -1;
    }
    __syncwarp();
    if (lane == 0) lengths[b] = 0;
  }
  if (threadIdx.x == 0) *free_count = min(carry, free_size);
}

// ---- storing --------------------------------------------------------------------------------------------------------------------
// Bound by memory: 2 (4 for fp32) bytes read and 1 written per element.  Rows that follow one another in a page are a group, found by
// its first row; the largest magnitude of the group and of each head decides the scale, so every element is looked at twice: the
// second time from registers, which hold 16 rows of 128 elements of 16 bits per warp, or from L1 where there are more rows.
// A warp works on one group, head and tensor; where a page holds more rows than its registers, two or four warps share a group.
// Measured: 7 prompts of up to 4096 tokens, 16 heads of 128, pages of 16, stored and read back, 94 us (the bytes: 77); a block that went through a
// group's heads one after the other took 324.  One token of each of 96 sequences: two launches, host time.
constexpr int kStoreThreads = 256, kStoreWarps = kStoreThreads / 32;
constexpr int kHeld = 8;      // 16-byte loads that a thread keeps

struct PutParams {
  long long k_row, k_head, v_row, v_head;
  long long rows, pages;
  int kv_heads, shift;
  int segment, team, heads_per_block;      // set at launch
};

// What differs between the types: 16 bytes to magnitudes (as integers, which order as they do), and to codes.
template <typename T> struct Raw;
template <typename T> struct Raw16 {
  static constexpr int kCodes = 8;
  static __device__ __forceinline__ uint4 load(const T* p, bool wide) {
    if (wide) return *reinterpret_cast<const uint4*>(p);
    const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
    return make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
  }
  static __device__ __forceinline__ uint32_t top(uint32_t m, uint4 x) {      // two magnitudes side by side
    m = __vmaxu2(m, __vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu));
    return __vmaxu2(m, __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
  }
  static __device__ __forceinline__ uint32_t one(uint32_t m) { return max(m & 0xffffu, m >> 16); }
  static __device__ __forceinline__ uint32_t finite(uint32_t x) {
    const uint32_t lo = x & 0x7fffu, hi = x >> 16 & 0x7fffu;
    return (lo < Raw<T>::kInf ? lo : 0u) | (hi < Raw<T>::kInf ? hi << 16 : 0u);
  }
  static __device__ __forceinline__ uint32_t pair(float2 x, float inv) { return __nv_cvt_float2_to_fp8x2(make_float2(x.x * inv, x.y * inv), __NV_SATFINITE, __NV_E4M3); }
  static __device__ __forceinline__ void put(unsigned char* p, uint4 x, float inv) {
    const uint32_t a = pair(Raw<T>::two(x.x), inv) | pair(Raw<T>::two(x.y), inv) << 16, b = pair(Raw<T>::two(x.z), inv) | pair(Raw<T>::two(x.w), inv) << 16;
    *reinterpret_cast<uint2*>(p) = make_uint2(a, b);
  }
};
template <> struct Raw<__nv_bfloat16> : Raw16<__nv_bfloat16> {
  static constexpr uint32_t kInf = 0x7f80;
  static __device__ __forceinline__ float value(uint32_t m) { return __uint_as_float(m << 16); }
  static __device__ __forceinline__ float2 two(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
};
template <> struct Raw<__half> : Raw16<__half> {
  static constexpr uint32_t kInf = 0x7c00;
  static __device__ __forceinline__ float value(uint32_t m) { return __half2float(__ushort_as_half(static_cast<unsigned short>(m))); }
  static __device__ __forceinline__ float2 two(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
};
template <> struct Raw<float> {
  static constexpr int kCodes = 4;
  static constexpr uint32_t kInf = 0x7f800000u;
  static __device__ __forceinline__ uint4 load(const float* p, bool wide) {
    if (wide) return *reinterpret_cast<const uint4*>(p);
    const unsigned* u = reinterpret_cast<const unsigned*>(p);
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  static __device__ __forceinline__ uint32_t top(uint32_t m, uint4 x) {
    return max(max(m, max(x.x & 0x7fffffffu, x.y & 0x7fffffffu)), max(x.z & 0x7fffffffu, x.w & 0x7fffffffu));
  }
  static __device__ __forceinline__ uint32_t one(uint32_t m) { return m; }
  static __device__ __forceinline__ uint32_t finite(uint32_t x) { return (x & 0x7fffffffu) < kInf ? x & 0x7fffffffu : 0u; }
  static __device__ __forceinline__ float value(uint32_t m) { return __uint_as_float(m); }
  static __device__ __forceinline__ void put(unsigned char* p, uint4 x, float inv) {
    *reinterpret_cast<uint32_t*>(p) =
        __nv_cvt_float2_to_fp8x2(make_float2(__uint_as_float(x.x) * inv, __uint_as_float(x.y) * inv), __NV_SATFINITE, __NV_E4M3) |
        static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(__uint_as_float(x.z) * inv, __uint_as_float(x.w) * inv), __NV_SATFINITE, __NV_E4M3)) << 16;
  }
};

// The page's older codes re-rounded to a larger scale: code * 2^(old - new).
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * i)), __NV_E4M3);
    const float2 x = __half22float2(__half2(h));
    out |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(x.x * ratio, x.y * ratio), __NV_SATFINITE, __NV_E4M3)) << (16 * i);
  }
  return out;
}

// One tensor's part of a group: rows [0, n) of one head from src go to page offsets [off, off + n).  The team is `warps` warps, this one
// its `me`-th; with several, all teams of the block come here together (n = 0: only for the barriers).
template <typename T, int D>
__device__ void store_group(const T* src, long long row_stride, bool wide, unsigned char* dst, float* scale, int off, int n, int me, int warps, uint32_t* shared_top) {
  using R = Raw<T>;
  constexpr int L = D / R::kCodes, RP = 32 / L;      // lanes of a row, rows of a load
  const int lane = threadIdx.x & 31, first = me * RP + lane / L, step = warps * RP, at = lane % L * R::kCodes;
  uint4 held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int r = first + i * step;
    held[i] = r < n ? R::load(src + r * row_stride + at, wide) : make_uint4(0, 0, 0, 0);
  }
  const float before = n > 0 && off > 0 ? *scale : 0.0f;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) m = R::top(m, held[i]);
  for (int r = first + kHeld * step; r < n; r += step) m = R::top(m, R::load(src + r * row_stride + at, wide));
  m = R::one(m);
  if (__any_sync(0xffffffffu, m >= R::kInf)) {      // once more without what is not finite
    m = 0;
    for (int r = first; r < n; r += step) {
      const uint4 x = R::load(src + r * row_stride + at, wide);
      m = R::top(m, make_uint4(R::finite(x.x), R::finite(x.y), R::finite(x.z), R::finite(x.w)));
    }
    m = R::one(m);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (warps > 1) {
    const int warp = threadIdx.x >> 5;
    __syncthreads();      // the group before may still be read
    if (lane == 0) shared_top[warp] = m;
    __syncthreads();      // and every warp has read the old scale
    for (int w = 0; w < warps; ++w) m = max(m, shared_top[warp - me + w]);
  }
  if (n == 0) return;
  __syncwarp();
  int e = st::page_exponent(R::value(m));
  const int old = off > 0 ? st::scale_exponent(before) : st::kMinExponent;
  e = max(e, old);
  const float inv = st::exp2_int(-e);
  if (e > old && off > 0) {
    const float ratio = st::exp2_int(old - e);      // 2^-120 at least
    for (int i = me * 32 + lane; i < off * (D / 4); i += warps * 32) {
      uint32_t* p = reinterpret_cast<uint32_t*>(dst) + i;
      *p = rescale4(*p, ratio);
    }
  }
  if (me == 0 && lane == 0) *scale = st::exp2_int(e);
  unsigned char* out = dst + static_cast<long long>(off) * D + at;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int r = first + i * step;
    if (r < n) R::put(out + r * D, held[i], inv);
  }
  for (int r = first + kHeld * step; r < n; r += step) R::put(out + r * D, R::load(src + r * row_stride + at, wide), inv);
  __syncwarp();
}

// Block (segment of at most a page's rows, heads_per_block heads).
template <typename T, int D>
__global__ void __launch_bounds__(kStoreThreads) store_kernel(const T* __restrict__ k, const T* __restrict__ v, unsigned char* kc, unsigned char* vc, float* ks, float* vs,
                                                              const long long* __restrict__ slots, const PutParams p, bool wide, unsigned* err) {
  chain_begin(k, v, slots);
  __shared__ uint32_t goes_on[2 * kStoreThreads / 32];      // a bit per row of the segment and of the page's length behind it: it follows the row before in its page
  __shared__ int first_row[kStoreThreads], group_rows[kStoreThreads];
  __shared__ long long first_slot[kStoreThreads];
  __shared__ int groups;
  __shared__ uint32_t shared_top[kStoreWarps];
  const long long r0 = static_cast<long long>(blockIdx.x) * p.segment;
  const int P = 1 << p.shift, warp = threadIdx.x >> 5;
  const long long limit = p.pages << p.shift;
  if (threadIdx.x == 0) groups = 0;
  bool leads = false;
  long long mine = -1;
  for (int j = threadIdx.x, part = 0; part < (p.segment + P + kStoreThreads - 1) / kStoreThreads; j += kStoreThreads, ++part) {
    const long long r = r0 + j, s = r < p.rows ? slots[r] : -1;
    const bool goes = s >= 0 && (s & (P - 1)) != 0 && r > 0 && slots[r - 1] == s - 1;
    const uint32_t bits = __ballot_sync(0xffffffffu, goes);
    if ((threadIdx.x & 31) == 0) goes_on[j >> 5] = bits;
    if (part == 0) {
      leads = j < p.segment && s >= 0 && s < limit && !goes;
      mine = s;
      if (j < p.segment && s >= limit && blockIdx.y == 0) st::report_error(err, st::ERR_BOUNDS, 0x7002);
    }
  }
  __syncthreads();
  if (leads) {
    int j = threadIdx.x + 1, w = j >> 5;
    uint32_t ends = ~goes_on[w] >> (j & 31);
    if (ends) j += __ffs(ends) - 1;
    else {
      const int last = (p.segment + P - 1) >> 5;
      for (++w; w <= last && goes_on[w] == 0xffffffffu; ++w) {}
      j = w > last ? 32 * w : 32 * w + __ffs(~goes_on[w]) - 1;
    }
    const int at = atomicAdd(&groups, 1);      // which warp takes which group does not change results
    first_row[at] = threadIdx.x, group_rows[at] = min(j - static_cast<int>(threadIdx.x), P - static_cast<int>(mine & (P - 1))), first_slot[at] = mine;
  }
  __syncthreads();
  const int n_groups = groups, h0 = blockIdx.y * p.heads_per_block, heads = min(p.heads_per_block, p.kv_heads - h0);
  auto work = [&](int group, int unit, int me, int warps) {
    const bool any = unit < 2 * heads;
    const int h = h0 + (any ? unit >> 1 : 0), second = unit & 1;
    const long long row = r0 + first_row[group], s = first_slot[group], at = (s >> p.shift) * p.kv_heads + h;
    store_group<T, D>(second ? v + row * p.v_row + h * p.v_head : k + row * p.k_row + h * p.k_head, second ? p.v_row : p.k_row, wide, (second ? vc : kc) + at * P * D,
                      (second ? vs : ks) + at, static_cast<int>(s & (P - 1)), any ? group_rows[group] : 0, me, warps, shared_top);
  };
  if (p.team > 1 && n_groups <= 2) {
    for (int g = 0; g < n_groups; ++g) work(g, warp / p.team, warp % p.team, p.team);
  } else {
    for (int i = warp; i < n_groups * 2 * heads; i += kStoreWarps) work(i / (2 * heads), i % (2 * heads), 0, 1);
  }
}

template <typename T>
int launch_store(const void* k, const void* v, void* kc, void* vc, float* ks, float* vs, const long long* slots, PutParams p, int dim, cudaStream_t stream) {
  const long long strides = p.k_row | p.k_head | p.v_row | p.v_head;
  const bool wide = (strides * static_cast<long long>(sizeof(T))) % 16 == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
  // four warps to a page's rows of a head, two where its rows are few; 8 warps work on the keys and values of 1, 2 or 4 heads
  p.team = p.shift >= 6 ? 4 : p.shift == 5 ? 2 : 1;
  p.heads_per_block = 4 / p.team;
  const int y = (p.kv_heads + p.heads_per_block - 1) / p.heads_per_block;
  // a page's rows to a block, fewer while that leaves the chip short of blocks: down to a warp per row, head and tensor
  int segment = 1 << p.shift;
  while (segment * p.heads_per_block > 4 && (p.rows + segment - 1) / segment * y < 2 * st::sm_count()) segment /= 2;
  p.segment = segment;
  const long long blocks = (p.rows + segment - 1) / segment;
  if (blocks > 2147483647LL) return st::fail(ST_ERR_TOO_LARGE, "paged store: too many rows");
  const dim3 grid(static_cast<unsigned>(blocks), y);
  const cudaError_t e = st::chained(dim == 64 ? store_kernel<T, 64> : store_kernel<T, 128>, grid, dim3(kStoreThreads), 0, stream)(
      static_cast<const T*>(k), static_cast<const T*>(v), static_cast<unsigned char*>(kc), static_cast<unsigned char*>(vc), ks, vs, slots, p, wide, st::error_word());
  if (e != cudaSuccess) return st::fail_cuda(e, "paged store");
  return ST_OK;
}

// ---- reading --------------------------------------------------------------------------------------------------------------------
// code * scale of the first `room` tokens of every sequence, zeros behind its length: 1 byte read, 2 (4) written per element.
// Sixteen elements a thread; the threads of a block run along a head's row, then its tokens.
template <typename OUT, int D>
__global__ void __launch_bounds__(256) read_kernel(const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc, const float* __restrict__ ks,
                                                   const float* __restrict__ vs, const int* __restrict__ table, const int* __restrict__ lengths, long long table_row, int width,
                                                   int shift, long long pages, int kv_heads, int room, OUT* ko, OUT* vo, unsigned* err) {
  chain_begin(kc, vc, ks, vs, table, lengths);
  constexpr int L = D / 16, TOK = 256 / L;
  const int b = blockIdx.z >> 1, which = blockIdx.z & 1, h = blockIdx.y, P = 1 << shift;
  const int tok = blockIdx.x * TOK + threadIdx.x / L, lane = threadIdx.x % L;
  if (tok >= room) return;
  const int block = tok >> shift;
  uint4 w = make_uint4(0, 0, 0, 0);
  float scale = 0.0f;
  if (tok < lengths[b] && block < width) {
    const long long page = table[b * table_row + block];
    if (page >= 0 && page < pages) {
      const long long at = page * kv_heads + h;
      w = *reinterpret_cast<const uint4*>((which ? vc : kc) + (at * P + (tok & (P - 1))) * D + lane * 16);
      scale = (which ? vs : ks)[at];
    } else if (lane == 0) {
      st::report_error(err, st::ERR_BOUNDS, 0x7003);
    }
  }
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
  float f[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2_raw x = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(words[i / 2] >> (16 * (i & 1))), __NV_E4M3);
    const float2 y = __half22float2(__half2(x));
    f[2 * i] = y.x * scale, f[2 * i + 1] = y.y * scale;
  }
  OUT* out = (which ? vo : ko) + ((static_cast<long long>(b) * room + tok) * kv_heads + h) * D + lane * 16;
  if constexpr (sizeof(OUT) == 2) {
    uint4 o[2];
    uint32_t* q = reinterpret_cast<uint32_t*>(o);
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = st::pack_bf16x2(f[2 * i], f[2 * i + 1]);
    reinterpret_cast<uint4*>(out)[0] = o[0];
    reinterpret_cast<uint4*>(out)[1] = o[1];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(out)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
  }
}
}  // namespace

ST_API int st_paged_max_sequences() { return kMaxSequences; }

// Pages for `added` more tokens of every sequence, taken from the end of free_list[0 .. *free_count) and written to the block table [B, width]
// (row stride table_row), and the maps of a step of `rows` rows: starts [B + 1], position and slot (page * page size + offset) of every row, rows
// behind the last sequence 0 and -1; lengths and free count after it.  free_after below 0: that many pages were missing; their blocks and rows get -1.
ST_API int st_paged_plan(const int* lengths, const int* added, int* table, long long table_row, int width, const int* free_list, const int* free_count, int free_size,
                         int page_size, int B, long long rows, int* starts, int* positions, long long* slots, int* lengths_after, int* free_after, void* stream_v) {
  const int shift = st::page_shift(page_size);
  if (shift < 0 || B < 0 || B > kMaxSequences || width < 0 || rows < 0 || rows > 2147483647LL)
    return st::fail(ST_ERR_INVALID, "paged plan: sizes out of range");
  if ((reinterpret_cast<uintptr_t>(positions) | reinterpret_cast<uintptr_t>(slots)) & 15) return st::fail(ST_ERR_INVALID, "paged plan: maps must be 16-byte aligned");
  const long long want = (rows + 4 * kPlanThreads - 1) / (4 * kPlanThreads);
  const int blocks = static_cast<int>(want < 1 ? 1 : want > 4 * st::sm_count() ? 4 * st::sm_count() : want);
  const size_t smem = 2 * (static_cast<size_t>(B) + 1) * sizeof(int);
  // once, for the most sequences: the 48 KB that need no opting in are for the sums and what the kernel declares itself together
  static bool opted[st::kMaxDevices];
  if (bool& done = opted[st::current_device()]; !done) {
    ST_CUDA_CHECK(cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(2 * (kMaxSequences + 1) * sizeof(int))));
    done = true;
  }
  const cudaError_t e = st::chained(plan_kernel, dim3(blocks), dim3(kPlanThreads), smem, reinterpret_cast<cudaStream_t>(stream_v))(
      lengths, added, table, table_row, width, free_list, free_count, free_size, shift, B, rows, starts, positions, slots, lengths_after, free_after);
  if (e != cudaSuccess) return st::fail_cuda(e, "paged plan");
  return ST_OK;
}

// Pages of the sequences with done[b] != 0 back to free_list (free_size entries), their table entries -1, their lengths 0.
ST_API int st_paged_release(int* lengths, const void* done, int* table, long long table_row, int width, int* free_list, int* free_count, int free_size, int page_size, int B,
                            void* stream_v) {
  const int shift = st::page_shift(page_size);
  if (shift < 0 || B < 0 || B > kMaxSequences || width < 0) return st::fail(ST_ERR_INVALID, "paged release: sizes out of range");
  if (B == 0) return ST_OK;
  const cudaError_t e = st::chained(release_kernel, dim3(1), dim3(kPlanThreads), static_cast<size_t>(B) * sizeof(int), reinterpret_cast<cudaStream_t>(stream_v))(
      lengths, static_cast<const unsigned char*>(done), table, table_row, width, free_list, free_count, free_size, shift, B, st::error_word());
  if (e != cudaSuccess) return st::fail_cuda(e, "paged release");
  return ST_OK;
}

// Rows k, v [rows, kv_heads, dim] (dim contiguous, strides in elements) into the pages; slots [rows]: page * page size + offset, below 0: not stored.
// Rows of one page follow one another; a group that starts at offset 0 begins the page anew.  type: 0 bf16, 1 fp16, 2 fp32.
ST_API int st_paged_store(const void* k, const void* v, void* k_codes, void* v_codes, float* k_scale, float* v_scale, const long long* slots, long long rows, int kv_heads,
                          int dim, int page_size, long long pages, long long k_row, long long k_head, long long v_row, long long v_head, int type, void* stream_v) {
  const int shift = st::page_shift(page_size);
  if (shift < 0 || rows < 0 || kv_heads < 1 || kv_heads > 65535 || pages < 0 || (dim != 64 && dim != 128))
    return st::fail(ST_ERR_INVALID, "paged store: sizes out of range (page 16 to 256, dim 64 or 128)");
  if ((reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes)) & 15) return st::fail(ST_ERR_INVALID, "paged store: codes must be 16-byte aligned");
  if (rows == 0) return ST_OK;
  const PutParams p{k_row, k_head, v_row, v_head, rows, pages, kv_heads, shift, 0, 0, 0};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  switch (type) {
    case 0: return launch_store<__nv_bfloat16>(k, v, k_codes, v_codes, k_scale, v_scale, slots, p, dim, stream);
    case 1: return launch_store<__half>(k, v, k_codes, v_codes, k_scale, v_scale, slots, p, dim, stream);
    case 2: return launch_store<float>(k, v, k_codes, v_codes, k_scale, v_scale, slots, p, dim, stream);
  }
  return st::fail(ST_ERR_INVALID, "paged store: unknown type");
}

// k, v [B, room, kv_heads, dim] (contiguous; bf16, or fp32 where wide_out) of the tokens below each length, zeros behind it.
ST_API int st_paged_read(const void* k_codes, const void* v_codes, const float* k_scale, const float* v_scale, const int* table, const int* lengths, long long table_row, int width,
                         int B, int room, int kv_heads, int dim, int page_size, long long pages, void* k_out, void* v_out, int wide_out, void* stream_v) {
  const int shift = st::page_shift(page_size);
  if (shift < 0 || B < 0 || B > 32767 || room < 0 || kv_heads < 1 || kv_heads > 65535 || pages < 0 || (dim != 64 && dim != 128))
    return st::fail(ST_ERR_INVALID, "paged read: sizes out of range (page 16 to 256, dim 64 or 128)");
  if (B == 0 || room == 0) return ST_OK;
  const int tok = 256 / (dim / 16);
  const dim3 grid((room + tok - 1) / tok, kv_heads, 2 * B);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  const unsigned char *kc = static_cast<const unsigned char*>(k_codes), *vc = static_cast<const unsigned char*>(v_codes);
  cudaError_t e;
  if (wide_out)
    e = st::chained(dim == 64 ? read_kernel<float, 64> : read_kernel<float, 128>, grid, dim3(256), 0, stream)(
        kc, vc, k_scale, v_scale, table, lengths, table_row, width, shift, pages, kv_heads, room, static_cast<float*>(k_out), static_cast<float*>(v_out), st::error_word());
  else
    e = st::chained(dim == 64 ? read_kernel<__nv_bfloat16, 64> : read_kernel<__nv_bfloat16, 128>, grid, dim3(256), 0, stream)(
        kc, vc, k_scale, v_scale, table, lengths, table_row, width, shift, pages, kv_heads, room, static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out),
        st::error_word());
  if (e != cudaSuccess) return st::fail_cuda(e, "paged read");
  return ST_OK;
}
