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
// second time from the registers of the team that works on the group, or from L1 where the group is larger.
constexpr int kStoreThreads = 256;

struct PutParams {
  long long k_row, k_head, v_row, v_head;
  long long rows;
  int kv_heads, shift, segment;
  long long pages;
};

template <typename T> __device__ __forceinline__ void load8f(const T* p, bool wide, float (&f)[8]);
template <> __device__ __forceinline__ void load8f(const float* p, bool wide, float (&f)[8]) {
  if (wide) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = p[i];
  }
}
template <> __device__ __forceinline__ void load8f(const __half* p, bool wide, float (&f)[8]) {
  if (wide) {
    uint4 u = *reinterpret_cast<const uint4*>(p);
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 x = __half22float2(h[i]); f[2 * i] = x.x, f[2 * i + 1] = x.y; }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __half2float(p[i]);
  }
}
template <> __device__ __forceinline__ void load8f(const __nv_bfloat16* p, bool wide, float (&f)[8]) {
  if (wide) {
    uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 x = st::unpack_bf16x2(w[i]); f[2 * i] = x.x, f[2 * i + 1] = x.y; }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __bfloat162float(p[i]);
  }
}

__device__ __forceinline__ float finite_max(float m, const float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(f[i]);
    m = a < INFINITY ? fmaxf(m, a) : m;      // false for NaN too
  }
  return m;
}

// Eight codes of values times a power of two; the conversion saturates and keeps NaN.
__device__ __forceinline__ uint2 codes8(const float (&f)[8], float inv) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i] * inv, f[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}

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

// One tensor's part of a group: rows [r0, r0 + n) of one head go to page offsets [off, off + n).  A team of TEAM threads (a warp or the
// block); L = D / 8 lanes hold a row.
template <typename T, int D, int TEAM>
__device__ void store_group(const T* src, long long row_stride, bool wide, unsigned char* dst, float* scale, int off, int n, float* shared_max, unsigned* err) {
  constexpr int L = D / 8, RPT = TEAM / L, HELD = 4;      // rows a pass, passes held in registers
  const int me = TEAM == 32 ? threadIdx.x & 31 : threadIdx.x, lane = me % L, row = me / L;
  float held[HELD][8];
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const int r = row + i * RPT;
    if (r < n) load8f(src + r * row_stride + lane * 8, wide, held[i]);
    else
#pragma unroll
      for (int e = 0; e < 8; ++e) held[i][e] = 0.0f;
  }
  const float before = off > 0 ? *scale : 0.0f;
#pragma unroll
  for (int i = 0; i < HELD; ++i) m = finite_max(m, held[i]);
  for (int r = row + HELD * RPT; r < n; r += RPT) {
    float f[8];
    load8f(src + r * row_stride + lane * 8, wide, f);
    m = finite_max(m, f);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if constexpr (TEAM > 32) {
    __syncthreads();                                    // the one before may still be read
    if ((threadIdx.x & 31) == 0) shared_max[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TEAM / 32; ++w) m = fmaxf(m, shared_max[w]);
  }
  if constexpr (TEAM == 32) __syncwarp();               // every thread has read the old scale; one writes the new one
  int e = st::page_exponent(m);
  const int old = off > 0 ? st::scale_exponent(before) : st::kMinExponent;
  e = max(e, old);
  const float inv = st::exp2_int(-e);
  if (e > old && off > 0) {
    const float ratio = st::exp2_int(max(old - e, -126));
    for (int i = me; i < off * (D / 4); i += TEAM) {
      uint32_t* p = reinterpret_cast<uint32_t*>(dst) + i;
      *p = rescale4(*p, ratio);
    }
  }
  if (me == 0) *scale = st::exp2_int(e);
  unsigned char* out = dst + static_cast<long long>(off) * D + lane * 8;
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const int r = row + i * RPT;
    if (r < n) *reinterpret_cast<uint2*>(out + r * D) = codes8(held[i], inv);
  }
  for (int r = row + HELD * RPT; r < n; r += RPT) {
    float f[8];
    load8f(src + r * row_stride + lane * 8, wide, f);
    *reinterpret_cast<uint2*>(out + r * D) = codes8(f, inv);
  }
  if constexpr (TEAM == 32) __syncwarp();
}

// Block (segment of rows, head).  Few groups in the segment: the block takes them one after another; many (decoding: a group is a row):
// a warp each.
template <typename T, int D>
__global__ void __launch_bounds__(kStoreThreads) store_kernel(const T* __restrict__ k, const T* __restrict__ v, unsigned char* kc, unsigned char* vc, float* ks, float* vs,
                                                              const long long* __restrict__ slots, const PutParams p, bool wide, unsigned* err) {
  chain_begin(k, v, slots);
  __shared__ int first_row[kStoreThreads], group_rows[kStoreThreads];
  __shared__ int groups;
  __shared__ float shared_max[kStoreThreads / 32];
  const long long r0 = static_cast<long long>(blockIdx.x) * p.segment;
  const int h = blockIdx.y, P = 1 << p.shift;
  const long long limit = p.pages << p.shift;
  if (threadIdx.x == 0) groups = 0;
  __syncthreads();
  const long long r = r0 + threadIdx.x;
  if (threadIdx.x < p.segment && r < p.rows) {
    const long long s = slots[r];
    if (s >= limit) {
      if (h == 0) st::report_error(err, st::ERR_BOUNDS, 0x7002);
    } else if (s >= 0 && ((s & (P - 1)) == 0 || r == 0 || slots[r - 1] != s - 1)) {
      const int off = static_cast<int>(s & (P - 1));
      int n = 1;
      while (n < P - off && r + n < p.rows && slots[r + n] == s + n) ++n;
      const int at = atomicAdd(&groups, 1);      // which team takes which group does not change results
      first_row[at] = threadIdx.x, group_rows[at] = n;
    }
  }
  __syncthreads();
  const int n_groups = groups, warp = threadIdx.x >> 5;
  const bool by_warp = n_groups > 2;
  for (int i = by_warp ? warp : 0; i < n_groups; i += by_warp ? kStoreThreads / 32 : 1) {
    const long long row = r0 + first_row[i], s = slots[row], page = s >> p.shift, at = page * gridDim.y + h;
    const int off = static_cast<int>(s & (P - 1)), n = group_rows[i];
    const T *sk = k + row * p.k_row + h * p.k_head, *sv = v + row * p.v_row + h * p.v_head;
    unsigned char *dk = kc + at * P * D, *dv = vc + at * P * D;
    if (by_warp) {
      store_group<T, D, 32>(sk, p.k_row, wide, dk, ks + at, off, n, shared_max, err);
      store_group<T, D, 32>(sv, p.v_row, wide, dv, vs + at, off, n, shared_max, err);
    } else {
      store_group<T, D, kStoreThreads>(sk, p.k_row, wide, dk, ks + at, off, n, shared_max, err);
      store_group<T, D, kStoreThreads>(sv, p.v_row, wide, dv, vs + at, off, n, shared_max, err);
    }
  }
}

template <typename T>
int launch_store(const void* k, const void* v, void* kc, void* vc, float* ks, float* vs, const long long* slots, PutParams p, int dim, cudaStream_t stream) {
  const long long strides = p.k_row | p.k_head | p.v_row | p.v_head;
  const bool wide = (strides * static_cast<long long>(sizeof(T))) % 16 == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
  // a page's rows to a block, fewer while that leaves the chip short of blocks
  int segment = 1 << p.shift;
  while (segment > 8 && (p.rows + segment - 1) / segment * p.kv_heads < 2 * st::sm_count()) segment /= 2;
  p.segment = segment;
  const long long blocks = (p.rows + segment - 1) / segment;
  if (blocks > 2147483647LL) return st::fail(ST_ERR_TOO_LARGE, "paged store: too many rows");
  const dim3 grid(static_cast<unsigned>(blocks), p.kv_heads);
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
  if (smem > 48 * 1024) ST_CUDA_CHECK(cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
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
  const PutParams p{k_row, k_head, v_row, v_head, rows, kv_heads, shift, 0, pages};
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
