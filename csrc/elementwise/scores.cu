// Scores of given tokens: log probability, entropy of the distribution and the likeliest tokens, from logits in one pass, and the gradient.
//
//   m = max x,  y = (x - m) log2 e,  S = sum 2^y,  T = sum 2^y y,  log p_j = x_j - m - ln S,  entropy = (log2 S - T / S) ln 2
//   dx_j = sum_i g_i [j = id_i] - p_j (sum_i g_i + g_entropy (log p_j + entropy)),  i over the given token and the likeliest ones
//
// Bound by memory: a row is read once (forward; the gradient reads it again and writes as much).  Every thread keeps m, S and T of what it has seen, and what
// its largest element is; they are joined at the end.  Of the threads' largest elements the `top` best give a bound, which only elements of these threads can
// reach: those are read again (25 vectors each of a row of 50304, out of L2) and what reaches the bound is ranked.
// Measured: 8192 x 50304 in bf16 139 to 141 us, 5.9 TB/s of the 6.6 that a copy reaches; with 20 alternatives 198 to 201, 4.2; forward and gradient 395, the gradient 256 of it (6.4).  In fp16
// 139, 195 and 394; in fp32 242 (6.8 TB/s), 315 and 744.
// At 2048 x 50304 the XU pipe, whose exponentials come next, is busy 70%, and the alternatives are 30% of the instructions.
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "../common/chain.cuh"
#include <cuda_fp16.h>
#include <type_traits>

namespace {
using st::chain_begin;

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kMostTop = 32;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f, kLowest = -3.402823466e38f;
constexpr float kMargin = 4.0f;       // how far an element may lie above a thread's m before that follows it: e^4 rows of S are far from overflow
// y is one multiplication and addition, x log2 e - (m log2 e), the second rounded once for all of a block; that rounding must stay below 1, so |m| below kUsual = 2^20, and
// it is known, so that it is taken out of the block's sums.  Elements below the least usual one, -inf among them, count as that, which keeps 2^y y from being 0
// times infinity.  Where m is not usual the sums are formed again with care: y = (x - m) log2 e.
constexpr float kUsual = 1048576.0f;
constexpr float kFar = -1.0e4f;       // 2^kFar is 0
template <typename T> constexpr float kLeast = -kUsual;
template <> constexpr float kLeast<__half> = -65504.0f;
template <typename T> __device__ __forceinline__ bool is_usual(float m) { return m > 0.9f * kLeast<T> && m < kUsual; }      // and what counts as the least is nothing beside it
__device__ __forceinline__ float scaled(float m) { return __fmul_rn(m, kLog2e); }
__device__ __forceinline__ float off_by(float m) { return -fmaf(m, kLog2e, -scaled(m)); }      // what is added to x log2 e - scaled(m) for (x - m) log2 e

struct ScoreParams {
  long long row, rows;      // elements between rows
  int vocab, top, parts;
};

template <typename T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float(float x) { return x; }
template <> __device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float(float x) { return x; }
template <> __device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }

template <typename T> __device__ __forceinline__ float at_least(float x) { return x < kLeast<T> ? kLeast<T> : x; }      // NaN stays

// 16 bytes of a row.
template <typename T>
struct alignas(16) Vec {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
  __device__ __forceinline__ void pairs(float2 (&f)[N / 2]) const {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) f[i] = make_float2(to_float(v[2 * i]), to_float(v[2 * i + 1]));
  }
};
template <int N>
__device__ __forceinline__ float largest_of(const float2 (&f)[N]) {
  if constexpr (N == 4) return fmaxf(st::max3(f[0].x, f[0].y, f[1].x), fmaxf(st::max3(f[1].y, f[2].x, f[2].y), fmaxf(f[3].x, f[3].y)));
  return fmaxf(fmaxf(f[0].x, f[0].y), fmaxf(f[1].x, f[1].y));
}

// The elements of a vector as pairs, none below the least usual one.
template <typename T>
__device__ __forceinline__ void usual_pairs(const Vec<T>& v, float2 (&f)[Vec<T>::N / 2]) {
  if constexpr (sizeof(T) == 4) {
    v.pairs(f);
#pragma unroll
    for (int i = 0; i < Vec<T>::N / 2; ++i) f[i] = make_float2(at_least<T>(f[i].x), at_least<T>(f[i].y));
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {      // two at a time before they are fp32
    const __nv_bfloat162 least = __float2bfloat162_rn(kLeast<T>);
    const uint4 bits = *reinterpret_cast<const uint4*>(&v);
    const uint32_t word[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 c = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&word[i]), least);
      const uint32_t u = *reinterpret_cast<const uint32_t*>(&c);
      f[i] = make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
    }
  } else {
    const __half2 least = __float2half2_rn(kLeast<T>);
    const uint4 bits = *reinterpret_cast<const uint4*>(&v);
    const uint32_t word[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __half22float2(__hmax2_nan(*reinterpret_cast<const __half2*>(&word[i]), least));
  }
}

// Vectors v, v + step, ... below end, four of them on their way while others are worked on.
template <typename T, typename F>
__device__ __forceinline__ void stream(const Vec<T>* from, int v, int end, int step, F&& work) {
  constexpr int kAhead = 4;
  Vec<T> next[kAhead];
  if (v + (kAhead - 1) * step < end) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) next[i] = from[v + i * step];
    for (; v + (2 * kAhead - 1) * step < end; v += kAhead * step)
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const Vec<T> own = next[i];
        next[i] = from[v + (i + kAhead) * step];
        work(own, v + i * step);
      }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) work(next[i], v + i * step);
    v += kAhead * step;
  }
#pragma unroll
  for (int i = 0; i < kAhead - 1; ++i)
    if (v + i * step < end) next[i] = from[v + i * step];
#pragma unroll
  for (int i = 0; i < kAhead - 1; ++i)
    if (v + i * step < end) work(next[i], v + i * step);
}

// ---- running sums -------------------------------------------------------------------------------------------------------------------
struct Sums {
  float m = kLowest, S = 0.0f, T = 0.0f;
  __device__ __forceinline__ void shift(float y) {      // by 2^y, to a larger m
    const float f = st::exp2_ftz(y);
    T = f > 0.0f ? f * fmaf(S, y, T) : f * S;           // f = 0: what was seen counts for nothing, and S y may be infinite
    S *= f;
  }
  __device__ __forceinline__ void move(float to, bool usual) {
    shift(to == m ? 0.0f : usual ? scaled(m) - scaled(to) : (m - to) * kLog2e);
    m = to;
  }
  __device__ __forceinline__ void add(float x) {        // with care
    if (x > m + kMargin) shift((m - x) * kLog2e), m = x;
    const float y = (x - m) * kLog2e, e = st::exp2_ftz(y);      // NaN, and infinity less infinity, make S NaN
    S += e;
    T = fmaf(e, fmaxf(y, kFar), T);
  }
  __device__ __forceinline__ void join(float m2, float S2, float T2) {      // with care
    Sums o;
    o.m = m2, o.S = S2, o.T = T2;
    if (m2 > m) move(m2, false);
    else o.move(m, false);
    S += o.S;
    T += o.T;
  }
};
// Two elements at a time.
template <typename E>
struct PairSums {
  float m = kLeast<E>;
  float2 S = make_float2(0.0f, 0.0f), T = make_float2(0.0f, 0.0f);
  template <int N>
  __device__ __forceinline__ void add(const float2 (&x)[N], float largest) {
    if (largest > m + kMargin) {
      Sums a, b;
      a.S = S.x, a.T = T.x, b.S = S.y, b.T = T.y;
      const float y = scaled(m) - scaled(largest);
      a.shift(y), b.shift(y);
      m = largest, S = make_float2(a.S, b.S), T = make_float2(a.T, b.T);
    }
    const float2 less = st::splat2(-scaled(m));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float2 y = st::fma2(x[i], st::splat2(kLog2e), less), e = make_float2(st::exp2_ftz(y.x), st::exp2_ftz(y.y));
      S = st::add2(S, e);
      T = st::fma2(e, y, T);
    }
  }
};
// Sums of a warp's lanes, or of the first `lanes` (a power of two) of them, in the same for all of these: the largest m first, then one shift each.
__device__ __forceinline__ void join_lanes(Sums& s, int lanes, bool usual) {
  float m = s.m;
  for (int o = lanes / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  s.move(m, usual);
  for (int o = lanes / 2; o > 0; o >>= 1) {
    s.S += __shfl_xor_sync(0xffffffffu, s.S, o);
    s.T += __shfl_xor_sync(0xffffffffu, s.T, o);
  }
}

// ---- the likeliest tokens -----------------------------------------------------------------------------------------------------------
// A key orders elements by value, equal ones by the lower index, and NaN before all: no two are equal, and none is 0.
__device__ __forceinline__ unsigned long long key_of(float x, int index) {
  const uint32_t b = __float_as_uint(x + 0.0f);      // -0 counts as 0
  const uint32_t o = x != x ? 0xFFFFFFFFu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return static_cast<unsigned long long>(o) << 32 | ~static_cast<uint32_t>(index);
}
__device__ __forceinline__ float value_of(unsigned long long key) {
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  return o == 0xFFFFFFFFu ? __uint_as_float(0x7FC00000u) : __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ unsigned long long warp_largest(unsigned long long key) {
  const uint32_t high = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(key >> 32));
  const uint32_t low = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(key >> 32) == high ? static_cast<uint32_t>(key) : 0u);
  return static_cast<unsigned long long>(high) << 32 | low;
}

// W warps on one row.
template <int W>
struct Joined {
  float sums[W][3], total[3];
};
// Without alternatives only what is joined has room.  kRoom keys, of which a round of the careful pass fills half.
template <int W>
struct Candidates : Joined<W> {
  static constexpr int kEach = 4, kRound = W * 32 * kEach, kRoom = 2 * kRound;      // elements of a thread, and of all, in a round
  unsigned long long key[kRoom];
  unsigned long long best[kMostTop];
  unsigned long long bound[W], thread[W * 32];      // thread: largest elements of those that may be among the best
  uint32_t reach;                                   // in the order of the keys: what the `top` best threads' largest elements reach; 0: fewer threads have any
  int threads, owners, count, kept;
  uint16_t owner[W * 32];                           // threads whose largest element reaches that
};

template <int W> __device__ __forceinline__ void sync() {
  if (W == 1) __syncwarp();
  else __syncthreads();
}

// A key that at least `top` of the threads' keys reach: in every warp the ceil(top / W)-th largest, of these the least.
template <int W>
__device__ __forceinline__ unsigned long long bound_of(Candidates<W>& c, unsigned long long key, int top, int warp, int lane) {
  unsigned long long at = 0;
  for (int i = 0; i < (top + W - 1) / W; ++i) {
    at = warp_largest(key);
    if (key == at) key = 0;
  }
  if (W == 1) return at;
  if (lane == 0) c.bound[warp] = at;
  sync<W>();
#pragma unroll
  for (int i = 0; i < W; ++i) at = min(at, c.bound[i]);
  sync<W>();
  return at;
}

// The `top` largest of the first c.count keys to c.best, in order.  All threads; the keys are in place.
template <int W>
__device__ void select(Candidates<W>& c, int top, int tid) {
  constexpr int kOwn = Candidates<W>::kRoom / (W * 32);
  const int warp = tid >> 5, lane = tid & 31;
  int n = c.count;
  if (n > 2 * kMostTop) {      // those that reach a bound: a few more than `top`
    unsigned long long own[kOwn], largest = 0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int at = i * W * 32 + tid;
      own[i] = at < n ? c.key[at] : 0;
      largest = max(largest, own[i]);
    }
    sync<W>();
    if (tid == 0) c.count = 0;
    const unsigned long long bound = max(bound_of(c, largest, top, warp, lane), 1ull);
    sync<W>();
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
      if (own[i] >= bound) c.key[atomicAdd(&c.count, 1)] = own[i];
    sync<W>();
    n = c.count;
  }
  for (int i = tid; i < n; i += W * 32) {
    const unsigned long long key = c.key[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += c.key[j] > key;
    if (rank < top) c.best[rank] = key;
  }
  sync<W>();
}

// Any row, whatever its order: every round's elements that are larger than the `top` best so far, then the best again.
template <typename T, int W>
__device__ __noinline__ void select_carefully(Candidates<W>& c, const T* x, int from, int to, int top, int tid) {
  unsigned long long bound = 0;
  sync<W>();      // the count may be what brought the row here: all have read it
  if (tid == 0) c.count = 0;
  sync<W>();
  for (int at = from; at < to; at += Candidates<W>::kRound) {
    for (int i = 0; i < Candidates<W>::kEach; ++i) {
      const int j = at + i * W * 32 + tid;
      if (j < to) {
        const unsigned long long key = key_of(to_float(x[j]), j);
        if (key > bound) c.key[atomicAdd(&c.count, 1)] = key;
      }
    }
    sync<W>();
    if (c.count > Candidates<W>::kRound) {
      select(c, top, tid);
      if (tid < top) c.key[tid] = c.best[tid];
      if (tid == 0) c.count = top;
      bound = c.best[top - 1];
    }
    sync<W>();
  }
}

// The sums of all of a row's threads, in all of them.
template <int W>
__device__ __forceinline__ void join_group(Candidates<W>& c, Sums& s, int warp, int lane, bool usual) {
  join_lanes(s, 32, usual);
  if (W == 1) return;
  if (lane == 0) c.sums[warp][0] = s.m, c.sums[warp][1] = s.S, c.sums[warp][2] = s.T;
  sync<W>();
  if (warp == 0) {
    const int i = lane & (W - 1);
    s.m = c.sums[i][0], s.S = c.sums[i][1], s.T = c.sums[i][2];
    join_lanes(s, W, usual);
    if (lane == 0) c.total[0] = s.m, c.total[1] = s.S, c.total[2] = s.T;
  }
  sync<W>();
  s.m = c.total[0], s.S = c.total[1], s.T = c.total[2];
}

// The elements, of vectors v0 to v1, that may be among the `top` largest, to c.key; best: the thread's largest element, none below the least usual one.
template <typename T, int W>
__device__ __noinline__ void gather_likeliest(Candidates<W>& c, const T* x, float best, int head, int v0, int v1, int top, int single, int tid) {
  constexpr int N = Vec<T>::N, kGroup = W * 32;
  const Vec<T>* xv = reinterpret_cast<const Vec<T>*>(x + head);
  const int warp = tid >> 5, lane = tid & 31;
  const unsigned long long key = v0 + tid < v1 || single >= 0 ? key_of(best, tid) : 0;
  const uint32_t loose = static_cast<uint32_t>(bound_of(c, key, top, warp, lane) >> 32);      // and the counts are 0 for all
  sync<W>();
  if (key != 0 && static_cast<uint32_t>(key >> 32) >= loose) c.thread[atomicAdd(&c.threads, 1)] = key;
  sync<W>();
  const int n = c.threads;
  if (tid == 0 && n < top) c.reach = 0;
  if (tid < n) {
    const unsigned long long own = c.thread[tid];
    int rank = 0, above = 0;      // among the threads, and of larger values: equal ones may hold a lower index
    for (int j = 0; j < n; ++j) {
      const unsigned long long other = c.thread[j];
      rank += other > own;
      above += static_cast<uint32_t>(other >> 32) > static_cast<uint32_t>(own >> 32);
    }
    if (rank == top - 1) c.reach = static_cast<uint32_t>(own >> 32);
    if (above < top) c.owner[atomicAdd(&c.owners, 1)] = static_cast<uint16_t>(~static_cast<uint32_t>(own));
  }
  sync<W>();
  const uint32_t reach = c.reach;
  const float limit = reach ? value_of(static_cast<unsigned long long>(reach) << 32) : -INFINITY;
  const auto keep = [&](float value, int index) {
    if (!(value >= limit)) return;
    const int at = atomicAdd(&c.count, 1);
    if (at < Candidates<W>::kRoom) c.key[at] = key_of(value, index);
  };
  if (single >= 0) keep(to_float(x[single]), single);
  // the owners' vectors, two to a thread at a time
  const int each = (v1 - v0 + kGroup - 1) / kGroup, all = c.owners * each;
  for (int i = tid; i < all; i += 2 * kGroup) {
    Vec<T> again[2];
    int at[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int item = i + h * kGroup, o = item / each;
      at[h] = item < all ? v0 + c.owner[o] + (item - o * each) * kGroup : v1;
      if (at[h] < v1) again[h] = xv[at[h]];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (at[h] >= v1) continue;
      float2 f[N / 2];
      again[h].pairs(f);
      if (!(largest_of(f) >= limit)) continue;
#pragma unroll
      for (int k = 0; k < N; ++k) keep(k % 2 ? f[k / 2].y : f[k / 2].x, head + at[h] * N + k);
    }
  }
}

// One row (or, in a cluster, one part of it) per W warps.
template <typename T, int W, bool TOP>
__global__ void __launch_bounds__(W == 1 ? kThreads : W * 32, W == 1 ? 1 : 32 / W)
    scores_kernel(const T* logits, const long long* targets, float* logprob, float* entropy, float2* stats, long long* top_ids, float* top_logprobs, const ScoreParams p) {
  extern __shared__ __align__(16) uint8_t room[];
  chain_begin(logits, targets, logprob, entropy, stats, top_ids, top_logprobs);
  constexpr int N = Vec<T>::N, kGroup = W * 32;
  Candidates<W>& c = reinterpret_cast<Candidates<W>*>(room)[W == 1 ? threadIdx.x >> 5 : 0];
  const int tid = threadIdx.x % kGroup, warp = tid >> 5, lane = tid & 31;
  const int part = W == 1 ? 0 : blockIdx.x % p.parts;
  const long long row = W == 1 ? static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5) : blockIdx.x / p.parts;
  if (row >= p.rows) return;
  const T* x = logits + row * p.row;
  // elements before the first 16-byte boundary and behind the last one go one by one, to the first threads of the first part
  const int head = min(p.vocab, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)));
  const int vectors = (p.vocab - head) / N, rest = head + vectors * N, singles = head + p.vocab - rest;
  const int share = (vectors + p.parts - 1) / p.parts, v0 = part * share, v1 = min(vectors, v0 + share);
  const Vec<T>* xv = reinterpret_cast<const Vec<T>*>(x + head);
  if (TOP && tid == 0) c.threads = c.owners = c.count = 0;
  PairSums<T> pairs;
  Sums s;
  float best = -INFINITY;      // the thread's largest element
  const int one = tid < head ? tid : rest + tid - head;
  const bool has_single = part == 0 && tid < singles;
  const float single = has_single ? to_float(x[one]) : 0.0f;
  const long long target = tid == 0 && part == 0 ? targets[row] : -1;
  const float given = target >= 0 && target < p.vocab ? to_float(x[target]) : 0.0f;

  stream(xv, v0 + tid, v1, kGroup, [&](const Vec<T>& vec, int) {
    float2 f[N / 2];
    usual_pairs(vec, f);
    const float largest = largest_of(f);
    if (TOP) best = fmaxf(best, largest);
    pairs.add(f, largest);
  });
  s.m = pairs.m, s.S = pairs.S.x + pairs.S.y, s.T = pairs.T.x + pairs.T.y;
  if (has_single) {
    const float x1 = at_least<T>(single);
    if (x1 > s.m + kMargin) s.shift(scaled(s.m) - scaled(x1)), s.m = x1;
    const float y = fmaf(x1, kLog2e, -scaled(s.m)), e = st::exp2_ftz(y);
    s.S += e, s.T = fmaf(e, y, s.T);
  }

  if (TOP) gather_likeliest<T, W>(c, x, has_single ? fmaxf(best, at_least<T>(single)) : best, head, v0, v1, p.top, has_single ? one : -1, tid);

  // sums of the row (part): in every thread
  join_group(c, s, warp, lane, true);
  if (is_usual<T>(s.m)) {
    s.shift(off_by(s.m));
  } else {      // whatever the sums are: beyond 2.3e38 a finite m's y is infinite, and differences of two such are NaN
    s = Sums();
    for (int v = v0 + tid; v < v1; v += kGroup)
      for (int k = 0; k < N; ++k) s.add(to_float(x[head + v * N + k]));
    if (has_single) s.add(single);
    sync<W>();
    join_group(c, s, warp, lane, false);
  }
  if (TOP) {
    sync<W>();
    // With care: a NaN hides from comparisons (and an infinity makes S one); keys that found no room are lost; of elements that count as the least usual one, a
    // thread has not kept the largest.
    const uint32_t reach = c.reach;
    if (c.count > Candidates<W>::kRoom || s.S != s.S || (reach && !(value_of(static_cast<unsigned long long>(reach) << 32) > kLeast<T>))) {
      if (part == 0) {      // its single elements too: with one part these are the row
        if (p.parts == 1) {
          select_carefully<T, W>(c, x, 0, p.vocab, p.top, tid);
        } else {
          select_carefully<T, W>(c, x, 0, head + v1 * N, p.top, tid);
          if (tid < p.vocab - rest) c.key[atomicAdd(&c.count, 1)] = key_of(to_float(x[rest + tid]), rest + tid);
        }
      } else {
        select_carefully<T, W>(c, x, head + v0 * N, head + v1 * N, p.top, tid);
      }
      sync<W>();
    }
    select(c, p.top, tid);
  }
  if (W > 1 && p.parts > 1) {      // the parts of a row: blocks of a cluster, read by the first
    const int n = TOP ? min(c.count, p.top) : 0;
    sync<W>();
    if (tid == 0) {
      c.sums[0][0] = s.m, c.sums[0][1] = s.S, c.sums[0][2] = s.T;
      if (TOP) c.kept = n;
    }
    st::cluster_sync();
    if (part == 0) {
      s = Sums();
      for (int r = 0; r < p.parts; ++r) {
        float f[3];
#pragma unroll
        for (int i = 0; i < 3; ++i)
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f[i]) : "r"(st::cluster_map(st::smem_u32(&c.sums[0][i]), r)));
        s.join(f[0], f[1], f[2]);
      }
      if (TOP) {
        sync<W>();
        if (tid == 0) c.count = 0;
        sync<W>();
        for (int r = warp; r < p.parts; r += W) {      // up to 32 keys of each
          unsigned long long key = 0;
          int have;
          asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(have) : "r"(st::cluster_map(st::smem_u32(&c.kept), r)));
          if (lane < have) asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key) : "r"(st::cluster_map(st::smem_u32(&c.best[lane]), r)));
          if (key) c.key[atomicAdd(&c.count, 1)] = key;
        }
        sync<W>();
        select(c, p.top, tid);
      }
    }
    st::cluster_sync();
    if (part != 0) return;
  }

  // an empty row, all -inf: no probability anywhere
  const bool empty = s.S == 0.0f;
  const float log_S = empty ? INFINITY : log2f(s.S), m = empty ? 0.0f : s.m;
  const auto log_p = [&](float v) { return fmaf(-log_S, kLn2, v - m); };
  if (tid == 0) {
    logprob[row] = target >= 0 && target < p.vocab ? log_p(given) : 0.0f;
    entropy[row] = empty ? 0.0f : (log_S - s.T / s.S) * kLn2;
    if (stats) stats[row] = make_float2(m, log_S);
  }
  if (TOP && tid < p.top) {
    const unsigned long long key = c.best[tid];
    top_ids[row * p.top + tid] = static_cast<long long>(~static_cast<uint32_t>(key));
    top_logprobs[row * p.top + tid] = log_p(value_of(key));
  }
}

// ---- gradient -----------------------------------------------------------------------------------------------------------------------
struct GradParams {
  long long row, out_row, rows;
  int vocab, top, parts;
};

// Probabilities below 2^-126 count as 0, as their exponentials are: what that leaves out of an element is below 10^-35 of the row's gradients.
// Blocks share a row in `parts` pieces of whole vectors; WIDE: rows of logits and gradient are at the same place between 16-byte boundaries.
template <typename T, int W, bool WIDE>
__global__ void __launch_bounds__(kThreads) scores_grad_kernel(const T* logits, const long long* targets, const float2* stats, const float* entropy,
                                                               const long long* top_ids, const float* g_logprob, const float* g_entropy, const float* g_top, T* out,
                                                               const GradParams p) {
  __shared__ float weight[kWarps][kMostTop + 1];
  __shared__ int id[kWarps][kMostTop + 1];
  chain_begin(logits, targets, stats, entropy, top_ids, g_logprob, g_entropy, g_top, out);
  constexpr int N = Vec<T>::N, kGroup = W * 32;
  const int slot = W == 1 ? threadIdx.x >> 5 : 0, tid = threadIdx.x % kGroup;
  const int part = W == 1 ? 0 : blockIdx.x % p.parts;
  const long long row = W == 1 ? static_cast<long long>(blockIdx.x) * kWarps + slot : blockIdx.x / p.parts;
  if (row >= p.rows) return;
  const T* x = logits + row * p.row;
  T* y = out + row * p.out_row;
  const float2 ms = stats[row];
  const bool empty = ms.y == INFINITY;
  const float m = ms.x, log_S = ms.y, H = entropy[row], gH = g_entropy ? g_entropy[row] : 0.0f;
  const int n = 1 + (g_top ? p.top : 0);
  // the tokens with a gradient of their own
  for (int i = tid; i < n; i += kGroup) {
    long long t = i == 0 ? targets[row] : top_ids[row * p.top + i - 1];
    const bool given = t >= 0 && t < p.vocab && (i > 0 || g_logprob);
    id[slot][i] = given ? static_cast<int>(t) : -1;
    weight[slot][i] = !given ? 0.0f : i == 0 ? g_logprob[row] : g_top[row * p.top + i - 1];
  }
  sync<W>();
  float all = 0.0f;
  for (int i = 0; i < n; ++i) all += weight[slot][i];
  // what the distribution contributes: p (factor log2 p + rest)
  const bool usual = is_usual<T>(m);
  const float factor = -gH * kLn2, rest_of = -fmaf(gH, H, all), less = off_by(m) - log_S;
  const auto shared = [&](float v) {
    const float y = (v - m) * kLog2e - log_S;
    return st::exp2_ftz(y) * fmaf(factor, fmaxf(y, kFar), rest_of);
  };
  const auto shared_pair = [&](float2 v) {
    const float2 y = st::add2(st::fma2(v, st::splat2(kLog2e), st::splat2(-scaled(m))), st::splat2(less));
    return st::mul2(make_float2(st::exp2_ftz(y.x), st::exp2_ftz(y.y)), st::fma2(st::splat2(factor), y, st::splat2(rest_of)));
  };
  if (WIDE) {
    const int head = min(p.vocab, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)));
    const int vectors = (p.vocab - head) / N, rest = head + vectors * N, singles = head + p.vocab - rest;
    const int share_v = (vectors + p.parts - 1) / p.parts, v0 = part * share_v, v1 = min(vectors, v0 + share_v);
    const Vec<T>* xv = reinterpret_cast<const Vec<T>*>(x + head);
    Vec<T>* yv = reinterpret_cast<Vec<T>*>(y + head);
    if (part == 0 && tid < singles) {
      const int at = tid < head ? tid : rest + tid - head;
      y[at] = from_float<T>(empty ? 0.0f : shared(to_float(x[at])));
    }
    if (empty || !usual) {
      for (int v = v0 + tid; v < v1; v += kGroup)
        for (int k = 0; k < N; ++k) y[head + v * N + k] = from_float<T>(empty ? 0.0f : shared(to_float(x[head + v * N + k])));
    } else {
      stream(xv, v0 + tid, v1, kGroup, [&](const Vec<T>& vec, int v) {
        float2 f[N / 2];
        usual_pairs(vec, f);
        Vec<T> g;
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {
          const float2 d = shared_pair(f[k]);
          g.v[2 * k] = from_float<T>(d.x), g.v[2 * k + 1] = from_float<T>(d.y);
        }
        yv[v] = g;
      });
    }
  } else {
    const int share_e = (p.vocab + p.parts - 1) / p.parts;
    for (int j = part * share_e + tid; j < min(p.vocab, (part + 1) * share_e); j += kGroup) y[j] = from_float<T>(empty ? 0.0f : shared(to_float(x[j])));
  }
  if (empty) return;
  // elements of those tokens, as a whole and rounded once, by the block that wrote them
  sync<W>();
  for (int i = tid; i < n; i += kGroup) {
    const int at = id[slot][i];
    if (at < 0) continue;
    if (p.parts > 1) {
      const int head = min(p.vocab, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T))), vectors = (p.vocab - head) / N;
      const int share_v = (vectors + p.parts - 1) / p.parts, share_e = (p.vocab + p.parts - 1) / p.parts;
      const int owner = !WIDE ? at / share_e : at < head || at >= head + vectors * N ? 0 : (at - head) / N / share_v;
      if (owner != part) continue;
    }
    float own = 0.0f;
    for (int k = 0; k < n; ++k) own += id[slot][k] == at ? weight[slot][k] : 0.0f;
    y[at] = from_float<T>(own + shared(to_float(x[at])));
  }
}

// How many blocks share a row: rows that leave SMs without a block are split, to no less than 32768 elements a block, whose start and join (in a cluster) take as
// long as 16384.  One row of 262144 with 1 block 18.7 us, 2 13.5, 4 10.3, 8 9.4; of 50304 7.5, 7.9, 7.7, 8.5.
int parts_of(long long rows, int vocab) {
  int parts = 1;
  while (parts < 8 && rows * parts * 2 <= 2 * st::sm_count() && vocab / (2 * parts) >= 32768) parts *= 2;
  return parts;
}

// Rows of up to as many elements go to a warp each, longer ones to 8 (or 4, below).  us by 8 warps and by one, with 5 alternatives: 1 x 1024 6.2 and 5.5, 1 x 2048 5.5 and 6.3, 1 x 4096 5.7
// and 7.9; 8192 x 2048 70 and 28, 8192 x 4096 75 and 38, 8192 x 8192 83 and 57; without, 8192 x 2048 21 and 17, 8192 x 3000 23 and 24; the gradient of 1 x 1024 4.0 and 3.8, of 1 x 2048 4.0
// and 4.5, of 8192 x 2048 45 and 16, of 8192 x 8192 66 and 50.  One row has its border between 1024 and 2048, many have theirs beyond 8192, where the one would lose half its time again.
constexpr int kWarpRow = 2048;

template <typename T, int W, bool TOP>
int forward(const void* logits, const long long* targets, float* logprob, float* entropy, float2* stats, long long* top_ids, float* top_logprobs, ScoreParams p,
            cudaStream_t stream) {
  p.parts = W == 1 ? 1 : parts_of(p.rows, p.vocab);
  const long long blocks = W == 1 ? (p.rows + kWarps - 1) / kWarps : p.rows * p.parts;
  if (blocks > 2147483647LL) return st::fail(ST_ERR_TOO_LARGE, "scores: too many rows");
  const size_t smem = (TOP ? sizeof(Candidates<W>) : sizeof(Joined<W>)) * (W == 1 ? kWarps : 1);
  static_assert(sizeof(Candidates<W>) * (W == 1 ? kWarps : 1) <= 48 * 1024, "candidates need no opting in");
  const cudaError_t e = st::chained(scores_kernel<T, W, TOP>, dim3(static_cast<unsigned>(blocks)), dim3(W == 1 ? kThreads : W * 32), smem, stream, p.parts)(
      static_cast<const T*>(logits), targets, logprob, entropy, stats, top_ids, top_logprobs, p);
  return e == cudaSuccess ? ST_OK : st::fail_cuda(e, "token scores");
}

template <typename T>
int forward(const void* logits, const long long* targets, float* logprob, float* entropy, float2* stats, long long* top_ids, float* top_logprobs, const ScoreParams& p,
            cudaStream_t stream) {
  if (p.vocab <= kWarpRow)
    return p.top ? forward<T, 1, true>(logits, targets, logprob, entropy, stats, top_ids, top_logprobs, p, stream)
                 : forward<T, 1, false>(logits, targets, logprob, entropy, stats, top_ids, top_logprobs, p, stream);
  if (p.top) return forward<T, kWarps, true>(logits, targets, logprob, entropy, stats, top_ids, top_logprobs, p, stream);
  // 4 warps to a row from 16 rows an SM (2368) on, where the SMs have many turns.  us with 8 and with 4: 4096 elements, 300 rows 4.4 and 4.4, 1200 9.0 and 7.1, 8192 41 and 26; 16384, 300 6.1 and 7.0,
  // 1200 14.6 and 14.1, 8192 68 and 57; 50304, 300 11.9 and 14.1, 1776 42 and 46, 2368 52 and 51, 8192 147 and 140; 131072, 1776 87 and 99, 3000 135 and 139.  With alternatives 8192 x 50304 200 and 211.
  return p.rows >= 16 * st::sm_count() ? forward<T, 4, false>(logits, targets, logprob, entropy, stats, top_ids, top_logprobs, p, stream)
                                      : forward<T, kWarps, false>(logits, targets, logprob, entropy, stats, top_ids, top_logprobs, p, stream);
}

template <typename T, int W, bool WIDE>
int backward(const void* logits, const long long* targets, const float2* stats, const float* entropy, const long long* top_ids, const float* g_logprob,
             const float* g_entropy, const float* g_top, void* out, GradParams p, cudaStream_t stream) {
  p.parts = W == 1 ? 1 : parts_of(p.rows, p.vocab);
  const long long blocks = W == 1 ? (p.rows + kWarps - 1) / kWarps : p.rows * p.parts;
  if (blocks > 2147483647LL) return st::fail(ST_ERR_TOO_LARGE, "scores: too many rows");
  const cudaError_t e = st::chained(scores_grad_kernel<T, W, WIDE>, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, stream)(
      static_cast<const T*>(logits), targets, stats, entropy, top_ids, g_logprob, g_entropy, g_top, static_cast<T*>(out), p);
  return e == cudaSuccess ? ST_OK : st::fail_cuda(e, "token scores gradient");
}

template <typename T>
int backward(const void* logits, const long long* targets, const float2* stats, const float* entropy, const long long* top_ids, const float* g_logprob,
             const float* g_entropy, const float* g_top, void* out, const GradParams& p, cudaStream_t stream) {
  const bool wide = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(out)) % 16 == 0 && (p.row - p.out_row) * static_cast<long long>(sizeof(T)) % 16 == 0;
#define ST_GRAD(WW, FF) backward<T, WW, FF>(logits, targets, stats, entropy, top_ids, g_logprob, g_entropy, g_top, out, p, stream)
  if (p.vocab <= kWarpRow) return wide ? ST_GRAD(1, true) : ST_GRAD(1, false);
  return wide ? ST_GRAD(kWarps, true) : ST_GRAD(kWarps, false);
#undef ST_GRAD
}
}  // namespace

struct StTokenScoresArgs {
  const void* logits;
  const long long* targets;
  float* logprob;
  float* entropy;
  void* stats;
  long long* top_ids;
  float* top_logprobs;
  long long rows, row;
  int vocab, top, type;
};

// Scores of rows of `vocab` logits (type 0 bf16, 1 fp16, 2 fp32; `row` elements apart): log probability of targets[i] (0 where that is no token), entropy, and the
// `top` (0 to 32) likeliest tokens with their log probabilities.  stats (may be null; on an 8-byte boundary): 2 floats a row for the gradient.
ST_API int st_token_scores(const StTokenScoresArgs* a, void* stream_v) {
  if (a->rows < 0 || a->vocab < 1 || a->vocab > 1 << 30 || a->top < 0 || a->top > kMostTop || a->top > a->vocab) return st::fail(ST_ERR_INVALID, "scores: sizes out of range");
  if (reinterpret_cast<uintptr_t>(a->stats) & 7) return st::fail(ST_ERR_INVALID, "scores: stats must lie on an 8-byte boundary");
  if (a->rows == 0) return ST_OK;
  const ScoreParams p{a->row, a->rows, a->vocab, a->top, 1};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  float2* ms = static_cast<float2*>(a->stats);
  switch (a->type) {
    case 0: return forward<__nv_bfloat16>(a->logits, a->targets, a->logprob, a->entropy, ms, a->top_ids, a->top_logprobs, p, stream);
    case 1: return forward<__half>(a->logits, a->targets, a->logprob, a->entropy, ms, a->top_ids, a->top_logprobs, p, stream);
    case 2: return forward<float>(a->logits, a->targets, a->logprob, a->entropy, ms, a->top_ids, a->top_logprobs, p, stream);
  }
  return st::fail(ST_ERR_INVALID, "scores: unknown type");
}

struct StTokenScoresGradArgs {
  const void* logits;
  const long long* targets;
  const void* stats;
  const float* entropy;
  const long long* top_ids;
  const float* g_logprob;
  const float* g_entropy;
  const float* g_top;
  void* out;
  long long rows, row, out_row;
  int vocab, top, type;
};

// Gradient of the logits from those of log probability, entropy and the likeliest tokens' log probabilities (each may be null: 0).
ST_API int st_token_scores_grad(const StTokenScoresGradArgs* a, void* stream_v) {
  if (a->rows < 0 || a->vocab < 1 || a->vocab > 1 << 30 || a->top < 0 || a->top > kMostTop || a->top > a->vocab) return st::fail(ST_ERR_INVALID, "scores: sizes out of range");
  if (reinterpret_cast<uintptr_t>(a->stats) & 7) return st::fail(ST_ERR_INVALID, "scores: stats must lie on an 8-byte boundary");
  if (a->rows == 0) return ST_OK;
  const GradParams p{a->row, a->out_row, a->rows, a->vocab, a->top, 1};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  const float2* ms = static_cast<const float2*>(a->stats);
  switch (a->type) {
    case 0: return backward<__nv_bfloat16>(a->logits, a->targets, ms, a->entropy, a->top_ids, a->g_logprob, a->g_entropy, a->g_top, a->out, p, stream);
    case 1: return backward<__half>(a->logits, a->targets, ms, a->entropy, a->top_ids, a->g_logprob, a->g_entropy, a->g_top, a->out, p, stream);
    case 2: return backward<float>(a->logits, a->targets, ms, a->entropy, a->top_ids, a->g_logprob, a->g_entropy, a->g_top, a->out, p, stream);
  }
  return st::fail(ST_ERR_INVALID, "scores: unknown type");
}
