// What the kernels of attention over pages share: how the work is counted and divided, what a block hands on, the joining of parts.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "paged.cuh"

namespace {
using st::chain_begin;

constexpr int kTile = 128;            // keys of a unit
template <int R> constexpr int kThreadsOf = R == 128 ? 640 : R == 32 ? 384 : 256;      // of a block
constexpr int kMaxWarps = 20;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoMax = -3e38f;      // before a row has seen a key: below all scores but fp32's very last
constexpr float kLag = 6.0f, kLift = 9.0f;

struct AttnParams {
  const void* q;
  const unsigned char *kc, *vc;
  const float *ks, *vs;
  const int *table, *starts, *lengths;
  void* out;
  float *lse, *parts;
  int* notes;
  long long q_row, q_head, o_row, o_head, table_row, pages;
  long long rows;      // of q and out
  int width, shift, B, heads, kv_heads, group;
  float scale;
  int causal, zero_tail, whole;      // whole: items are not split
  unsigned* err;
};

// What the beginning and the end of an item count, in units.  Of a block alone on its SM (one sequence, one key head of 128, whole; from 4 to 20 units, less
// 2.5 us of a launch) they take 8000 cycles with 8 rows, 20000 with 16, 23000 with 32 and 18000 with 128, and a unit 1600, 2300, 4000 and 3300; where two
// blocks share an SM a unit takes 2100, 3300 and 6800.  That is a run's first item; later ones begin beside the end of the one before.  With 128 rows
// of those tried: 4 sequences of 256 tokens behind up to 4000, 3 units 40.0 us, 5 40.9, 8 43.7, 12 46.4.  16 rows count as 8 do.
template <int N> constexpr int kItemCost = N == 128 ? 3 : N == 32 ? 4 : 2;

struct Seq {
  int start, n, len, row_blocks, tiles, size, units;      // size: what an item counts
};
template <int N>
__device__ __forceinline__ Seq sequence(const AttnParams& p, int b) {
  Seq s;
  const int rows = static_cast<int>(p.rows), a = p.starts[b], e = p.starts[b + 1], len = max(p.lengths[b], 0);
  s.start = max(a, 0);
  s.n = max(min(e, rows) - s.start, 0);
  s.len = min(len, p.width << p.shift);
  s.row_blocks = (s.n * p.group + N - 1) / N;
  s.tiles = max((s.len + kTile - 1) / kTile, 1);      // a sequence without keys still gets its zero rows
  s.size = p.whole ? 1 : s.tiles + kItemCost<N>;
  s.units = s.row_blocks * s.size * p.kv_heads;
  return s;
}

// Where the block's share begins: the sequence that holds a unit, and the number of the sequence's first one.
struct Found {
  int b, first;
};
template <int WARPS>
__device__ __forceinline__ int scan_block(int mine, int* shared, int& total) {      // sum of the threads before, and of all
  int s = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) >= o) s += u;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 31) shared[threadIdx.x >> 5] = s;
  __syncthreads();
  int before = s - mine;
  total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < static_cast<int>(threadIdx.x >> 5)) before += shared[w];
    total += shared[w];
  }
  return before;
}
// The block's share [u0, u1) of the units, if it has one, and where unit u0 lies.  Up to a block's threads of sequences are looked at once.
template <int N>
__device__ bool find_share(const AttnParams& p, int* shared, Found* found, int& all, int& runs, int& u0, int& u1, Found& f) {
  constexpr int kThreads = kThreadsOf<N>, kWarps = kThreads / 32;
  int mine = 0, total = 0, before = 0;
#pragma unroll 1
  for (int b = threadIdx.x; b < p.B; b += kThreads) mine += sequence<N>(p, b).units;
  before = scan_block<kWarps>(mine, shared, total);
  all = total;
  runs = min(static_cast<int>(gridDim.x), all);      // none of them empty
  const int me = blockIdx.x;
  if (me >= runs) return false;
  // floor(all * block / runs) without the product
  const unsigned each = static_cast<unsigned>(all) / static_cast<unsigned>(runs), rest = all - each * runs;
  u0 = me * each + me * rest / runs, u1 = (me + 1) * each + (me + 1) * rest / runs;
  if (p.B <= kThreads) {
    if (u0 >= before && u0 < before + mine) *found = Found{static_cast<int>(threadIdx.x), before};      // one thread
  } else {
    int base = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < p.B && u0 >= base; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      mine = b < p.B ? sequence<N>(p, b).units : 0;
      before = base + scan_block<kWarps>(mine, shared, total);
      if (u0 >= before && u0 < before + mine) *found = Found{b, before};
      base += total;
    }
  }
  __syncthreads();
  f = *found;
  return true;
}

// Eight 16-bit elements, wherever they begin.
template <typename T> __device__ __forceinline__ uint4 load8(const T* p, bool wide) {
  if (wide) return *reinterpret_cast<const uint4*>(p);
  const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
  return make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
}
template <typename T> __device__ __forceinline__ float2 two_floats(uint32_t u);
template <> __device__ __forceinline__ float2 two_floats<__nv_bfloat16>(uint32_t u) { return st::unpack_bf16x2(u); }
template <> __device__ __forceinline__ float2 two_floats<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }

constexpr int kInvalid = -1000, kBehind = -2147483647 - 1;      // of a page: none by that number; none, as the keys end before it

// An item, or the part of it that the block's run covers: units [t0, t1) of one head's rows [row0, row_end) of a sequence.
struct Item {
  const int* table;
  int start, n, len, h, row0, row_end, t0, t1, tiles;
  int keys;      // that the last row sees
  int next;      // number of the unit behind it
  // Units to work on: those behind the last key are left out, one stays.
  __device__ __forceinline__ int steps() const { return max(min(t1, (keys + kTile - 1) / kTile) - t0, 1); }
};
// The first item with work at or behind unit u of the run that ends at u1; false: there is none.
template <int N>
__device__ __forceinline__ bool item_at(Item& it, const AttnParams& p, int u, int u1, Found& f, Seq& sq) {
#pragma unroll 1
  while (u < u1) {
    while (u >= f.first + sq.units) {
      f.first += sq.units;
      sq = sequence<N>(p, ++f.b);
    }
    // unit -> (key head, row block, tile): row blocks of one head next to each other, as they read the same pages
    const unsigned size = sq.size, in = u - f.first, item = in / size;
    const int at = in - item * size, end = min(static_cast<int>(size), at + (u1 - u));
    u += end - at;
    it.t0 = p.whole ? 0 : max(at - kItemCost<N>, 0), it.t1 = p.whole ? sq.tiles : end - kItemCost<N>;
    if (it.t1 <= it.t0) continue;      // nothing but the count for its beginning
    it.next = u;
    it.h = item / static_cast<unsigned>(sq.row_blocks);
    int rb = item - it.h * sq.row_blocks;
    // a prompt's first rows see few keys, its last ones many, and each item counts the same: they take turns, so that runs are alike
    // (first, last, second, ...; a prompt of 2048 tokens, 32 heads over 8: 132 us, 104 so)
    if (N == 128) rb = rb / 2 + (rb & 1) * (sq.row_blocks - 1 - rb / 2 * 2);
    it.tiles = sq.tiles, it.start = sq.start, it.n = sq.n, it.len = sq.len;
    it.row0 = rb * N, it.row_end = min(sq.n * p.group, it.row0 + N);
    it.table = p.table + f.b * p.table_row;
    it.keys = max(it.len - (p.causal ? it.n - 1 - (it.row_end - 1) / p.group : 0), 0);
    return true;
  }
  return false;
}

template <int THREADS>
__device__ __forceinline__ void soft_sync() { asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory"); }
template <int THREADS>
__device__ __forceinline__ bool soft_any(bool x) {      // of the softmax threads; a barrier too
  uint32_t y;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.u32 p, %1, 0;\n"
      "barrier.cta.red.or.pred q, 1, %2, p;\n"
      "selp.u32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(y)
      : "r"(static_cast<uint32_t>(x)), "n"(THREADS)
      : "memory");
  return y != 0;
}
// Bytes of e4m3 that are no number, as 0x80 in their places.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// What a block notes about the border behind its run: the item that it is inside of (parts 0: none).
struct Note {
  int parts, first, border;      // parts of the item, block of the first one, place of this border among the item's
  int rows, start, row0, h;      // live rows, and where they belong
  int unused;
};
// The note about a run that ends, with unit u1, inside an item.
__device__ __forceinline__ Note note_of(const Item& it, int u1, int runs, int all) {
  // Block b holds a part if its run begins before the item's end, all * b / runs < end, which is all * b < end * runs, and ends behind its first unit.
  const long long first_unit = u1 - it.t1, end = first_unit + it.tiles;
  Note n{};
  n.first = static_cast<int>(((first_unit + 1) * runs - 1) / all);
  n.parts = static_cast<int>((end * runs - 1) / all) - n.first + 1;
  n.border = static_cast<int>(blockIdx.x) - n.first;
  n.rows = it.row_end - it.row0, n.start = it.start, n.row0 = it.row0, n.h = it.h;
  return n;
}

template <int R>
__device__ __forceinline__ float* part_of(const AttnParams& p, int D, long long slot) {      // [R][D] output, [R] reference, [R] sum
  return p.parts + slot * (R * (D + 2));
}

// After a wait ran out: what the block's last `turns` turns set going, a ring of barriers long, gets a millisecond to come to its end.
template <int STAGES>
__device__ __forceinline__ void settle(unsigned long long (&bars)[STAGES], uint32_t turns) {
  const uint64_t t0 = st::globaltimer_ns();
#pragma unroll 1
  for (uint32_t i = turns > STAGES ? turns - STAGES : 0; i < turns; ++i)
    while (!st::mbar_try_wait(st::smem_u32(&bars[i % STAGES]), i / STAGES & 1) && st::globaltimer_ns() - t0 < 1000000) {}
}

// Rows before the first sequence and behind the last one, by one warp of every block: 0, unless the output is one that the caller gave, and a
// log-sum-exp of no keys.
template <typename T, int D>
__device__ __forceinline__ void blank_rows(const AttnParams& p) {
  if (!p.zero_tail && p.lse == nullptr) return;
  const int lane = threadIdx.x & 31, vectors = p.zero_tail ? p.heads * (D / 2) : 0;
  const int rows = static_cast<int>(p.rows), before = p.B > 0 ? min(max(p.starts[0], 0), rows) : 0, skip = (p.B > 0 ? max(p.starts[p.B], 0) : 0) - before;
#pragma unroll 1
  for (unsigned i = blockIdx.x;; i += gridDim.x) {
    const unsigned at = i < before ? i : i + skip;
    if (at >= rows) break;
    const long long row = at;
    T* o = static_cast<T*>(p.out) + row * p.o_row;
#pragma unroll 1
    for (int j = lane; j < vectors; j += 32) {
      T* at = o + j / (D / 2) * p.o_head + j % (D / 2) * 2;
      at[0] = at[1] = from_f<T>(0.0f);
    }
    if (p.lse != nullptr)
      for (int j = lane; j < p.heads; j += 32) p.lse[row * p.heads + j] = -INFINITY;
  }
}

// Joins the parts of the items that several blocks worked on.  A block per border; an item of P parts has P - 1 of them, which share its rows.
// With few parts a warp does a row; with many, the block's warps share the parts of a row.  Large items have several blocks to a border (the grid's second extent).
constexpr int kJoinThreads = 128, kWarps = kJoinThreads / 32;
template <typename T, int D, int N>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(AttnParams p) {
  constexpr int E = D / 32;
  extern __shared__ float weight[];      // [kWarps][few] or [parts]
  __shared__ float red[2][kWarps], rows[kWarps][D];
  const float* parts = p.parts;
  const Note* notes = reinterpret_cast<const Note*>(p.notes);
  chain_begin(parts, notes);
  const Note n = notes[blockIdx.x];
  if (n.parts < 2) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr long long kSlot = N * (D + 2);
  constexpr int kFew = 8;
  const float* base = parts + 2LL * n.first * kSlot;      // part 0 lies in its block's second slot, the others in the first slots of their blocks
  const bool few = n.parts <= kFew;
  const int members = few ? kWarps : 1, me = few ? warp : 0, width = few ? 32 : kJoinThreads, at = few ? lane : threadIdx.x;
  for (int r = (n.border * gridDim.y + blockIdx.y) * members + me; r < n.rows; r += (n.parts - 1) * gridDim.y * members) {      // few: warps go their own ways, without barriers
    float m = -INFINITY;
    for (int i = at; i < n.parts; i += width) {
      const float* part = base + (2LL * i + (i == 0 ? 1 : 0)) * kSlot + N * D;
      if (part[N + r] != 0.0f) m = fmaxf(m, part[r]);      // a sum of 0: saw nothing
    }
    m = st::warp_max(m);
    if (!few) {
      __syncthreads();
      if (lane == 0) red[0][warp] = m;
      __syncthreads();
      m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    }
    float l = 0.0f, *w = weight + (few ? warp * kFew : 0);
    for (int i = at; i < n.parts; i += width) {
      const float* part = base + (2LL * i + (i == 0 ? 1 : 0)) * kSlot + N * D;
      const float pl = part[N + r], e = pl == 0.0f ? 0.0f : st::exp2_ftz(part[r] - m);
      w[i] = e;
      l += pl * e;
    }
    l = st::warp_sum(l);
    if (few) {
      __syncwarp();
    } else {
      if (lane == 0) red[1][warp] = l;
      __syncthreads();
      l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    }
    float x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = 0.0f;
#pragma unroll 8
    for (int i = few ? 0 : warp; i < n.parts; i += few ? 1 : kWarps) {
      const float e = w[i];
      const float* part = base + (2LL * i + (i == 0 ? 1 : 0)) * kSlot + r * D + lane * E;
      if constexpr (E == 4) {
        const float4 y = *reinterpret_cast<const float4*>(part);
        x[0] = fmaf(y.x, e, x[0]), x[1] = fmaf(y.y, e, x[1]), x[2] = fmaf(y.z, e, x[2]), x[3] = fmaf(y.w, e, x[3]);
      } else {
        const float2 y = *reinterpret_cast<const float2*>(part);
        x[0] = fmaf(y.x, e, x[0]), x[1] = fmaf(y.y, e, x[1]);
      }
    }
    const int fr = n.row0 + r;
    const long long row = n.start + fr / p.group;
    const int head = n.h * p.group + fr % p.group;
    T* o = static_cast<T*>(p.out) + row * p.o_row + head * p.o_head;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (few) {
#pragma unroll
      for (int e = 0; e < E; ++e) o[lane * E + e] = from_f<T>(x[e] * inv);
      __syncwarp();
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) rows[warp][lane * E + e] = x[e];
      __syncthreads();
      const int d = threadIdx.x;
      if (d < D) o[d] = from_f<T>(((rows[0][d] + rows[1][d]) + (rows[2][d] + rows[3][d])) * inv);
    }
    if (at == 0 && p.lse != nullptr) p.lse[row * p.heads + head] = l == 0.0f ? -INFINITY : (m + kLift + log2f(l)) / kLog2e;
  }
}
}  // namespace
