// Attention of the newest tokens of every sequence over an 8-bit paged cache (decoding, checking drafted tokens, parts of prompts).
//
//   s = scale * q . k * 2^a,  p = softmax(s) over the visible keys,  o = sum p v * 2^b      (a, b: exponents of the page's scales)
//
// What bounds it: a key is 2 * D bytes and 4 * D operations per query row, so for the rows of one decoding step (the query
// heads of one key head) it is bound by reading the cache once.
//
// Work.  The rows of a sequence that share a key head are its n tokens times the G query heads of the group; N = 8, 16 or 32 of them
// are an item together with one (sequence, key head), and 64 keys of an item are a unit.  All units of the call are numbered through and
// every block takes an equal run of them, whatever the lengths are: the split needs nothing from the host but the shapes, so a captured
// launch stays right while the sequences grow, and one long sequence fills the chip as well as many short ones.  Each block finds its run
// by a prefix sum over the sequences.  Where a run ends inside an item, the block leaves (maximum, sum, output) in the workspace,
// and a second kernel joins the parts of such items in their order, so results do not depend on timing.
//
// Inner loop.  A warp takes 16 keys of a unit at a time straight from global memory to registers: each thread loads 16 bytes of
// contiguous codes, and the order of the head elements inside the matrix instructions is chosen so that those bytes are its own
// fragments (keys as the rows of A, S^T = K Q^T; values transposed by byte permutes, O^T = V^T P^T), converted to fp16, which holds e4m3
// exactly.  So nothing passes through shared memory, and the queries are the N side of m16n8k16, which wastes nothing from 8 rows on.
// Queries are scaled by a power of two per row so that fp16 holds bf16's bits too.  The softmax runs over x + b instead of x
// (b: the page's value exponent): the weights exp2(x + b - max) are those that multiply the codes, at most 1, and fp16 keeps 11 bits
// of them; the sum takes exp2(-b) back out.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "paged.cuh"

namespace {
using st::chain_begin;

constexpr int kWarps = 4, kThreads = 32 * kWarps, kTile = 16 * kWarps;      // keys of a unit
constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
  const void* q;
  const unsigned char *kc, *vc;
  const float *ks, *vs;
  const int *table, *starts, *lengths;
  void* out;
  float *lse, *parts;
  long long q_row, q_head, o_row, o_head, table_row, pages;
  long long rows;      // of q and out
  int width, shift, B, heads, kv_heads, group;
  float scale;
  int causal, zero_tail;
  unsigned* err;
};

struct Seq {
  int start, n, len, row_blocks, tiles;
  long long units;
};
template <int N>
__device__ __forceinline__ Seq sequence(const AttnParams& p, int b) {
  Seq s;
  const long long a = p.starts[b], e = p.starts[b + 1];
  s.start = static_cast<int>(a < 0 ? 0 : a);
  const long long end = e < p.rows ? e : p.rows;
  s.n = end > s.start ? static_cast<int>(end - s.start) : 0;
  const long long room = static_cast<long long>(p.width) << p.shift;
  const int len = max(p.lengths[b], 0);
  s.len = len < room ? len : static_cast<int>(room);
  s.row_blocks = (static_cast<long long>(s.n) * p.group + N - 1) / N;
  s.tiles = max((s.len + kTile - 1) / kTile, 1);      // a sequence without keys still gets its zero rows
  s.units = static_cast<long long>(s.row_blocks) * s.tiles * p.kv_heads;
  return s;
}

// Units of all sequences, and of those before `want`: the sequence that holds unit `want` and the number of its first one.
struct Found {
  int b;
  long long first;
};
template <int N>
__device__ long long units_in_all(const AttnParams& p, long long* shared) {
  long long sum = 0;
  for (int b = threadIdx.x; b < p.B; b += kThreads) sum += sequence<N>(p, b).units;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sum += shared[w];
  __syncthreads();
  return sum;
}
template <int N>
__device__ Found find_unit(const AttnParams& p, long long want, long long* shared, Found* found) {
  long long before = 0;
  for (int base = 0; base < p.B; base += kThreads) {
    const int b = base + threadIdx.x;
    const long long mine = b < p.B ? sequence<N>(p, b).units : 0;
    long long s = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, s, o);
      if ((threadIdx.x & 31) >= o) s += u;
    }
    if ((threadIdx.x & 31) == 31) shared[threadIdx.x >> 5] = s;
    __syncthreads();
    long long first = before + s - mine;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < (threadIdx.x >> 5)) first += shared[w];
      before += shared[w];
    }
    if (want >= first && want < first + mine) *found = Found{b, first};      // one thread at most
    __syncthreads();
    if (want < before) break;
  }
  return *found;
}

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t pair) {      // of the low 16 bits
  uint32_t d;
  asm("{ .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, lo; }" : "=r"(d) : "r"(pair));
  return d;
}
__device__ __forceinline__ uint32_t e4m3x2_hi_to_f16x2(uint32_t pair) {   // of the high 16 bits
  uint32_t d;
  asm("{ .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, hi; }" : "=r"(d) : "r"(pair));
  return d;
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint4 load_stream(const unsigned char* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 load_stream8(const unsigned char* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
// Bytes of e4m3 that are no number, as 0x80 in their places.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ void load4f(const T* p, float (&f)[4]);
template <> __device__ __forceinline__ void load4f(const __nv_bfloat16* p, float (&f)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __bfloat162float(p[i]);
}
template <> __device__ __forceinline__ void load4f(const __half* p, float (&f)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __half2float(p[i]);
}
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }

// 16 keys of one head: codes of keys and values as this thread's fragments take them, and the page's exponents.
template <int D>
struct Chunk {
  static constexpr int W = D / 16;      // words per key row part / value row part
  uint32_t k[2][W], v[4][D / 32];
  float ks;
  int ve;
  bool valid;
};

template <int D, int NT>
struct Shared {
  static constexpr int N = 8 * NT;
  static constexpr int OUT_ROW = D + 8;
  uint2 q[NT][D / 16][32];
  float out[kWarps][N][OUT_ROW];
  float m[kWarps][N], l[kWarps][N], mx[N], inv[N];
  float factor[N];
  int limit[N];
  long long sums[kWarps];
  Found found;
};

template <int D>
__device__ __forceinline__ void load_chunk(Chunk<D>& c, const AttnParams& p, const int* table, int key0, int keys, int h, int g, int q4) {
  c.valid = key0 < keys;
  c.ks = 0.0f;
  c.ve = 0;
  if (!c.valid) return;
  const long long page = table[key0 >> p.shift];
  if (page < 0 || page >= p.pages) {
    if ((threadIdx.x & 31) == 0) st::report_error(p.err, st::ERR_BOUNDS, 0x7004);
    c.valid = false;
    return;
  }
  const long long at = page * p.kv_heads + h;
  const long long base = ((at << p.shift) + (key0 & ((1 << p.shift) - 1))) * D;
  const unsigned char *kp = p.kc + base, *vp = p.vc + base;
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      const uint4 x = load_stream(kp + (g + 8 * r) * D + 64 * j + 16 * q4);
      c.k[r][4 * j] = x.x, c.k[r][4 * j + 1] = x.y, c.k[r][4 * j + 2] = x.z, c.k[r][4 * j + 3] = x.w;
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned char* row = vp + (2 * q4 + (i & 1) + 8 * (i >> 1)) * D + g * (D / 8);
    if constexpr (D == 128) {
      const uint4 x = load_stream(row);
      c.v[i][0] = x.x, c.v[i][1] = x.y, c.v[i][2] = x.z, c.v[i][3] = x.w;
    } else {
      const uint2 x = load_stream8(row);
      c.v[i][0] = x.x, c.v[i][1] = x.y;
    }
  }
  c.ks = p.ks[at];
  c.ve = st::scale_exponent(p.vs[at]);
}

template <int D, int NT>
struct Running {
  float o[D / 16][NT][4];
  float m[NT][2], l[NT][2];
};

// One chunk of 16 keys: scores, running maximum and sum, weights times values.
template <int D, int NT>
__device__ __forceinline__ void process(Chunk<D>& c, Running<D, NT>& st_, const Shared<D, NT>& sh, const uint2 (&qreg)[D / 16], int key0, int keys, int limit_min, int g, int q4) {
  float s[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 0; k < D / 16; ++k) {
    const uint32_t a0 = e4m3x2_to_f16x2(c.k[0][k]), a1 = e4m3x2_to_f16x2(c.k[1][k]), a2 = e4m3x2_hi_to_f16x2(c.k[0][k]), a3 = e4m3x2_hi_to_f16x2(c.k[1][k]);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint2 b = NT == 1 ? qreg[k] : sh.q[n][k][lane];
      mma(s[n], a0, a1, a2, a3, b.x, b.y);
    }
  }
  const bool edge = key0 + 16 > limit_min;      // some row does not see some of these keys
  const float ve = static_cast<float>(c.ve), take = st::exp2_int(-c.ve);
  uint32_t pw[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r0 = 8 * n + 2 * q4;
    const float f0 = sh.factor[r0] * c.ks, f1 = sh.factor[r0 + 1] * c.ks;
    float x0 = fmaf(s[n][0], f0, ve), x1 = fmaf(s[n][1], f1, ve), x2 = fmaf(s[n][2], f0, ve), x3 = fmaf(s[n][3], f1, ve);
    if (edge) {
      const int l0 = sh.limit[r0], l1 = sh.limit[r0 + 1];
      if (key0 + g >= l0) x0 = -INFINITY;
      if (key0 + g >= l1) x1 = -INFINITY;
      if (key0 + g + 8 >= l0) x2 = -INFINITY;
      if (key0 + g + 8 >= l1) x3 = -INFINITY;
    }
    float m0 = fmaxf(x0, x2), m1 = fmaxf(x1, x3);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
      m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
    }
    m0 = fmaxf(m0, st_.m[n][0]), m1 = fmaxf(m1, st_.m[n][1]);
    if (__any_sync(0xffffffffu, m0 > st_.m[n][0] || m1 > st_.m[n][1])) {
      const float a0 = m0 > st_.m[n][0] ? exp2f(st_.m[n][0] - m0) : 1.0f, a1 = m1 > st_.m[n][1] ? exp2f(st_.m[n][1] - m1) : 1.0f;
      st_.m[n][0] = m0, st_.m[n][1] = m1;
      st_.l[n][0] *= a0, st_.l[n][1] *= a1;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) st_.o[i][n][0] *= a0, st_.o[i][n][1] *= a1, st_.o[i][n][2] *= a0, st_.o[i][n][3] *= a1;
    }
    const float z0 = m0 == -INFINITY ? 0.0f : m0, z1 = m1 == -INFINITY ? 0.0f : m1;      // nothing seen so far: weights 0, not NaN
    const float w0 = exp2f(x0 - z0), w1 = exp2f(x1 - z1), w2 = exp2f(x2 - z0), w3 = exp2f(x3 - z1);
    st_.l[n][0] = fmaf(w0 + w2, take, st_.l[n][0]);
    st_.l[n][1] = fmaf(w1 + w3, take, st_.l[n][1]);
    pw[n][0] = transpose8x8(pack_f16x2(w0, w1));
    pw[n][1] = transpose8x8(pack_f16x2(w2, w3));
  }
  if (edge) {
    // what lies behind the end is no value; a value that is no number counts only for the rows that see it
    uint32_t some = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool behind = key0 + 2 * q4 + (i & 1) + 8 * (i >> 1) >= keys;
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        if (behind) c.v[i][w] = 0;
        some |= nan_bytes(c.v[i][w]);
      }
    }
    if (__any_sync(0xffffffffu, some != 0)) {
      uint32_t bad[4];      // a bit per element of the thread's part of a key's row
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        bad[i] = 0;
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
          const uint32_t nb = nan_bytes(c.v[i][w]);
          bad[i] |= ((nb >> 7 & 1) | (nb >> 14 & 2) | (nb >> 21 & 4) | (nb >> 28 & 8)) << (4 * w);
          c.v[i][w] &= ~((nb >> 7) * 255u);
        }
      }
#pragma unroll
      for (int src = 0; src < 4; ++src)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t bits = __shfl_sync(0xffffffffu, bad[i], (lane & ~3) | src);
          const int key = key0 + 2 * src + (i & 1) + 8 * (i >> 1);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r)
              if (bits && key < sh.limit[8 * n + 2 * q4 + r])
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                  if (bits >> (2 * d) & 1) st_.o[d][n][r] = NAN;
                  if (bits >> (2 * d + 1) & 1) st_.o[d][n][2 + r] = NAN;
                }
        }
    }
  }
#pragma unroll
  for (int d = 0; d < D / 16; ++d) {
    const int w = d / 2;
    const uint32_t sel = d & 1 ? 0x7362 : 0x5140;
    const uint32_t lo = __byte_perm(c.v[0][w], c.v[1][w], sel), hi = __byte_perm(c.v[2][w], c.v[3][w], sel);
    const uint32_t a0 = e4m3x2_to_f16x2(lo), a1 = e4m3x2_hi_to_f16x2(lo), a2 = e4m3x2_to_f16x2(hi), a3 = e4m3x2_hi_to_f16x2(hi);
#pragma unroll
    for (int n = 0; n < NT; ++n) mma(st_.o[d][n], a0, a1, a2, a3, pw[n][0], pw[n][1]);
  }
}

template <int D, int NT>
__device__ __forceinline__ float* part_of(const AttnParams& p, long long slot) {      // [N][D] output, [N] maximum, [N] sum
  return p.parts + slot * (8 * NT * (D + 2));
}

// Where an output element stands in a row of Shared::out: element 16 g + 2 i + e (D = 128) at 16 i + 2 g + e.
template <int D>
__device__ __forceinline__ int out_at(int d) {
  constexpr int PER = D / 8;
  return (d % PER / 2) * 16 + (d / PER) * 2 + (d & 1);
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads) paged_attn_kernel(AttnParams p) {
  constexpr int N = 8 * NT;
  extern __shared__ __align__(16) unsigned char raw[];
  Shared<D, NT>& sh = *reinterpret_cast<Shared<D, NT>*>(raw);
  chain_begin(p.kc, p.vc, p.ks, p.vs, p.table, p.starts, p.lengths);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q4 = lane & 3;
  const T* q = static_cast<const T*>(p.q);
  T* out = static_cast<T*>(p.out);

  if (p.zero_tail) {      // rows behind the last sequence
    const long long from = p.B > 0 ? max(p.starts[p.B], 0) : 0, per = static_cast<long long>(p.heads) * D;
    for (long long i = from * per + blockIdx.x * kThreads + threadIdx.x; i < p.rows * per; i += static_cast<long long>(gridDim.x) * kThreads) {
      const long long row = i / per, e = i - row * per;
      out[row * p.o_row + e / D * p.o_head + e % D] = from_f<T>(0.0f);
      if (p.lse != nullptr && e % D == 0) p.lse[row * p.heads + e / D] = -INFINITY;
    }
  }
  const long long all = units_in_all<N>(p, sh.sums);
  const int runs = static_cast<int>(min(static_cast<long long>(gridDim.x), all));      // none of them empty
  if (static_cast<int>(blockIdx.x) >= runs) return;
  const long long u0 = all * blockIdx.x / runs, u1 = all * (blockIdx.x + 1) / runs;
  Found f = find_unit<N>(p, u0, sh.sums, &sh.found);
  Seq sq = sequence<N>(p, f.b);

  for (long long u = u0; u < u1;) {
    while (u >= f.first + sq.units) {
      f.first += sq.units;
      sq = sequence<N>(p, ++f.b);
    }
    // unit -> (key head, row block, tile): row blocks of one head next to each other, as they read the same pages
    const long long in = u - f.first;
    const int t0 = static_cast<int>(in % sq.tiles);
    const long long item = in / sq.tiles;
    const int rb = static_cast<int>(item % sq.row_blocks), h = static_cast<int>(item / sq.row_blocks);
    const int t1 = static_cast<int>(min(static_cast<long long>(sq.tiles), t0 + (u1 - u)));
    const int row0 = rb * N, row_end = min(sq.n * p.group, row0 + N);
    const int* table = p.table + f.b * p.table_row;
    // keys that row r sees: all of the sequence, or those up to its own place
    const int hidden = p.causal ? sq.n - 1 - row0 / p.group : 0, hidden_last = p.causal ? sq.n - 1 - (row_end - 1) / p.group : 0;
    const int limit_min = max(sq.len - hidden, 0), keys = max(sq.len - hidden_last, 0);

    Chunk<D> next;
    int key0 = t0 * kTile + warp * 16;
    load_chunk(next, p, table, key0, min(keys, t1 * kTile), h, g, q4);
    __syncthreads();      // the item before is done with the shared memory
    for (int r = warp; r < N; r += kWarps) {
      float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      const int fr = row0 + r;
      const bool live = fr < row_end;
      if (live && 4 * lane < D) load4f(q + (sq.start + fr / p.group) * p.q_row + (h * p.group + fr % p.group) * p.q_head + 4 * lane, x);
      const float top = st::warp_max(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
      // the largest to [2^13, 2^14): exact for bf16 and fp16 down to 2^-27 of it; a row with infinities stays as it is
      int e = static_cast<int>((__float_as_uint(top) >> 23) & 255) - 127 - 13;
      e = top < INFINITY ? max(e, -100) : 0;
      const float mul = st::exp2_int(-e);
      if (4 * lane < D) {
        const int d = 4 * lane, k = d / 64 * 4 + d % 16 / 4, c = d % 64 / 16;
        sh.q[r / 8][k][(r % 8) * 4 + c] = make_uint2(pack_f16x2(x[0] * mul, x[1] * mul), pack_f16x2(x[2] * mul, x[3] * mul));
      }
      if (lane == 0) {
        sh.factor[r] = p.scale * kLog2e * st::exp2_int(e);
        sh.limit[r] = live ? max(sq.len - (p.causal ? sq.n - 1 - fr / p.group : 0), 0) : 0x7fffffff;      // rows that are none are not written
      }
    }
    __syncthreads();
    uint2 qreg[D / 16];
    if constexpr (NT == 1)
#pragma unroll
      for (int k = 0; k < D / 16; ++k) qreg[k] = sh.q[0][k][lane];
    Running<D, NT> s;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      s.m[n][0] = s.m[n][1] = -INFINITY;
      s.l[n][0] = s.l[n][1] = 0.0f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) s.o[d][n][0] = s.o[d][n][1] = s.o[d][n][2] = s.o[d][n][3] = 0.0f;
    }
    for (int t = t0; t < t1; ++t) {
      Chunk<D> c = next;
      const int at = key0;
      key0 += kTile;
      load_chunk(next, p, table, key0, min(keys, t1 * kTile), h, g, q4);
      if (c.valid) process<D, NT>(c, s, sh, qreg, at, keys, limit_min, g, q4);
    }

    // join the warps
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) s.l[n][r] += __shfl_xor_sync(0xffffffffu, s.l[n][r], o);
        if (g == 0) sh.m[warp][8 * n + 2 * q4 + r] = s.m[n][r], sh.l[warp][8 * n + 2 * q4 + r] = s.l[n][r];
      }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float a[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = 8 * n + 2 * q4 + r;
        const float mx = fmaxf(fmaxf(sh.m[0][row], sh.m[1][row]), fmaxf(sh.m[2][row], sh.m[3][row]));
        a[r] = s.l[n][r] == 0.0f ? 0.0f : exp2f(s.m[n][r] - mx);      // 0: saw nothing; a score that is no number leaves a sum that is none
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int r = 0; r < 2; ++r)
          *reinterpret_cast<float2*>(&sh.out[warp][8 * n + 2 * q4 + r][16 * d + 2 * g]) = make_float2(s.o[d][n][r] * a[r], s.o[d][n][2 + r] * a[r]);
    }
    if (threadIdx.x < N) {
      const int row = threadIdx.x;
      const float mx = fmaxf(fmaxf(sh.m[0][row], sh.m[1][row]), fmaxf(sh.m[2][row], sh.m[3][row]));
      float l = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) l += sh.l[w][row] == 0.0f ? 0.0f : sh.l[w][row] * exp2f(sh.m[w][row] - mx);
      sh.mx[row] = mx, sh.inv[row] = l;
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == sq.tiles;
    float* part = whole ? nullptr : part_of<D, NT>(p, 2LL * blockIdx.x + (t0 == 0 ? 1 : 0));
    for (int i = threadIdx.x; i < N * (D / 2); i += kThreads) {
      const int row = i / (D / 2), d = i % (D / 2) * 2, at = out_at<D>(d);
      if (row >= row_end - row0) break;
      float2 x = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 y = *reinterpret_cast<const float2*>(&sh.out[w][row][at]);
        x.x += y.x, x.y += y.y;
      }
      const float l = sh.inv[row];
      if (whole) {
        const int fr = row0 + row;
        T* o = out + (sq.start + fr / p.group) * p.o_row + (h * p.group + fr % p.group) * p.o_head + d;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        o[0] = from_f<T>(x.x * inv), o[1] = from_f<T>(x.y * inv);
        if (d == 0 && p.lse != nullptr)
          p.lse[(sq.start + fr / p.group) * static_cast<long long>(p.heads) + h * p.group + fr % p.group] = l == 0.0f ? -INFINITY : (sh.mx[row] + log2f(l)) / kLog2e;
      } else {
        *reinterpret_cast<float2*>(part + row * D + d) = x;
        if (d == 0) part[N * D + row] = sh.mx[row], part[N * D + N + row] = l;
      }
    }
    u += t1 - t0;
  }
}

// Joins the parts of an item that several blocks worked on, a block (border, row): border c is the one between the runs of blocks c and
// c + 1, and the first border inside an item stands for the item.  All parts' maxima and sums are read at once; then each warp adds up its
// share of the parts, D / 32 elements a thread, with as many loads in flight as it has parts.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads) paged_join_kernel(AttnParams p, int most_runs) {
  constexpr int N = 8 * NT, E = D / 32;
  extern __shared__ float weight[];      // [parts]
  __shared__ long long sums[kWarps];
  __shared__ Found found;
  __shared__ float red[2][kWarps], rows[kWarps][D];
  chain_begin(p.table, p.starts, p.lengths);
  const long long all = units_in_all<N>(p, sums);
  const int runs = static_cast<int>(min(static_cast<long long>(most_runs), all)), c = blockIdx.x;
  if (c + 1 >= runs) return;
  const long long u0 = all * c / runs, u1 = all * (c + 1) / runs;
  const Found f = find_unit<N>(p, u1, sums, &found);
  const Seq sq = sequence<N>(p, f.b);
  const long long in = u1 - f.first;
  const int t = static_cast<int>(in % sq.tiles), r = blockIdx.y;
  if (t == 0 || u1 - t < u0) return;
  const long long end = u1 - t + sq.tiles, item = in / sq.tiles;
  const int rb = static_cast<int>(item % sq.row_blocks), h = static_cast<int>(item / sq.row_blocks);
  const int row0 = rb * N, row_end = min(sq.n * p.group, row0 + N);
  if (r >= row_end - row0) return;
  // block b holds a part if its run begins before the end: all * b / runs < end, which is all * b < end * runs
  const int parts = static_cast<int>((end * runs - 1) / all) - c + 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr long long kSlot = N * (D + 2);
  const float* base = p.parts + (2LL * c) * kSlot;      // part 0 lies in the block's second slot, the others in the first slots of their blocks

  float m = -INFINITY;
  for (int i = threadIdx.x; i < parts; i += kThreads) {
    const float* part = base + (2LL * i + (i == 0 ? 1 : 0)) * kSlot + N * D;
    if (part[N + r] != 0.0f) m = fmaxf(m, part[r]);      // a sum of 0: saw nothing
  }
  m = st::warp_max(m);
  if (lane == 0) red[0][warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, red[0][w]);
  float l = 0.0f;
  for (int i = threadIdx.x; i < parts; i += kThreads) {
    const float* part = base + (2LL * i + (i == 0 ? 1 : 0)) * kSlot + N * D;
    const float pl = part[N + r], e = pl == 0.0f ? 0.0f : exp2f(part[r] - m);
    weight[i] = e;
    l += pl * e;
  }
  l = st::warp_sum(l);
  if (lane == 0) red[1][warp] = l;
  __syncthreads();
  l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);

  float x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = 0.0f;
#pragma unroll 8
  for (int i = warp; i < parts; i += kWarps) {
    const float w = weight[i];
    const float* part = base + (2LL * i + (i == 0 ? 1 : 0)) * kSlot + r * D + lane * E;
    if constexpr (E == 4) {
      const float4 y = *reinterpret_cast<const float4*>(part);
      x[0] = fmaf(y.x, w, x[0]), x[1] = fmaf(y.y, w, x[1]), x[2] = fmaf(y.z, w, x[2]), x[3] = fmaf(y.w, w, x[3]);
    } else {
      const float2 y = *reinterpret_cast<const float2*>(part);
      x[0] = fmaf(y.x, w, x[0]), x[1] = fmaf(y.y, w, x[1]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) rows[warp][lane * E + e] = x[e];
  __syncthreads();
  const int d = threadIdx.x, fr = row0 + r;
  const long long row = sq.start + fr / p.group;
  const int head = h * p.group + fr % p.group;
  if (d < D) {
    const float sum = (rows[0][d] + rows[1][d]) + (rows[2][d] + rows[3][d]);
    static_cast<T*>(p.out)[row * p.o_row + head * p.o_head + d] = from_f<T>(l == 0.0f ? 0.0f : sum / l);
  }
  if (d == 0 && p.lse != nullptr) p.lse[row * p.heads + head] = l == 0.0f ? -INFINITY : (m + log2f(l)) / kLog2e;
}

// Row tiles of 8 by the rows that the longest step of a sequence has.
int row_tiles(long long max_queries, int group) {
  const long long rows = max_queries * group;
  return rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
}
int runs_of(int nt) { return st::sm_count() * (nt == 4 ? 2 : 3); }

template <typename T, int D, int NT>
int launch(const AttnParams& p, cudaStream_t stream) {
  const int runs = runs_of(NT);
  constexpr int smem = sizeof(Shared<D, NT>);
  auto kernel = paged_attn_kernel<T, D, NT>;
  if (smem > 48 * 1024) ST_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  cudaError_t e = st::chained(kernel, dim3(runs), dim3(kThreads), smem, stream)(p);
  if (e != cudaSuccess) return st::fail_cuda(e, "paged attention");
  e = st::chained(paged_join_kernel<T, D, NT>, dim3(runs - 1, 8 * NT), dim3(kThreads), runs * sizeof(float), stream)(p, runs);
  if (e != cudaSuccess) return st::fail_cuda(e, "paged attention: join");
  return ST_OK;
}
template <typename T>
int dispatch(const AttnParams& p, int dim, int nt, cudaStream_t stream) {
  if (dim == 64) return nt == 1 ? launch<T, 64, 1>(p, stream) : nt == 2 ? launch<T, 64, 2>(p, stream) : launch<T, 64, 4>(p, stream);
  return nt == 1 ? launch<T, 128, 1>(p, stream) : nt == 2 ? launch<T, 128, 2>(p, stream) : launch<T, 128, 4>(p, stream);
}
}  // namespace

// Floats of workspace that st_paged_attention takes.
ST_API long long st_paged_attention_workspace(int max_queries, int heads, int kv_heads, int dim) {
  if (kv_heads < 1 || heads < kv_heads) return 0;
  const int nt = row_tiles(max_queries, heads / kv_heads);
  return 2LL * runs_of(nt) * 8 * nt * (dim + 2);
}

// q, out [rows, heads, dim] (dim contiguous, strides in elements): row starts[b] + i is the i-th of the newest tokens of sequence b, whose keys and values,
// these tokens' included, are the first lengths[b] of the pages in table[b].  lse [rows, heads] or null.  max_queries: the most rows of a sequence, by which
// the row tile is chosen; more are computed too.  zero_tail: rows behind the last sequence become 0 (else they stay as they were).  type: 0 bf16, 1 fp16.
ST_API int st_paged_attention(const void* q, const void* k_codes, const void* v_codes, const float* k_scale, const float* v_scale, const int* table, const int* starts,
                              const int* lengths, void* out, float* lse, float* workspace, long long q_row, long long q_head, long long o_row, long long o_head,
                              long long table_row, long long pages, long long rows, int width, int page_size, int B, int heads, int kv_heads, int dim, int max_queries, float scale,
                              int causal, int zero_tail, int type, void* stream_v) {
  const int shift = st::page_shift(page_size);
  if (shift < 0 || B < 0 || rows < 0 || rows > 2147483647LL || width < 0 || (static_cast<long long>(width) << shift) > 2147483647LL || kv_heads < 1 || heads < kv_heads ||
      heads % kv_heads || (dim != 64 && dim != 128) || pages < 0 || max_queries < 1 || (type != 0 && type != 1) || rows * (heads / kv_heads) > 2147483647LL)
    return st::fail(ST_ERR_INVALID, "paged attention: sizes out of range (page 16 to 256, dim 64 or 128, heads a multiple of kv_heads)");
  if ((reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return st::fail(ST_ERR_INVALID, "paged attention: codes must be 16-byte aligned");
  if (rows == 0) return ST_OK;
  const AttnParams p{q, static_cast<const unsigned char*>(k_codes), static_cast<const unsigned char*>(v_codes), k_scale, v_scale, table, starts, lengths, out, lse, workspace,
                     q_row, q_head, o_row, o_head, table_row, pages, rows, width, shift, B, heads, kv_heads, heads / kv_heads, scale, causal, zero_tail, st::error_word()};
  const int nt = row_tiles(max_queries, heads / kv_heads);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  return type == 0 ? dispatch<__nv_bfloat16>(p, dim, nt, stream) : dispatch<__half>(p, dim, nt, stream);
}
