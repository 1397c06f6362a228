// Attention of the newest tokens of every sequence over an 8-bit paged cache (decoding, checking drafted tokens, parts of prompts).
//
//   s = scale * q . k * 2^a,  p = softmax(s) over the visible keys,  o = sum p v * 2^b      (a, b: exponents of the page's scales)
//
// What bounds it: a key is 2 * D bytes and 4 * D operations per query row, so for the rows of one decoding step (the query
// heads of one key head) it is bound by reading the cache once.
//
// Work.  The rows of a sequence that share a key head are its n tokens times the G query heads of the group; N = 8, 16 or 32 of them
// are an item together with one (sequence, key head), and 128 keys of an item are a unit.  All units of the call are numbered through and
// every block takes an equal run of them, whatever the lengths are: the split needs nothing from the host but the shapes, so a captured
// launch stays right while the sequences grow, and one long sequence fills the chip as well as many short ones.  Each block finds its run
// by a prefix sum over the sequences.  Where a run ends inside an item, the block leaves (maximum, sum, output) in the workspace,
// and a second kernel joins the parts of such items in their order, so results do not depend on timing.  It finds them by the notes
// that the blocks leave about the border between their run and the next.
//
// Inner loop.  A warp takes 32 keys of a unit at a time through rings of its own in shared memory, two slots of 4 KB (for heads of 128) for keys
// and two for values, which one lane fills by tiled copies: the keys two steps ahead are asked for as soon as the scores of this step are
// formed, the values when its products are, and the run's next item follows the last one without a pause.
// The order of the head elements inside the matrix instructions is chosen so that 16 contiguous bytes of a key are a thread's
// fragments (keys as the rows of A, S^T = K Q^T; values transposed by byte permutes, O^T = V^T P^T), the order of the keys so that no two
// lanes' loads from the swizzled rows meet in a bank (key_of below).  Codes become fp16, which holds e4m3 exactly, and the queries are the
// N side of m16n8k16, which wastes nothing from 8 rows on.  (m16n8k32 on the codes themselves, with a query as the sum of two e4m3 values, is
// no gain: it takes more instructions than the conversion, 78 us against 75 on the case of 64 sequences.)  Queries are scaled by a power of two
// per row so that fp16 holds bf16's bits too.  The softmax runs over x + b instead of x (b: the page's value exponent): the weights exp2(x + b - max) are those that
// multiply the codes, at most 1, and fp16 keeps 11 bits of them; the sum takes exp2(-b) back out.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "paged.cuh"

namespace {
using st::chain_begin;

constexpr int kWarps = 4, kThreads = 32 * kWarps, kTile = 32 * kWarps;      // keys of a unit
constexpr float kLog2e = 1.4426950408889634f;

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

// Where the block's share begins: the sequence that holds a unit, and the number of the sequence's first one.
struct Found {
  int b;
  long long first;
};
__device__ __forceinline__ long long scan_block(long long mine, long long* shared, long long& total) {      // sum of the threads before, and of all
  long long s = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) >= o) s += u;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 31) shared[threadIdx.x >> 5] = s;
  __syncthreads();
  long long before = s - mine;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < static_cast<int>(threadIdx.x >> 5)) before += shared[w];
    total += shared[w];
  }
  return before;
}
// The block's share [u0, u1) of the units, if it has one, and where unit u0 lies.  Up to a block's threads of sequences are looked at once.
template <int N>
__device__ bool find_share(const AttnParams& p, long long* shared, Found* found, long long& all, int& runs, long long& u0, long long& u1, Found& f) {
  long long mine = 0, total = 0, before = 0;
  for (int b = threadIdx.x; b < p.B; b += kThreads) mine += sequence<N>(p, b).units;
  before = scan_block(mine, shared, total);
  all = total;
  runs = static_cast<int>(min(static_cast<long long>(gridDim.x), all));      // none of them empty
  if (static_cast<int>(blockIdx.x) >= runs) return false;
  u0 = all * blockIdx.x / runs, u1 = all * (blockIdx.x + 1) / runs;
  if (p.B <= kThreads) {
    if (u0 >= before && u0 < before + mine) *found = Found{static_cast<int>(threadIdx.x), before};      // one thread
  } else {
    long long base = 0;
    for (int b0 = 0; b0 < p.B && u0 >= base; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      mine = b < p.B ? sequence<N>(p, b).units : 0;
      before = base + scan_block(mine, shared, total);
      if (u0 >= before && u0 < before + mine) *found = Found{b, before};
      base += total;
    }
  }
  __syncthreads();
  f = *found;
  return true;
}
// a / b and a % b, by 32-bit arithmetic where both fit.
__device__ __forceinline__ long long divide(long long a, int b, int& rest) {
  if (a >> 32 == 0) {
    const unsigned q = static_cast<unsigned>(a) / static_cast<unsigned>(b);
    rest = static_cast<int>(static_cast<unsigned>(a) - q * b);
    return q;
  }
  const long long q = a / b;
  rest = static_cast<int>(a - q * b);
  return q;
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

// What the page (WIDE: pages of 32 tokens and more) or the two pages of 32 keys say of them.
template <bool WIDE>
struct Info {
  static constexpr int PAGES = WIDE ? 1 : 2;
  int page[PAGES];      // -1: nothing there
  float ks[PAGES];      // the keys' scale
  int ve[PAGES];        // the values' exponent
  __device__ __forceinline__ bool valid(int piece) const { return page[WIDE ? 0 : piece] >= 0; }
  __device__ __forceinline__ bool any() const { return WIDE ? page[0] >= 0 : page[0] >= 0 || page[PAGES - 1] >= 0; }
  __device__ __forceinline__ float key_scale(int piece) const { return ks[WIDE ? 0 : piece]; }
  __device__ __forceinline__ int value_exponent(int piece) const { return ve[WIDE ? 0 : piece]; }
};
// One lane's share of the page numbers and scales of the warp's next 16 steps: piece lane % 2 of step lane / 2.
struct PieceList {
  int page;
  float ks;
  int ve;
};

// A slot of a warp's ring: 32 keys (or values), as the copies leave them: lines of 128 bytes (a token, or two of 64 elements) whose 16-byte
// parts are swizzled by the line's number.
template <int D>
struct Slot {
  unsigned char piece[2][16 * D];
};
// The key of a piece that stands at row g (0..7) of a matrix fragment, and how far behind it that of row g + 8 is.  A quarter warp's 16-byte loads of
// keys are rows (2i, 2i + 1) with parts 0..3 or 4..7; its loads of values rows 0, 2, 4, 6 (or 1, 3, 5, 7) with two neighbouring parts: both touch
// all eight parts of the swizzled lines once.
template <int D>
__device__ __forceinline__ int key_of(int g) {
  return D == 128 ? (g & 1 ? g ^ 4 : g) : 4 * (g >> 1) + (g & 1);
}
template <int D>
constexpr int kSecond = D == 128 ? 8 : 2;
// Byte of element 16 * part of token `key` of a piece.
template <int D>
__device__ __forceinline__ int at_part(int key, int part) {
  if constexpr (D == 128) return key * 128 + ((part ^ (key & 7)) << 4);
  return (key >> 1) * 128 + (((4 * (key & 1) + part) ^ (key >> 1 & 7)) << 4);
}

template <int D, int NT>
struct Shared {
  static constexpr int N = 8 * NT;
  static constexpr int OUT_ROW = D + 4;      // lanes' stores of outputs in 32 banks
  Slot<D> ring[kWarps][2][2];                // keys, values
  float out[2][N][OUT_ROW];
  uint2 q[NT][D / 16][32];
  unsigned long long full[kWarps][2][2];     // barriers of the slots
  float m[kWarps][N], l[kWarps][N], mx[N], sum[N];
  float factor[N];
  int limit[N];
  long long place[N];                        // of a row in the output
  long long sums[kWarps];
  Found found;
  int abort;
};

// An item, or the part of it that the block's run covers: units [t0, t1) of one head's rows [row0, row_end) of a sequence.
struct Item {
  const int* table;
  int start, n, len, h, row0, row_end, t0, t1, tiles;
  __device__ __forceinline__ int steps() const { return t1 - t0; }
};
template <int N>
__device__ __forceinline__ Item item_at(const AttnParams& p, long long u, long long u1, Found& f, Seq& sq) {
  while (u >= f.first + sq.units) {
    f.first += sq.units;
    sq = sequence<N>(p, ++f.b);
  }
  // unit -> (key head, row block, tile): row blocks of one head next to each other, as they read the same pages
  Item it;
  int rb;
  it.h = static_cast<int>(divide(divide(u - f.first, sq.tiles, it.t0), sq.row_blocks, rb));
  it.t1 = static_cast<int>(min(static_cast<long long>(sq.tiles), it.t0 + (u1 - u)));
  it.tiles = sq.tiles, it.start = sq.start, it.n = sq.n, it.len = sq.len;
  it.row0 = rb * N, it.row_end = min(sq.n * p.group, it.row0 + N);
  it.table = p.table + f.b * p.table_row;
  return it;
}
// Keys that a row sees: all of the sequence, or those up to its own place.
__device__ __forceinline__ int keys_of(const AttnParams& p, const Item& it, int row) { return max(it.len - (p.causal ? it.n - 1 - row / p.group : 0), 0); }

// Lane i: piece i % 2 of the warp's step first + i / 2.
__device__ __forceinline__ PieceList list_pieces(const AttnParams& p, const Item& it, int first, int keys) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long key = (it.t0 + first + lane / 2) * static_cast<long long>(kTile) + warp * 32 + 16 * (lane & 1);
  PieceList l{-1, 0.0f, 0};
  if (key < keys && first + lane / 2 < it.steps()) {
    const int page = it.table[key >> p.shift];
    if (page < 0 || page >= p.pages) {
      st::report_error(p.err, st::ERR_BOUNDS, 0x7004);
    } else {
      const long long at = static_cast<long long>(page) * p.kv_heads + it.h;
      l.page = page;
      l.ks = p.ks[at];
      l.ve = st::scale_exponent(p.vs[at]);
    }
  }
  return l;
}
template <bool WIDE>
__device__ __forceinline__ Info<WIDE> info_of(const PieceList& list, int step) {
  Info<WIDE> c;
#pragma unroll
  for (int j = 0; j < Info<WIDE>::PAGES; ++j) {
    const int lane = 2 * (step & 15) + j;
    c.page[j] = __shfl_sync(0xffffffffu, list.page, lane);
    c.ks[j] = __shfl_sync(0xffffffffu, list.ks, lane);
    c.ve[j] = __shfl_sync(0xffffffffu, list.ve, lane);
  }
  return c;
}
// Starts the copies of 32 keys (or values) into a slot: one page, or two of 16 tokens.  What lies behind the last key is masked.
template <int D, bool WIDE>
__device__ __forceinline__ void copy_keys(Slot<D>& slot, uint32_t bar, const CUtensorMap* map, const AttnParams& p, const Info<WIDE>& c, int h, int key0) {
  if ((threadIdx.x & 31) != 0) return;
  if constexpr (WIDE) {
    st::mbar_arrive_expect_tx(bar, c.page[0] >= 0 ? sizeof(Slot<D>) : 0);
    if (c.page[0] < 0) return;
    const long long row = ((static_cast<long long>(c.page[0]) * p.kv_heads + h) << p.shift) + (key0 & ((1 << p.shift) - 1));
    st::tma_load_2d(st::smem_u32(slot.piece), map, bar, 0, static_cast<int>(row * D / 128));
  } else {
    st::mbar_arrive_expect_tx(bar, ((c.page[0] >= 0) + (c.page[1] >= 0)) * static_cast<int>(sizeof(Slot<D>) / 2));
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (c.page[j] >= 0)
        st::tma_load_2d(st::smem_u32(slot.piece[j]), map, bar, 0, static_cast<int>((static_cast<long long>(c.page[j]) * p.kv_heads + h) * (16 * D / 128)));
  }
}

template <int D, int NT>
struct Running {
  float o[D / 16][NT][4];
  float m[NT][2], l[NT][2];
};

// Scores of KS pieces of 16 keys.
template <int D, int NT, int KS>
__device__ __forceinline__ void scores(float (&s)[KS][NT][4], const Slot<D>& slot, int piece0, const Shared<D, NT>& sh, const uint2 (&qreg)[D / 16], int g, int q4) {
  constexpr int KW = D / 16;      // words of a key row's part
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < KS; ++j) {
    uint32_t k0[KW], k1[KW];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const uint4 x = *reinterpret_cast<const uint4*>(slot.piece[piece0 + j] + at_part<D>(key_of<D>(g), 4 * i + q4));
      const uint4 y = *reinterpret_cast<const uint4*>(slot.piece[piece0 + j] + at_part<D>(key_of<D>(g) + kSecond<D>, 4 * i + q4));
      k0[4 * i] = x.x, k0[4 * i + 1] = x.y, k0[4 * i + 2] = x.z, k0[4 * i + 3] = x.w;
      k1[4 * i] = y.x, k1[4 * i + 1] = y.y, k1[4 * i + 2] = y.z, k1[4 * i + 3] = y.w;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) s[j][n][0] = s[j][n][1] = s[j][n][2] = s[j][n][3] = 0.0f;
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      const uint32_t a0 = e4m3x2_to_f16x2(k0[k]), a1 = e4m3x2_to_f16x2(k1[k]), a2 = e4m3x2_hi_to_f16x2(k0[k]), a3 = e4m3x2_hi_to_f16x2(k1[k]);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint2 b = NT == 1 ? qreg[k] : sh.q[n][k][lane];
        mma(s[j][n], a0, a1, a2, a3, b.x, b.y);
      }
    }
  }
}

// Running maximum and sum, and the weights in fp16, transposed to fragments.  edge: some row does not see some of these keys.
template <int D, int NT, int KS, bool WIDE>
__device__ __forceinline__ void weights(uint32_t (&pw)[KS][NT][2], float (&s)[KS][NT][4], Running<D, NT>& run, const Info<WIDE>& info, int piece0, const Shared<D, NT>& sh,
                                        const float (&freg)[2], int key0, bool edge, int g, int q4) {
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r0 = 8 * n + 2 * q4;
    const float f0 = NT == 1 ? freg[0] : sh.factor[r0], f1 = NT == 1 ? freg[1] : sh.factor[r0 + 1];
    float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      const float ks = info.key_scale(piece0 + j), a0 = f0 * ks, a1 = f1 * ks, ve = static_cast<float>(info.value_exponent(piece0 + j));
      float (&x)[4] = s[j][n];
      x[0] = fmaf(x[0], a0, ve), x[1] = fmaf(x[1], a1, ve), x[2] = fmaf(x[2], a0, ve), x[3] = fmaf(x[3], a1, ve);
      if (edge) {
        const bool valid = info.valid(piece0 + j);
        const int key = key0 + 16 * j + key_of<D>(g), l0 = valid ? sh.limit[r0] : 0, l1 = valid ? sh.limit[r0 + 1] : 0;
        if (key >= l0) x[0] = -INFINITY;
        if (key >= l1) x[1] = -INFINITY;
        if (key + kSecond<D> >= l0) x[2] = -INFINITY;
        if (key + kSecond<D> >= l1) x[3] = -INFINITY;
      }
      m0 = st::max3(m0, x[0], x[2]), m1 = st::max3(m1, x[1], x[3]);
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
      m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
    }
    m0 = fmaxf(m0, run.m[n][0]), m1 = fmaxf(m1, run.m[n][1]);
    if (__any_sync(0xffffffffu, m0 > run.m[n][0] || m1 > run.m[n][1])) {
      const float a0 = m0 > run.m[n][0] ? st::exp2_ftz(run.m[n][0] - m0) : 1.0f, a1 = m1 > run.m[n][1] ? st::exp2_ftz(run.m[n][1] - m1) : 1.0f;
      run.m[n][0] = m0, run.m[n][1] = m1;
      run.l[n][0] *= a0, run.l[n][1] *= a1;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) run.o[i][n][0] *= a0, run.o[i][n][1] *= a1, run.o[i][n][2] *= a0, run.o[i][n][3] *= a1;
    }
    const float z0 = m0 == -INFINITY ? 0.0f : m0, z1 = m1 == -INFINITY ? 0.0f : m1;      // nothing seen so far: weights 0, not NaN
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      const float (&x)[4] = s[j][n];
      // fp16 ends at 2^-24, so exp2's subnormal results, from 2^-126 on, are 0 anyway
      const float w0 = st::exp2_ftz(x[0] - z0), w1 = st::exp2_ftz(x[1] - z1), w2 = st::exp2_ftz(x[2] - z0), w3 = st::exp2_ftz(x[3] - z1);
      const float take = st::exp2_int(-info.value_exponent(piece0 + j));
      run.l[n][0] = fmaf(w0 + w2, take, run.l[n][0]);
      run.l[n][1] = fmaf(w1 + w3, take, run.l[n][1]);
      pw[j][n][0] = transpose8x8(pack_f16x2(w0, w1));
      pw[j][n][1] = transpose8x8(pack_f16x2(w2, w3));
    }
  }
}

// Weights times values.
template <int D, int NT, int KS, bool WIDE>
__device__ __forceinline__ void values(Running<D, NT>& run, const uint32_t (&pw)[KS][NT][2], const Slot<D>& slot, const Info<WIDE>& info, int piece0, const Shared<D, NT>& sh,
                                       int key0, int keys, bool edge, int g, int q4) {
  constexpr int VW = D / 32;      // words of a value row's part
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < KS; ++j) {
    uint32_t v[4][VW];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = key_of<D>(2 * q4 + (i & 1)) + kSecond<D> * (i >> 1);
      if constexpr (D == 128) {
        const uint4 x = *reinterpret_cast<const uint4*>(slot.piece[piece0 + j] + at_part<D>(key, g));
        v[i][0] = x.x, v[i][1] = x.y, v[i][2] = x.z, v[i][3] = x.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(slot.piece[piece0 + j] + at_part<D>(key, g >> 1) + 8 * (g & 1));
        v[i][0] = x.x, v[i][1] = x.y;
      }
    }
    if (edge) {
      // what lies behind the end is no value; a value that is no number counts only for the rows that see it
      const int first = key0 + 16 * j;
      uint32_t some = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool behind = !info.valid(piece0 + j) || first + key_of<D>(2 * q4 + (i & 1)) + kSecond<D> * (i >> 1) >= keys;
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          if (behind) v[i][w] = 0;
          some |= nan_bytes(v[i][w]);
        }
      }
      if (__any_sync(0xffffffffu, some != 0)) {
        uint32_t bad[4];      // a bit per element of the thread's part of a key's row
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bad[i] = 0;
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            const uint32_t nb = nan_bytes(v[i][w]);
            bad[i] |= ((nb >> 7 & 1) | (nb >> 14 & 2) | (nb >> 21 & 4) | (nb >> 28 & 8)) << (4 * w);
            v[i][w] &= ~((nb >> 7) * 255u);
          }
        }
#pragma unroll 1
        for (int src = 0; src < 4; ++src)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t bits = __shfl_sync(0xffffffffu, bad[i], (lane & ~3) | src);
            const int key = first + key_of<D>(2 * src + (i & 1)) + kSecond<D> * (i >> 1);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int r = 0; r < 2; ++r)
                if (bits && key < sh.limit[8 * n + 2 * q4 + r])
#pragma unroll
                  for (int d = 0; d < D / 16; ++d) {
                    if (bits >> (2 * d) & 1) run.o[d][n][r] = NAN;
                    if (bits >> (2 * d + 1) & 1) run.o[d][n][2 + r] = NAN;
                  }
          }
      }
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      const int w = d / 2;
      const uint32_t sel = d & 1 ? 0x7362 : 0x5140;
      const uint32_t lo = __byte_perm(v[0][w], v[1][w], sel), hi = __byte_perm(v[2][w], v[3][w], sel);
      const uint32_t a0 = e4m3x2_to_f16x2(lo), a1 = e4m3x2_hi_to_f16x2(lo), a2 = e4m3x2_to_f16x2(hi), a3 = e4m3x2_hi_to_f16x2(hi);
#pragma unroll
      for (int n = 0; n < NT; ++n) mma(run.o[d][n], a0, a1, a2, a3, pw[j][n][0], pw[j][n][1]);
    }
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

// Blocks of an SM: by registers (128 to 255 a thread) and 32 or 64 KB of rings.
template <int D, int NT> constexpr int kBlocks = NT == 4 ? 2 : (D == 64 ? 5 : 4) - NT;

// What a block notes about the border behind its run: the item that it is inside of (parts 0: none).
struct Note {
  int parts, first, border;      // parts of the item, block of the first one, place of this border among the item's
  int rows, start, row0, h;      // live rows, and where they belong
  int unused;
};

template <typename T, int D, int NT, bool WIDE>
__global__ void __launch_bounds__(kThreads, kBlocks<D, NT>) paged_attn_kernel(AttnParams p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  constexpr int N = 8 * NT;
  extern __shared__ __align__(1024) unsigned char raw[];      // the swizzle counts lines from multiples of 1024
  Shared<D, NT>& sh = *reinterpret_cast<Shared<D, NT>*>(raw);
  if (threadIdx.x == 0) {
    st::tma_prefetch_desc(&k_map);
    st::tma_prefetch_desc(&v_map);
    for (int i = 0; i < 4 * kWarps; ++i) st::mbar_init(st::smem_u32(&sh.full[0][0][0] + i), 1);
    st::fence_barrier_init();
    sh.abort = 0;
  }
  chain_begin(p.ks, p.vs, p.table, p.starts, p.lengths);
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
  long long all, u0, u1;
  int runs;
  Found f;
  Note* note = reinterpret_cast<Note*>(p.notes) + blockIdx.x;
  if (!find_share<N>(p, sh.sums, &sh.found, all, runs, u0, u1, f)) {
    if (threadIdx.x == 0) note->parts = 0;
    return;
  }
  Seq sq = sequence<N>(p, f.b);
  const uint32_t k_bar = st::smem_u32(&sh.full[warp][0][0]), v_bar = k_bar + 16;
  Slot<D>(&k_ring)[2] = sh.ring[warp][0];
  Slot<D>(&v_ring)[2] = sh.ring[warp][1];
  uint32_t turn = 0;      // steps that the warp has worked on: slot turn % 2 of the rings, for the (turn / 2)-th time

  long long u = u0;
  Item it = item_at<N>(p, u, u1, f, sq), after;
  int keys = min(keys_of(p, it, it.row_end - 1), it.t1 * kTile);      // what the run's part of the item is about, of what its last row sees
  PieceList list = list_pieces(p, it, 0, keys), list_more{-1, 0.0f, 0}, list_after{-1, 0.0f, 0};
  Info<WIDE> info[2];      // of this step and the next one
  int asked = 0, keys_after = 0;
  for (;;) {
    const int steps = it.steps(), key0 = it.t0 * kTile + warp * 32;
    for (; asked < 2 && asked < steps; ++asked) {
      const Info<WIDE> c = info_of<WIDE>(list, asked);
      const uint32_t to = (turn + asked) & 1;
      if (asked == 0) info[0] = c; else info[1] = c;
      copy_keys<D, WIDE>(k_ring[to], k_bar + 8 * to, &k_map, p, c, it.h, key0 + asked * kTile);
      copy_keys<D, WIDE>(v_ring[to], v_bar + 8 * to, &v_map, p, c, it.h, key0 + asked * kTile);
    }
    const bool more = u + steps < u1;
    __syncthreads();      // the item before is done with the queries and the rows' places
    for (int r = warp; r < N; r += kWarps) {
      float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      const int fr = it.row0 + r, i = fr / p.group, head = it.h * p.group + fr - i * p.group;
      const bool live = fr < it.row_end;
      if (live && 4 * lane < D) load4f(q + (it.start + i) * p.q_row + head * p.q_head + 4 * lane, x);
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
        sh.limit[r] = live ? max(it.len - (p.causal ? it.n - 1 - i : 0), 0) : 0x7fffffff;      // rows that are none are not written
        sh.place[r] = (it.start + i) * p.o_row + head * p.o_head;
      }
    }
    if (more) {      // the loads are in flight while this item is worked on
      after = item_at<N>(p, u + steps, u1, f, sq);
      keys_after = min(keys_of(p, after, after.row_end - 1), after.t1 * kTile);
      list_after = list_pieces(p, after, 0, keys_after);
    }
    __syncthreads();
    const int limit_min = sh.limit[0];      // rows come in order
    uint2 qreg[D / 16];
    if constexpr (NT == 1)
#pragma unroll
      for (int k = 0; k < D / 16; ++k) qreg[k] = sh.q[0][k][lane];
    const float freg[2] = {sh.factor[2 * q4], sh.factor[2 * q4 + 1]};
    Running<D, NT> s;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      s.m[n][0] = s.m[n][1] = -INFINITY;
      s.l[n][0] = s.l[n][1] = 0.0f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) s.o[d][n][0] = s.o[d][n][1] = s.o[d][n][2] = s.o[d][n][3] = 0.0f;
    }
    asked = 0;      // of the next item's steps
    if (steps == 1 && more) {
      info[1] = info_of<WIDE>(list_after, 0);
      const uint32_t to = (turn + 1) & 1;
      copy_keys<D, WIDE>(k_ring[to], k_bar + 8 * to, &k_map, p, info[1], after.h, after.t0 * kTile + warp * 32);
      copy_keys<D, WIDE>(v_ring[to], v_bar + 8 * to, &v_map, p, info[1], after.h, after.t0 * kTile + warp * 32);
      asked = 1;
    }
    for (int i = 0; i < steps; ++i) {
      // the step after the next, of this item or of the next one
      const int ahead = i + 2, over = ahead - steps, at = key0 + i * kTile;
      if ((ahead & 15) == 8) list_more = list_pieces(p, it, (ahead & ~15) + 16, keys);
      if ((ahead & 15) == 0) list = list_more;
      Info<WIDE> coming = info[1];
      const bool ask = over < 0 || (more && over < after.steps());
      if (ask) coming = over < 0 ? info_of<WIDE>(list, ahead) : info_of<WIDE>(list_after, over);
      const int ask_h = over < 0 ? it.h : after.h, ask_key = over < 0 ? at + 2 * kTile : after.t0 * kTile + warp * 32 + over * kTile;

      const uint32_t now = turn & 1, phase = turn >> 1 & 1;
      const bool edge = at + 32 > limit_min || !info[0].valid(0) || !info[0].valid(1);
      bool here = st::mbar_wait_warp(k_bar + 8 * now, phase, &sh.abort);
      if constexpr (NT <= 2) {
        float sc[2][NT][4];
        uint32_t pw[2][NT][2];
        const bool any = here && info[0].any();
        if (any) scores<D, NT, 2>(sc, k_ring[now], 0, sh, qreg, g, q4);
        __syncwarp();      // every lane is done with the keys
        if (ask) copy_keys<D, WIDE>(k_ring[now], k_bar + 8 * now, &k_map, p, coming, ask_h, ask_key);
        if (any) weights<D, NT, 2, WIDE>(pw, sc, s, info[0], 0, sh, freg, at, edge, g, q4);
        here = st::mbar_wait_warp(v_bar + 8 * now, phase, &sh.abort) && here;
        if (any && here) values<D, NT, 2, WIDE>(s, pw, v_ring[now], info[0], 0, sh, at, keys, edge, g, q4);
      } else {      // a piece at a time: two do not fit the registers
        here = st::mbar_wait_warp(v_bar + 8 * now, phase, &sh.abort) && here;
#pragma unroll 1
        for (int j = 0; j < 2; ++j) {
          if (!here || !info[0].valid(j)) continue;
          float sc[1][NT][4];
          uint32_t pw[1][NT][2];
          scores<D, NT, 1>(sc, k_ring[now], j, sh, qreg, g, q4);
          weights<D, NT, 1, WIDE>(pw, sc, s, info[0], j, sh, freg, at + 16 * j, edge, g, q4);
          values<D, NT, 1, WIDE>(s, pw, v_ring[now], info[0], j, sh, at + 16 * j, keys, edge, g, q4);
        }
        __syncwarp();
        if (ask) copy_keys<D, WIDE>(k_ring[now], k_bar + 8 * now, &k_map, p, coming, ask_h, ask_key);
      }
      __syncwarp();      // and with the values
      if (ask) {
        copy_keys<D, WIDE>(v_ring[now], v_bar + 8 * now, &v_map, p, coming, ask_h, ask_key);
        if (over >= 0) ++asked;
      }
      if (!here && lane == 0) st::report_error(p.err, st::ERR_MBAR_TIMEOUT, 0x7005);
      ++turn;
      info[0] = info[1];
      info[1] = coming;
    }

    // join the warps: two write their outputs, the others add theirs
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
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = 8 * n + 2 * q4 + r;
        const float mx = fmaxf(fmaxf(sh.m[0][row], sh.m[1][row]), fmaxf(sh.m[2][row], sh.m[3][row]));
        const float a = s.l[n][r] == 0.0f ? 0.0f : st::exp2_ftz(s.m[n][r] - mx);      // 0: saw nothing; a score that is no number leaves a sum that is none
#pragma unroll
        for (int d = 0; d < D / 16; ++d) s.o[d][n][r] *= a, s.o[d][n][2 + r] *= a;
      }
    if (threadIdx.x < N) {
      const int row = threadIdx.x;
      const float mx = fmaxf(fmaxf(sh.m[0][row], sh.m[1][row]), fmaxf(sh.m[2][row], sh.m[3][row]));
      float l = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) l += sh.l[w][row] == 0.0f ? 0.0f : sh.l[w][row] * st::exp2_ftz(sh.m[w][row] - mx);
      sh.mx[row] = mx, sh.sum[row] = l;
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (warp / 2 == half)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float2* to = reinterpret_cast<float2*>(&sh.out[warp & 1][8 * n + 2 * q4 + r][16 * d + 2 * g]);
              float2 x = make_float2(s.o[d][n][r], s.o[d][n][2 + r]);
              if (half == 1) x.x += to->x, x.y += to->y;
              *to = x;
            }
      __syncthreads();
    }
    const int rows = it.row_end - it.row0;
    const bool whole = it.t0 == 0 && it.t1 == it.tiles;
    float* part = whole ? nullptr : part_of<D, NT>(p, 2LL * blockIdx.x + (it.t0 == 0 ? 1 : 0));
    for (int i = threadIdx.x; i < rows * (D / 2); i += kThreads) {
      const int row = i / (D / 2), d = i % (D / 2) * 2, from = out_at<D>(d);
      const float2 x = *reinterpret_cast<const float2*>(&sh.out[0][row][from]), y = *reinterpret_cast<const float2*>(&sh.out[1][row][from]);
      const float l = sh.sum[row];
      if (whole) {
        T* o = out + sh.place[row] + d;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        o[0] = from_f<T>((x.x + y.x) * inv), o[1] = from_f<T>((x.y + y.y) * inv);
        if (d == 0 && p.lse != nullptr) {
          const int fr = it.row0 + row;
          p.lse[(it.start + fr / p.group) * static_cast<long long>(p.heads) + it.h * p.group + fr % p.group] = l == 0.0f ? -INFINITY : (sh.mx[row] + log2f(l)) / kLog2e;
        }
      } else {
        *reinterpret_cast<float2*>(part + row * D + d) = make_float2(x.x + y.x, x.y + y.y);
        if (d == 0) part[N * D + row] = sh.mx[row], part[N * D + N + row] = l;
      }
    }
    u += steps;
    if (!more) break;
    it = after, keys = keys_after, list = list_after;
  }
  if (threadIdx.x == 0) {
    Note n{};
    if (it.t1 < it.tiles) {
      // block b holds a part if its run begins before the item's end, all * b / runs < end, which is all * b < end * runs, and ends behind its first unit
      const long long first_unit = u1 - it.t1, end = first_unit + it.tiles;
      n.first = static_cast<int>(((first_unit + 1) * runs - 1) / all);
      n.parts = static_cast<int>((end * runs - 1) / all) - n.first + 1;
      n.border = static_cast<int>(blockIdx.x) - n.first;
      n.rows = it.row_end - it.row0, n.start = it.start, n.row0 = it.row0, n.h = it.h;
    }
    *note = n;
  }
}

// Joins the parts of the items that several blocks worked on.  A block per border; an item of P parts has P - 1 of them, which share its rows.
// With few parts a warp does a row; with many, the block's warps share the parts of a row.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads) paged_join_kernel(AttnParams p) {
  constexpr int N = 8 * NT, E = D / 32;
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
  const int members = few ? kWarps : 1, me = few ? warp : 0, width = few ? 32 : kThreads, at = few ? lane : threadIdx.x;
  for (int r = n.border * members + me; r < n.rows; r += (n.parts - 1) * members) {      // few: warps go their own ways, without barriers
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
    if (at == 0 && p.lse != nullptr) p.lse[row * p.heads + head] = l == 0.0f ? -INFINITY : (m + log2f(l)) / kLog2e;
  }
}

// Row tiles of 8 by the rows that the longest step of a sequence has.
int row_tiles(long long max_queries, int group) {
  const long long rows = max_queries * group;
  return rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
}
int runs_of(int nt, int dim) {
  return st::sm_count() * (dim == 64 ? nt == 1 ? kBlocks<64, 1> : nt == 2 ? kBlocks<64, 2> : kBlocks<64, 4> : nt == 1 ? kBlocks<128, 1> : nt == 2 ? kBlocks<128, 2> : kBlocks<128, 4>);
}

template <typename T, int D, int NT, bool WIDE>
int launch(const AttnParams& p, cudaStream_t stream) {
  const int runs = runs_of(NT, D);
  constexpr int smem = sizeof(Shared<D, NT>);
  CUtensorMap maps[2];
  const uint64_t dims[2] = {128, (static_cast<uint64_t>(p.pages) * p.kv_heads << p.shift) * D / 128}, strides[1] = {128};
  const uint32_t box[2] = {128, (WIDE ? 32u : 16u) * D / 128};
  for (int i = 0; i < 2; ++i)
    if (!st::encode_tmap(&maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, i == 0 ? p.kc : p.vc, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return ST_ERR_CUDA;
  auto kernel = paged_attn_kernel<T, D, NT, WIDE>;
  static bool opted[st::kMaxDevices];
  if (bool& done = opted[st::current_device()]; !done) {
    ST_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    done = true;
  }
  // in order: blocks that come early pile up on the SMs that fall free first (64 sequences: 98 us a pass against 80)
  cudaError_t e = st::in_order(kernel, dim3(runs), dim3(kThreads), smem, stream)(p, maps[0], maps[1]);
  if (e != cudaSuccess) return st::fail_cuda(e, "paged attention");
  e = st::chained(paged_join_kernel<T, D, NT>, dim3(runs - 1), dim3(kThreads), runs * sizeof(float), stream)(p);
  if (e != cudaSuccess) return st::fail_cuda(e, "paged attention: join");
  return ST_OK;
}
template <typename T, int D>
int dispatch(const AttnParams& p, int nt, cudaStream_t stream) {
  if (p.shift >= 5) return nt == 1 ? launch<T, D, 1, true>(p, stream) : nt == 2 ? launch<T, D, 2, true>(p, stream) : launch<T, D, 4, true>(p, stream);
  return nt == 1 ? launch<T, D, 1, false>(p, stream) : nt == 2 ? launch<T, D, 2, false>(p, stream) : launch<T, D, 4, false>(p, stream);
}
}  // namespace

// Floats of workspace that st_paged_attention takes.
ST_API long long st_paged_attention_workspace(int max_queries, int heads, int kv_heads, int dim) {
  if (kv_heads < 1 || heads < kv_heads) return 0;
  const int nt = row_tiles(max_queries, heads / kv_heads);
  return (2LL * 8 * nt * (dim + 2) + sizeof(Note) / sizeof(float)) * runs_of(nt, dim);
}

// q, out [rows, heads, dim] (dim contiguous, strides in elements): row starts[b] + i is the i-th of the newest tokens of sequence b, whose keys and values,
// these tokens' included, are the first lengths[b] of the pages in table[b].  lse [rows, heads] or null.  max_queries: the most rows of a sequence, by which
// the row tile is chosen; more are computed too.  zero_tail: rows behind the last sequence become 0 (else they stay as they were).  type: 0 bf16, 1 fp16.
ST_API int st_paged_attention(const void* q, const void* k_codes, const void* v_codes, const float* k_scale, const float* v_scale, const int* table, const int* starts,
                              const int* lengths, void* out, float* lse, float* workspace, long long q_row, long long q_head, long long o_row, long long o_head,
                              long long table_row, long long pages, long long rows, int width, int page_size, int B, int heads, int kv_heads, int dim, int max_queries, float scale,
                              int causal, int zero_tail, int type, void* stream_v) {
  const int shift = st::page_shift(page_size);
  if (shift < 0 || B < 0 || rows < 0 || rows > 2147483647LL || width < 0 || (static_cast<long long>(width) << shift) > 2147480000LL || kv_heads < 1 || heads < kv_heads ||
      heads % kv_heads || (dim != 64 && dim != 128) || pages < 1 || (pages * kv_heads << shift) > 2147483647LL || max_queries < 1 || (type != 0 && type != 1) || rows * (heads / kv_heads) > 2147483647LL)
    return st::fail(ST_ERR_INVALID, "paged attention: sizes out of range (page 16 to 256, dim 64 or 128, heads a multiple of kv_heads, 1 to 2^31 - 1 tokens times kv_heads)");
  if ((reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return st::fail(ST_ERR_INVALID, "paged attention: codes must be 16-byte aligned");
  if (rows == 0) return ST_OK;
  const int nt = row_tiles(max_queries, heads / kv_heads);
  int* notes = reinterpret_cast<int*>(workspace + 2LL * 8 * nt * (dim + 2) * runs_of(nt, dim));      // behind the parts
  const AttnParams p{q, static_cast<const unsigned char*>(k_codes), static_cast<const unsigned char*>(v_codes), k_scale, v_scale, table, starts, lengths, out, lse, workspace, notes,
                     q_row, q_head, o_row, o_head, table_row, pages, rows, width, shift, B, heads, kv_heads, heads / kv_heads, scale, causal, zero_tail, st::error_word()};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  if (type == 0) return dim == 64 ? dispatch<__nv_bfloat16, 64>(p, nt, stream) : dispatch<__nv_bfloat16, 128>(p, nt, stream);
  return dim == 64 ? dispatch<__half, 64>(p, nt, stream) : dispatch<__half, 128>(p, nt, stream);
}
