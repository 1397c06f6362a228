// Attention of the newest tokens of every sequence over an 8-bit paged cache (decoding, checking drafted tokens, parts of prompts).
//
//   s = scale * q . k * 2^a,  p = softmax(s) over the visible keys,  o = sum p v * 2^b      (a, b: exponents of the page's scales)
//
// What bounds it: a key is 2 * D bytes and 4 * D operations per query row, so for the rows of one decoding step (the query
// heads of one key head) it is bound by reading the cache once.
//
// Work.  The rows of a sequence that share a key head are its n tokens times the G query heads of the group; R = 8, 16 or 32 of them
// are an item together with one (sequence, key head), and 128 keys of an item are a unit.  All units of the call are numbered through and
// every block takes an equal run of them, whatever the lengths are: the split needs nothing from the host but the shapes, so a captured
// launch stays right while the sequences grow, and one long sequence fills the chip as well as many short ones.  Each block finds its run
// by a prefix sum over the sequences.  An item counts some units more than it has, for what its beginning and end cost a block: without
// them blocks in short sequences took up to a third longer than those in long ones.  Where a run ends inside an item, the block leaves (maximum, sum, output) in the workspace,
// and a second kernel joins the parts of such items in their order, so results do not depend on timing.  It finds them by the notes
// that the blocks leave about the border between their run and the next.
//
// Where the table holds few units for a sequence, an item is not split: nothing has to be joined then, and a block is through with it in the time
// that the second kernel takes.
//
// Products.  Both run on tcgen05 with the codes as they lie in the cache: no code is ever converted or passes through a register.  A unit's keys
// are the 128 rows of S^T = K Q^T (keys in lanes, so a thread has all rows' scores of its key), its values, read along the tokens,
// those of O^T = V^T P^T.  The other operands, queries and weights, are fp16 numbers written as sums of e5m2 numbers, whose three
// significant bits are those of fp16's upper byte: the byte, the byte of what it leaves, and so on; three hold bf16's 8 bits, four fp16's
// 11.  The parts stand side by side in N; those of a score are added by its thread, those of an output when the item is done.  So the products are exact
// and a unit costs a warp about 150 instructions; with mma.sync on codes converted in registers it was 650 (64 sequences: 87 us against 71).
// Queries are scaled by a power of two per row to use fp16's range.  The softmax runs over x + b instead of x (b: the page's value
// exponent): the weights exp2(x + b - M) are those that multiply the codes, and the sum takes exp2(-b) back out.  M is not the running
// maximum but some number that no x + b exceeds by more than 6: it moves, and the outputs with it, in the first unit and rarely after, and the
// weights, times 2^9, stay below 2^15.  What lies 2^126 below is flushed: with value scales of one sequence up to 2^98 apart that takes no weight
// above 2^-28 of the largest (scales further apart: values of 10^14 next to pages of zeros).
//
// Blocks: four warps for the softmax, one that copies keys (a tiled copy per page and unit) and issues scores, one that copies values, one that
// issues the products with them, one that prepares the queries of the next item, so that a run's items follow one another without a pause: with that in the
// softmax warps' way an item cost them 4500 cycles more.  Heads of 64: the copies lay two tokens side by side, 64 rows of 128, and the weights of
// even and odd tokens have columns of their own; half of each product is not used.
//
// Measured (device time in a graph, 128-wide heads if not said): 64 sequences of up to 8192 tokens, 32 heads over 8, 67 us, 5.5 TB/s of the 6.5 that a copy
// reaches; two of up to 131001, 32 over 4, 39 us, 4.4 TB/s, of which the parts' way through the workspace and the joining take about 8; one of 777, 16 heads, 12 us: seven
// units one after the other behind a beginning of 5000 cycles, most of it spent on instructions that have to be fetched; 12 sequences of 5 drafted tokens
// behind up to 2049, 12 heads of 64, fp16, 19 us.
#include "paged_prompt.cuh"

namespace {
// Warps of the softmax: with 32 rows twice as many, each of which has half of the rows (4 sequences of 256 tokens: 118 us with four warps, 86 with eight);
// then come one that copies keys and issues scores, one that issues the products with values, one that prepares queries, one that copies values.
template <int R> constexpr int kSoftWarps = R == 32 ? 8 : 4;
static_assert(kThreadsOf<8> == 32 * (kSoftWarps<8> + 4) && kThreadsOf<32> == 32 * (kSoftWarps<32> + 4));
constexpr int kParts = 4;             // e5m2 numbers of a weight

__device__ __forceinline__ void umma_codes(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n"
      ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// A is e4m3 (0), B e5m2 (1), the sums fp32.
constexpr uint32_t codes_idesc(int M, int N, bool mn_major) {
  return (1u << 4) | (0u << 7) | (1u << 10) | (static_cast<uint32_t>(mn_major) << 15) | (static_cast<uint32_t>(mn_major) << 16) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}
// Descriptor of a tile whose rows are WIDTH bytes, swizzled over that width: rows of K-major operands, or the K of MN-major ones; 8 rows are a group.
// `block`: distance of the next WIDTH bytes along M or N.
template <int WIDTH>
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, uint32_t block = 16) {
  static_assert(WIDTH == 32 || WIDTH == 64 || WIDTH == 128);
  constexpr uint64_t kind = WIDTH == 128 ? 2 : WIDTH == 64 ? 4 : 6;
  return ((addr & 0x3FFFF) >> 4) | static_cast<uint64_t>(block >> 4) << 16 | static_cast<uint64_t>(8 * WIDTH >> 4) << 32 | 1ull << 46 | kind << 61;
}
// Byte of 16-byte part `part` of row `row` in such a tile.
template <int WIDTH>
__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t part) {
  constexpr uint32_t mask = WIDTH / 16 - 1;
  return row * WIDTH + ((part ^ (row * WIDTH >> 7 & mask)) << 4);
}
__device__ __forceinline__ void tmem_ld_8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st_8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// Splits off the upper bytes, e5m2 numbers, of eight fp16 numbers: returns them side by side, and leaves the rest (exactly).
__device__ __forceinline__ uint2 split_off(__half2 (&x)[4]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u[i] = *reinterpret_cast<const uint32_t*>(&x[i]);
    const uint32_t high = u[i] & 0xff00ff00u;
    x[i] = __hsub2(x[i], *reinterpret_cast<const __half2*>(&high));
  }
  return make_uint2(__byte_perm(u[0], u[1], 0x7531), __byte_perm(u[2], u[3], 0x7531));
}

// e5m2 numbers of a query element: bf16 has 8 bits, fp16 11.
template <typename T> constexpr int kQueryParts = 3;
template <> constexpr int kQueryParts<__half> = 4;

template <int D, int R, int QP>
struct Layout {
  // Parts of the queries that stand side by side in N; with 32 rows two, as tensor memory has no room for more, and the others follow in the sum.
  // (One product of N = 16 takes 90 cycles before the next can add to it: with all 12 of a unit in a row it took a block 1900 cycles.)
  static constexpr int WAYS = R == 32 ? 2 : QP, SETS = (QP + WAYS - 1) / WAYS;
  static constexpr int S_N = (WAYS * R + 15) / 16 * 16;                // columns of the scores
  static constexpr int SIDES = D == 64 ? 2 : 1;                        // tokens side by side
  static constexpr int P_N = SIDES * kParts * R;                       // columns of the products with values
  static constexpr int P_WIDTH = P_N < 128 ? P_N : 128;                // bytes of a swizzled row of weights
  static constexpr int P_ROWS = kTile / SIDES;
  static constexpr int P_BYTES = P_ROWS * P_N;
  static constexpr int COLUMNS = 2 * S_N + P_N <= 64 ? 64 : 2 * S_N + P_N <= 128 ? 128 : 2 * S_N + P_N <= 256 ? 256 : 512;
  static constexpr int BLOCKS = COLUMNS == 512 ? 1 : 2;                // of an SM
  static constexpr int Q_BYTES = QP * R * D;
  // What fits the shared memory of two blocks (111 KB each, 2 KB of them for the small things): queries twice before a third stage of values, that
  // before weights twice, and a third one of keys last.
  static constexpr int ROOM = (BLOCKS == 2 ? 113 * 1024 : 226 * 1024) - 3 * 1024, ONE = kTile * D;
  static constexpr int Q_BUFS = (D == 64 ? 4 : 2) * 2 * ONE + P_BYTES + 2 * Q_BYTES <= ROOM ? 2 : 1;
  static constexpr int P_BUFS = (D == 64 ? 4 : 2) * 2 * ONE + 2 * P_BYTES + Q_BUFS * Q_BYTES <= ROOM ? 2 : 1;
  static constexpr int V_STAGES = D == 64 ? 4 : 5 * ONE + P_BUFS * P_BYTES + Q_BUFS * Q_BYTES <= ROOM ? 3 : 2;
  static constexpr int K_STAGES = D == 64 ? 4 : (3 + V_STAGES) * ONE + P_BUFS * P_BYTES + Q_BUFS * Q_BYTES <= ROOM ? 3 : 2;
};

// An item as the query warp hands it over.
template <int D, int R>
struct alignas(16) Rows {
  Item item;
  alignas(16) float factor[R];
  alignas(16) int limit[R];
  long long place[R];
};

template <int D, int R, int QP>
struct Shared {
  using L = Layout<D, R, QP>;
  unsigned char k[L::K_STAGES][kTile * D], v[L::V_STAGES][kTile * D];
  unsigned char p[L::P_BUFS][L::P_BYTES];
  unsigned char q[L::Q_BUFS][QP][R * D];
  // s_full: the scores of a stage's keys are there, which are not read any more; pv_done: the same for values
  unsigned long long k_full[L::K_STAGES], s_full[L::K_STAGES], v_full[L::V_STAGES], pv_done[L::V_STAGES], p_full[2], q_full[L::Q_BUFS], q_empty[L::Q_BUFS];
  float ks[L::V_STAGES][8];      // of the unit's pages
  int ve[L::V_STAGES][8];        // kInvalid: no such page
  Rows<D, R> rows[L::Q_BUFS];
  float m[4][R], sum[R];       // largest x of each warp's keys, less 9
  alignas(16) float ref[2][R == 32 ? R : 1];
  uint32_t bad[R][D / 32];     // outputs that a value which is no number reaches though not all rows see it
  int sums[kMaxWarps];
  Found found;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(Shared<128, 8, 3>) <= 113 * 1024 && sizeof(Shared<128, 16, 3>) <= 113 * 1024 && sizeof(Shared<128, 32, 3>) <= 113 * 1024 && sizeof(Shared<128, 8, 4>) <= 113 * 1024 &&
              sizeof(Shared<128, 16, 4>) <= 113 * 1024 && sizeof(Shared<128, 32, 4>) <= 113 * 1024 && sizeof(Shared<64, 16, 4>) <= 113 * 1024 && sizeof(Shared<64, 32, 4>) <= 226 * 1024);

// ---- copies -------------------------------------------------------------------------------------------------------------------------
// The run's units one after another, for keys or for values.  Page numbers and scales are looked up for 32 pages at a time (4 units of 8 pages
// of 16 tokens to 32 units of one page), a batch ahead of the copies: two loads that wait for one another, 1400 cycles, at every unit set the
// pace before.  A copy takes its warp about 110 cycles, so keys and values have warps of their own.
template <typename L, int D, int R, bool VALUES, typename S>
struct Copier {
  static constexpr int ST = VALUES ? L::V_STAGES : L::K_STAGES;
  struct Batch {
    int t, n, h;      // units [t, t + n) of an item (n 0: the end), its key head
    int page;         // the lane's: page lane % pages of unit lane / pages; -1: none
    float ks;
    int ve;
  };
  S& sh;
  const AttnParams& p;
  const CUtensorMap* map;
  int u, u1, t = 0, end = 0;      // behind the next batch
  Found f;
  Seq sq;
  Item it;
  int lane, rows, pages, mine, at_page, i = 0;
  uint32_t turn = 0;
  Batch now, next;

  __device__ __forceinline__ Copier(S& sh_, const AttnParams& p_, const CUtensorMap* map_, int u0, int u1_, Found f_, const Seq& sq_)
      : sh(sh_), p(p_), map(map_), u(u0), u1(u1_), f(f_), sq(sq_), lane(threadIdx.x & 31), rows(min(1 << p.shift, kTile)), pages(kTile / rows), mine(lane / pages), at_page(lane % pages) {
    now = look_pages();
    look_scales(now);
    next = look_pages();
  }
  __device__ __forceinline__ Batch look_pages() {
    Batch b{0, 0, 0, -1, 0.0f, kInvalid};
    if (t >= end) {
      if (!item_at<R>(it, p, u, u1, f, sq)) return b;
      u = it.next, t = it.t0, end = it.t0 + it.steps();
    }
    b.t = t, b.n = min(32 / pages, end - t), b.h = it.h;
    const int key = (t + mine) * kTile + at_page * rows;
    if (mine < b.n && key < it.keys) b.page = it.table[key >> p.shift];
    else b.page = kBehind;
    t += b.n;
    return b;
  }
  __device__ __forceinline__ void look_scales(Batch& b) {
    if (b.page < 0 || b.page >= p.pages) {
      if (VALUES && b.n > 0 && b.page != kBehind) st::report_error(p.err, st::ERR_BOUNDS, 0x7004);
      b.page = -1;
      return;
    }
    if (!VALUES) return;
    const long long at = static_cast<long long>(b.page) * p.kv_heads + b.h;
    b.ks = p.ks[at], b.ve = st::scale_exponent(p.vs[at]);
  }
  // The next unit into its stage, once that is free; false: there is none, or a wait ran out.
  __device__ __forceinline__ bool copy() {
    if (now.n == 0) return false;
    const int slot = turn % ST;
    const bool live = mine == i && now.page >= 0;
    const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, live)) * rows * D;
    const long long token = (((static_cast<long long>(now.page) * p.kv_heads + now.h) << p.shift)) + (((now.t + i) * kTile + at_page * rows) & ((1 << p.shift) - 1));
    const uint32_t full = st::smem_u32(VALUES ? &sh.v_full[slot] : &sh.k_full[slot]);
    if (!st::mbar_wait_warp(st::smem_u32(VALUES ? &sh.pv_done[slot] : &sh.s_full[slot]), (turn / ST & 1) ^ 1, &sh.abort)) return false;
    if (live) st::tma_load_2d(st::smem_u32(VALUES ? sh.v[slot] : sh.k[slot]) + at_page * rows * D, map, full, 0, static_cast<int>(VALUES ? token * D / 128 : token));
    if (VALUES && mine == i) sh.ks[slot][at_page] = now.ks, sh.ve[slot][at_page] = now.ve;      // the scales may still be on their way
    __syncwarp();
    if (lane == 0) st::mbar_arrive_expect_tx(full, bytes);      // what has come before counts
    ++turn;
    if (++i == 1) look_scales(next);      // the page numbers have come by now
    if (i == now.n) {
      now = next, i = 0;
      next = look_pages();
    }
    return true;
  }
};

// ---- products -----------------------------------------------------------------------------------------------------------------------
// N is a multiple of 16: three parts of 8 rows are followed by 8 columns that nobody reads, from whatever lies behind them.  Each of the two products has
// a warp of its own: an instruction or a wait takes the issuing lane 70 to 130 cycles, a unit's scores 600, its outputs 700.

// The number of an item's units, 0 behind the last one, once its queries are there; -1: a wait ran out.
template <typename L, typename S>
__device__ __forceinline__ int steps_of(S& sh, uint32_t item) {
  if (!st::mbar_wait_warp(st::smem_u32(&sh.q_full[item % L::Q_BUFS]), item / L::Q_BUFS & 1, &sh.abort)) return -1;
  const Item& it = sh.rows[item % L::Q_BUFS].item;
  return it.t1 > it.t0 ? it.steps() : 0;
}

// Copies keys and issues scores, two units ahead of the softmax at most.  Returns the units that it copied and those whose scores it issued.
template <typename L, int D, int R, int QP, typename S>
__device__ __forceinline__ uint2 score_warp(S& sh, const AttnParams& p, const CUtensorMap* map, uint32_t tmem_, int u0, int u1, Found f, const Seq& sq) {
  Copier<L, D, R, false, S> keys(sh, p, map, u0, u1, f, sq);
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_, 0);
  const bool leader = st::elect_one();
#pragma unroll 1
  for (int i = 0; i < L::K_STAGES; ++i) keys.copy();
  uint32_t turn = 0;
  for (uint32_t item = 0;; ++item) {
    const int steps = steps_of<L>(sh, item);
    if (steps <= 0) return make_uint2(keys.turn, turn);
    const bool more = sh.rows[item % L::Q_BUFS].item.next < u1;
#pragma unroll 1
    for (int i = 0; i < steps; ++i, ++turn) {
      const int slot = turn % L::K_STAGES;
      if (!st::mbar_wait_warp(st::smem_u32(&sh.k_full[slot]), turn / L::K_STAGES & 1, &sh.abort)) return make_uint2(keys.turn, turn);
      // the columns are free again once the softmax has written the weights of the unit before last
      if (turn > 1 && !st::mbar_wait_warp(st::smem_u32(&sh.p_full[turn & 1]), (turn - 2) >> 1 & 1, &sh.abort)) return make_uint2(keys.turn, turn);
      st::tc_fence_after();
      if (leader) {
        const uint64_t a = tile_desc<D>(st::smem_u32(sh.k[slot]));
#pragma unroll
        for (int j = 0; j < L::SETS; ++j) {
          const int ways = min(L::WAYS, QP - j * L::WAYS);
          const uint64_t b = tile_desc<D>(st::smem_u32(sh.q[item % L::Q_BUFS][j * L::WAYS]));
#pragma unroll
          for (int k = 0; k < D / 32; ++k) umma_codes(tmem + (turn & 1) * L::S_N, a + 2 * k, b + 2 * k, codes_idesc(128, (ways * R + 15) / 16 * 16, false), j + k > 0);
        }
        st::umma_commit(st::smem_u32(&sh.s_full[slot]));
      }
      __syncwarp();
      if (turn > 0) keys.copy();      // into the stage of the unit before, whose scores are there by now
    }
    if (!more) return make_uint2(keys.turn, turn);
  }
}

// Issues the products with values; returns of how many units.
template <typename L, int D, int R, typename S>
__device__ __forceinline__ uint32_t value_warp(S& sh, uint32_t tmem_, int u1) {
  constexpr uint32_t idesc = codes_idesc(128, L::P_N, true);
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_, 0);
  const bool leader = st::elect_one();
  uint32_t turn = 0;
  for (uint32_t item = 0;; ++item) {
    const int steps = steps_of<L>(sh, item);
    if (steps <= 0) return turn;
    const bool more = sh.rows[item % L::Q_BUFS].item.next < u1;
#pragma unroll 1
    for (int i = 0; i < steps; ++i, ++turn) {
      const int slot = turn % L::V_STAGES;
      if (!st::mbar_wait_warp(st::smem_u32(&sh.v_full[slot]), turn / L::V_STAGES & 1, &sh.abort)) return turn;
      if (!st::mbar_wait_warp(st::smem_u32(&sh.p_full[turn & 1]), turn >> 1 & 1, &sh.abort)) return turn;
      st::tc_fence_after();
      if (leader) {
        // 32 rows of K (tokens, or pairs of them) at a time: 4 groups of 8
        const uint64_t a = tile_desc<128>(st::smem_u32(sh.v[slot])), b = tile_desc<L::P_WIDTH>(st::smem_u32(sh.p[turn % L::P_BUFS]), L::P_ROWS * L::P_WIDTH);
#pragma unroll
        for (int k = 0; k < L::P_ROWS / 32; ++k) umma_codes(tmem + 2 * L::S_N, a + k * (32 * 128 >> 4), b + k * (32 * L::P_WIDTH >> 4), idesc, i + k > 0);
        st::umma_commit(st::smem_u32(&sh.pv_done[slot]));
      }
      __syncwarp();
    }
    if (!more) return turn;
  }
}

// ---- the warp that prepares queries -------------------------------------------------------------------------------------------------
template <typename T, typename L, int D, int R, int QP, typename S>
__device__ __forceinline__ void query_warp(S& sh, const AttnParams& p, int u0, int u1, Found f, Seq sq) {
  const int lane = threadIdx.x & 31;
  const T* q = static_cast<const T*>(p.q);
  const bool wide = ((p.q_row | p.q_head) & 7) == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
  uint32_t item = 0;
  Item it;
  for (int u = u0; u < u1; ++item) {
    if (!item_at<R>(it, p, u, u1, f, sq)) {      // the last word: no more items; no rows either, so nothing is read
      it = Item{};
      it.next = u1;
    }
    u = it.next;
    const int buf = item % L::Q_BUFS;
    if (!st::mbar_wait_warp(st::smem_u32(&sh.q_empty[buf]), (item / L::Q_BUFS & 1) ^ 1, &sh.abort)) return;
    Rows<D, R>& to = sh.rows[buf];
    if (lane == 0) to.item = it;
    // four lanes to a row, a quarter of it each; loops as they are, as code that runs once per item costs its way into the instruction cache
#pragma unroll 1
    for (int r = lane / 4; r < R; r += 8) {
      constexpr int VECS = D / 32;      // 8 elements each
      const int fr = it.row0 + r, i = fr / p.group, head = it.h * p.group + fr - i * p.group;
      const bool live = fr < it.row_end;
      const T* from = q + (it.start + i) * p.q_row + head * p.q_head + (lane & 3) * (D / 4);
      uint4 raw[VECS];
#pragma unroll
      for (int k = 0; k < VECS; ++k) raw[k] = live ? load8(from + 8 * k, wide) : make_uint4(0, 0, 0, 0);
      float top = 0.0f;
#pragma unroll
      for (int k = 0; k < VECS; ++k) {
        const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 x = two_floats<T>(w[j]);
          top = st::max3(top, fabsf(x.x), fabsf(x.y));
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the largest to [2^14, 2^15): exact down to 2^-14 of e5m2, 2^-28 of the largest; a row with infinities gives NaN
      int e = static_cast<int>((__float_as_uint(top) >> 23) & 255) - 127 - 14;
      e = top < INFINITY ? max(e, -100) : 0;
      const float mul = top < INFINITY ? st::exp2_int(-e) : NAN;
#pragma unroll
      for (int k = 0; k < VECS; ++k) {
        const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
        __half2 h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 x = two_floats<T>(w[j]);
          h[j] = __floats2half2_rn(x.x * mul, x.y * mul);
        }
        const int d = (lane & 3) * (D / 4) + 8 * k;
#pragma unroll
        for (int j = 0; j < QP; ++j) *reinterpret_cast<uint2*>(sh.q[buf][j] + swizzled<D>(r, d / 16) + d % 16) = split_off(h);
      }
      if ((lane & 3) == 0) {
        to.factor[r] = p.scale * kLog2e * st::exp2_int(e);
        to.limit[r] = live ? max(it.len - (p.causal ? it.n - 1 - i : 0), 0) : 0x7fffffff;      // rows that are none are not written
        to.place[r] = (it.start + i) * p.o_row + head * p.o_head;
      }
    }
    st::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) st::mbar_arrive(st::smem_u32(&sh.q_full[buf]));
  }
}

// ---- the softmax -------------------------------------------------------------------------------------------------------------------
// The largest over a warp; NaN counts only where all are.
__device__ __forceinline__ float warp_top(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// COLUMNS of this warp's lanes.
template <int COLUMNS>
__device__ __forceinline__ void tmem_ld_columns(uint32_t taddr, uint32_t (&r)[COLUMNS]) {
  if constexpr (COLUMNS == 8) tmem_ld_8(taddr, r);
  else if constexpr (COLUMNS == 16) st::tmem_ld_32x16(taddr, r);
  else st::tmem_ld_32x32(taddr, r);
}

// Keys that not all rows see, in a unit's values: what lies behind the end becomes 0; a value that is no number becomes 0 too, and the
// outputs of the rows that see it are noted.  One key a thread.
template <int D, int R, typename S>
__device__ __forceinline__ void clean_values(S& sh, const Rows<D, R>& of, int slot, int key, bool there, int limit_min) {
  constexpr int SIDES = D == 64 ? 2 : 1, PARTS = D / 16;
  const int t = threadIdx.x & 127, line = t / SIDES, side = t % SIDES * PARTS;
  if (!there) {
#pragma unroll
    for (int c = 0; c < PARTS; ++c) *reinterpret_cast<uint4*>(sh.v[slot] + swizzled<128>(line, side + c)) = make_uint4(0, 0, 0, 0);
    return;
  }
  if (key < limit_min) return;      // all rows see it
#pragma unroll 1
  for (int c = 0; c < PARTS; ++c) {
    uint4* at = reinterpret_cast<uint4*>(sh.v[slot] + swizzled<128>(line, side + c));
    const uint4 x = *at;
    uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t nb = nan_bytes(w[i]);
      bits |= ((nb >> 7 & 1) | (nb >> 14 & 2) | (nb >> 21 & 4) | (nb >> 28 & 8)) << (4 * i);
      w[i] &= ~((nb >> 7) * 255u);
    }
    if (bits == 0) continue;
    for (int r = 0; r < R; ++r)
      if (key < of.limit[r]) atomicOr(&sh.bad[r][c / 2], bits << (16 * (c & 1)));
    *at = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <typename T, typename L, int D, int R, typename S>
__device__ __forceinline__ void soft_warps(S& sh, const AttnParams& p, uint32_t tmem_all, Note* note, int u1, int runs, int all) {
  // a thread has RT rows from `low` on of one key
  constexpr int SOFT = 32 * kSoftWarps<R>, RT = R * 128 / SOFT;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5 & 3, t = threadIdx.x & 127, half = threadIdx.x >> 7, low = half * RT;
  const uint32_t tmem = tmem_all + (warp << 21);                                                          // the warp's 32 lanes
  const uint32_t o_cols = tmem + 2 * L::S_N + (D == 64 && warp >= 2 ? kParts * R : 0);                      // lanes 64..127 of heads of 64: the odd tokens'
  const int page_at = t >> min(p.shift, 7);
  T* out = static_cast<T*>(p.out);
  // A wait that runs out sets the abort flag, and all later ones return at once: the warps finish the item together and stop at the next one.
  uint32_t turn = 0, item = 0;
  // The rows' references are the same for all keys: registers, or with 32 rows, which leave none, shared memory, the old ones and the new ones.
  constexpr bool kShared = R == 32;
  int flip = 0;
  for (int i = threadIdx.x; i < R * (D / 32); i += SOFT) sh.bad[i / (D / 32)][i % (D / 32)] = 0;
  for (;; ++item) {
    const Rows<D, R>& of = sh.rows[item % L::Q_BUFS];
    if (kShared && threadIdx.x < R) sh.ref[flip][threadIdx.x] = kNoMax;
    if (soft_any<SOFT>(!st::mbar_wait_warp(st::smem_u32(&sh.q_full[item % L::Q_BUFS]), item / L::Q_BUFS & 1, &sh.abort))) return;
    if (of.item.t1 <= of.item.t0) return;      // no more items
    const int steps = of.item.steps(), t0 = of.item.t0, keys = of.item.keys, next = of.item.next;
    const int limit_min = of.limit[0];      // rows come in order
    float own_ref[kShared ? 1 : RT]{}, l[RT];
    auto ref = [&](int r) { return kShared ? sh.ref[flip][low + r] : own_ref[kShared ? 0 : r]; };      // M - 9
    bool unseen = false;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      if (!kShared) own_ref[kShared ? 0 : r] = kNoMax;
      l[r] = 0.0f;
    }

    for (int i = 0; i < steps; ++i, ++turn) {
      const int slot = turn % L::V_STAGES, key = (t0 + i) * kTile + t;
      st::mbar_wait_warp(st::smem_u32(&sh.v_full[slot]), turn / L::V_STAGES & 1, &sh.abort);
      const float ks = sh.ks[slot][page_at];
      const int ve_or_not = sh.ve[slot][page_at];
      const bool there = ve_or_not != kInvalid && key < keys;
      const int ve = there ? ve_or_not : 0;
      const bool gone = (t0 + i + 1) * kTile > limit_min || !there;      // of this unit's keys some row may not see this one
      st::mbar_wait_warp(st::smem_u32(&sh.s_full[turn % L::K_STAGES]), turn / L::K_STAGES & 1, &sh.abort);
      st::tc_fence_after();
      uint32_t raw[L::WAYS][RT];
#pragma unroll
      for (int w = 0; w < L::WAYS; ++w) tmem_ld_columns<RT>(tmem + (turn & 1) * L::S_N + w * R + low, raw[w]);
      st::tmem_ld_wait();
      float x[RT];
      const float lift = static_cast<float>(ve);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float sum = __uint_as_float(raw[L::WAYS - 1][r]);      // the smallest first
#pragma unroll
        for (int w = L::WAYS - 2; w >= 0; --w) sum += __uint_as_float(raw[w][r]);
        x[r] = fmaf(sum, of.factor[low + r] * ks, lift);
      }
      if (gone) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
          if (!there || key >= of.limit[low + r]) x[r] = -INFINITY;
      }
      // the reference moves where a weight would be too large; the first unit sets it, or a later one for a row that saw nothing before
      const bool fresh = i == 0 || unseen;
      bool move = fresh;
      if (!fresh) {
        float over = -INFINITY;
#pragma unroll
        for (int r = 0; r < RT; ++r) x[r] -= ref(r);
#pragma unroll
        for (int r = 0; r < RT; r += 2) over = st::max3(over, x[r], x[r + 1]);
        move = soft_any<SOFT>(over > kLag + kLift);
      }
      if (move) {
        if (!fresh) {
#pragma unroll
          for (int r = 0; r < RT; ++r) x[r] += ref(r);
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float top = warp_top(x[r]);
          if (lane == 0) sh.m[warp][low + r] = top - kLift;
        }
        soft_sync<SOFT>();
        if (i > 0) {
          st::mbar_wait_warp(st::smem_u32(&sh.pv_done[(turn - 1) % L::V_STAGES]), (turn - 1) / L::V_STAGES & 1, &sh.abort);
          st::tc_fence_after();
        }
        bool none = false;
#pragma unroll
        for (int c = 0; c < RT / 8; ++c) {
          float b[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const int row = 8 * c + r;
            const float from = ref(row), to = fmaxf(from, fmaxf(fmaxf(sh.m[0][low + row], sh.m[1][low + row]), fmaxf(sh.m[2][low + row], sh.m[3][low + row])));
            b[r] = st::exp2_ftz(from - to);
            none = none || to == kNoMax;
            if (!kShared) own_ref[kShared ? 0 : row] = to;
            else if (t == 0) sh.ref[flip ^ 1][low + row] = to;
            l[row] *= b[r];
            x[row] -= to;
          }
          if (i > 0)
#pragma unroll
            for (int j = 0; j < kParts; ++j) {
              uint32_t o[8];
              tmem_ld_8(o_cols + j * R + low + 8 * c, o);
              st::tmem_ld_wait();
#pragma unroll
              for (int r = 0; r < 8; ++r) o[r] = __float_as_uint(__uint_as_float(o[r]) * b[r]);
              tmem_st_8(o_cols + j * R + low + 8 * c, o);
            }
        }
        if (i > 0) st::tmem_st_wait();
        unseen = soft_any<SOFT>(none);      // and the maxima are read
        flip ^= 1;
      }
      if (gone && half == 0) clean_values<D, R>(sh, of, slot, key, there, limit_min);
      // the buffer's last products are done
      if (L::P_BUFS == 2 && turn > 1) st::mbar_wait_warp(st::smem_u32(&sh.pv_done[(turn - 2) % L::V_STAGES]), (turn - 2) / L::V_STAGES & 1, &sh.abort);
      if (L::P_BUFS == 1 && turn > 0) st::mbar_wait_warp(st::smem_u32(&sh.pv_done[(turn - 1) % L::V_STAGES]), (turn - 1) / L::V_STAGES & 1, &sh.abort);
      const float take = st::exp2_int(-ve - static_cast<int>(kLift));
      unsigned char* to = sh.p[turn % L::P_BUFS];
      const uint32_t row = t / L::SIDES, first = t % L::SIDES * kParts * R + low;
#pragma unroll
      for (int c = 0; c < RT / 8; ++c) {
        __half2 w[4];
#pragma unroll
        for (int r = 0; r < 8; r += 2) {
          const float y = st::exp2_ftz(x[8 * c + r]), z = st::exp2_ftz(x[8 * c + r + 1]);
          l[8 * c + r] = fmaf(y, take, l[8 * c + r]), l[8 * c + r + 1] = fmaf(z, take, l[8 * c + r + 1]);
          w[r / 2] = __floats2half2_rn(y, z);
        }
#pragma unroll
        for (int j = 0; j < kParts; ++j) {
          const uint32_t byte = first + j * R + 8 * c;
          *reinterpret_cast<uint2*>(to + byte / 128 * (L::P_ROWS * 128) + swizzled<L::P_WIDTH>(row, byte % 128 / 16) + byte % 16) = split_off(w);
        }
      }
      st::fence_proxy_async_smem();
      st::tc_fence_before();
      st::mbar_arrive(st::smem_u32(&sh.p_full[turn & 1]));
    }

    // the item's outputs, and the sums over all keys, through the room of the weights, which no product reads now
    st::mbar_wait_warp(st::smem_u32(&sh.pv_done[(turn - 1) % L::V_STAGES]), (turn - 1) / L::V_STAGES & 1, &sh.abort);
    st::tc_fence_after();
    const Item& it = of.item;
    const int rows = it.row_end - it.row0;
    const bool whole = it.t0 == 0 && it.t1 == it.tiles;
    float* part = whole ? nullptr : part_of<R>(p, D, 2LL * blockIdx.x + (it.t0 == 0 ? 1 : 0));
    float* room = reinterpret_cast<float*>(sh.p[0]);      // [R][128]
#pragma unroll
    for (int r = 0; r < RT; ++r) room[(low + r) * 128 + t] = l[r];
    soft_sync<SOFT>();
    {      // SOFT / R threads to a row; where they begin keeps them out of one another's banks
      constexpr int TPR = SOFT / R, KEYS = 128 / TPR;
      const int r = threadIdx.x / TPR, first = threadIdx.x % TPR * KEYS;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < KEYS / 4; ++i) {
        const float4 y = *reinterpret_cast<const float4*>(room + r * 128 + first + 4 * ((i + t) % (KEYS / 4)));
        sum += (y.x + y.y) + (y.z + y.w);
      }
#pragma unroll
      for (int o = TPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (threadIdx.x % TPR == 0) sh.sum[r] = sum;
    }
    soft_sync<SOFT>();
    room += half * 512;
#pragma unroll
    for (int c = 0; c < RT / 8; ++c) {
      float o[8];
      if constexpr (R == 8) {      // the parts of 8 rows are 32 neighbouring columns
        uint32_t raw[32];
        st::tmem_ld_32x32(o_cols, raw);
        st::tmem_ld_wait();
#pragma unroll
        for (int r = 0; r < 8; ++r) o[r] = (__uint_as_float(raw[r]) + __uint_as_float(raw[8 + r])) + (__uint_as_float(raw[16 + r]) + __uint_as_float(raw[24 + r]));
      } else {
        uint32_t raw[kParts][8];
#pragma unroll
        for (int j = 0; j < kParts; ++j) tmem_ld_8(o_cols + j * R + low + 8 * c, raw[j]);
        st::tmem_ld_wait();
#pragma unroll
        for (int r = 0; r < 8; ++r) o[r] = (__uint_as_float(raw[0][r]) + __uint_as_float(raw[1][r])) + (__uint_as_float(raw[2][r]) + __uint_as_float(raw[3][r]));
      }
      if constexpr (D == 64) {
        if (warp >= 2)
#pragma unroll
          for (int r = 0; r < 8; ++r) room[r * 64 + t - 64] = o[r];
        soft_sync<SOFT>();
        if (warp < 2)
#pragma unroll
          for (int r = 0; r < 8; ++r) o[r] += room[r * 64 + t];
        if (c + 1 < RT / 8) soft_sync<SOFT>();
      }
      if (D == 128 || warp < 2) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int row = low + 8 * c + r;
          if (row >= rows) continue;
          const float sum = sh.sum[row];
          float y = o[r] * (1.0f / 512.0f);      // 2^-9
          if (sh.bad[row][t / 32] >> (t & 31) & 1) y = NAN;
          if (whole) out[of.place[row] + t] = from_f<T>(sum == 0.0f ? 0.0f : __fdividef(y, sum));
          else part[row * D + t] = y;
          if (t == 0) {
            if (!whole) part[R * D + row] = ref(8 * c + r), part[R * D + R + row] = sum;
            else if (p.lse != nullptr) {
              const int fr = it.row0 + row;
              p.lse[(it.start + fr / p.group) * static_cast<long long>(p.heads) + it.h * p.group + fr % p.group] = sum == 0.0f ? -INFINITY : (ref(8 * c + r) + kLift + log2f(sum)) / kLog2e;
            }
          }
        }
      }
    }
    if (threadIdx.x == 0 && it.t1 < it.tiles) *note = note_of(it, u1, runs, all);      // the run ends inside the item; never where items are whole, which have no notes
    st::tc_fence_before();
    soft_sync<SOFT>();      // everything of the item is read
    if (next >= u1) return;
    for (int i = threadIdx.x; i < R * (D / 32); i += SOFT) sh.bad[i / (D / 32)][i % (D / 32)] = 0;
    if (threadIdx.x == 0) st::mbar_arrive(st::smem_u32(&sh.q_empty[item % L::Q_BUFS]));
  }
}

template <typename T, int D, int R>
__global__ void __launch_bounds__(kThreadsOf<R>, Layout<D, R, kQueryParts<T>>::BLOCKS) paged_attn_kernel(AttnParams p, const __grid_constant__ CUtensorMap k_map,
                                                                                                     const __grid_constant__ CUtensorMap v_map) {
  constexpr int QP = kQueryParts<T>, SW = kSoftWarps<R>;
  using L = Layout<D, R, QP>;
  extern __shared__ __align__(1024) unsigned char raw[];      // swizzles count rows from multiples of 1024
  using S = Shared<D, R, QP>;
  S& sh = *reinterpret_cast<S*>(raw);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    st::tma_prefetch_desc(&k_map);
    st::tma_prefetch_desc(&v_map);
    for (int i = 0; i < L::K_STAGES; ++i) st::mbar_init(st::smem_u32(&sh.k_full[i]), 1), st::mbar_init(st::smem_u32(&sh.s_full[i]), 1);
    for (int i = 0; i < L::V_STAGES; ++i) st::mbar_init(st::smem_u32(&sh.v_full[i]), 1), st::mbar_init(st::smem_u32(&sh.pv_done[i]), 1);
    for (int i = 0; i < 2; ++i) st::mbar_init(st::smem_u32(&sh.p_full[i]), 32 * SW);
    for (int i = 0; i < L::Q_BUFS; ++i) st::mbar_init(st::smem_u32(&sh.q_full[i]), 1), st::mbar_init(st::smem_u32(&sh.q_empty[i]), 1);
    st::fence_barrier_init();
    sh.abort = 0;
  }
  chain_begin(p.ks, p.vs, p.table, p.starts, p.lengths);

  if (warp == SW + 1) {
    st::tmem_alloc(st::smem_u32(&sh.tmem), L::COLUMNS);
    st::tmem_relinquish();
  }
  st::tc_fence_before();      // before the barriers of the scan
  int all, u0, u1, runs;
  Found f;
  Note* note = reinterpret_cast<Note*>(p.notes) + blockIdx.x;
  const bool share = find_share<R>(p, sh.sums, &sh.found, all, runs, u0, u1, f);
  st::tc_fence_after();
  const uint32_t tmem = sh.tmem;
  if (threadIdx.x == 0 && !p.whole) note->parts = 0;
  if (!share) {
    if (warp == SW + 3) blank_rows<T, D>(p);
    if (warp == SW + 1) st::tmem_dealloc(tmem, L::COLUMNS);
    return;
  }
  const Seq sq = sequence<R>(p, f.b);
  // With 16 rows and more the softmax takes registers from the other warps: 176 and 80 of the 128 of the launch, with 32 rows 88
  // (of two warpgroups) and 64 of 80.
  constexpr bool kShift = R >= 16 && L::BLOCKS == 2;
  uint2 under_way = make_uint2(0, 0);
  if (warp >= SW) {
    if constexpr (kShift) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R == 32 ? 64 : 80));
    if (warp == SW) {
      under_way = score_warp<L, D, R, QP>(sh, p, &k_map, tmem, u0, u1, f, sq);
    } else if (warp == SW + 1) {
      under_way.y = value_warp<L, D, R>(sh, tmem, u1);
    } else if (warp == SW + 2) {
      query_warp<T, L, D, R, QP>(sh, p, u0, u1, f, sq);
    } else {
      Copier<L, D, R, true, S> values(sh, p, &v_map, u0, u1, f, sq);
      while (values.copy()) {}
      under_way.x = values.turn;
      blank_rows<T, D>(p);
    }
  } else {
    if constexpr (kShift) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R == 32 ? 88 : 176));
    soft_warps<T, L, D, R>(sh, p, tmem, note, u1, runs, all);
    if (threadIdx.x == 0 && sh.abort) st::report_error(p.err, st::ERR_MBAR_TIMEOUT, 0x7005);
  }
  st::tc_fence_before();
  __syncthreads();
  if (sh.abort) {
    if (warp == SW) settle(sh.k_full, under_way.x), settle(sh.s_full, under_way.y);
    if (warp == SW + 1) settle(sh.pv_done, under_way.y);
    if (warp == SW + 3) settle(sh.v_full, under_way.x);
    __syncthreads();
  }
  if (warp == SW + 1) st::tmem_dealloc(tmem, L::COLUMNS);
}

// Rows of an item, by those that the longest step of a sequence has for a key head.  Two items of 32 rows against one of 128 at 40 rows: 16 sequences at 6000
// 118 us and 91, 64 at 1000 with heads of 64 107 and 67.
int item_rows(long long max_queries, int group) {
  const long long rows = max_queries * group;
  return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : kPromptRows;
}
// Blocks that run at once: two to an SM, one where the products take all columns of tensor memory.
int runs_of(int rows, int dim) { return st::sm_count() * (rows == kPromptRows ? 1 : dim == 64 && rows == 32 ? Layout<64, 32, 4>::BLOCKS : Layout<128, 32, 4>::BLOCKS); }

// Whether items of sequences of up to `tokens` tokens are whole: then no second kernel is launched (4 us of the host) and no parts pass through the
// workspace.  Split ones share the chip evenly.  Device us, whole and split, 8 key heads of 128, every sequence as long as the table:
//                          1 sequence       16             64 sequences
//     8 rows,  7 units    13.2   13.1    15.3   18.0    30.6   36.5
//             14          19.6   12.8    21.1   21.0    47.0   51.9
//    16 rows,  7          21.4   16.3    23.5   26.7    45.9   66.0
//             14          30.9   18.2    33.3   32.1    67.4   87.8
//    32 rows,  7          29.9   21.3    31.2   43.6    77.3   95.8
//             18          53.5   23.1    56.8   61.1   153.6  159.6
//   128 rows, 12          31.9   19.8    33.0   45.8   127.3  130.6
//             18          41.8   21.3    44.2   58.1   175.3  172.9
// The limits are for the 16, which fill part of the chip: there whole items gain up to them.  A single sequence loses by them, 30 us at 18 units of 32 rows (with
// the host's part 55 and 26 us), and so do lengths that differ (64 sequences of 300 to 2304 tokens, 32 rows: 137 and 115); the shapes that the host knows
// tell neither the lengths nor, where the workspace is sized, how many sequences there are.
bool not_split(int rows, long long tokens) { return tokens <= (rows == 32 ? 18 : rows == kPromptRows ? 12 : 7) * kTile; }

template <typename T, int D, int R>
int launch_join(const AttnParams& p, cudaStream_t stream) {
  if (p.whole) return ST_OK;
  const int runs = runs_of(R, D);
  const cudaError_t e = st::chained(paged_join_kernel<T, D, R>, dim3(runs - 1, R == kPromptRows ? 16 : 1), dim3(kJoinThreads), runs * sizeof(float), stream)(p);
  return e == cudaSuccess ? ST_OK : st::fail_cuda(e, "paged attention: join");
}
template <typename T, int D>
int launch_prompt(const AttnParams& p, cudaStream_t stream) {
  constexpr int smem = sizeof(PromptShared<D>);
  auto kernel = paged_prompt_kernel<T, D>;
  static bool opted[st::kMaxDevices];
  if (bool& done = opted[st::current_device()]; !done) {
    ST_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    done = true;
  }
  const cudaError_t e = st::in_order(kernel, dim3(runs_of(kPromptRows, D)), dim3(kThreadsOf<kPromptRows>), smem, stream)(p);
  if (e != cudaSuccess) return st::fail_cuda(e, "paged attention");
  return launch_join<T, D, kPromptRows>(p, stream);
}
template <typename T, int D, int R>
int launch(const AttnParams& p, cudaStream_t stream) {
  const int runs = runs_of(R, D);
  constexpr int smem = sizeof(Shared<D, R, kQueryParts<T>>);
  // keys: rows of one token, swizzled over its D bytes; values: lines of 128 bytes; a copy takes a page's tokens, or a unit's
  CUtensorMap maps[2];
  const uint64_t tokens = static_cast<uint64_t>(p.pages) * p.kv_heads << p.shift;
  const uint32_t rows = p.shift < 7 ? 1u << p.shift : kTile;
  for (int i = 0; i < 2; ++i) {
    const uint64_t width = i == 0 ? D : 128, dims[2] = {width, tokens * D / width}, strides[1] = {width};
    const uint32_t box[2] = {static_cast<uint32_t>(width), static_cast<uint32_t>(rows * D / width)};
    if (!st::encode_tmap(&maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, i == 0 ? p.kc : p.vc, dims, strides, box,
                         width == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B))
      return ST_ERR_CUDA;
  }
  auto kernel = paged_attn_kernel<T, D, R>;
  static bool opted[st::kMaxDevices];
  if (bool& done = opted[st::current_device()]; !done) {
    ST_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    done = true;
  }
  // in order: blocks that come early pile up on the SMs that fall free first
  const cudaError_t e = st::in_order(kernel, dim3(runs), dim3(kThreadsOf<R>), smem, stream)(p, maps[0], maps[1]);
  if (e != cudaSuccess) return st::fail_cuda(e, "paged attention");
  return launch_join<T, D, R>(p, stream);
}
template <typename T, int D>
int dispatch(const AttnParams& p, int rows, cudaStream_t stream) {
  return rows == 8 ? launch<T, D, 8>(p, stream) : rows == 16 ? launch<T, D, 16>(p, stream) : rows == 32 ? launch<T, D, 32>(p, stream) : launch_prompt<T, D>(p, stream);
}
}  // namespace

// Floats of workspace that st_paged_attention takes.
ST_API long long st_paged_attention_workspace(int max_queries, int heads, int kv_heads, int dim, int width, int page_size) {
  if (kv_heads < 1 || heads < kv_heads || not_split(item_rows(max_queries, heads / kv_heads), static_cast<long long>(width) * page_size)) return 0;
  const int r = item_rows(max_queries, heads / kv_heads);
  return (2LL * r * (dim + 2) + sizeof(Note) / sizeof(float)) * runs_of(r, dim);
}

// q, out [rows, heads, dim] (dim contiguous, strides in elements): row starts[b] + i is the i-th of the newest tokens of sequence b, whose keys and values,
// these tokens' included, are the first lengths[b] of the pages in table[b].  lse [rows, heads] or null.  max_queries: the most rows of a sequence, by which
// the row tile is chosen; more are computed too.  zero_tail: rows before the first
// sequence and behind the last one become 0 (else they stay as they were); their lse is -inf.  type: 0 bf16, 1 fp16.
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
  const int r = item_rows(max_queries, heads / kv_heads);
  // units are counted in 32 bits
  if ((rows * (heads / kv_heads) / r + B) * (((static_cast<long long>(width) << shift) + kTile - 1) / kTile + 1 + kItemCost<32>) * kv_heads > 2147483647LL)
    return st::fail(ST_ERR_TOO_LARGE, "paged attention: rows times the table's width is too large for one call");
  int* notes = reinterpret_cast<int*>(workspace + 2LL * r * (dim + 2) * runs_of(r, dim));      // behind the parts
  const AttnParams p{q, static_cast<const unsigned char*>(k_codes), static_cast<const unsigned char*>(v_codes), k_scale, v_scale, table, starts, lengths, out, lse, workspace, notes,
                     q_row, q_head, o_row, o_head, table_row, pages, rows, width, shift, B, heads, kv_heads, heads / kv_heads, scale, causal, zero_tail, not_split(r, static_cast<long long>(width) << shift), st::error_word()};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  if (type == 0) return dim == 64 ? dispatch<__nv_bfloat16, 64>(p, r, stream) : dispatch<__nv_bfloat16, 128>(p, r, stream);
  return dim == 64 ? dispatch<__half, 64>(p, r, stream) : dispatch<__half, 128>(p, r, stream);
}
