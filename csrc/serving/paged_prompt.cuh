// Attention over pages for parts of prompts: items of 128 rows.
//
// With many rows to a key head the products bound it, 4 * 128 * D * 128 operations a unit and item, 1024 cycles of an SM's fp16 rate for D = 128, and beside them the
// exponentials, as many cycles.  So here the rows are the 128 lanes of S = Q K^T and O = P V, one thread has a row and no row's softmax needs another
// thread, and codes are converted to fp16 (exactly) once per unit for all rows: warps of their own read them from the pages into registers and write them to
// shared memory, swizzled as the products read them.  Weights go to tensor memory, over the scores that they were made from.
//
// Two groups of softmax warps take turns: a unit's turn decides which group has it, with scores, weights, outputs and a reference of its own, so the products of one
// group's unit run beside the softmax of the other's.  At the end of an item both read both outputs, half of the columns each, and add them up.
//
// The softmax is that of the other items: x = s * f + b over the codes' scores with f = scale * 2^a (queries are fp16 numbers, scaled by a power of two per row and
// by the scale's sign, so f >= 0 and a page's largest x comes from its largest score), weights exp2(x - reference) below 2^15, the reference behind the
// maximum by 9 at first and 15 at most, and the sum takes exp2(-b) back out per 16 keys.
//
// Measured: 4 sequences of 256 tokens behind up to 4000, 16 heads over 4 of 128: 41 us, where two products' operations take 6.  A unit takes a block 3200 cycles:
// a group's scores, weights and outputs follow one another (1000 for the maximum, 2500 for the weights, 400 until the last warp is there, 1900 for the two
// products), and two groups are what tensor memory has room for.  Before: items of 32 rows on codes 87, this with masks in the same code as the rest 77.  Tried without
// gain: maximum and weights in one pass with corrections behind it (46), halves of 64 keys, which need half as many product instructions more (48), more of the
// loops unrolled (48 to 58): instructions come from a cache that the block's kinds of warps share (waiting for them took 4.2 of 17 cycles an instruction at 58 us, 1.0 of 13 now).  A beginning takes 11000 cycles for the same reason.
#pragma once
#include "paged_work.cuh"

namespace {
constexpr int kPromptRows = 128;
constexpr int kNoRow = 1 << 30;

template <int D>
struct PromptShared {
  static constexpr int TILE = 128 * D * 2;      // rows of 128 bytes, one or two of them side by side: 128 rows of the first 64 elements, then of the others
  unsigned char q[2][TILE], k[2][TILE], v[2][TILE];
  // of the two turns: keys and values are converted, a unit's scales are there, its scores, weights, outputs
  unsigned long long k_full[2], v_full[2], scales[2], s_full[2], p_full[2], pv_done[2], q_full[2], q_empty[2];
  alignas(16) float ks[2][8], lift[2][8], take[2][8];      // of 16 keys: 2^a, b (-inf: no such page), 2^(-b - 9)
  Item item[2];
  float factor[2][kPromptRows];
  float2 stat[2][kPromptRows];      // a group's references and sums
  int bad[4][D], some_bad[4];       // first row that a value reaches which is no number though not all rows see it; whether there are such
  int sums[kMaxWarps];
  Found found;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(PromptShared<128>) <= 226 * 1024);

// Instruction descriptor: fp16 products, fp32 sums.
constexpr uint32_t half_idesc(int N, bool b_mn_major) { return 1u << 4 | static_cast<uint32_t>(b_mn_major) << 16 | static_cast<uint32_t>(N >> 3) << 17 | 128u >> 4 << 24; }

// Two e4m3 numbers as fp16, exactly; no number stays none.
__device__ __forceinline__ uint32_t two_halves(uint32_t codes) {
  uint32_t h;
  asm("{\n.reg .b16 c;\ncvt.u16.u32 c, %1;\ncvt.rn.f16x2.e4m3x2 %0, c;\n}\n" : "=r"(h) : "r"(codes));
  return h;
}

// ---- keys or values: pages -> registers -> fp16 in shared memory ---------------------------------------------------------------------
// Four warps for keys and four for values, in the same code: with code for each, and with more of the rest unrolled, a quarter of the time went to waiting for
// instructions.  Each warp has 32 keys of a unit, at most two pages.
template <int D, typename S>
__device__ __forceinline__ void convert_warp(S& sh, const AttnParams& p, bool values, int u, int u1, Found f, Seq sq) {
  constexpr int VECS = D / 16, PER = 32 / VECS, LOADS = 32 / PER;      // 16-byte vectors of a key, keys of a load
  const int lane = threadIdx.x & 31, first = (threadIdx.x >> 5 & 3) * 32;
  // eight lanes write parts of two neighbouring rows, whose swizzles keep them in different banks
  const int vec = D == 64 ? lane & 3 : (lane & 3) | (lane >> 1 & 4), at = D == 64 ? lane >> 2 : (lane >> 2 & 1) | (lane >> 3 & 2);
  const unsigned char* codes = (values ? p.vc : p.kc) + at * D + vec * 16;
  const int mask = (1 << p.shift) - 1;
  // A unit ahead of the one that is converted its codes and scales are on their way, two ahead its page numbers.
  struct Unit {
    int key, h, keys;          // its first key (-1: no more), key head, keys that the item sees
    int all, sees, item;       // keys of it that all rows see, first row that sees its first key
    int page;                  // one to 16 lanes
  };
  Item it;
  int t = 0, end = 0, items = -1;
  auto advance = [&](Unit& x) {
    if (++t >= end) {
      if (!item_at<kPromptRows>(it, p, u, u1, f, sq)) {
        u = u1, t = end - 1, x = Unit{-1, 0, 0, kTile, 0, 0, kBehind};
        return;
      }
      u = it.next, t = it.t0, end = it.t0 + it.steps(), ++items;
    }
    x.key = t * kTile, x.h = it.h, x.keys = it.keys, x.item = items & 3;
    x.all = max(it.len - (p.causal ? it.n - 1 - it.row0 / p.group : 0), 0) - x.key, x.sees = (x.key + it.n - it.len) * p.group - it.row0;
    const int key = x.key + first + (lane & 16);
    x.page = key < it.keys ? it.table[key >> p.shift] : kBehind;
  };
  uint4 raw[LOADS];
  float ks = 0.0f, vs = 0.0f;
  const unsigned char* from[2];
  int live[2];      // keys of 16 that there are
  auto look = [&](Unit& x) {
    if (x.page < 0 || x.page >= p.pages) {
      if (values && x.page != kBehind && (lane & 15) == 0) st::report_error(p.err, st::ERR_BOUNDS, 0x7004);
      x.page = -1;
    } else if (values) {
      const long long scale = static_cast<long long>(x.page) * p.kv_heads + x.h;
      ks = p.ks[scale], vs = p.vs[scale];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int pg = __shfl_sync(0xffffffffu, x.page, 16 * h), key = x.key + first + 16 * h;
      from[h] = codes + (((static_cast<long long>(pg) * p.kv_heads + x.h) << p.shift) + (key & mask)) * D;
      live[h] = pg >= 0 ? x.keys - key : 0;
    }
  };
  auto load = [&](int j) {
    const int h = j * PER / 16, in = j * PER % 16;
    raw[j] = make_uint4(0, 0, 0, 0);
    if (in + at < live[h]) raw[j] = *reinterpret_cast<const uint4*>(from[h] + in * D);
  };
  Unit now, next;
  advance(now);
  if (now.key < 0) return;
  advance(next);
  look(now);
#pragma unroll
  for (int j = 0; j < LOADS; ++j) load(j);
  uint32_t turn = 0;
#pragma unroll 1
  for (;; ++turn) {
    const int g = turn & 1;
    const uint32_t before = (turn >> 1 & 1) ^ 1;
    if (values) {
      if (!st::mbar_wait_warp(st::smem_u32(&sh.p_full[g]), before, &sh.abort)) return;      // the scales of the turn before last are read
      if ((lane & 15) == 0) {
        const int group = (first + lane) / 16, b = st::scale_exponent(vs);
        const bool there = now.page >= 0;
        sh.ks[g][group] = there ? ks : 0.0f;
        sh.lift[g][group] = there ? static_cast<float>(b) : -INFINITY;
        sh.take[g][group] = there ? st::exp2_int(-b - static_cast<int>(kLift)) : 0.0f;
        st::mbar_arrive(st::smem_u32(&sh.scales[g]));
      }
      __syncwarp();
    }
    if (values && now.all < kTile) {      // values that are no numbers and not for all rows: 0, and a note of the first row that sees them
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
        const int row = first + j * PER + at;
        if ((nan_bytes(w[0]) | nan_bytes(w[1]) | nan_bytes(w[2]) | nan_bytes(w[3])) == 0 || row < now.all) continue;
        sh.some_bad[now.item] = 1;
#pragma unroll 1
        for (int c = 0; c < 16; ++c) {
          const uint32_t x = c < 4 ? w[0] : c < 8 ? w[1] : c < 12 ? w[2] : w[3];
          if (nan_bytes(x) >> (8 * (c & 3) + 7) & 1) atomicMin(&sh.bad[now.item][vec * 16 + c], max(now.sees + row * p.group, 0));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] &= ~((nan_bytes(w[i]) >> 7) * 255u);
        raw[j] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    if (!st::mbar_wait_warp(st::smem_u32(values ? &sh.pv_done[g] : &sh.s_full[g]), before, &sh.abort)) return;
    const bool more = next.key >= 0;
    now = next;
    look(now);
    unsigned char* to = (values ? sh.v[g] : sh.k[g]) + vec / 4 * (128 * 128) + (first + at) * 128;
    const uint32_t part = (vec % 4 * 2 ^ at) * 16;      // swizzled; at < 8
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w}, swizzle = j * PER % 8 * 16;
      load(j);
      *reinterpret_cast<uint4*>(to + j * PER * 128 + (part ^ swizzle)) = make_uint4(two_halves(w[0]), two_halves(w[0] >> 16), two_halves(w[1]), two_halves(w[1] >> 16));
      *reinterpret_cast<uint4*>(to + j * PER * 128 + (part ^ swizzle ^ 16)) = make_uint4(two_halves(w[2]), two_halves(w[2] >> 16), two_halves(w[3]), two_halves(w[3] >> 16));
    }
    st::fence_proxy_async_smem();
    st::mbar_arrive(st::smem_u32(values ? &sh.v_full[g] : &sh.k_full[g]));
    if (!more) return;
    advance(next);
  }
}

// ---- products ------------------------------------------------------------------------------------------------------------------------
// Returns the turns whose scores and whose outputs it issued.  Scores go two turns ahead; they overwrite the weights of the turn before last, whose
// product was issued before by the same thread.
template <int D, typename S>
__device__ __forceinline__ uint2 product_warp(S& sh, uint32_t tmem_, int u1) {
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_, 0);
  constexpr uint32_t hi = st::smem_desc_hi(1024), score = half_idesc(128, false), value = half_idesc(D, true);
  const bool leader = st::elect_one();
  struct Cursor {
    uint32_t turn, item;
    int left, at;
    bool more;
  };
  Cursor s{0, 0, 0, 0, true}, v{0, 0, 0, 0, true};
  bool failed = false;
  // The cursor's next unit: whether there is one.
  auto step = [&](Cursor& c) {
    if (c.left == 0) {
      if (!c.more) return false;
      const Item& it = sh.item[c.item & 1];
      if (!st::mbar_wait_warp(st::smem_u32(&sh.q_full[c.item & 1]), c.item >> 1 & 1, &sh.abort)) {
        failed = true;
        return false;
      }
      c.left = it.t1 > it.t0 ? it.steps() : 0, c.at = 0, c.more = c.left > 0 && it.next < u1;
      if (c.left == 0) return false;
      ++c.item;
    }
    return true;
  };
  auto scores = [&] {
    if (!step(s)) return;
    const int g = s.turn & 1;
    if (!st::mbar_wait_warp(st::smem_u32(&sh.k_full[g]), s.turn >> 1 & 1, &sh.abort)) {
      failed = true;
      return;
    }
    st::tc_fence_after();
    if (leader) {
      const uint32_t a = st::smem_desc_lo(st::smem_u32(sh.q[(s.item - 1) & 1]), 16), b = st::smem_desc_lo(st::smem_u32(sh.k[g]), 16);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t off = (k / 4 * (128 * 128) + k % 4 * 32) >> 4;
        st::umma_bf16_ss_split(tmem + g * 128, a + off, hi, b + off, hi, score, k > 0);
      }
      st::umma_commit(st::smem_u32(&sh.s_full[g]));
    }
    __syncwarp();
    ++s.turn, --s.left;
  };
  scores();
  if (!failed) scores();
  while (!failed && step(v)) {
    const int g = v.turn & 1;
    if (!st::mbar_wait_warp(st::smem_u32(&sh.v_full[g]), v.turn >> 1 & 1, &sh.abort) || !st::mbar_wait_warp(st::smem_u32(&sh.p_full[g]), v.turn >> 1 & 1, &sh.abort)) break;
    st::tc_fence_after();
    if (leader) {
      const uint32_t b = st::smem_desc_lo(st::smem_u32(sh.v[g]), 128 * 128);
#pragma unroll
      for (int k = 0; k < 8; ++k) st::umma_bf16_ts_split(tmem + 256 + g * D, tmem + g * 128 + k * 8, b + (k * (16 * 128) >> 4), hi, value, v.at > 1 || k > 0);
      st::umma_commit(st::smem_u32(&sh.pv_done[g]));
    }
    __syncwarp();
    ++v.turn, ++v.at, --v.left;
    scores();
  }
  return make_uint2(s.turn, v.turn);
}

// ---- queries -------------------------------------------------------------------------------------------------------------------------
// Three warps.  Each row's largest element to [2^14, 2^15): fp16 holds bf16's 8 bits down to 2^-28 of it.
template <typename T, int D, typename S>
__device__ __forceinline__ void prompt_query_warp(S& sh, const AttnParams& p, int w, int u0, int u1, Found f, Seq sq) {
  constexpr int VECS = D / 32;      // of a lane: four to a row
  const int lane = threadIdx.x & 31;
  const T* q = static_cast<const T*>(p.q);
  const bool wide = ((p.q_row | p.q_head) & 7) == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
  const float sign = p.scale < 0.0f ? -1.0f : 1.0f;
  uint32_t item = 0;
  Item it;
  for (int u = u0; u < u1; ++item) {
    if (!item_at<kPromptRows>(it, p, u, u1, f, sq)) {      // the last word: no more items, and no rows
      it = Item{};
      it.next = u1;
    }
    u = it.next;
    const int buf = item & 1;
    if (!st::mbar_wait_warp(st::smem_u32(&sh.q_empty[buf]), (item >> 1 & 1) ^ 1, &sh.abort)) return;
    if (w == 0 && lane == 0) sh.item[buf] = it;
#pragma unroll 1
    for (int r = 8 * w + lane / 4; r < kPromptRows; r += 24) {
      const int fr = it.row0 + r, i = fr / p.group, head = it.h * p.group + fr - i * p.group;
      const bool live = fr < it.row_end;
      const T* from = q + (it.start + i) * p.q_row + head * p.q_head + (lane & 3) * (D / 4);
      uint4 raw[VECS];
#pragma unroll
      for (int k = 0; k < VECS; ++k) raw[k] = live ? load8(from + 8 * k, wide) : make_uint4(0, 0, 0, 0);
      float top = 0.0f;
#pragma unroll
      for (int k = 0; k < VECS; ++k) {
        const uint32_t x[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 y = two_floats<T>(x[j]);
          top = st::max3(top, fabsf(y.x), fabsf(y.y));
        }
      }
      const uint32_t four = 0xfu << (lane & 28);      // a warp's last rows may be none
      top = fmaxf(top, __shfl_xor_sync(four, top, 1));
      top = fmaxf(top, __shfl_xor_sync(four, top, 2));
      int e = static_cast<int>((__float_as_uint(top) >> 23) & 255) - 127 - 14;
      e = top < INFINITY ? max(e, -100) : 0;
      const float mul = top < INFINITY ? sign * st::exp2_int(-e) : NAN;      // a row with infinities gives NaN
#pragma unroll
      for (int k = 0; k < VECS; ++k) {
        const uint32_t x[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 y = two_floats<T>(x[j]);
          const __half2 z = __floats2half2_rn(y.x * mul, y.y * mul);
          h[j] = *reinterpret_cast<const uint32_t*>(&z);
        }
        const int d = (lane & 3) * (D / 4) + 8 * k;
        *reinterpret_cast<uint4*>(sh.q[buf] + d / 64 * (128 * 128) + st::sw128_offset(r, d % 64 / 8)) = make_uint4(h[0], h[1], h[2], h[3]);
      }
      if ((lane & 3) == 0) sh.factor[buf][r] = fabsf(p.scale) * kLog2e * st::exp2_int(e);
    }
    st::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) st::mbar_arrive(st::smem_u32(&sh.q_full[buf]));
  }
}

// ---- the softmax ---------------------------------------------------------------------------------------------------------------------
// The largest x of a row's scores.  MASKED: keys from `end` on do not count, nor those of pages that are none.
template <bool MASKED>
__device__ __forceinline__ float prompt_top(uint32_t s_cols, float factor, const float* ks, const float* lift, int end) {
  float top = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    uint32_t raw[32];
    st::tmem_ld_32x32(s_cols + 32 * c, raw);
    const float2 k = *reinterpret_cast<const float2*>(ks + 2 * c), b = *reinterpret_cast<const float2*>(lift + 2 * c);
    st::tmem_ld_wait();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = MASKED && 32 * c + 16 * h + j >= end ? -INFINITY : __uint_as_float(raw[16 * h + j]);
      float m = st::max3(x[0], x[1], x[2]), n = st::max3(x[3], x[4], x[5]);
      m = st::max3(m, x[6], x[7]), n = st::max3(n, x[8], x[9]);
      m = st::max3(m, x[10], x[11]), n = st::max3(n, x[12], x[13]);
      m = st::max3(m, x[14], x[15]);
      top = fmaxf(top, fmaf(fmaxf(m, n), factor * (h ? k.y : k.x), h ? b.y : b.x));
    }
  }
  return top;
}
// Weights over the scores that they are made from; returns the sum with them.  x - reference is one multiplication and addition, which holds the product
// whole where the reference is rounded: of scores beyond kLarge, MASKED rounds x as the reference's was.
constexpr float kLarge = 4194304.0f;      // 2^22: half a unit in the last place is 2^-2, and weights below 2^15 stay below fp16's 2^16 by it
template <bool MASKED>
__device__ __forceinline__ float prompt_weights(uint32_t s_cols, float factor, float ref, float sum, const float* ks, const float* lift, const float* take, int end) {
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    uint32_t raw[32], w[16];
    st::tmem_ld_32x32(s_cols + 32 * c, raw);
    const float2 k = *reinterpret_cast<const float2*>(ks + 2 * c), b = *reinterpret_cast<const float2*>(lift + 2 * c), t = *reinterpret_cast<const float2*>(take + 2 * c);
    st::tmem_ld_wait();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float lifted = h ? b.y : b.x;
      const float2 fs = st::splat2(factor * (h ? k.y : k.x)), bs = st::splat2(MASKED ? lifted : lifted - ref);
      const bool none = MASKED && lifted == -INFINITY;
      float2 part = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        float2 x = st::fma2(make_float2(__uint_as_float(raw[16 * h + j]), __uint_as_float(raw[16 * h + j + 1])), fs, bs);
        if (MASKED) x = st::add2(x, st::splat2(-ref));
        x.x = st::exp2_ftz(x.x), x.y = st::exp2_ftz(x.y);
        if (MASKED && (none || 32 * c + 16 * h + j >= end)) x.x = 0.0f;
        if (MASKED && (none || 32 * c + 16 * h + j + 1 >= end)) x.y = 0.0f;
        part = st::add2(part, x);
        const __half2 y = __floats2half2_rn(x.x, x.y);
        w[8 * h + j / 2] = *reinterpret_cast<const uint32_t*>(&y);
      }
      sum = fmaf(part.x + part.y, h ? t.y : t.x, sum);
    }
    st::tmem_st_32x16(s_cols + 16 * c, w);
  }
  return sum;
}

template <typename T, int D, typename S>
__device__ __forceinline__ void prompt_soft_warps(S& sh, const AttnParams& p, uint32_t tmem_all, Note* note, int u1, int runs, int all) {
  const int row = threadIdx.x & 127, g = threadIdx.x >> 7;
  const uint32_t lanes = tmem_all + ((threadIdx.x >> 5 & 3) << 21), s_cols = lanes + g * 128, o_cols = lanes + 256 + g * D;
  T* out = static_cast<T*>(p.out);
  const bool wide = ((p.o_row | p.o_head) & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0;
  uint32_t first = 0;      // turn of the item's first unit
#pragma unroll 1
  for (uint32_t item = 0;; ++item) {
    // a wait that runs out sets the abort flag: the warps finish the item together and stop at the next one
    if (soft_any<256>(!st::mbar_wait_warp(st::smem_u32(&sh.q_full[item & 1]), item >> 1 & 1, &sh.abort))) return;
    const Item& it = sh.item[item & 1];
    if (it.t1 <= it.t0) return;      // no more items
    const int steps = it.steps(), t0 = it.t0, next = it.next, rows = it.row_end - it.row0;
    const float factor = sh.factor[item & 1][row];
    const int fr = it.row0 + row, query = fr / p.group;
    const int limit = row < rows ? max(it.len - (p.causal ? it.n - 1 - query : 0), 0) : it.len;
    const int limit_min = max(it.len - (p.causal ? it.n - 1 - it.row0 / p.group : 0), 0);
    float ref = kNoMax, sum = 0.0f;      // the reference, maximum less 9 and behind, and the weights' sum over it
    const int mine = (first ^ g) & 1;      // the group's first unit
#pragma unroll 1
    for (int i = mine; i < steps; i += 2) {
      const uint32_t turn = first + i, phase = turn >> 1 & 1;
      st::mbar_wait_warp(st::smem_u32(&sh.scales[g]), phase, &sh.abort);
      bool none = false;
#pragma unroll
      for (int c = 0; c < 8; ++c) none = none || sh.lift[g][c] == -INFINITY;
      const bool gone = none || (t0 + i + 1) * kTile > limit_min;      // some row may not see some key
      const int end = limit - (t0 + i) * kTile;      // keys of the unit that the row sees
      st::mbar_wait_warp(st::smem_u32(&sh.s_full[g]), phase, &sh.abort);
      st::tc_fence_after();
      const float top = gone ? prompt_top<true>(s_cols, factor, sh.ks[g], sh.lift[g], end) : prompt_top<false>(s_cols, factor, sh.ks[g], sh.lift[g], end);
      if (__any_sync(0xffffffffu, top - ref > kLag + kLift)) {
        const float to = fmaxf(ref, top - kLift), shrink = st::exp2_ftz(ref - to);
        ref = to, sum *= shrink;
        if (i > 1) {
          st::mbar_wait_warp(st::smem_u32(&sh.pv_done[g]), phase ^ 1, &sh.abort);      // of the turn before last
          st::tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            st::tmem_ld_32x16(o_cols + 16 * c, o);
            st::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * shrink);
            st::tmem_st_32x16(o_cols + 16 * c, o);
          }
          st::tmem_st_wait();
        }
      }
      sum = gone || __any_sync(0xffffffffu, fabsf(top) > kLarge) ? prompt_weights<true>(s_cols, factor, ref, sum, sh.ks[g], sh.lift[g], sh.take[g], end) : prompt_weights<false>(s_cols, factor, ref, sum, sh.ks[g], sh.lift[g], sh.take[g], end);
      st::tmem_st_wait();
      st::tc_fence_before();
      st::mbar_arrive(st::smem_u32(&sh.p_full[g]));
    }

    // both groups' outputs, half of the columns each
    sh.stat[g][row] = make_float2(ref, sum);
    // A group waits for its own last unit and the barrier does the rest: another's parity may stand two turns back, where a wait would not hold.
    const int last = steps - 1 - ((first + steps - 1 ^ g) & 1);
    if (last >= 0) st::mbar_wait_warp(st::smem_u32(&sh.pv_done[g]), (first + last) >> 1 & 1, &sh.abort);
    st::tc_fence_before();
    soft_sync<256>();
    st::tc_fence_after();
    const float2 other = sh.stat[g ^ 1][row];
    const float m = fmaxf(ref, other.x);
    const float w_own = st::exp2_ftz(ref - m), w_other = st::exp2_ftz(other.x - m);
    const float all_sum = sum * w_own + other.y * w_other;
    const bool whole = it.t0 == 0 && it.t1 == it.tiles;
    const float by = 1.0f / 512.0f * (whole ? (all_sum == 0.0f ? 0.0f : 1.0f / all_sum) : 1.0f);
    const float scale[2] = {(g == 0 ? w_own : w_other) * by, (g == 0 ? w_other : w_own) * by};
    const bool has[2] = {steps > 1 || (first & 1) == 0, steps > 1 || (first & 1) == 1};
    float* part = whole ? nullptr : part_of<kPromptRows>(p, D, 2LL * blockIdx.x + (it.t0 == 0 ? 1 : 0));
    const int head = it.h * p.group + fr - query * p.group, lane = threadIdx.x & 31;
    const long long place = (it.start + query) * p.o_row + head * p.o_head;
    const bool check = sh.some_bad[item & 3] != 0;
    // a quarter of the columns at a time through the room of the item's queries, which no product reads now: a warp's own eighth of it, whole rows to a store
    constexpr int WIDE = D / 4, LANES = WIDE / 4;      // columns, lanes of a row
    static_assert(8 * 32 * WIDE * sizeof(float) == S::TILE);
    float* room = reinterpret_cast<float*>(sh.q[item & 1]) + (threadIdx.x >> 5) * (32 * WIDE);
#pragma unroll 1
    for (int c = 0; c < 2; ++c) {
      const int d0 = g * (D / 2) + WIDE * c;
#pragma unroll 1
      for (int part16 = 0; part16 < WIDE / 16; ++part16) {
        const int d = d0 + 16 * part16;
        uint32_t o[2][16];
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (has[k]) st::tmem_ld_32x16(lanes + 256 + k * D + d, o[k]);
        st::tmem_ld_wait();
        float y[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float a = has[0] ? __uint_as_float(o[0][j]) * scale[0] : 0.0f;
          y[j] = has[1] ? fmaf(__uint_as_float(o[1][j]), scale[1], a) : a;
          if (whole && all_sum == 0.0f) y[j] = 0.0f;
        }
        if (check)
          for (int j = 0; j < 16; ++j)
            if (row >= sh.bad[item & 3][d + j]) y[j] = NAN;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<float4*>(room + WIDE * lane + 4 * ((4 * part16 + j) ^ (lane & (LANES - 1)))) = make_float4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
      }
      __syncwarp();
#pragma unroll 1
      for (int k = 0; k < LANES; ++k) {
        const int r = 32 / LANES * k + lane / LANES, at = lane & (LANES - 1), in = (threadIdx.x >> 5 & 3) * 32 + r, d = d0 + 4 * at;
        const float4 y = *reinterpret_cast<const float4*>(room + WIDE * r + 4 * (at ^ (r & (LANES - 1))));
        const long long to = __shfl_sync(0xffffffffu, place, r);
        if (in >= rows) continue;
        if (!whole) {
          *reinterpret_cast<float4*>(part + in * D + d) = y;
        } else {
          const T h[4] = {from_f<T>(y.x), from_f<T>(y.y), from_f<T>(y.z), from_f<T>(y.w)};
          if (wide) *reinterpret_cast<uint2*>(out + to + d) = *reinterpret_cast<const uint2*>(h);
          else
            for (int j = 0; j < 4; ++j) out[to + d + j] = h[j];
        }
      }
      __syncwarp();
    }
    if (g == 0 && row < rows) {
      if (!whole) part[kPromptRows * D + row] = m, part[kPromptRows * D + kPromptRows + row] = all_sum;
      else if (p.lse != nullptr) p.lse[(it.start + query) * static_cast<long long>(p.heads) + head] = all_sum == 0.0f ? -INFINITY : (m + kLift + log2f(all_sum)) / kLog2e;
    }
    if (threadIdx.x == 0 && it.t1 < it.tiles) *note = note_of(it, u1, runs, all);      // the run ends inside the item
    st::tc_fence_before();
    soft_sync<256>();      // everything of the item is read
    if (next >= u1) return;
    if (check) {
      if (threadIdx.x < D) sh.bad[item & 3][threadIdx.x] = kNoRow;
      if (threadIdx.x == 0) sh.some_bad[item & 3] = 0;
    }
    if (threadIdx.x == 0) st::mbar_arrive(st::smem_u32(&sh.q_empty[item & 1]));
    first += steps;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreadsOf<kPromptRows>, 1) paged_prompt_kernel(AttnParams p) {
  extern __shared__ __align__(1024) unsigned char raw[];
  using S = PromptShared<D>;
  S& sh = *reinterpret_cast<S*>(raw);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      st::mbar_init(st::smem_u32(&sh.k_full[i]), 128), st::mbar_init(st::smem_u32(&sh.v_full[i]), 128), st::mbar_init(st::smem_u32(&sh.scales[i]), 8);
      st::mbar_init(st::smem_u32(&sh.s_full[i]), 1), st::mbar_init(st::smem_u32(&sh.p_full[i]), 128), st::mbar_init(st::smem_u32(&sh.pv_done[i]), 1);
      st::mbar_init(st::smem_u32(&sh.q_full[i]), 3), st::mbar_init(st::smem_u32(&sh.q_empty[i]), 1);
    }
    st::fence_barrier_init();
    sh.abort = 0;
  }
  if (threadIdx.x < 4) sh.some_bad[threadIdx.x] = 0;
  if (threadIdx.x < 4 * D) sh.bad[threadIdx.x / D][threadIdx.x % D] = kNoRow;
  chain_begin(p.ks, p.vs, p.table, p.starts, p.lengths);
  if (warp == 16) {
    st::tmem_alloc(st::smem_u32(&sh.tmem), 512);
    st::tmem_relinquish();
  }
  st::tc_fence_before();      // before the barriers of the scan
  int all, u0, u1, runs;
  Found f;
  Note* note = reinterpret_cast<Note*>(p.notes) + blockIdx.x;
  const bool share = find_share<kPromptRows>(p, sh.sums, &sh.found, all, runs, u0, u1, f);
  st::tc_fence_after();
  const uint32_t tmem = sh.tmem;
  if (threadIdx.x == 0 && !p.whole) note->parts = 0;
  if (!share) {
    if (warp == 19) blank_rows<T, D>(p);
    if (warp == 16) st::tmem_dealloc(tmem, 512);
    return;
  }
  const Seq sq = sequence<kPromptRows>(p, f.b);
  uint2 under_way = make_uint2(0, 0);
  if (warp >= 16) {
    if (warp == 16) under_way = product_warp<D>(sh, tmem, u1);
    else prompt_query_warp<T, D>(sh, p, warp - 17, u0, u1, f, sq);
    if (warp == 19) blank_rows<T, D>(p);
  } else if (warp >= 8) {
    convert_warp<D>(sh, p, warp >= 12, u0, u1, f, sq);
  } else {
    prompt_soft_warps<T, D>(sh, p, tmem, note, u1, runs, all);
    if (threadIdx.x == 0 && sh.abort) st::report_error(p.err, st::ERR_MBAR_TIMEOUT, 0x7006);
  }
  st::tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    if (sh.abort) settle(sh.s_full, under_way.x), settle(sh.pv_done, under_way.y);
    st::tmem_dealloc(tmem, 512);
  }
}
}  // namespace
