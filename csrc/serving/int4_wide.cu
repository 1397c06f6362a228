// Products of many rows with weights of four bits on tcgen05:  y = act(x W^T + bias) + residual  and  dx = dy W.
//
// The weights are the 128-row operand and lie in tensor memory: warps take codes from shared memory, make them numbers q s of the input's type (exact), and write
// them from registers in the order in which they come (int4.cuh).  The rows of x (or dy) are the other operand, up to 192 of them, by tiled copies.  So
// a tile's sums stand as [weight row or column][token], and a weight is converted once for 192 tokens and never passes through shared memory as 16 bits.
// dx contracts over the weights' rows: the same tiles, each 8 x 8 block turned over in registers.
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "../common/chain.cuh"
#include "int4.cuh"
#include "int4_wide.h"

namespace {
using namespace st4;

constexpr int kRing = 4;                     // weight operands in tensor memory, 32 columns each, behind two results
constexpr int kMostTokens = 192;             // of a tile: 2 * 192 + 4 * 32 = 512 columns
constexpr int kMostStages = 12;
constexpr int kTeams = 3;                    // of 4 warps, one for each 32 lanes of tensor memory, that take weights in turn
constexpr int kThreads = 256 + kTeams * 128; // warps: 0 copies, 1 products, 4-7 results, from 8 on weights
constexpr int kRoom = 200 * 1024;            // of shared memory for stages

struct alignas(16) Shared {
  unsigned char out[4][2048];      // 32 tokens by 32 rows of the result for each of its warps
  unsigned long long full[kMostStages], empty[kMostStages], ready[kRing], taken[kRing], done[2], drained[2];
  uint32_t tmem;
  int abort;
};

struct WideParams {
  const void* bias;
  const void* residual;
  void* y;
  long long residual_row, y_row;
  int tokens, outs, depth;      // outs: rows of the result's weights side; depth: chunks of 64 of the contraction
  int nt, stages, tiles_down, tiles, parts, act;
  bool wide_rows;      // rows of y lie on 16-byte boundaries and are whole vectors
  unsigned* err;
};

// A whole warp's bounded wait, as st::mbar_wait_warp, but the clock is first read after 64 polls: every hop of this kernel's ring is short, and a read of the
// global timer takes longer than it.
__device__ __forceinline__ bool wait(const unsigned long long& barrier, uint32_t parity, volatile int* abort_flag) {
  const uint32_t bar = st::smem_u32(&barrier);
  bool ok = st::mbar_try_wait(bar, parity);
  uint64_t t0 = 0;
  for (uint32_t i = 1; !ok; ++i) {
    ok = st::mbar_try_wait(bar, parity);
    if (ok || (i & 63u)) continue;
    if (*abort_flag) break;
    const uint64_t now = st::globaltimer_ns();
    if (t0 == 0) t0 = now;
    if (now - t0 > st::wait_limit_ns()) {
      *abort_flag = 1;
      break;
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// Codes times their scale, twice each, in the input's type.  bf16 in one step: 64 + code, whose unit is bit 1, times s less 72 s, both of which bf16 holds.  fp16 does not
// hold 72 s of large scales: the code first.
template <typename T> struct Scale;
template <> struct Scale<__nv_bfloat16> {
  __nv_bfloat162 s, less;
  __device__ __forceinline__ void set(uint32_t low16) {
    const uint32_t both = __byte_perm(low16, 0, 0x1010);
    s = *reinterpret_cast<const __nv_bfloat162*>(&both);
    less = __hmul2(s, __float2bfloat162_rn(-72.0f));
  }
  __device__ __forceinline__ uint32_t pair(uint32_t word, int e) const {
    const uint32_t v = ((e == 0 ? word << 1 : word >> (4 * e - 1)) & 0x001E001Eu) | 0x42804280u;
    const __nv_bfloat162 d = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&v), s, less);
    return *reinterpret_cast<const uint32_t*>(&d);
  }
};
template <> struct Scale<__half> {
  __half2 s;
  __device__ __forceinline__ void set(uint32_t low16) { s = __float2half2_rn(bf16_bits(low16 & 0xFFFFu)); }
  __device__ __forceinline__ uint32_t pair(uint32_t word, int e) const {
    const uint32_t v = codes_to_pair<__half>(word, e);
    const __half2 d = __hmul2(*reinterpret_cast<const __half2*>(&v), s);
    return *reinterpret_cast<const uint32_t*>(&d);
  }
};
__device__ __forceinline__ uint32_t turn_over(uint32_t block) {      // an 8 x 8 block of 16-bit numbers, a row per 4 lanes
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(block));
  return r;
}
// 16 lanes by 32 columns: registers 2 i and 2 i + 1 of lane l hold column 4 i + l % 4 of rows l / 4 and l / 4 + 8.
__device__ __forceinline__ void tmem_st_16x32(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
               "r"(r[14]), "r"(r[15])
               : "memory");
}

// A tile is 128 rows of the result's weights side by nt tokens.  In a cluster of `parts` blocks each contracts its share of the depth, and all of them join the sums.
template <typename T, bool TURN, int GROUP>
__global__ void __launch_bounds__(kThreads, 1) wide_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_codes,
                                                           const __grid_constant__ CUtensorMap map_scales, WideParams p) {
  extern __shared__ __align__(1024) unsigned char unaligned[];
  __shared__ Shared sh;
  unsigned char* raw = unaligned + (-st::smem_u32(unaligned) & 1023u);      // the swizzle counts from 1024-byte boundaries
  constexpr int kCodes = 4096;                                                     // bytes of a stage: 8 tiles of 512
  constexpr int kScaleGroups = TURN ? 128 / GROUP : GROUP == 32 ? 2 : 1;            // of a stage and tile of 16 rows
  constexpr int kScales = (TURN ? 4 : 8) * kScaleGroups * 32;
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  volatile int* abort_flag = &sh.abort;
  const int part = p.parts > 1 ? static_cast<int>(st::cluster_ctarank()) : 0;
  const int first_tile = blockIdx.x / p.parts, tile_step = gridDim.x / p.parts;
  const int c0 = p.depth * part / p.parts, c1 = p.depth * (part + 1) / p.parts;
  const uint32_t x_bytes = p.nt * 128, smem_x = st::smem_u32(raw), smem_codes = smem_x + p.stages * x_bytes, smem_scales = smem_codes + p.stages * kCodes;

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) st::mbar_init(st::smem_u32(&sh.full[i]), 1), st::mbar_init(st::smem_u32(&sh.empty[i]), 1);
    for (int i = 0; i < kRing; ++i) st::mbar_init(st::smem_u32(&sh.ready[i]), 4), st::mbar_init(st::smem_u32(&sh.taken[i]), 1);
    for (int i = 0; i < 2; ++i) st::mbar_init(st::smem_u32(&sh.done[i]), 1), st::mbar_init(st::smem_u32(&sh.drained[i]), 4);
    sh.abort = 0;
    st::fence_barrier_init();
    st::tma_prefetch_desc(&map_x), st::tma_prefetch_desc(&map_codes), st::tma_prefetch_desc(&map_scales);
  }
  // Tensor memory is asked for when the kernel before has given back its own, and before the next one's blocks may come and ask.  Blocks of other kernels
  // that hold some do not fit beside this one's shared memory, so that a cluster's blocks never wait for memory that waits for them.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 1) {
    st::tmem_alloc(st::smem_u32(&sh.tmem), 512);
    st::tmem_relinquish();
  }
  st::tc_fence_before();
  __syncthreads();
  st::tc_fence_after();
  const uint32_t tmem = sh.tmem, operands = tmem + 2 * kMostTokens;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == 0) {
    const bool leader = st::elect_one();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = first_tile; t < p.tiles && ok; t += tile_step) {
      const int down = t % p.tiles_down, m0 = t / p.tiles_down * p.nt;
      for (int c = c0; c < c1; ++c) {
        if (!(ok = wait(sh.empty[stage], phase ^ 1u, abort_flag))) break;
        if (leader) {
          const uint32_t bar = st::smem_u32(&sh.full[stage]);
          st::mbar_arrive_expect_tx(bar, x_bytes + kCodes + kScales);
          if (TURN) {      // 64 weight rows (4 tiles) by 128 columns (2 tiles)
            st::tma_load_2d(smem_codes + stage * kCodes, &map_codes, bar, down * 256, c * 4);
            st::tma_load_2d(smem_scales + stage * kScales, &map_scales, bar, down * (128 / GROUP) * 16, c * 4);
          } else {         // 128 weight rows by 64 columns
            st::tma_load_2d(smem_codes + stage * kCodes, &map_codes, bar, c * 128, down * 8);
            st::tma_load_2d(smem_scales + stage * kScales, &map_scales, bar, c * 64 / GROUP * 16, down * 8);
          }
          st::tma_load_2d(smem_x + stage * x_bytes, &map_x, bar, c * 64, m0);
        }
        if (++stage == p.stages) stage = 0, phase ^= 1u;
      }
    }
  } else if (warp == 1) {
    const bool leader = st::elect_one();
    const uint32_t idesc = st::make_idesc_bf16(128, p.nt, false, false) & ~(std::is_same<T, __half>::value ? (1u << 7 | 1u << 10) : 0u);
    const uint32_t high = st::smem_desc_hi(1024);
    int stage = 0, ring = 0, buf = 0;
    uint32_t phase = 0, ring_phase = 0, buf_phase = 0;
    bool ok = true;
    for (int t = first_tile; t < p.tiles && ok; t += tile_step) {
      if (!(ok = wait(sh.drained[buf], buf_phase ^ 1u, abort_flag))) break;
      st::tc_fence_after();
      for (int c = c0; c < c1; ++c) {
        if (!(ok = wait(sh.full[stage], phase, abort_flag))) break;
        if (!(ok = wait(sh.ready[ring], ring_phase, abort_flag))) break;
        st::tc_fence_after();
        if (leader) {
          const uint32_t low = st::smem_desc_lo(smem_x + stage * x_bytes, 16);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            st::umma_bf16_ts_split(tmem + buf * kMostTokens, operands + ring * 32 + k * 8, low + 2 * k, high, idesc, c > c0 || k > 0);
          st::umma_commit(st::smem_u32(&sh.empty[stage]));
          st::umma_commit(st::smem_u32(&sh.taken[ring]));
          if (c == c1 - 1) st::umma_commit(st::smem_u32(&sh.done[buf]));
        }
        __syncwarp();
        if (++stage == p.stages) stage = 0, phase ^= 1u;
        if (++ring == kRing) ring = 0, ring_phase ^= 1u;
      }
      if (++buf == 2) buf = 0, buf_phase ^= 1u;
    }
  } else if (warp >= 8) {
    const int quarter = warp & 3, team = (warp >> 2) - 2;
    const uint32_t to = operands + (static_cast<uint32_t>(quarter * 32) << 16);
    int n = team;                                          // the block's chunks count on from tile to tile
    int stage = team % p.stages, ring = team % kRing;
    uint32_t phase = 0, ring_phase = 0;
    const int own = c1 - c0, all = own * ((p.tiles - first_tile + tile_step - 1) / tile_step);
    for (; n < all; n += kTeams) {
      if (!wait(sh.full[stage], phase, abort_flag)) break;
      const unsigned char* codes = raw + (smem_codes - smem_x) + stage * kCodes;
      const unsigned char* scales = raw + (smem_scales - smem_x) + stage * kScales;
      uint32_t r[2][16];
#pragma unroll
      for (int half = 0; half < 2; ++half) {               // 16 lanes each
        if (TURN) {      // word `quarter % 2 * 2 + half` of column tile quarter / 2, from each of the 4 row tiles
          const int s = (quarter & 1) * 2 + half, group = ((quarter >> 1) * 64 + s * 16) / GROUP;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t word = *reinterpret_cast<const uint32_t*>(codes + (i * 2 + (quarter >> 1)) * kTileBytes + lane * 16 + s * 4);
            const uint32_t both = *reinterpret_cast<const uint32_t*>(scales + (i * kScaleGroups + group) * 32 + (lane >> 2) * 4);
            Scale<T> low, high;
            low.set(both), high.set(both >> 16);
            r[half][4 * i] = turn_over(low.pair(word, 0)), r[half][4 * i + 1] = turn_over(low.pair(word, 2));
            r[half][4 * i + 2] = turn_over(high.pair(word, 1)), r[half][4 * i + 3] = turn_over(high.pair(word, 3));
          }
        } else {
          const int u = quarter * 2 + half;
          const uint4 four = *reinterpret_cast<const uint4*>(codes + u * kTileBytes + lane * 16);
          const uint32_t word[4] = {four.x, four.y, four.z, four.w};
          Scale<T> low, high;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (i % (4 / kScaleGroups) == 0) {
              const uint32_t both = *reinterpret_cast<const uint32_t*>(scales + (u * kScaleGroups + i / (4 / kScaleGroups)) * 32 + (lane >> 2) * 4);
              low.set(both), high.set(both >> 16);
            }
            r[half][4 * i] = low.pair(word[i], 0), r[half][4 * i + 1] = high.pair(word[i], 1);
            r[half][4 * i + 2] = low.pair(word[i], 2), r[half][4 * i + 3] = high.pair(word[i], 3);
          }
        }
      }
      if (!wait(sh.taken[ring], ring_phase ^ 1u, abort_flag)) break;
      st::tc_fence_after();
      tmem_st_16x32(to + ring * 32, r[0]);
      tmem_st_16x32(to + (16u << 16) + ring * 32, r[1]);
      st::tmem_st_wait();
      st::tc_fence_before();
      __syncwarp();
      if (lane == 0) st::mbar_arrive(st::smem_u32(&sh.ready[ring]));
      stage += kTeams;
      while (stage >= p.stages) stage -= p.stages, phase ^= 1u;
      ring += kTeams;
      if (ring >= kRing) ring -= kRing, ring_phase ^= 1u;
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3;
    const T* bias = static_cast<const T*>(p.bias);
    const T* residual = static_cast<const T*>(p.residual);
    T* y = static_cast<T*>(p.y);
    unsigned char* out = sh.out[quarter];
    int buf = 0;
    uint32_t buf_phase = 0;
    for (int t = first_tile; t < p.tiles; t += tile_step) {
      if (!wait(sh.done[buf], buf_phase, abort_flag)) break;
      st::tc_fence_after();
      const int r0 = t % p.tiles_down * 128 + quarter * 32, r = r0 + lane, m0 = t / p.tiles_down * p.nt, end = min(p.nt, p.tokens - m0);
      const float b = bias != nullptr && p.parts == 1 && r < p.outs ? to_float(bias[r]) : 0.0f;
#pragma unroll 1
      for (int at = 0; at < end; at += 32) {
        uint32_t v[32];
        st::tmem_ld_32x32(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + buf * kMostTokens + at, v);
        st::tmem_ld_wait();
        if (p.parts > 1) {      // this block's share of the sums, for the cluster
          float* sums = reinterpret_cast<float*>(raw) + quarter * 32 + lane;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (at + i < end) sums[(at + i) * 128] = __uint_as_float(v[i]);
          continue;
        }
        float f[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(v[i]) + b;
        if (p.act == 1) {
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = activate(f[i], 1);
        } else if (p.act == 2) {
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = st::gelu_tanh(f[i]);
        }
        if (residual && r < p.outs) {
          const T* from = residual + (m0 + at) * p.residual_row + r;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (at + i < end) f[i] += to_float(*from);
            from += p.residual_row;
          }
        }
        // to rows of 32: a token's 64 bytes, which 4 lanes take to memory
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 32; ++i) *reinterpret_cast<T*>(out + i * 64 + lane * 2) = from_float<T>(f[i]);
        __syncwarp();
        T* to = y + (m0 + at) * p.y_row + r0;
        if (p.wide_rows) {
          const int col = (lane & 3) * 8;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int m = i * 8 + (lane >> 2);
            if (at + m < end && r0 + col < p.outs) *reinterpret_cast<uint4*>(to + m * p.y_row + col) = *reinterpret_cast<const uint4*>(out + m * 64 + col * 2);
          }
        } else if (r < p.outs) {
          for (int i = 0; i < 32 && at + i < end; ++i) to[i * p.y_row + lane] = *reinterpret_cast<const T*>(out + i * 64 + lane * 2);
        }
      }
      st::tc_fence_before();
      __syncwarp();
      if (lane == 0) st::mbar_arrive(st::smem_u32(&sh.drained[buf]));
      if (++buf == 2) buf = 0, buf_phase ^= 1u;
    }
  }
  st::tc_fence_before();
  __syncwarp();
  if (p.parts > 1) {
    // all copies have been read and all products are done, or a wait ran out and the result is void: the stages' memory holds the sums
    st::cluster_sync();
    const T* bias = static_cast<const T*>(p.bias);
    const T* residual = static_cast<const T*>(p.residual);
    T* y = static_cast<T*>(p.y);
    const int down = first_tile % p.tiles_down, m0 = first_tile / p.tiles_down * p.nt;
    const int r = down * 128 + (threadIdx.x & 127);
    for (int at = part + p.parts * (threadIdx.x >> 7); at < p.nt; at += p.parts * (kThreads / 128)) {
      const int m = m0 + at;
      if (m >= p.tokens || r >= p.outs) break;
      float f = 0.0f;
      for (int q = 0; q < p.parts; ++q) {
        float s;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(s) : "r"(st::cluster_map(smem_x + (at * 128 + (threadIdx.x & 127)) * 4, q)));
        f += s;
      }
      if (bias) f += to_float(bias[r]);
      f = activate(f, p.act);
      if (residual) f += to_float(residual[m * p.residual_row + r]);
      y[m * p.y_row + r] = from_float<T>(f);
    }
    st::cluster_sync();
  } else {
    __syncthreads();
  }
  if (*abort_flag) {
    if (threadIdx.x == 0) st::report_error(p.err, st::ERR_MBAR_TIMEOUT, 0x4B00u);
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);      // copies in flight land before their memory is given up
  }
  if (warp == 1) {
    st::tc_fence_after();
    st::tmem_dealloc(tmem, 512);
  }
}

template <typename T, bool TURN, int GROUP>
int launch(const st4::WideArgs& a, cudaStream_t stream) {
  const int sms = st::sm_count();
  WideParams p{a.bias, a.residual, a.y, a.residual_row, a.y_row, a.tokens, TURN ? a.cols : a.rows, ((TURN ? a.rows : a.cols) + 63) / 64, 0, 0, 0, 0, 1, a.act, false, st::error_word()};
  p.wide_rows = (reinterpret_cast<uintptr_t>(a.y) & 15) == 0 && a.y_row % 8 == 0 && p.outs % 8 == 0;
  p.tiles_down = (p.outs + 127) / 128;
  // tokens of a tile: the size whose rounds over the SMs take the fewest tokens' time; a tile of fewer than 64 takes as long as one of 64, its weights' conversion
  long long best = -1;
  for (int nt = kMostTokens; nt >= 16; nt -= 16) {
    const long long across = (a.tokens + nt - 1) / nt, rounds = (across * p.tiles_down + sms - 1) / sms, cost = rounds * (nt > 64 ? nt : 64);
    if (best < 0 || cost < best || (cost == best && across == (a.tokens + p.nt - 1) / p.nt)) best = cost, p.nt = nt;
  }
  const long long tiles = static_cast<long long>(p.tiles_down) * ((a.tokens + p.nt - 1) / p.nt);
  if (tiles > 1 << 30) return st::fail(ST_ERR_TOO_LARGE, "int4: too many rows");
  p.tiles = static_cast<int>(tiles);
  while (p.parts < 8 && p.tiles * p.parts * 2 <= sms && p.depth >= 4 * p.parts) p.parts *= 2;
  constexpr int kScales = (TURN ? 4 * (128 / GROUP) : 8 * (GROUP == 32 ? 2 : 1)) * 32;
  const int stage = p.nt * 128 + 4096 + kScales;
  p.stages = min(kMostStages, kRoom / stage);
  CUtensorMap mx, mc, ms;
  const uint64_t units = (a.rows + 15) / 16, chunks = (a.cols + 63) / 64, groups = (a.cols + GROUP - 1) / GROUP;
  {
    const uint64_t dims[2] = {static_cast<uint64_t>(TURN ? a.rows : a.cols), static_cast<uint64_t>(a.tokens)}, strides[1] = {static_cast<uint64_t>(a.x_row) * 2};
    const uint32_t box[2] = {64, static_cast<uint32_t>(p.nt)};
    if (!st::encode_tmap(&mx, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.x, dims, strides, box,
                         CU_TENSOR_MAP_SWIZZLE_128B))
      return ST_ERR_CUDA;
  }
  {
    const uint64_t dims[2] = {chunks * 128, units}, strides[1] = {chunks * 512};
    const uint32_t box[2] = {TURN ? 256u : 128u, TURN ? 4u : 8u};
    if (!st::encode_tmap(&mc, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, a.codes, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE)) return ST_ERR_CUDA;
  }
  {
    const uint64_t dims[2] = {groups * 16, units}, strides[1] = {groups * 32};
    const uint32_t box[2] = {static_cast<uint32_t>(TURN ? 128 / GROUP * 16 : GROUP == 32 ? 32 : 16), TURN ? 4u : 8u};
    if (!st::encode_tmap(&ms, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.scales, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE)) return ST_ERR_CUDA;
  }
  constexpr int smem = kRoom + 1024;      // always: one block per SM
  static bool opted[st::kMaxDevices];
  const int dev = st::current_device();
  if (!opted[dev]) {
    ST_CUDA_CHECK(cudaFuncSetAttribute(wide_kernel<T, TURN, GROUP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    opted[dev] = true;
  }
  const int blocks = p.parts > 1 ? p.tiles * p.parts : min(p.tiles, sms);
  const cudaError_t e = st::chained(wide_kernel<T, TURN, GROUP>, dim3(blocks), dim3(kThreads), smem, stream, p.parts)(mx, mc, ms, p);
  return e == cudaSuccess ? ST_OK : st::fail_cuda(e, "int4 wide");
}

template <typename T, bool TURN>
int by_group(const st4::WideArgs& a, cudaStream_t stream) {
  if (a.group == 32) return launch<T, TURN, 32>(a, stream);
  if (a.group == 64) return launch<T, TURN, 64>(a, stream);
  return launch<T, TURN, 128>(a, stream);
}
}  // namespace

int st4::wide(const WideArgs& a, int type, bool turn, cudaStream_t stream) {
  if (type == 0) return turn ? by_group<__nv_bfloat16, true>(a, stream) : by_group<__nv_bfloat16, false>(a, stream);
  return turn ? by_group<__half, true>(a, stream) : by_group<__half, false>(a, stream);
}
