// Products of many rows with weights of four bits on tcgen05:  y = act(x W^T + bias) + residual  and  dx = dy W.
//
// The weights are the 128-row operand and lie in tensor memory: warps take codes from shared memory, make them numbers q s of the input's type (exact), and write
// them from registers in the order in which they come (int4.cuh).  The rows of x (or dy) are the other operand, up to 192 of them, by tiled copies.  So
// a tile's sums stand as [weight row or column][token], and a weight is converted once for 192 tokens and never passes through shared memory as 16 bits.
// dx contracts over the weights' rows: the same tiles, each 8 x 8 block turned over in registers.
//
// Bound by the products where rows are many: 4096 rows, 2048 inputs to 8192 outputs, 98 to 103 us in two runs, 1337 to 1398 TFLOP/s of the 1678 that a library's product reaches in
// bursts, the tensor pipe busy 78%; the gradient 106 to 112, 72%.  777 rows, 2048 to 6144, 21 us: two rounds of tiles.  64 rows, 8192 to 2048, 11 to 12.  Few rows are bound by
// conversion: 32 rows, 8192 to 18944, take 26 us (the codes' bytes alone 13), which leaves some 720 cycles for each of a block's 64 steps; a team converts a step in 1250 cycles and stores it
// in 250, three teams at a time.  50304 x 2048 by 16, 32 and 64 rows 19.8, 20.5 and 22.5 us.  The gradient of one row to 64: 7.0 to 8.7 us at 2048 x 2048, 9.8 to 11.5 with four times the weights.
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "../common/chain.cuh"
#include "int4.cuh"
#include "int4_wide.h"

namespace {
using namespace st4;

constexpr int kMostRing = 6;                 // weight operands in tensor memory, 64 columns each, behind two results: as many as fit
constexpr int kMostTokens = 192;             // of a tile: 2 * 192 + 2 * 64 = 512 columns
constexpr int kMostStages = 8;
constexpr int kMostParts = 8;                // blocks of a cluster
constexpr int kCodes = 8192;                 // bytes of a stage: 128 rows by 128 columns of the weights, 8 by 2 tiles
constexpr int kTeams = 3;                    // of 4 warps, one for each 32 lanes of tensor memory, that take weights in turn
constexpr int kThreads = 256 + kTeams * 128; // warps: 0 copies, 1 products, 4-7 results, from 8 on weights
constexpr int kRoom = 200 * 1024;            // of shared memory for stages

struct alignas(16) Shared {
  unsigned char out[4][2048];      // 32 tokens by 32 rows of the result for each of its warps
  // Copies land in any order, and a team looks at every third stage only: with one barrier a stage it could come by before the turn ahead of its own had
  // landed, which the parity of its own would take for done.  Two barriers a stage, in turns: the turn before on the same one is long used up.
  unsigned long long full[2 * kMostStages], empty[kMostStages], ready[kMostRing], taken[kMostRing], done[2], drained[2];
  uint32_t tmem;
  int abort;
};

struct WideParams {
  const void* bias;
  const void* residual;
  void* y;
  long long residual_row, y_row;
  int tokens, outs, depth;      // outs: columns of the result; depth: steps of 128 of the contraction
  int nt, stages, ring, teams, tiles_down, tiles, parts, act;
  bool wide_rows;      // rows of y lie on 16-byte boundaries and are whole vectors
  unsigned* err;
};

__device__ __forceinline__ bool wait(const unsigned long long& barrier, uint32_t parity, volatile int* abort_flag) {      // the whole warp
  return st::mbar_wait_warp(st::smem_u32(&barrier), parity, abort_flag);
}
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
  constexpr int kScaleGroups = 128 / GROUP, kScales = 8 * kScaleGroups * 32;      // of a stage: groups of a tile row, bytes
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  volatile int* abort_flag = &sh.abort;
  const int part = p.parts > 1 ? static_cast<int>(st::cluster_ctarank()) : 0;
  const int first_tile = blockIdx.x / p.parts, tile_step = gridDim.x / p.parts;
  const int c0 = p.depth * part / p.parts, c1 = p.depth * (part + 1) / p.parts;
  const uint32_t x_bytes = p.nt * 256, smem_x = st::smem_u32(raw), smem_codes = smem_x + p.stages * x_bytes, smem_scales = smem_codes + p.stages * kCodes;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * p.stages; ++i) st::mbar_init(st::smem_u32(&sh.full[i]), 1);
    for (int i = 0; i < p.stages; ++i) st::mbar_init(st::smem_u32(&sh.empty[i]), 1);
    for (int i = 0; i < p.ring; ++i) st::mbar_init(st::smem_u32(&sh.ready[i]), 4), st::mbar_init(st::smem_u32(&sh.taken[i]), 1);
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
  const uint32_t tmem = sh.tmem, operands = tmem + 512 - 64 * p.ring;
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
          const uint32_t bar = st::smem_u32(&sh.full[stage + phase * p.stages]);
          st::mbar_arrive_expect_tx(bar, x_bytes + kCodes + kScales);
          const int row = TURN ? c : down, col = TURN ? down : c;      // of the 128 x 128 blocks of the weights
          st::tma_load_2d(smem_codes + stage * kCodes, &map_codes, bar, col * 256, row * 8);
          st::tma_load_2d(smem_scales + stage * kScales, &map_scales, bar, col * kScaleGroups * 16, row * 8);
          st::tma_load_2d(smem_x + stage * x_bytes, &map_x, bar, c * 128, m0);
          st::tma_load_2d(smem_x + stage * x_bytes + p.nt * 128, &map_x, bar, c * 128 + 64, m0);
        }
        if (++stage == p.stages) stage = 0, phase ^= 1u;
      }
    }
  } else if (warp == 1) {
    const bool leader = st::elect_one();
    const uint32_t idesc = st::make_idesc_bf16(128, p.nt, false, false) & ~(std::is_same<T, __half>::value ? (1u << 7 | 1u << 10) : 0u);
    const uint32_t high = st::smem_desc_hi(1024);
    int stage = 0, ring = 0, buf = 0;
    uint32_t ring_phase = 0, buf_phase = 0;
    bool ok = true;
    for (int t = first_tile; t < p.tiles && ok; t += tile_step) {
      if (!(ok = wait(sh.drained[buf], buf_phase ^ 1u, abort_flag))) break;
      st::tc_fence_after();
      for (int c = c0; c < c1; ++c) {
        if (!(ok = wait(sh.ready[ring], ring_phase, abort_flag))) break;      // its team has waited for the stage, x with it
        st::tc_fence_after();
        if (leader) {
          const uint32_t low = st::smem_desc_lo(smem_x + stage * x_bytes, 16);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            st::umma_bf16_ts_split(tmem + buf * p.nt, operands + ring * 64 + k * 8, low + (k >> 2) * p.nt * 8 + 2 * (k & 3), high, idesc, c > c0 || k > 0);
          st::umma_commit(st::smem_u32(&sh.empty[stage]));
          st::umma_commit(st::smem_u32(&sh.taken[ring]));
          if (c == c1 - 1) st::umma_commit(st::smem_u32(&sh.done[buf]));
        }
        __syncwarp();
        if (++stage == p.stages) stage = 0;
        if (++ring == p.ring) ring = 0, ring_phase ^= 1u;
      }
      if (++buf == 2) buf = 0, buf_phase ^= 1u;
    }
  } else if (warp >= 8) {
    const int quarter = warp & 3, team = (warp >> 2) - 2;
    const uint32_t to = operands + (static_cast<uint32_t>(quarter * 32) << 16);
    int n = team;                                          // the block's stages count on from tile to tile
    int stage = team % p.stages, filled = team, ring = team % p.ring;
    uint32_t fill_phase = 0, ring_phase = team / p.ring & 1;
    const int own = c1 - c0, all = own * ((p.tiles - first_tile + tile_step - 1) / tile_step);
    for (; n < all && team < p.teams; n += p.teams) {
      if (!wait(sh.full[filled], fill_phase, abort_flag)) break;
      const unsigned char* codes = raw + (smem_codes - smem_x) + stage * kCodes;
      const unsigned char* scales = raw + (smem_scales - smem_x) + stage * kScales;
      uint32_t r[2][2][16];      // [64 of the 128 numbers of every lane][16 lanes]
      if (TURN) {      // words `quarter % 2 * 2` and the next of column tile quarter / 2, 16 columns each, from the 8 row tiles; both lie in one group
        const int s = (quarter & 1) * 2, group = ((quarter >> 1) * 64 + s * 16) / GROUP;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint2 words = *reinterpret_cast<const uint2*>(codes + (i * 2 + (quarter >> 1)) * kTileBytes + lane * 16 + s * 4);
          const uint32_t both = *reinterpret_cast<const uint32_t*>(scales + (i * kScaleGroups + group) * 32 + (lane >> 2) * 4);
          Scale<T> low, high;
          low.set(both), high.set(both >> 16);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t word = half ? words.y : words.x;
            uint32_t* to = r[i >> 2][half] + 4 * (i & 3);
            to[0] = turn_over(low.pair(word, 0)), to[1] = turn_over(low.pair(word, 2));
            to[2] = turn_over(high.pair(word, 1)), to[3] = turn_over(high.pair(word, 3));
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int u = quarter * 2 + half;
            const uint4 four = *reinterpret_cast<const uint4*>(codes + (u * 2 + k) * kTileBytes + lane * 16);
            const uint32_t word[4] = {four.x, four.y, four.z, four.w};
            Scale<T> low, high;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (i == 0 || (GROUP == 32 && i == 2)) {
                const uint32_t both = *reinterpret_cast<const uint32_t*>(scales + (u * kScaleGroups + (k * 64 + i * 16) / GROUP) * 32 + (lane >> 2) * 4);
                low.set(both), high.set(both >> 16);
              }
              r[k][half][4 * i] = low.pair(word[i], 0), r[k][half][4 * i + 1] = high.pair(word[i], 1);
              r[k][half][4 * i + 2] = low.pair(word[i], 2), r[k][half][4 * i + 3] = high.pair(word[i], 3);
            }
          }
      }
      if (!wait(sh.taken[ring], ring_phase ^ 1u, abort_flag)) break;
      st::tc_fence_after();
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        tmem_st_16x32(to + ring * 64 + k * 32, r[k][0]);
        tmem_st_16x32(to + (16u << 16) + ring * 64 + k * 32, r[k][1]);
      }
      st::tmem_st_wait();
      st::tc_fence_before();
      __syncwarp();
      if (lane == 0) st::mbar_arrive(st::smem_u32(&sh.ready[ring]));
      stage = (stage + p.teams) % p.stages;
      filled += p.teams;
      if (filled >= 2 * p.stages) filled -= 2 * p.stages, fill_phase ^= 1u;
      ring += p.teams;
      while (ring >= p.ring) ring -= p.ring, ring_phase ^= 1u;
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
        st::tmem_ld_32x32(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + buf * p.nt + at, v);
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
      float s[kMostParts], f = 0.0f;
#pragma unroll
      for (int q = 0; q < kMostParts; ++q)      // all on their way before the first is used
        if (q < p.parts) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(s[q]) : "r"(st::cluster_map(smem_x + (at * 128 + (threadIdx.x & 127)) * 4, q)));
#pragma unroll
      for (int q = 0; q < kMostParts; ++q)
        if (q < p.parts) f += s[q];
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
  WideParams p{a.bias, a.residual, a.y, a.residual_row, a.y_row, a.tokens, TURN ? a.cols : a.rows, ((TURN ? a.rows : a.cols) + 127) / 128, 0, 0, 0, 0, 0, 0, 1, a.act, false, st::error_word()};
  p.wide_rows = (reinterpret_cast<uintptr_t>(a.y) & 15) == 0 && a.y_row % 8 == 0 && p.outs % 8 == 0;
  p.tiles_down = (p.outs + 127) / 128;
  constexpr int smem = kRoom + 1024;      // always: one block per SM
  static int clusters[st::kMaxDevices][kMostParts + 1];      // that run at the same time, by their size
  int (&at_once)[kMostParts + 1] = clusters[st::current_device()];
  if (at_once[1] == 0) {
    ST_CUDA_CHECK(cudaFuncSetAttribute(wide_kernel<T, TURN, GROUP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    for (int n = kMostParts; n > 0; --n) {
      cudaLaunchAttribute attr{};
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = n, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(n * sms), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = smem, cfg.attrs = &attr, cfg.numAttrs = 1;
      int found = 0;
      ST_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&found, wide_kernel<T, TURN, GROUP>, &cfg));
      at_once[n] = n > 1 ? found : sms;
    }
  }
  // Tokens of a tile, and blocks that share one, by what steps of 128 in a row cost: its tokens' time and that of 100 more, with fewer than 3 weight operands (above
  // 160 tokens) of 140 more; a cluster's start and join as much as 1150 (2.4 us).  4096 x 8192 x 2048 in tiles of 96 125 us, 128 112, 160 104, 176 111, 192 106;
  // 64 x 2048 x 8192 with 1 block to a tile 24.4 us, 2 17.8, 4 12.3, 6 10.7.  Clusters that do not all run at once take twice as long: with 8 blocks 18.4.
  long long best = -1;
  for (int nt = kMostTokens; nt >= 16; nt -= 16) {
    const long long tiles = static_cast<long long>(p.tiles_down) * ((a.tokens + nt - 1) / nt);
    for (int parts = 1; parts <= kMostParts && parts <= p.depth; ++parts) {
      if (parts > 1 && tiles > at_once[parts]) continue;
      const long long steps = parts > 1 ? (p.depth + parts - 1) / parts : (tiles + sms - 1) / sms * p.depth;
      const long long cost = steps * (nt + (nt > 160 ? 140 : 100)) + (parts > 1 ? 1150 : 0);
      if (best < 0 || cost < best) best = cost, p.nt = nt, p.parts = parts, p.tiles = static_cast<int>(min(tiles, 2147483647LL));
    }
  }
  if (p.tiles > 1 << 30) return st::fail(ST_ERR_TOO_LARGE, "int4: too many rows");
  const int stage = p.nt * 256 + kCodes + 8 * (128 / GROUP) * 32;
  p.stages = min(kMostStages, kRoom / stage);
  p.ring = min(kMostRing, (512 - 2 * p.nt) / 64);
  p.teams = min(kTeams, min(p.ring, p.stages));      // no more: a barrier tells one turn of a ring from the next, not from the one after
  // a stage two turns back is used up: the team's last operand waited for the product `ring` before it
  if (2 * p.stages < p.teams + p.ring) return st::fail(ST_ERR_INVALID, "int4: too few stages");
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
    const uint32_t box[2] = {256, 8};
    if (!st::encode_tmap(&mc, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, a.codes, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE)) return ST_ERR_CUDA;
  }
  {
    const uint64_t dims[2] = {groups * 16, units}, strides[1] = {groups * 32};
    const uint32_t box[2] = {128 / GROUP * 16, 8};
    if (!st::encode_tmap(&ms, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.scales, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE)) return ST_ERR_CUDA;
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
