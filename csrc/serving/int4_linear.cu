// Products with weights of four bits:  y = act(x W^T + bias) + residual,  W = q s  (int4.cuh): few rows here, by matrix instructions on codes converted in registers.
//
// At a floor of the codes' bytes no single thing bounds it: one row, 2048 inputs to 50304 outputs in groups of 128, takes 17.1 to 17.7 us in bf16, 3.1 TB/s.  60% of the issue slots are
// taken, and of what keeps a warp from issuing, waiting for memory is the most (1.9 warps an issue; instructions before 1.6, the ALU pipe 1.1, barriers 0.7).  A
// slice of 16 rows by 256 columns takes 378 instructions of a warp, half of which turn codes into numbers (a shift, a selection and a subtraction for two).  444 blocks take 3144 tile rows in 8
// turns where 7.08 would do, and a store of partial sums meets three bank conflicts.  In groups of 64 2048 to 2048 takes 3.5 us, 2048 to 8192 5.6 to 6.0, 8192 to 2048 7.3.
// tcgen05 needs the same instructions and a way through tensor memory (int4_wide.cu); is_wide says where it pays.
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "../common/chain.cuh"
#include "int4.cuh"
#include "int4_wide.h"

namespace {
using namespace st4;
using st::chain_begin;

struct LinearParams {
  const void* x;
  const uint8_t* codes;
  const __nv_bfloat16* scales;
  const void* bias;
  const void* residual;
  void* y;
  long long x_row, residual_row, y_row;      // in elements
  int tokens, rows, cols, groups, chunks, units, group, act;
  bool wide;      // rows of x lie on 16-byte boundaries
  int parts;      // blocks of a cluster
};

template <typename T> __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]);
template <> __device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
template <> __device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// x in shared memory: a token's 64 columns of a chunk are 128 bytes, in which the 16 bytes at 64 p + 16 t hold what lane t of a row's 4 takes to steps 2 p and 2 p + 1:
// columns 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of each.  Tokens are 64 bytes more than a whole number of 128 apart, so that 8 lanes read from all banks.
constexpr int kWarps = 8, kMostParts = 8;

// A thread takes 8 columns (step s, half h; word t of them goes to 16 (s / 2) + 4 t + 2 (s % 2) + h) of every second or of all tokens, four at a time.  What stands in the
// place of tokens that there are none of does not matter: they are columns of their own.
template <typename T, int COLUMNS>
__device__ __forceinline__ void stage_tokens(const T* x, long long x_row, uint32_t* to, int stride, int tokens, int k0, int cols, bool wide) {
  constexpr int kVectors = COLUMNS / 8, kRows = kWarps * 32 / kVectors, kAhead = 4;
  const int j = threadIdx.x % kVectors, k = k0 + j * 8;
  if (k >= (cols + 63) / 64 * 64) return;
  uint32_t* at = to + (j >> 3) * 32 + ((j >> 2) & 1) * 16 + ((j >> 1) & 1) * 2 + (j & 1);
  for (int m0 = threadIdx.x / kVectors; m0 < tokens; m0 += kAhead * kRows) {
    uint4 v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int m = m0 + i * kRows;
      const T* from = x + m * x_row + k;
      v[i] = make_uint4(0, 0, 0, 0);
      if (m >= tokens) continue;
      if (wide && k + 8 <= cols) {
        v[i] = *reinterpret_cast<const uint4*>(from);
      } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(from);
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k + e < cols) w[e / 2] |= static_cast<uint32_t>(h[e]) << (16 * (e % 2));
        v[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int m = m0 + i * kRows;
      if (m >= tokens) continue;
      at[m * stride] = v[i].x, at[m * stride + 4] = v[i].y, at[m * stride + 8] = v[i].z, at[m * stride + 12] = v[i].w;
    }
  }
}

// What a warp reads of a tile row: C chunks of codes side by side, 16 bytes a lane each, and their scales, 8 words (of 2 rows) to a group.
template <int C, int GROUP>
struct Slice {
  static constexpr int kScales = C * 64 / GROUP > 0 ? C * 64 / GROUP : 1, kWords = (kScales * 8 + 31) / 32;
  uint4 w[C];
  uint32_t s[kWords];
  // codes and scales: of the tile row
  __device__ __forceinline__ void load(const uint8_t* codes, const __nv_bfloat16* scales, int c0, int chunks, int groups, int lane) {
    const uint8_t* from = codes + static_cast<long long>(c0) * kTileBytes + lane * 16;
    const int g0 = c0 * 64 / GROUP;
    const uint32_t* words = reinterpret_cast<const uint32_t*>(scales) + g0 * 8 + lane;
    // groups of 32: the last chunk may have one, and what follows in memory are the next tile row's
    if (c0 + C <= chunks && (GROUP > 32 || g0 + kScales <= groups)) {
#pragma unroll
      for (int i = 0; i < C; ++i) w[i] = *reinterpret_cast<const uint4*>(from + i * kTileBytes);
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        if (kScales * 8 % 32 == 0 || i * 32 + lane < kScales * 8) s[i] = words[i * 32];
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i)
        if (c0 + i < chunks) w[i] = *reinterpret_cast<const uint4*>(from + i * kTileBytes);
#pragma unroll
      for (int i = 0; i < kWords; ++i) s[i] = i * 32 + lane < min(kScales, groups - g0) * 8 ? words[i * 32] : 0u;
    }
  }
  // of chunk i, half k of it where groups are halves
  __device__ __forceinline__ uint32_t scale(int i, int k, int lane) const {
    const int at = ((i * 64 + k * 32) / GROUP) * 8;
    return __shfl_sync(0xffffffffu, s[at / 32], at % 32 + (lane >> 2));
  }
};

// Blocks take tile rows (16 weight rows) in turns; their 8 warps share the columns, C chunks of 64 each: a stretch of 8 C.  Where there are more columns, a cluster's
// blocks take a stretch each (every eighth, beyond 8) and join their sums.  The weights are the matrix instruction's 16-row operand, NT times 8 tokens its
// columns.  The products of a group are summed on their own and take its scale in fp32, so codes enter as whole numbers of units.
// The next row's codes are on their way while one is multiplied.
template <typename T, int NT, int C, int GROUP>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 3 : 2) linear_kernel(const T* x, const uint8_t* codes, const __nv_bfloat16* scales, const T* bias, const T* residual, T* y,
                                                            const LinearParams p) {
  extern __shared__ __align__(16) uint32_t room[];
  chain_begin(x, codes, scales, bias, residual, y);
  constexpr int kTokens = NT * 8, kOuts = kTokens * kTileRows, kColumns = kWarps * C * kTileCols;
  constexpr int kStride = kColumns / 2 + 16;                   // words of a token
  constexpr int kGroups = GROUP >= 64 ? 1 : 2, kSteps = 4 / kGroups;      // groups of a chunk, steps of 16 columns in each
  uint32_t* tokens = room;
  float* part = reinterpret_cast<float*>(room + kTokens * kStride);       // two of [warp][token][row]
  float* total = part + 2 * kWarps * kOuts;                               // two of [token][row], in a cluster
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = p.parts > 1 ? static_cast<int>(st::cluster_ctarank()) : 0, stretches = (p.cols + kColumns - 1) / kColumns;
  const auto stage = [&](int ph) { stage_tokens<T, kColumns>(x, p.x_row, tokens, kStride, p.tokens, ph * kColumns, p.cols, p.wide); };
  const long long tile_row = static_cast<long long>(p.chunks) * kTileBytes, scale_row = static_cast<long long>(p.groups) * 16;
  constexpr int kOwn = (kOuts + kWarps * 32 - 1) / (kWarps * 32);      // elements of the result that a thread writes
  float acc[NT][4] = {}, off[kOwn], add[kOwn];
  const auto fetch = [&](Slice<C, GROUP>& to, int u, int ph) { to.load(codes + u * tile_row, scales + u * scale_row, (ph * kWarps + warp) * C, p.chunks, p.groups, lane); };
  const auto multiply = [&](const Slice<C, GROUP>& own, int ph) {
    const int count = min(C, p.chunks - (ph * kWarps + warp) * C);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      if (i >= count) break;
      const uint32_t word[4] = {own.w[i].x, own.w[i].y, own.w[i].z, own.w[i].w};
      uint4 b[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) b[n][h] = *reinterpret_cast<const uint4*>(tokens + (n * 8 + g) * kStride + (warp * C + i) * 32 + h * 16 + t * 4);
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        float sum[NT][4] = {};
#pragma unroll
        for (int j = k * kSteps; j < (k + 1) * kSteps; ++j) {
          const uint32_t a[4] = {codes_to_pair<T>(word[j], 0), codes_to_pair<T>(word[j], 1), codes_to_pair<T>(word[j], 2), codes_to_pair<T>(word[j], 3)};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 v = b[n][j / 2];
            mma<T>(sum[n], a, j % 2 ? v.z : v.x, j % 2 ? v.w : v.y, sum[n]);
          }
        }
        const uint32_t both = own.scale(i, k, lane);
        const float low = bf16_bits(both) * kUnits<T>, high = __uint_as_float(both & 0xFFFF0000u) * kUnits<T>;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          acc[n][0] = fmaf(low, sum[n][0], acc[n][0]);
          acc[n][1] = fmaf(low, sum[n][1], acc[n][1]);
          acc[n][2] = fmaf(high, sum[n][2], acc[n][2]);
          acc[n][3] = fmaf(high, sum[n][3], acc[n][3]);
        }
      }
    }
  };
  const auto addends = [&](int u) {      // on their way beside the codes
    if (bias == nullptr && residual == nullptr) return;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      const int i = j * kWarps * 32 + threadIdx.x, m = i / kTileRows, r = u * kTileRows + i % kTileRows;
      const bool in = i < kOuts && m < p.tokens && r < p.rows;
      off[j] = bias && in ? to_float(bias[r]) : 0.0f;
      add[j] = residual && in ? to_float(residual[m * p.residual_row + r]) : 0.0f;
    }
  };
  const auto finish = [&](int u, int flip) {      // the warps' sums, in the order of the warps; in a cluster then the blocks', in theirs
    float* mine = part + flip * kWarps * kOuts;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        mine[warp * kOuts + (n * 8 + 2 * t + (e & 1)) * kTileRows + g + 8 * (e >> 1)] = acc[n][e];
        acc[n][e] = 0.0f;
      }
    __syncthreads();
    if (p.parts > 1) {
#pragma unroll
      for (int j = 0; j < kOwn; ++j) {
        const int i = j * kWarps * 32 + threadIdx.x;
        if (i >= min(kOuts, p.tokens * kTileRows)) continue;
        float v = mine[i];
#pragma unroll
        for (int k = 1; k < kWarps; ++k) v += mine[k * kOuts + i];
        total[flip * kOuts + i] = v;
      }
      st::cluster_sync();
    }
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      const int i = j * kWarps * 32 + threadIdx.x, m = i / kTileRows, r = u * kTileRows + i % kTileRows;
      if (i >= kOuts || m >= p.tokens || r >= p.rows) continue;
      float v;
      if (p.parts > 1) {
        if (m % p.parts != rank) continue;      // a token's 16 rows by one of the blocks
        float f[kMostParts];
        const uint32_t at = st::smem_u32(total + flip * kOuts + i);
#pragma unroll
        for (int q = 0; q < kMostParts; ++q)
          if (q < p.parts) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f[q]) : "r"(st::cluster_map(at, q)));
        v = f[0];
#pragma unroll
        for (int q = 1; q < kMostParts; ++q)
          if (q < p.parts) v += f[q];
      } else {
        v = mine[i];
#pragma unroll
        for (int k = 1; k < kWarps; ++k) v += mine[k * kOuts + i];
      }
      y[m * p.y_row + r] = from_float<T>(activate(v + off[j], p.act) + add[j]);
    }
  };
#pragma unroll
  for (int j = 0; j < kOwn; ++j) off[j] = add[j] = 0.0f;
  Slice<C, GROUP> a, b;
  int u = blockIdx.x / p.parts;
  const int step = gridDim.x / p.parts;
  fetch(a, u, rank);
  if (rank + p.parts >= stretches) {      // this block's only stretch: its x stays
    addends(u);
    stage(rank);
    __syncthreads();
    for (;;) {      // two rows at a time: what is on its way needs no copy
      if (u + step < p.units) fetch(b, u + step, rank);
      multiply(a, rank);
      finish(u, 0);
      if ((u += step) >= p.units) break;
      addends(u);
      if (u + step < p.units) fetch(a, u + step, rank);
      multiply(b, rank);
      finish(u, 1);
      if ((u += step) >= p.units) break;
      addends(u);
    }
  } else {
    for (int flip = 0; u < p.units; u += step, flip ^= 1) {
      addends(u);
      for (int s = rank; s < stretches; s += p.parts) {
        __syncthreads();      // the stretch before has been read
        stage(s);
        __syncthreads();
        b = a;
        const bool more = s + p.parts < stretches;
        if (more || u + step < p.units) fetch(a, more ? u : u + step, more ? s + p.parts : rank);
        multiply(b, s);
      }
      finish(u, flip);
    }
  }
  if (p.parts > 1) st::cluster_sync();      // until then its sums are read
}

template <typename T, int NT, int C, int GROUP>
int launch(LinearParams p, cudaStream_t stream) {
  constexpr int kOuts = NT * 8 * kTileRows, kColumns = kWarps * C * kTileCols;
  constexpr int smem = NT * 8 * (kColumns / 2 + 16) * 4 + 2 * (kWarps + 1) * kOuts * 4;
  p.parts = min(kMostParts, (p.cols + kColumns - 1) / kColumns);
  static int resident[st::kMaxDevices][kMostParts + 1];      // clusters that run at once, by their size
  int& clusters = resident[st::current_device()][p.parts];
  if (clusters == 0) {
    if (smem > 48 * 1024) ST_CUDA_CHECK(cudaFuncSetAttribute(linear_kernel<T, NT, C, GROUP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = p.parts, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.parts * st::sm_count()), cfg.blockDim = dim3(kWarps * 32), cfg.dynamicSmemBytes = smem, cfg.attrs = &attr, cfg.numAttrs = 1;
    int n = 0;
    ST_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, linear_kernel<T, NT, C, GROUP>, &cfg));
    clusters = max(1, n);
  }
  const int grid = min(p.units, clusters) * p.parts;
  const cudaError_t e = st::chained(linear_kernel<T, NT, C, GROUP>, dim3(grid), dim3(kWarps * 32), smem, stream, p.parts)(
      static_cast<const T*>(p.x), p.codes, p.scales, static_cast<const T*>(p.bias), static_cast<const T*>(p.residual), static_cast<T*>(p.y), p);
  return e == cudaSuccess ? ST_OK : st::fail_cuda(e, "int4 linear");
}

template <typename T, int NT, int C>
int by_group(const LinearParams& p, cudaStream_t stream) {
  if (p.group == 32) return launch<T, NT, C, 32>(p, stream);
  if (p.group == 64) return launch<T, NT, C, 64>(p, stream);
  return launch<T, NT, C, 128>(p, stream);
}

template <typename T>
int dispatch(const LinearParams& p, cudaStream_t stream) {
  // 2 chunks a warp where that is the whole depth, 4 otherwise
  if (p.tokens <= 8) return p.chunks <= 2 * kWarps ? by_group<T, 1, 2>(p, stream) : by_group<T, 1, 4>(p, stream);
  return p.chunks <= 2 * kWarps ? by_group<T, 2, 2>(p, stream) : by_group<T, 2, 4>(p, stream);
}

// Whether products go through tcgen05 (int4_wide.cu): from 17 tokens on, and from 9 where the weights are more than 2^24.  us of this kernel and that one (outputs x inputs), 9 and 16 tokens:
//   2048 x 2048 5.3 / 7.0, 6.4 / 7.3     8192 x 2048 8.1 / 9.5, 9.4 / 9.5     2048 x 8192 9.4 / 9.2, 10.9 / 9.6     4096 x 4096 9.5 / 8.7, 11.2 / 9.0
//   12288 x 2048 10.1 / 9.7, 11.4 / 9.8  6144 x 4096 12.0 / 10.6, 14.0 / 11.0  8192 x 8192 23.0 / 15.7, 25.5 / 16.2  50304 x 2048 23.6 / 19.8, 25.6 / 20.1
// 2^24 weights (second to fourth) are even, all larger ones gain.  At 8 tokens tcgen05 is even from there to 2^25 (8192 x 2048 7.7 / 9.5, 4096 x 4096 9.1 / 8.7, 50304 x 2048 20.1 / 19.8) and gains
// by deep matrices beyond (8192 x 8192 18.7 / 15.5, 18944 x 4096 20.0 / 15.1): those are left here.
bool is_wide(int tokens, int rows, int cols) { return tokens > 16 || (tokens > 8 && static_cast<long long>(rows) * cols > 1 << 24); }

int aligned(const void* x, long long row, int cols) {
  if ((reinterpret_cast<uintptr_t>(x) & 15) == 0 && row % 8 == 0 && row >= cols) return ST_OK;
  return st::fail(ST_ERR_INVALID, "int4: rows must lie on 16-byte boundaries");
}
}  // namespace

struct StInt4LinearArgs {
  const void* x;
  const void* codes;
  const void* scales;
  const void* bias;
  const void* residual;
  void* y;
  long long x_row, residual_row, y_row;
  int tokens, rows, cols, group, act, type;
};

// y [tokens, rows] = act(x [tokens, cols] W^T + bias) + residual.  Columns are contiguous, rows the given numbers of elements apart; bias and residual may be
// null.  Where st_int4_is_wide() x lies on a 16-byte boundary, its rows a multiple of 8 elements apart.  act: 0 none, 1 relu, 2 gelu (tanh form); type of x, bias,
// residual and y: 0 bf16, 1 fp16.
ST_API int st_int4_linear(const StInt4LinearArgs* a, void* stream_v) {
  if (a->tokens < 0 || a->tokens > 1 << 30 || a->rows < 1 || a->cols < 1 || a->rows > 1 << 30 || a->cols > 1 << 30 || (a->group != 32 && a->group != 64 && a->group != 128) || a->act < 0 || a->act > 2)
    return st::fail(ST_ERR_INVALID, "int4: sizes out of range");
  if (a->type != 0 && a->type != 1) return st::fail(ST_ERR_INVALID, "int4: unknown type");
  if ((reinterpret_cast<uintptr_t>(a->codes) | reinterpret_cast<uintptr_t>(a->scales)) & 15) return st::fail(ST_ERR_INVALID, "int4: codes and scales must lie on 16-byte boundaries");
  if (a->tokens == 0) return ST_OK;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  if (is_wide(a->tokens, a->rows, a->cols)) {
    if (const int e = aligned(a->x, a->x_row, a->cols)) return e;
    return wide(WideArgs{a->x, a->codes, a->scales, a->bias, a->residual, a->y, a->x_row, a->residual_row, a->y_row, a->tokens, a->rows, a->cols, a->group, a->act}, a->type,
                false, stream);
  }
  const LinearParams p{a->x, static_cast<const uint8_t*>(a->codes), static_cast<const __nv_bfloat16*>(a->scales), a->bias, a->residual, a->y, a->x_row, a->residual_row,
                       a->y_row, a->tokens, a->rows, a->cols, (a->cols + a->group - 1) / a->group, (a->cols + kTileCols - 1) / kTileCols,
                       (a->rows + kTileRows - 1) / kTileRows, a->group, a->act,
                       (reinterpret_cast<uintptr_t>(a->x) & 15) == 0 && a->x_row % 8 == 0, 1};
  return a->type == 0 ? dispatch<__nv_bfloat16>(p, stream) : dispatch<__half>(p, stream);
}

// dx [tokens, cols] = dy [tokens, rows] W.  dy lies on a 16-byte boundary, its rows a multiple of 8 elements apart.
ST_API int st_int4_linear_grad(const void* dy, const void* codes, const void* scales, void* dx, int tokens, int rows, int cols, long long dy_row, long long dx_row,
                               int group, int type, void* stream_v) {
  if (tokens < 0 || tokens > 1 << 30 || rows < 1 || cols < 1 || rows > 1 << 30 || cols > 1 << 30 || (group != 32 && group != 64 && group != 128))
    return st::fail(ST_ERR_INVALID, "int4: sizes out of range");
  if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) & 15) return st::fail(ST_ERR_INVALID, "int4: codes and scales must lie on 16-byte boundaries");
  if (type != 0 && type != 1) return st::fail(ST_ERR_INVALID, "int4: unknown type");
  if (tokens == 0) return ST_OK;
  if (const int e = aligned(dy, dy_row, rows)) return e;
  return wide(WideArgs{dy, codes, scales, nullptr, nullptr, dx, dy_row, 0, dx_row, tokens, rows, cols, group, 0}, type, true, reinterpret_cast<cudaStream_t>(stream_v));
}

// Whether a product of these sizes goes through tcgen05 (x then as dy above).
ST_API int st_int4_is_wide(int tokens, int rows, int cols) { return is_wide(tokens, rows, cols); }
