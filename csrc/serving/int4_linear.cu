// Products with weights of four bits:  y = act(x W^T + bias) + residual,  W = q s  (int4.cuh).
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

// Elements k and k + 1 of a row of x as one word; what lies behind the row's end is zero.
template <typename T, bool PAIRS>
__device__ __forceinline__ uint32_t load_pair(const T* row, int k, int cols) {
  if (PAIRS) return k < cols ? *reinterpret_cast<const uint32_t*>(row + k) : 0u;
  const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
  return (k < cols ? h[k] : 0u) | (k + 1 < cols ? static_cast<uint32_t>(h[k + 1]) << 16 : 0u);
}

// A warp multiplies U tiles of 16 weight rows, one under another, by NT tiles of 8 tokens: chunk by chunk of 64 columns, those of the
// block's warps interleaved.  The weights are the matrix instruction's 16-row operand, the tokens its 8 columns.  The products of a group are
// summed on their own and take its scale in fp32, so codes enter as the whole numbers that they are.
template <typename T, int NT, int U, int GROUP, int WARPS, bool PAIRS>
__global__ void __launch_bounds__(WARPS * 32) linear_kernel(const T* x, const uint8_t* codes, const __nv_bfloat16* scales, const T* bias, const T* residual, T* y,
                                                            const LinearParams p) {
  extern __shared__ float part[];      // [warp][token][row]
  chain_begin(x, codes, scales, bias, residual, y);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int u0 = blockIdx.x * U, m0 = blockIdx.y * NT * 8;
  constexpr int kGroups = GROUP >= 64 ? 1 : 2, kSteps = 4 / kGroups;      // groups of a chunk, steps of 16 columns in each
  float acc[U][NT][4] = {};
  for (int c = warp; c < p.chunks; c += WARPS) {
    uint4 w[U];
    uint32_t s[U][kGroups];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const long long u = min(u0 + i, p.units - 1);
      w[i] = *reinterpret_cast<const uint4*>(codes + (u * p.chunks + c) * kTileBytes + lane * 16);
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        const int at = min(c * kTileCols / GROUP + k, p.groups - 1);
        s[i][k] = *reinterpret_cast<const uint32_t*>(scales + (u * p.groups + at) * 16 + 2 * g);
      }
    }
    uint32_t b[NT][8];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int m = m0 + n * 8 + g;
      const T* row = x + static_cast<long long>(m) * p.x_row;
#pragma unroll
      for (int h = 0; h < 8; ++h) b[n][h] = m < p.tokens ? load_pair<T, PAIRS>(row, c * kTileCols + 8 * h + 2 * t, p.cols) : 0u;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const uint32_t word[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        float sum[NT][4] = {};
#pragma unroll
        for (int j = k * kSteps; j < (k + 1) * kSteps; ++j) {
          const uint32_t a[4] = {codes_to_pair<T>(word[j], 0), codes_to_pair<T>(word[j], 1), codes_to_pair<T>(word[j], 2), codes_to_pair<T>(word[j], 3)};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma<T>(sum[n], a, b[n][2 * j], b[n][2 * j + 1], sum[n]);
        }
        const float low = bf16_bits(s[i][k]), high = bf16_bits(s[i][k] >> 16);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          acc[i][n][0] = fmaf(low, sum[n][0], acc[i][n][0]);
          acc[i][n][1] = fmaf(low, sum[n][1], acc[i][n][1]);
          acc[i][n][2] = fmaf(high, sum[n][2], acc[i][n][2]);
          acc[i][n][3] = fmaf(high, sum[n][3], acc[i][n][3]);
        }
      }
    }
  }
  // the warps' sums, in the order of the warps
  constexpr int kRows = U * kTileRows, kTokens = NT * 8;
#pragma unroll
  for (int i = 0; i < U; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[(warp * kTokens + n * 8 + 2 * t + (e & 1)) * kRows + i * kTileRows + g + 8 * (e >> 1)] = acc[i][n][e];
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * kTokens; i += WARPS * 32) {
    const int m = m0 + i / kRows;
    const int r = u0 * kTileRows + i % kRows;
    if (m >= p.tokens || r >= p.rows) continue;
    float v = part[i];
    for (int k = 1; k < WARPS; ++k) v += part[k * kRows * kTokens + i];
    if (bias) v += to_float(bias[r]);
    v = activate(v, p.act);
    if (residual) v += to_float(residual[m * p.residual_row + r]);
    y[m * p.y_row + r] = from_float<T>(v);
  }
}

template <typename T, int NT, int U, int GROUP, bool PAIRS>
int launch(const LinearParams& p, cudaStream_t stream) {
  constexpr int kWarps = 8;
  constexpr size_t smem = sizeof(float) * kWarps * NT * 8 * U * kTileRows;
  static_assert(smem <= 48 * 1024, "sums need no opting in");
  const dim3 grid((p.units + U - 1) / U, (p.tokens + NT * 8 - 1) / (NT * 8));
  if (grid.y > 65535) return st::fail(ST_ERR_TOO_LARGE, "int4: too many rows");
  const cudaError_t e = st::chained(linear_kernel<T, NT, U, GROUP, kWarps, PAIRS>, grid, dim3(kWarps * 32), smem, stream)(
      static_cast<const T*>(p.x), p.codes, p.scales, static_cast<const T*>(p.bias), static_cast<const T*>(p.residual), static_cast<T*>(p.y), p);
  return e == cudaSuccess ? ST_OK : st::fail_cuda(e, "int4 linear");
}

template <typename T, int NT, int U>
int by_group(const LinearParams& p, cudaStream_t stream) {
  const bool pairs = (reinterpret_cast<uintptr_t>(p.x) & 3) == 0 && p.x_row % 2 == 0 && p.cols % 2 == 0;
  if (p.group == 32) return pairs ? launch<T, NT, U, 32, true>(p, stream) : launch<T, NT, U, 32, false>(p, stream);
  if (p.group == 64) return pairs ? launch<T, NT, U, 64, true>(p, stream) : launch<T, NT, U, 64, false>(p, stream);
  return pairs ? launch<T, NT, U, 128, true>(p, stream) : launch<T, NT, U, 128, false>(p, stream);
}

template <typename T>
int dispatch(const LinearParams& p, cudaStream_t stream) {
  if (p.tokens <= 8) return by_group<T, 1, 1>(p, stream);
  return by_group<T, 2, 1>(p, stream);
}
constexpr int kWideFrom = 17;

int aligned(const void* x, long long row, int cols) {
  if ((reinterpret_cast<uintptr_t>(x) & 15) == 0 && row % 8 == 0 && row >= cols) return ST_OK;
  return st::fail(ST_ERR_INVALID, "int4: rows must lie on 16-byte boundaries");
}
}  // namespace

// y [tokens, rows] = act(x [tokens, cols] W^T + bias) + residual.  Columns are contiguous, rows the given numbers of elements apart; bias and residual may be
// null.  From st_int4_wide_from() tokens on x lies on a 16-byte boundary, its rows a multiple of 8 elements apart.  act: 0 none, 1 relu, 2 gelu (tanh form); type of x, bias, residual and y: 0 bf16, 1 fp16.
ST_API int st_int4_linear(const void* x, const void* codes, const void* scales, const void* bias, const void* residual, void* y, int tokens, int rows, int cols,
                          long long x_row, long long residual_row, long long y_row, int group, int act, int type, void* stream_v) {
  if (tokens < 0 || rows < 1 || cols < 1 || rows > 1 << 30 || cols > 1 << 30 || (group != 32 && group != 64 && group != 128) || act < 0 || act > 2)
    return st::fail(ST_ERR_INVALID, "int4: sizes out of range");
  if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) & 15) return st::fail(ST_ERR_INVALID, "int4: codes and scales must lie on 16-byte boundaries");
  if (tokens == 0) return ST_OK;
  const LinearParams p{x, static_cast<const uint8_t*>(codes), static_cast<const __nv_bfloat16*>(scales), bias, residual, y, x_row, residual_row, y_row,
                       tokens, rows, cols, (cols + group - 1) / group, (cols + kTileCols - 1) / kTileCols, (rows + kTileRows - 1) / kTileRows, group, act};
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  if (type != 0 && type != 1) return st::fail(ST_ERR_INVALID, "int4: unknown type");
  if (tokens >= kWideFrom) {
    if (const int e = aligned(x, x_row, cols)) return e;
    return wide(WideArgs{x, codes, scales, bias, residual, y, x_row, residual_row, y_row, tokens, rows, cols, group, act}, type, false, stream);
  }
  if (type == 0) return dispatch<__nv_bfloat16>(p, stream);
  return dispatch<__half>(p, stream);
}

// dx [tokens, cols] = dy [tokens, rows] W.  dy lies on a 16-byte boundary, its rows a multiple of 8 elements apart.
ST_API int st_int4_linear_grad(const void* dy, const void* codes, const void* scales, void* dx, int tokens, int rows, int cols, long long dy_row, long long dx_row,
                               int group, int type, void* stream_v) {
  if (tokens < 0 || rows < 1 || cols < 1 || rows > 1 << 30 || cols > 1 << 30 || (group != 32 && group != 64 && group != 128))
    return st::fail(ST_ERR_INVALID, "int4: sizes out of range");
  if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) & 15) return st::fail(ST_ERR_INVALID, "int4: codes and scales must lie on 16-byte boundaries");
  if (type != 0 && type != 1) return st::fail(ST_ERR_INVALID, "int4: unknown type");
  if (tokens == 0) return ST_OK;
  if (const int e = aligned(dy, dy_row, rows)) return e;
  return wide(WideArgs{dy, codes, scales, nullptr, nullptr, dx, dy_row, 0, dx_row, tokens, rows, cols, group, 0}, type, true, reinterpret_cast<cudaStream_t>(stream_v));
}

// From how many rows of x products go through tcgen05 (x then as dy above).
ST_API int st_int4_wide_from() { return kWideFrom; }
