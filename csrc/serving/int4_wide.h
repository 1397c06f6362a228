// The tcgen05 form of products with weights of four bits (int4_wide.cu), for the launchers of int4_linear.cu.
#pragma once
#include <cuda_runtime.h>

namespace st4 {

struct WideArgs {
  const void* x;      // [tokens, cols], or the gradient [tokens, rows]: on a 16-byte boundary, x_row a multiple of 8
  const void* codes;
  const void* scales;
  const void* bias;
  const void* residual;
  void* y;            // [tokens, rows], or [tokens, cols]
  long long x_row, residual_row, y_row;
  int tokens, rows, cols, group, act;
};

// type: 0 bf16, 1 fp16; turn: x W instead of x W^T, without bias, residual and activation.
int wide(const WideArgs& a, int type, bool turn, cudaStream_t stream);

}  // namespace st4
