// Norms of queries and keys for each head with the rotation of positions, forward and backward (rotary.cu).
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r w,  y = n rotated: each pair (a, b) of the first 2 * half columns becomes
//   (a cos - b sin, b cos + a sin) with the angle of its position and place; pairs are columns (i, i + half), or (2i, 2i + 1)
//   where interleaved.  Columns behind 2 * half are not rotated.
//   Backward: t = dy rotated back, dw = sum over rows of t x r, g = t w, dx = r (g - x r mean(g x r)).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace pccl {

constexpr int kRotaryMaxDim = 256;

struct RotaryTensor {
  void* p;
  int64_t sb, ss, sh;              // strides in elements: batch, row, head
};

struct RotaryArgs {
  RotaryTensor x[2], y[2], dy[2];  // [0] queries, [1] keys.  Forward: x -> y.  Backward: x, dy -> y (the gradient of x)
  const void* w[2];
  void* dw[2];
  int w_type;                      // 0 bf16, 1 fp16, 2 fp32: weights and their gradients
  int is_bf16;                     // x, y, dy; else fp16
  const float* cos;
  const float* sin;                // [table, half]
  const void* positions;           // [batch, rows], or nullptr: the row's number
  int positions64;
  int64_t table;
  int half, interleaved;
  int B, S, D, H[2];
  int heads_per_item, chunks[2];   // a thread group works on so many heads of one row at a time
  int q_blocks;                    // the first blocks work on queries, the others on keys
  float eps;
  float* partial;                  // backward: rotary_blocks(...) * D floats
};

// How the work is cut; sets heads_per_item, chunks and q_blocks, returns the number of blocks.
int rotary_blocks(RotaryArgs& a, bool backward, int sm_count);
cudaError_t launch_rotary_forward(const RotaryArgs& a, int blocks, cudaStream_t s);
cudaError_t launch_rotary_backward(const RotaryArgs& a, int blocks, cudaStream_t s);

}  // namespace pccl
