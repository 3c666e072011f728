// Attention, forward and backward (attention_fwd.cu, attention_bwd.cu).
//
//   s_ij = scale * <q_i, k_j>,   p_ij = exp(s_ij - lse_i),   lse_i = log(sum_j exp(s_ij)),   o_i = sum_j p_ij v_j
//   dv_j = sum_i p_ij do_i,   ds_ij = p_ij (<do_i, v_j> - <do_i, o_i>),   dq_i = scale * sum_j ds_ij k_j,   dk_j = scale * sum_i ds_ij q_i
//
// Causal: query i of a sequence sees the keys j <= i + (keys - queries) of it.  A query that sees no key has o = 0 and
// lse = -inf and adds nothing to any gradient.  H query heads share H / Hk key/value heads in groups of neighbours; the
// gradients of a shared head are summed over its group.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace pccl {

// A [batch, row, head, column] tensor of 16-bit elements whose columns are contiguous; strides in elements.
struct AttnTensor {
  const void* p;
  int64_t sb, ss, sh;
};

struct AttnArgs {
  AttnTensor q, k, v, o;             // o: written by the forward pass, read by the backward pass
  AttnTensor dout, dq, dk, dv;       // backward pass
  float* lse;                        // [batch, head, row], or [head, row] of packed sequences
  float* delta;                      // <do_i, o_i>, laid out like lse (backward pass: scratch)
  int is_bf16;                       // else fp16
  int B, H, Hk, D;                   // B = 1 for packed sequences
  int Sq, Sk;                        // rows of each batch entry, or of all packed sequences together
  const int* cu_q;                   // packed: nseq + 1 starts of the sequences (device), nullptr where not packed
  const int* cu_k;
  int nseq;
  int causal;
  int zero_tail;                     // packed: rows behind the last sequence are set to 0 (lse: -inf); else they are left alone
  float scale;
  int* error;
};

constexpr int kAttnMaxDim = 128;     // columns of a head: a multiple of 8 up to this

cudaError_t launch_attention_forward(const AttnArgs& a, cudaStream_t stream);
cudaError_t launch_attention_backward(const AttnArgs& a, cudaStream_t stream);

}  // namespace pccl
