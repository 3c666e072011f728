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
  int2* order_q;                     // packed: which sequence and which of its tiles each tile number stands for (scratch; forward:
  int2* order_k;                     // order_q; backward: both)
  int causal;
  int zero_tail;                     // packed: rows behind the last sequence are set to 0; else they are left alone (lse there is -inf)
  float scale;
  int* error;
  // Work split over a long axis (not for packed sequences), where there are too few tiles for the device: the parts of one
  // tile's sum go to partial, [part][batch][head][row][D] in fp32, and are added up by a small kernel.
  int parts_o, parts_dq, parts_dkv;  // 1: not split
  float* partial;
  float* partial_lse;                // forward: lse of each part, [part][batch][head][row]
};

constexpr int kAttnMaxDim = 128;     // columns of a head: a multiple of 8 up to this

// How many parts to cut each tile's work into: fills in parts_* and returns what partial, partial_lse (floats) and order_* need.
struct AttnScratch {
  int64_t partial, partial_lse;
  int64_t order_q, order_k;          // entries
};
AttnScratch plan_attention_forward(AttnArgs& a, int sm_count);
AttnScratch plan_attention_backward(AttnArgs& a, int sm_count);
// kernels: goes up by one with each kernel launched.
cudaError_t launch_attention_forward(const AttnArgs& a, cudaStream_t stream, int64_t& kernels);
cudaError_t launch_attention_backward(const AttnArgs& a, cudaStream_t stream, int64_t& kernels);

}  // namespace pccl
