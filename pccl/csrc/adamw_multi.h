// AdamW over a list of tensors in one launch, states in 32 or in 8 bits (adamw_multi.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace pccl {

constexpr int kAdamBlock = 256;            // elements that share a scale; every tensor's state starts on such a block
constexpr int kAdamTensors = 768;          // tensors in one launch (the argument block may hold 32,764 bytes)

struct AdamTensor {
  void* param;
  float* master;                           // the 32-bit copy, or nullptr: param itself is 32-bit
  const void* grad;
  int64_t n;
  float decay;
  uint32_t first;                          // first block of its state, counted from the launch's first block
};

struct AdamMultiArgs {
  void* m;                                 // fp32, or int8 codes
  void* v;                                 // fp32, or uint8 codes
  float* m_scale;                          // 8 bits: largest size in each block
  float* v_scale;
  uint64_t first_block;                    // where the launch's first tensor lies in the state
  uint32_t blocks;                         // of all tensors of the launch
  uint32_t key;                            // chooses the rounding noise: from the seed and the step
  float lr, beta1, beta2, one_minus_beta1, one_minus_beta2, eps, bias1, bias2, grad_scale, max_grad_norm;
  const float* total_sq_norm;              // nullptr: no clipping
};

enum AdamType : int { kAdamBf16 = 0, kAdamF16 = 1, kAdamF32 = 2 };

// The smallest eps that 8-bit states take, 2^-35 / sqrt(1 - beta2): adamw_multi.cu has the reason.
double adamw_least_eps(double beta2);
uint32_t adamw_noise_key(uint64_t seed, int64_t step);
cudaError_t launch_adamw_multi(const AdamMultiArgs& a, const AdamTensor* tensors, int count, int param_type, int grad_type, bool bits8,
                               int sm_count, cudaStream_t s);
// The values that 8-bit states stand for, n (a multiple of kAdamBlock) elements.
cudaError_t launch_adamw_dequantize(const int8_t* m, const float* m_scale, const uint8_t* v, const float* v_scale, float* m_out,
                                    float* v_out, int64_t n, cudaStream_t s);

}  // namespace pccl
