// A mixture-of-experts layer for a few tokens: router, choice, ReLU^2 experts, shared expert (moe_tokens.cu).
#pragma once
#include <cuda_runtime_api.h>
#include <stdint.h>

constexpr int NT_MOE_TOKENS_MOST = 64, NT_MOE_TOKENS_EXPERTS = 512, NT_MOE_TOKENS_CHOICES = 16, NT_MOE_TOKENS_WIDTH = 8192;

struct MoeTokensArgs {
  const void* x = nullptr;         // [T, d], rows x_stride elements apart
  int64_t x_stride = 0;
  const float* router = nullptr;   // [E, d]
  const float* bias = nullptr;     // [E] or null
  const void *w_fc = nullptr, *w_proj = nullptr;            // [E, F, d], [E, d, F]
  const void *shared_fc = nullptr, *shared_proj = nullptr;  // [Fs, d], [d, Fs] or null
  void* y = nullptr;               // [T, d]
  void* workspace = nullptr;
  int T = 0, d = 0, F = 0, Fs = 0, E = 0, k = 0, sms = 0;
  bool fp16 = false;
};
// Bytes of scratch a call needs; it holds nothing between calls.
size_t nt_moe_tokens_workspace(const MoeTokensArgs& a);
// 0, or -1 for an unsupported shape.
int nt_moe_tokens(const MoeTokensArgs& a, cudaStream_t s);
