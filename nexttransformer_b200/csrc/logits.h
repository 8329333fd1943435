// Penalties for repeated tokens, sparse biases and a grammar mask on next-token logits (logits.cu).
#pragma once
#include <cuda_runtime_api.h>
#include <stdint.h>

enum LogitsType { LOGITS_BF16 = 0, LOGITS_FP16 = 1, LOGITS_FP32 = 2 };

struct LogitsArgs {
  const void* logits = nullptr;  // [B, V], rows row_stride elements apart
  int64_t row_stride = 0;
  float* out = nullptr;          // [B, V] contiguous
  const int* tokens = nullptr;   // [B, L] or null
  const int* length = nullptr;   // [B]: tokens that count (null: L)
  const int* prompt = nullptr;   // [B]: of these, the first that are the prompt's (null: 0)
  const float *repetition = nullptr, *presence = nullptr, *frequency = nullptr;  // [B] or null
  const int* bias_ids = nullptr;  // [B, K] or null
  const float* bias = nullptr;    // [B, K]
  const int* allowed = nullptr;   // [B, words] bits, 1 = allowed, or null
  int B = 0, V = 0, L = 0, K = 0, words = 0, type = 0, sms = 0;
};
// 0, or -1 for an unsupported shape.
int nt_adjust_logits(const LogitsArgs& a, cudaStream_t s);
