// A token for each row of logits: temperature, top-k, top-p, min-p, and the draw from a given number (sampling.cu).
#pragma once
#include <cuda_runtime_api.h>
#include <stdint.h>

#include "logits.h"

struct RowValue {               // one value for all rows, or one for each
  const void* rows = nullptr;   // fp32 or int32 [B], or null
  double all = 0;
};

struct SampleArgs {
  const void* logits = nullptr;  // [B, V], rows row_stride elements apart
  int64_t row_stride = 0;
  const float* uniform = nullptr;  // [B]
  RowValue temperature, top_k, top_p, min_p;
  int64_t* tokens = nullptr;     // [B]
  float* logprobs = nullptr;     // [B]
  int B = 0, V = 0, type = 0, sms = 0;
};
// The largest vocabulary (up to 131072 logits a row are held on chip, of longer rows each pass reads them again).
int nt_sample_most();
// 0, or -1 for an unsupported shape.
int nt_sample_logits(const SampleArgs& a, cudaStream_t s);
