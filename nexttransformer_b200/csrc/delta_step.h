// Recurrent form of the gated delta rule with a carried fp32 state (delta_step.cu).
#pragma once
#include <cuda_runtime_api.h>
#include <stdint.h>

enum DeltaStepType { DELTA_STEP_BF16 = 0, DELTA_STEP_FP16 = 1, DELTA_STEP_FP32 = 2 };

// q, k, v, o [B, T, H, D] (D 64 or 128, o contiguous); strides of row, token, head in elements, the head
// dimension contiguous.  beta [B, T, H] in the type of q or fp32; g (log decay) fp32 [B, T, H] or
// [B, T, H, D] (gate 1 or 2; 0: none).  state fp32 [states, H, D, D] is updated in place; row b works on
// state slots[b] (null: b; negative: none).  Tokens from count[b] on (null: T) do nothing and give zeros.
struct DeltaStepArgs {
  const void *q = nullptr, *k = nullptr, *v = nullptr, *beta = nullptr;
  const float* g = nullptr;
  int64_t qs[3] = {}, ks[3] = {}, vs[3] = {}, bs[3] = {}, gs[3] = {};
  float* state = nullptr;
  void* o = nullptr;
  const int *slots = nullptr, *count = nullptr;
  int64_t states = 0;
  int B = 0, T = 0, H = 0, D = 0, gate = 0, type = 0, sms = 0;
  bool beta_f32 = false, l2norm = false;
  float scale = 1.f;
  void* workspace = nullptr;  // 16-byte aligned; holds nothing between calls
};
size_t nt_delta_step_workspace(const DeltaStepArgs& a);
// 0, or -1 for an unsupported shape.
int nt_delta_step(const DeltaStepArgs& a, cudaStream_t s);
// Error word (reading clears it): 1 = a bounded device wait ran out, 2 = a slot outside the states, `where` is the row.
int nt_delta_step_read_error(unsigned* where);
