// Paged key-value cache (paged.cu): appending rotated keys and values, and attention over the pages.
// 16-bit tensors (bf16 or fp16), heads of 64 or 128.  Pages hold [Hk, page, D] keys (or values); token
// p of row b lives in page table[b, p / page] at slot p % page.  Strides are in elements, the head
// dimension is contiguous.  The launchers return 0, or -1 for an unsupported shape.
#pragma once
#include <cuda_runtime_api.h>
#include <stdint.h>

struct PagedCacheArgs {
  void* k = nullptr;
  void* v = nullptr;
  int64_t page_stride_k = 0, head_stride_k = 0, slot_stride_k = 0;
  int64_t page_stride_v = 0, head_stride_v = 0, slot_stride_v = 0;
  const int* table = nullptr;  // [B, columns]
  int columns = 0;
  int64_t pages = 0;
  int page = 0;                // tokens per page, a multiple of 16
};

struct PagedAppendArgs {
  PagedCacheArgs cache;
  const void *q = nullptr, *kin = nullptr, *vin = nullptr;  // [B, t, heads, D]
  int64_t qs[3] = {}, ks[3] = {}, vs[3] = {};               // strides of row, token, head
  const void* ve = nullptr;                                 // [B, t, Hk, D] or null
  const void* ve_gate = nullptr;                            // [B, t, Hk]
  int64_t es[3] = {}, gs[3] = {};
  void* q_out = nullptr;                                    // [B, t, H, D] contiguous
  const int *start = nullptr, *count = nullptr;             // [B]; count null: t
  const void *cos = nullptr, *sin = nullptr;                // [rope_rows, D / 2]
  int rope_rows = 0;
  int B = 0, t = 0, H = 0, Hk = 0, D = 0, sms = 0;
  bool norm = false, fp16 = false;
  float scale = 1.f;
};
int nt_paged_append(const PagedAppendArgs& a, cudaStream_t s);

struct PagedAttnArgs {
  PagedCacheArgs cache;
  const void* q = nullptr;  // [B, t, H, D]
  int64_t qs[3] = {};
  void* out = nullptr;      // [B, t, H, D] contiguous
  const int *start = nullptr, *count = nullptr;
  int B = 0, t = 0, H = 0, Hk = 0, D = 0, window = -1, sms = 0;
  bool fp16 = false;
  float scale = 1.f;
  float* workspace = nullptr;
  unsigned* counters = nullptr;
};
// Bytes of scratch a call needs (0: none; then no counters either); it holds nothing between calls.
size_t nt_paged_attn_workspace(const PagedAttnArgs& a);
// Counters a call needs.  They have to be 0 before a call, which leaves them 0; calls that may run at the same
// time must not share them.
int nt_paged_attn_counters(int sms);
int nt_paged_attn(const PagedAttnArgs& a, cudaStream_t s);

// Error word of this unit (reading clears it): 1 = a position behind the row's page table, 2 = a page number
// outside the cache, 3 = a position behind the rotary table; `where` is the row.
int nt_paged_read_error(unsigned* where);
