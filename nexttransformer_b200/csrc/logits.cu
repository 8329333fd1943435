// K23: what a serving loop does to next-token logits before it samples, in one pass:
//
//   seen in prompt or answer   x <- x / r where x > 0, x r elsewhere
//   n times in the answer      x <- x - frequency n - presence [n > 0]
//   listed                     x <- x + bias (an id's entries are added in their order)
//   not allowed                x <- -inf
//
// A CTA owns a piece of one row.  It streams the piece through first, masked but otherwise as it is, which waits
// for nothing but its loads; meanwhile it counts the row's tokens that fall into the piece in shared memory
// (whole-number atomics: their order does not matter) and then mends the few entries that tokens or biases
// concern.  Reading and writing V (in + 4) bytes a row bounds it; the token list is read again by each piece, from L2.
//
// Measured on one B200, 224 rows of 65536 bf16 logits, up to 2048 tokens, 48 biases, a mask: 23 us, where its 92 MB
// take 14 at the copy rate; an earlier build took 20 without tokens, biases and mask.  One row of 32768: 3 us.  With
// counts and biases applied inside the stream it took 43 us (every piece waited for its counts).  Entries of 4 a thread
// let a warp store whole lines.
#include "logits.h"
#include "common.cuh"

#include <cuda_fp16.h>

namespace nt {
namespace logits {

constexpr int THREADS = 256;
constexpr uint32_t PROMPT = 0x80000000u;  // with the answer's count in the lower bits

template <class T> struct In;
template <> struct In<__nv_bfloat16> {
  static NT_DEVICE float f(__nv_bfloat16 v) { return __bfloat162float(v); }
};
template <> struct In<__half> {
  static NT_DEVICE float f(__half v) { return __half2float(v); }
};
template <> struct In<float> {
  static NT_DEVICE float f(float v) { return v; }
};
template <class T, int N>
struct alignas(N * sizeof(T)) Vec {
  T x[N];
};
// PIECE logits a CTA, in vectors of VEC (4: a warp stores whole lines; or 1 where rows do not start on one).
template <class T, int PIECE, int VEC>
__global__ void __launch_bounds__(THREADS) adjust_kernel(const LogitsArgs a) {
  constexpr int N = PIECE / THREADS / VEC, EARLY = 4;
  __shared__ __align__(16) uint32_t counts[PIECE];
  const int b = blockIdx.y, c0 = blockIdx.x * PIECE, tid = threadIdx.x, lane = tid & 31;
  const int width = min(PIECE, a.V - c0);
  const T* in = static_cast<const T*>(a.logits) + b * a.row_stride + c0;
  const int* allowed = a.allowed ? a.allowed + static_cast<int64_t>(b) * a.words : nullptr;
  float* out = a.out + static_cast<int64_t>(b) * a.V + c0;

  // the loads that depend on nothing are all asked for first
  Vec<T, VEC> x[N];
  uint32_t word[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = (i * THREADS + tid) * VEC;
    word[i] = 0xffffffffu;
    if (at < width) {
      x[i] = *reinterpret_cast<const Vec<T, VEC>*>(in + at);
      if (allowed) word[i] = static_cast<uint32_t>(allowed[(c0 + at) >> 5]) >> (at & 31);
    }
  }
  const int n = a.length ? min(a.length[b], a.L) : a.L, prompt = a.prompt ? a.prompt[b] : 0;
  const int* row = a.tokens + static_cast<int64_t>(b) * a.L;
  int early[EARLY];
#pragma unroll
  for (int i = 0; i < EARLY; ++i) early[i] = i * THREADS + tid < n ? row[i * THREADS + tid] : -1;
  const float r = a.repetition ? a.repetition[b] : 1.f;
  const float presence = a.presence ? a.presence[b] : 0.f, frequency = a.frequency ? a.frequency[b] : 0.f;
  const bool adds_bias = a.K && tid >= THREADS - 32;  // one warp: repeated ids are added in their order
  const int64_t entry = static_cast<int64_t>(b) * a.K + lane;
  int bias_id = adds_bias && lane < a.K ? a.bias_ids[entry] : -1;
  float bias_value = adds_bias && lane < a.K ? a.bias[entry] : 0.f;

  auto count = [&](int i, int token) {
    const uint32_t at = static_cast<uint32_t>(token - c0);
    if (i < n && at < static_cast<uint32_t>(width)) {
      if (i < prompt) atomicOr(counts + at, PROMPT);
      else atomicAdd(counts + at, 1u);
    }
  };
  if (a.tokens)
    for (int i = tid; i < PIECE / 4; i += THREADS) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = (i * THREADS + tid) * VEC;
    if (at >= width) continue;
    float y[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) y[e] = (word[i] >> e) & 1u ? In<T>::f(x[i].x[e]) : -INFINITY;
    if (VEC >= 4) {
#pragma unroll
      for (int e = 0; e < VEC / 4; ++e)
        reinterpret_cast<float4*>(out + at)[e] = make_float4(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
    } else {
      out[at] = y[0];
    }
  }
  if (!a.tokens && !a.K) return;
  __syncthreads();
  if (a.tokens) {
#pragma unroll
    for (int i = 0; i < EARLY; ++i) count(i * THREADS + tid, early[i]);
#pragma unroll 4
    for (int i = EARLY * THREADS + tid; i < n; i += THREADS) count(i, row[i]);
    __syncthreads();
  }

  auto is_allowed = [&](uint32_t at) { return !allowed || (static_cast<uint32_t>(allowed[(c0 + at) >> 5]) >> ((c0 + at) & 31)) & 1u; };
  auto mend = [&](int i, int token) {  // whoever takes an entry's count mends it
    const uint32_t at = static_cast<uint32_t>(token - c0);
    if (i >= n || at >= static_cast<uint32_t>(width)) return;
    const uint32_t c = atomicExch(counts + at, 0u), times = c & ~PROMPT;
    if (c == 0 || !is_allowed(at)) return;
    float v = In<T>::f(in[at]);
    v = v > 0.f ? v / r : v * r;
    if (times) v = v - frequency * static_cast<float>(times) - presence;
    out[at] = v;
  };
  if (a.tokens) {
#pragma unroll 1
    for (int i = 0; i < EARLY; ++i) {
      int token = early[0];
#pragma unroll
      for (int e = 1; e < EARLY; ++e) token = i == e ? early[e] : token;
      mend(i * THREADS + tid, token);
    }
    for (int i = EARLY * THREADS + tid; i < n; i += THREADS) mend(i, row[i]);
    if (a.K) __syncthreads();
  }
  if (!adds_bias) return;
  for (int i = 0; i < a.K; i += 32) {
    const int id = bias_id;
    const float v = bias_value;
    const bool more = i + 32 + lane < a.K;
    bias_id = more ? a.bias_ids[entry + i + 32] : -1;
    bias_value = more ? a.bias[entry + i + 32] : 0.f;
    const uint32_t at = static_cast<uint32_t>(id - c0);
    const bool mine = id >= 0 && at < static_cast<uint32_t>(width);
    if (!__any_sync(0xffffffffu, mine)) continue;
    unsigned same = __match_any_sync(0xffffffffu, mine ? at : 0xffffffffu);
    const bool first = (same & ((1u << lane) - 1u)) == 0;
    if (!mine) same = 0;
    float sum = mine ? out[at] : 0.f;
    while (__any_sync(0xffffffffu, same)) {
      const float w = __shfl_sync(0xffffffffu, v, same ? __ffs(same) - 1 : 0);
      if (same) sum += w;
      same &= same - (same ? 1u : 0u);
    }
    if (mine && first && is_allowed(at)) out[at] = sum;
    __syncwarp();
  }
}

template <class T, int PIECE>
static int launch(const LogitsArgs& a, cudaStream_t s) {
  constexpr int VEC = 4;
  const dim3 grid((a.V + PIECE - 1) / PIECE, a.B);
  if (a.V % VEC == 0 && a.row_stride % VEC == 0 && reinterpret_cast<uintptr_t>(a.logits) % (4 * sizeof(T)) == 0)
    adjust_kernel<T, PIECE, VEC><<<grid, THREADS, 0, s>>>(a);
  else
    adjust_kernel<T, PIECE, 1><<<grid, THREADS, 0, s>>>(a);
  return 0;
}
template <class T>
static int by_piece(const LogitsArgs& a, cudaStream_t s) {
  // large pieces read the token list less often (224 x 65536: 6 % faster than pieces of 4096), small ones reach
  // more SMs (1 x 32768: 16 instead of 4)
  if (static_cast<int64_t>(a.B) * ((a.V + 8191) / 8192) >= 2 * a.sms) return launch<T, 8192>(a, s);
  return launch<T, 2048>(a, s);
}

}  // namespace logits
}  // namespace nt

using namespace nt::logits;

int nt_adjust_logits(const LogitsArgs& a, cudaStream_t s) {
  if (a.B == 0 || a.V == 0) return 0;
  if (a.B > 65535) return -1;
  if (a.type == LOGITS_BF16) return by_piece<__nv_bfloat16>(a, s);
  if (a.type == LOGITS_FP16) return by_piece<__half>(a, s);
  if (a.type == LOGITS_FP32) return by_piece<float>(a, s);
  return -1;
}
