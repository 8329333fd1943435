// K23: what a serving loop does to next-token logits before it samples, in one pass:
//
//   seen in prompt or answer   x <- x / r where x > 0, x r elsewhere
//   n times in the answer      x <- x - frequency n - presence [n > 0]
//   listed                     x <- x + bias (an id's entries are added in their order)
//   not allowed                x <- -inf
//
// A CTA owns a piece of one row.  It asks for the piece's logits first, counts the row's tokens that fall
// into the piece in shared memory while they travel (whole-number atomics: the order does not matter), and
// writes fp32.  Reading and writing V (in + 4) bytes a row bounds it; the token list is read again by each
// piece, from L2.
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
template <class T>
struct alignas(4 * sizeof(T)) Four {
  T x[4];
};

// PIECE logits a CTA, in vectors of VEC (4, or 1 where rows do not start on a vector).
template <class T, int PIECE, int VEC>
__global__ void __launch_bounds__(THREADS) adjust_kernel(const LogitsArgs a) {
  constexpr int N = PIECE / THREADS / VEC;
  extern __shared__ uint32_t smem[];
  const int b = blockIdx.y, c0 = blockIdx.x * PIECE, tid = threadIdx.x;
  const int width = min(PIECE, a.V - c0);
  uint32_t* counts = smem;
  float* bias = reinterpret_cast<float*>(smem + (a.tokens ? PIECE : 0));

  const T* in = static_cast<const T*>(a.logits) + b * a.row_stride + c0;
  T x[N][VEC];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = (i * THREADS + tid) * VEC;
    if (VEC == 4) {
      if (at < width) *reinterpret_cast<Four<T>*>(x[i]) = *reinterpret_cast<const Four<T>*>(in + at);
    } else if (at < width) {
      x[i][0] = in[at];
    }
  }
  if (a.tokens || a.K) {
    if (a.tokens)
      for (int i = tid; i < PIECE; i += THREADS) counts[i] = 0;
    if (a.K)
      for (int i = tid; i < PIECE; i += THREADS) bias[i] = 0.f;
    __syncthreads();
    if (a.tokens) {
      const int n = a.length ? min(a.length[b], a.L) : a.L, prompt = a.prompt ? a.prompt[b] : 0;
      const int* row = a.tokens + static_cast<int64_t>(b) * a.L;
#pragma unroll 4
      for (int i = tid; i < n; i += THREADS) {
        const uint32_t at = static_cast<uint32_t>(row[i] - c0);
        if (at < static_cast<uint32_t>(width)) {
          if (i < prompt) atomicOr(counts + at, PROMPT);
          else atomicAdd(counts + at, 1u);
        }
      }
    }
    if (a.K && tid < 32) {
      for (int i = 0; i < a.K; i += 32) {
        const bool live = i + tid < a.K;
        const int64_t e = static_cast<int64_t>(b) * a.K + i + tid;
        const uint32_t at = live ? static_cast<uint32_t>(a.bias_ids[e] - c0) : 0xffffffffu;
        const float v = live ? a.bias[e] : 0.f;
        const uint32_t same = __match_any_sync(0xffffffffu, at);
        float sum = at < static_cast<uint32_t>(width) ? bias[at] : 0.f;
#pragma unroll
        for (int l = 0; l < 32; ++l) {
          const float w = __shfl_sync(0xffffffffu, v, l);
          if ((same >> l) & 1u) sum += w;
        }
        if (at < static_cast<uint32_t>(width) && (same & ((1u << tid) - 1u)) == 0) bias[at] = sum;
        __syncwarp();
      }
    }
    __syncthreads();
  }
  const float r = a.repetition ? a.repetition[b] : 1.f;
  const float presence = a.presence ? a.presence[b] : 0.f, frequency = a.frequency ? a.frequency[b] : 0.f;
  const int* allowed = a.allowed ? a.allowed + static_cast<int64_t>(b) * a.words : nullptr;
  float* out = a.out + static_cast<int64_t>(b) * a.V + c0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = (i * THREADS + tid) * VEC;
    if (at >= width) continue;
    const uint32_t word = allowed ? static_cast<uint32_t>(allowed[(c0 + at) >> 5]) >> (at & 31) : 0xffffffffu;
    float y[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float v = In<T>::f(x[i][e]);
      if (a.tokens) {
        const uint32_t c = counts[at + e], n = c & ~PROMPT;
        if (c) v = v > 0.f ? v / r : v * r;
        if (n) v = v - frequency * static_cast<float>(n) - presence;
      }
      if (a.K) v += bias[at + e];
      y[e] = (word >> e) & 1u ? v : -INFINITY;
    }
    if (VEC == 4) *reinterpret_cast<float4*>(out + at) = make_float4(y[0], y[VEC > 1 ? 1 : 0], y[VEC > 2 ? 2 : 0], y[VEC > 3 ? 3 : 0]);
    else out[at] = y[0];
  }
}

template <class T, int PIECE>
static int launch(const LogitsArgs& a, cudaStream_t s) {
  const dim3 grid((a.V + PIECE - 1) / PIECE, a.B);
  const int smem = PIECE * 4 * ((a.tokens ? 1 : 0) + (a.K ? 1 : 0));
  const bool vec = a.V % 4 == 0 && a.row_stride % 4 == 0 &&
                   reinterpret_cast<uintptr_t>(a.logits) % (4 * sizeof(T)) == 0;
  if (vec) {
    static std::atomic<uint64_t> done{0};
    if (smem_limit(done, adjust_kernel<T, PIECE, 4>, PIECE * 8) != cudaSuccess) return -1;
    adjust_kernel<T, PIECE, 4><<<grid, THREADS, smem, s>>>(a);
  } else {
    static std::atomic<uint64_t> done{0};
    if (smem_limit(done, adjust_kernel<T, PIECE, 1>, PIECE * 8) != cudaSuccess) return -1;
    adjust_kernel<T, PIECE, 1><<<grid, THREADS, smem, s>>>(a);
  }
  return 0;
}
template <class T>
static int by_piece(const LogitsArgs& a, cudaStream_t s) {
  // large pieces read the token list less often, small ones reach more SMs
  if (static_cast<int64_t>(a.B) * ((a.V + 4095) / 4096) >= 2 * a.sms) return launch<T, 4096>(a, s);
  return launch<T, 1024>(a, s);
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
