// K10c: the gated delta rule token by token, for decoding and short prompts:
//
//   S <- diag(a) S,   u = beta (v - k^T S),   S <- S + k u^T,   o = q^T S,     a = e^g (per head or per feature)
//
// The columns of S do not meet, so a warp keeps 8 of them in registers (a thread: one column, a quarter of
// its rows) from the call's first token to its last; the state is read once and written once.  With
// k^T (a S) and q^T (a S) taken in one pass,  o = q^T (a S) + (q . k) u  needs no second one: a token costs
// two shuffles in a row and the update, which the next token's pass follows register by register.
//
// One token: the state's 8 D D bytes a head bound it; a thread's 32 loads are all in flight before the first
// is used.  Many tokens: the chain of pass, shuffles and update bounds it.  A CTA holds 32 columns (128
// threads), so one row of 12 heads already loads 48 SMs.
#include "delta_step.h"
#include "common.cuh"

#include <cuda_fp16.h>

namespace nt {
namespace dstep {

constexpr int THREADS = 128, COLS = 32, CHUNK = 8;  // tokens prepared at a time

NT_DEVICE float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
NT_DEVICE float to_f(__half v) { return __half2float(v); }
NT_DEVICE float to_f(float v) { return v; }
template <class T> NT_DEVICE T from_f(float v);
template <> NT_DEVICE __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> NT_DEVICE __half from_f(float v) { return __float2half_rn(v); }
template <> NT_DEVICE float from_f(float v) { return v; }

template <class T, int N>
struct alignas(N * sizeof(T)) Vec {
  T x[N];
};

template <int D, int GATE>
struct Token {  // as fp32 in shared memory; quarters of the features lie in different banks
  static constexpr int Q = D / 4 + 4;
  alignas(16) float k[4 * Q];
  alignas(16) float q[4 * Q];
  alignas(16) float a[GATE == 2 ? 4 * Q : 4];
  float v[COLS];
  float beta, decay, qk, unused;
};

template <class T, int D, int GATE>
struct Raw {  // one token in registers: D / 32 features a lane
  static constexpr int E = D / 32;
  float q[E], k[E], a[GATE == 2 ? E : 1], v, beta;
};

template <class T, int D, int GATE>
__global__ void __launch_bounds__(THREADS) delta_step_kernel(const DeltaStepArgs p) {
  constexpr int E = D / 32, R = D / 4, BLOCKS = D / COLS, PER_WARP = CHUNK / (THREADS / 32);
  using Tok = Token<D, GATE>;
  __shared__ Tok toks[2][CHUNK];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cb = blockIdx.x % BLOCKS;
  const int bh = blockIdx.x / BLOCKS;
  const int b = bh / p.H, h = bh - b * p.H;
  const int64_t slot = p.slots ? p.slots[b] : b;
  int n = p.count ? min(max(p.count[b], 0), p.T) : p.T;
  if (slot < 0 || slot >= p.states) {
    if (slot >= p.states && threadIdx.x == 0) record_error(1, b);
    n = 0;
  }
  const int col = cb * COLS + warp * 8 + (lane & 7), quarter = lane >> 3;
  float* sp = p.state + ((n ? slot : 0) * p.H + h) * D * D + static_cast<int64_t>(quarter) * R * D + col;
  T* op = static_cast<T*>(p.o) + (static_cast<int64_t>(b) * p.T * p.H + h) * D + col;
  const int64_t ostep = static_cast<int64_t>(p.H) * D;

  if (n > 0) {
    float2 S[R / 2];
#pragma unroll
    for (int r = 0; r < R / 2; ++r) S[r] = make_float2(sp[2 * r * D], sp[(2 * r + 1) * D]);

    Raw<T, D, GATE> raw[PER_WARP];
    auto load = [&](int base) {
#pragma unroll
      for (int i = 0; i < PER_WARP; ++i) {
        const int64_t t = base + warp * PER_WARP + i;
        if (t >= n) break;
        const auto qv = *reinterpret_cast<const Vec<T, E>*>(static_cast<const T*>(p.q) + b * p.qs[0] + t * p.qs[1] +
                                                            h * p.qs[2] + lane * E);
        const auto kv = *reinterpret_cast<const Vec<T, E>*>(static_cast<const T*>(p.k) + b * p.ks[0] + t * p.ks[1] +
                                                            h * p.ks[2] + lane * E);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          raw[i].q[e] = to_f(qv.x[e]);
          raw[i].k[e] = to_f(kv.x[e]);
        }
        if (GATE == 2) {
          const auto gv = *reinterpret_cast<const Vec<float, E>*>(p.g + b * p.gs[0] + t * p.gs[1] + h * p.gs[2] + lane * E);
#pragma unroll
          for (int e = 0; e < E; ++e) raw[i].a[e] = gv.x[e];
        } else if (GATE == 1) {
          raw[i].a[0] = p.g[b * p.gs[0] + t * p.gs[1] + h * p.gs[2]];
        }
        raw[i].v = to_f(static_cast<const T*>(p.v)[b * p.vs[0] + t * p.vs[1] + h * p.vs[2] + cb * COLS + lane]);
        const int64_t at = b * p.bs[0] + t * p.bs[1] + h * p.bs[2];
        raw[i].beta = p.beta_f32 ? static_cast<const float*>(p.beta)[at] : to_f(static_cast<const T*>(p.beta)[at]);
      }
    };
    auto store = [&](int buf, int base) {
#pragma unroll
      for (int i = 0; i < PER_WARP; ++i) {
        if (base + warp * PER_WARP + i >= n) break;
        Tok& tk = toks[buf][warp * PER_WARP + i];
        float qq = 0.f, kk = 0.f, qk = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          qq = fmaf(raw[i].q[e], raw[i].q[e], qq);
          kk = fmaf(raw[i].k[e], raw[i].k[e], kk);
          qk = fmaf(raw[i].q[e], raw[i].k[e], qk);
        }
        qk = warp_sum(qk);
        float fq = p.scale, fk = 1.f;
        if (p.l2norm) {
          fq = p.scale / fmaxf(sqrtf(warp_sum(qq)), 1e-12f);
          fk = 1.f / fmaxf(sqrtf(warp_sum(kk)), 1e-12f);
        }
        const int f = lane * E, at = (f / R) * Tok::Q + f % R;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          tk.q[at + e] = raw[i].q[e] * fq;
          tk.k[at + e] = raw[i].k[e] * fk;
          if (GATE == 2) tk.a[at + e] = expf(raw[i].a[e]);
        }
        tk.v[lane] = raw[i].v;
        if (lane == 0) {
          tk.beta = raw[i].beta;
          tk.decay = GATE == 1 ? expf(raw[i].a[0]) : 1.f;
          tk.qk = qk * fq * fk;
        }
      }
    };

    load(0);
    store(0, 0);
    __syncthreads();
    for (int base = 0, buf = 0; base < n; base += CHUNK, buf ^= 1) {
      const bool more = base + CHUNK < n;
      if (more) load(base + CHUNK);
      const int m = min(CHUNK, n - base);
      for (int i = 0; i < m; ++i) {
        const Tok& tk = toks[buf][i];
        const float4* k4 = reinterpret_cast<const float4*>(tk.k + quarter * Tok::Q);
        const float4* q4 = reinterpret_cast<const float4*>(tk.q + quarter * Tok::Q);
        const float4* a4 = reinterpret_cast<const float4*>(tk.a + (GATE == 2 ? quarter * Tok::Q : 0));
        float2 dk[2] = {{0.f, 0.f}, {0.f, 0.f}}, dq[2] = {{0.f, 0.f}, {0.f, 0.f}};
        float4 kv[R / 4];
#pragma unroll
        for (int r = 0; r < R / 4; ++r) {
          const float4 qv = q4[r];
          kv[r] = k4[r];
          if (GATE == 2) {
            const float4 av = a4[r];
            S[2 * r] = mul2(S[2 * r], make_float2(av.x, av.y));
            S[2 * r + 1] = mul2(S[2 * r + 1], make_float2(av.z, av.w));
          }
          dk[0] = fma2(S[2 * r], make_float2(kv[r].x, kv[r].y), dk[0]);
          dk[1] = fma2(S[2 * r + 1], make_float2(kv[r].z, kv[r].w), dk[1]);
          dq[0] = fma2(S[2 * r], make_float2(qv.x, qv.y), dq[0]);
          dq[1] = fma2(S[2 * r + 1], make_float2(qv.z, qv.w), dq[1]);
        }
        dk[0] = add2(dk[0], dk[1]);
        dq[0] = add2(dq[0], dq[1]);
        float ks = dk[0].x + dk[0].y, qs = dq[0].x + dq[0].y;
#pragma unroll
        for (int o = 8; o < 32; o <<= 1) {
          ks += __shfl_xor_sync(0xffffffffu, ks, o);
          qs += __shfl_xor_sync(0xffffffffu, qs, o);
        }
        const float decay = GATE == 1 ? tk.decay : 1.f;
        const float u = tk.beta * fmaf(-decay, ks, tk.v[warp * 8 + (lane & 7)]);
        const float2 u2 = make_float2(u, u), d2 = make_float2(decay, decay);
#pragma unroll
        for (int r = 0; r < R / 4; ++r) {
          const float2 lo = make_float2(kv[r].x, kv[r].y), hi = make_float2(kv[r].z, kv[r].w);
          if (GATE == 1) {
            S[2 * r] = fma2(S[2 * r], d2, mul2(lo, u2));
            S[2 * r + 1] = fma2(S[2 * r + 1], d2, mul2(hi, u2));
          } else {
            S[2 * r] = fma2(lo, u2, S[2 * r]);
            S[2 * r + 1] = fma2(hi, u2, S[2 * r + 1]);
          }
        }
        if (quarter == 0) op[(base + i) * ostep] = from_f<T>(fmaf(tk.qk, u, decay * qs));
      }
      if (more) {
        store(buf ^ 1, base + CHUNK);
        __syncthreads();
      }
    }
#pragma unroll
    for (int r = 0; r < R / 2; ++r) {
      sp[2 * r * D] = S[r].x;
      sp[(2 * r + 1) * D] = S[r].y;
    }
  }
  if (quarter == 0)
    for (int t = n; t < p.T; ++t) op[t * ostep] = from_f<T>(0.f);
}

template <class T, int D>
static void launch(const DeltaStepArgs& a, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(a.B * a.H * (D / COLS));
  if (a.gate == 0) delta_step_kernel<T, D, 0><<<grid, THREADS, 0, s>>>(a);
  else if (a.gate == 1) delta_step_kernel<T, D, 1><<<grid, THREADS, 0, s>>>(a);
  else delta_step_kernel<T, D, 2><<<grid, THREADS, 0, s>>>(a);
}
template <class T>
static int by_width(const DeltaStepArgs& a, cudaStream_t s) {
  if (a.D == 128) launch<T, 128>(a, s);
  else if (a.D == 64) launch<T, 64>(a, s);
  else return -1;
  return 0;
}

}  // namespace dstep
}  // namespace nt

using namespace nt::dstep;

int nt_delta_step(const DeltaStepArgs& a, cudaStream_t s) {
  if (a.B == 0 || a.T == 0 || a.H == 0) return 0;
  if (static_cast<int64_t>(a.B) * a.H * 4 > INT32_MAX || a.gate < 0 || a.gate > 2) return -1;
  if (a.type == DELTA_STEP_BF16) return by_width<__nv_bfloat16>(a, s);
  if (a.type == DELTA_STEP_FP16) return by_width<__half>(a, s);
  if (a.type == DELTA_STEP_FP32) return by_width<float>(a, s);
  return -1;
}

int nt_delta_step_read_error(unsigned* where) {
  nt::ErrorWord e{};
  cudaMemcpyFromSymbol(&e, nt::g_nt_error, sizeof(e));
  if (where) *where = e.where;
  if (e.code) {
    const nt::ErrorWord z{};
    cudaMemcpyToSymbol(nt::g_nt_error, &z, sizeof(z));
  }
  return static_cast<int>(e.code);
}
