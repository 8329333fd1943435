// K10c: the gated delta rule with a carried state, for decoding and short prompts:
//
//   S <- diag(a) S,   u = beta (v - k^T S),   S <- S + k u^T,   o = q^T S,     a = e^g (per head or per feature)
//
// The columns of S do not meet, so a CTA takes 32 of them and one row of 12 heads already loads 48 SMs.  With
// k^T (a S) and q^T (a S) taken in one pass,  o = q^T (a S) + (q . k) u  needs no second one.
//
// step_kernel (one token): the state's 8 D D bytes a head bound it.  A lane holds a column and a warp a quarter
// of its rows, so that every access is a full line; a thread's loads of the state are all in flight before the
// first is used, and the quarters, the norms of q and k included, meet at one barrier.
//
// block_kernel (more tokens): eight tokens at a time.  With c_i the decay from the block's start through token i and
// c_ij that behind token j through token i,
//   u_i = beta_i (v_i - (k_i c_i)^T S - sum_{j<i} M_ij u_j),     M_ij = k_i^T c_ij k_j
//   o_i = (q_i c_i)^T S + sum_{j<=i} N_ij u_j,                   N_ij = q_i^T c_ij k_j
//   S  <- c_7 S + sum_j (c_7j k_j) u_j^T
// so the chain through S, its reduction and its update is walked once for eight tokens.  Decays are products of a
// (never quotients or differences of sums), so none overflows and a decay of 0 is one.  Four warps hold the columns
// in registers (a lane: CPL columns, an eighth of their rows) and read the block's vectors from shared memory, each
// 16 bytes for 4 CPL products; four more prepare the next block meanwhile, a thread for each feature.  The state is
// read once and written once.
#include "delta_step.h"
#include "common.cuh"

#include <cuda_fp16.h>

namespace nt {
namespace dstep {

constexpr int COLS = 32, C = 8;

NT_DEVICE float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
NT_DEVICE float to_f(__half v) { return __half2float(v); }
NT_DEVICE float to_f(float v) { return v; }
template <class T> NT_DEVICE T from_f(float v);
template <> NT_DEVICE __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> NT_DEVICE __half from_f(float v) { return __float2half_rn(v); }
template <> NT_DEVICE float from_f(float v) { return v; }

// What a row of the call has to do: its state and its number of tokens.
NT_DEVICE int tokens_of(const DeltaStepArgs& p, int b, bool report, int64_t& slot) {
  slot = p.slots ? p.slots[b] : b;
  if (slot >= 0 && slot < p.states) return p.count ? min(max(p.count[b], 0), p.T) : p.T;
  if (slot >= p.states && report) record_error(1, b);
  return 0;
}
template <class T>
NT_DEVICE float beta_of(const DeltaStepArgs& p, int64_t at) {
  return p.beta_f32 ? static_cast<const float*>(p.beta)[at] : to_f(static_cast<const T*>(p.beta)[at]);
}

// ------------------------------------------------------------------------------------ one token
template <class T, int D, int GATE>
__global__ void __launch_bounds__(128) step_kernel(const DeltaStepArgs p) {
  constexpr int R = D / 4, BLOCKS = D / COLS;  // rows of a warp
  __shared__ __align__(16) float ks[4][R], qs[4][R], as[4][GATE == 2 ? R : 4];
  __shared__ float dots[4][2][COLS], norms[4][3];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cb = blockIdx.x % BLOCKS, bh = blockIdx.x / BLOCKS;
  const int b = bh / p.H, h = bh - b * p.H;
  int64_t slot;
  const int n = tokens_of(p, b, threadIdx.x == 0, slot);
  const int col = cb * COLS + lane;
  T* op = static_cast<T*>(p.o) + static_cast<int64_t>(bh) * D + col;
  if (n == 0) {
    if (warp == 0) *op = from_f<T>(0.f);
    return;
  }
  float* sp = p.state + (slot * p.H + h) * D * D + static_cast<int64_t>(warp * R) * D + col;
  float S[R];
#pragma unroll
  for (int r = 0; r < R; ++r) S[r] = sp[r * D];
  float kr = 0.f, qr = 0.f;
  if (lane < R) {
    const int f = warp * R + lane;
    kr = to_f(static_cast<const T*>(p.k)[b * p.ks[0] + h * p.ks[2] + f]);
    qr = to_f(static_cast<const T*>(p.q)[b * p.qs[0] + h * p.qs[2] + f]);
    ks[warp][lane] = kr;
    qs[warp][lane] = qr;
    if (GATE == 2) as[warp][lane] = expf(p.g[b * p.gs[0] + h * p.gs[2] + f]);
  }
  const float decay = GATE == 1 ? expf(p.g[b * p.gs[0] + h * p.gs[2]]) : 1.f;
  const float beta = beta_of<T>(p, b * p.bs[0] + h * p.bs[2]);
  const float v = to_f(static_cast<const T*>(p.v)[b * p.vs[0] + h * p.vs[2] + col]);
  const float kk = warp_sum(kr * kr), qq = warp_sum(qr * qr), qk = warp_sum(qr * kr);
  if (lane == 0) {
    norms[warp][0] = kk;
    norms[warp][1] = qq;
    norms[warp][2] = qk;
  }
  __syncwarp();
  float dk = 0.f, dq = 0.f;
#pragma unroll
  for (int r = 0; r < R; r += 4) {
    const float4 k4 = *reinterpret_cast<const float4*>(&ks[warp][r]), q4 = *reinterpret_cast<const float4*>(&qs[warp][r]);
    if (GATE == 2) {
      const float4 a4 = *reinterpret_cast<const float4*>(&as[warp][r]);
      S[r] *= a4.x; S[r + 1] *= a4.y; S[r + 2] *= a4.z; S[r + 3] *= a4.w;
    }
    dk = fmaf(k4.x, S[r], dk); dk = fmaf(k4.y, S[r + 1], dk); dk = fmaf(k4.z, S[r + 2], dk); dk = fmaf(k4.w, S[r + 3], dk);
    dq = fmaf(q4.x, S[r], dq); dq = fmaf(q4.y, S[r + 1], dq); dq = fmaf(q4.z, S[r + 2], dq); dq = fmaf(q4.w, S[r + 3], dq);
  }
  dots[warp][0][lane] = dk;
  dots[warp][1][lane] = dq;
  __syncthreads();
  dk = dots[0][0][lane] + dots[1][0][lane] + dots[2][0][lane] + dots[3][0][lane];
  dq = dots[0][1][lane] + dots[1][1][lane] + dots[2][1][lane] + dots[3][1][lane];
  float fk = 1.f, fq = p.scale;
  if (p.l2norm) {
    fk = 1.f / fmaxf(sqrtf(norms[0][0] + norms[1][0] + norms[2][0] + norms[3][0]), 1e-12f);
    fq = p.scale / fmaxf(sqrtf(norms[0][1] + norms[1][1] + norms[2][1] + norms[3][1]), 1e-12f);
  }
  const float u = beta * fmaf(-decay * fk, dk, v), ku = fk * u;
#pragma unroll
  for (int r = 0; r < R; r += 4) {
    const float4 k4 = *reinterpret_cast<const float4*>(&ks[warp][r]);
    sp[r * D] = fmaf(k4.x, ku, decay * S[r]);
    sp[(r + 1) * D] = fmaf(k4.y, ku, decay * S[r + 1]);
    sp[(r + 2) * D] = fmaf(k4.z, ku, decay * S[r + 2]);
    sp[(r + 3) * D] = fmaf(k4.w, ku, decay * S[r + 3]);
  }
  if (warp == 0)
    *op = from_f<T>(fq * fmaf(norms[0][2] + norms[1][2] + norms[2][2] + norms[3][2], ku, decay * dq));
}

// ---------------------------------------------------------------------------------- more tokens
constexpr int PAIRS = C * (C + 1) / 2;  // (i, j) with j <= i, at i (i + 1) / 2 + j
constexpr int SUMS = 2 * PAIRS + C;     // k_i c_ij k_j, q_i c_ij k_j, q_i q_i

template <int D, int GATE, int COLS_>
struct Block {  // eight tokens; the eighths of a vector lie in different banks
  static constexpr int R = D / 8, SL = R + 4, ROW = 8 * SL;
  alignas(16) float k[C][ROW];    // c_i k_i
  alignas(16) float q[C][ROW];    // c_i q_i
  alignas(16) float kc[C][ROW];   // c_7j k_j
  alignas(16) float c7[GATE == 2 ? ROW : 4];
  alignas(16) float Mt[C][C];     // Mt[j][i] = M_ij
  alignas(16) float N[C][C];      // 0 above the diagonal
  alignas(16) float beta[C];
  float v[C][COLS_];
};

// Sums of N values a lane over the warp: lane l (l % 16 for 16 values) gets the l-th sum.
template <int N>
NT_DEVICE float reduce_scatter(float (&x)[N], int lane) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) {
    const bool upper = lane & o;
#pragma unroll
    for (int e = 0; e < o; ++e) {
      const float other = __shfl_xor_sync(0xffffffffu, upper ? x[e] : x[e + o], o);
      x[e] = (upper ? x[e + o] : x[e]) + other;
    }
  }
  if (N == 16) x[0] += __shfl_xor_sync(0xffffffffu, x[0], 16);
  return x[0];
}
// The place of token pair e (compile-time after unrolling).
NT_DEVICE constexpr int pair_i(int e) {
  int i = 0;
  while ((i + 1) * (i + 2) / 2 <= e) ++i;
  return i;
}
NT_DEVICE constexpr int pair_j(int e) { return e - pair_i(e) * (pair_i(e) + 1) / 2; }

template <class T, int D, int GATE, int CPL>
__global__ void __launch_bounds__(256, 1) block_kernel(const DeltaStepArgs p) {
  constexpr int W = 16 * CPL, BLOCKS = D / W, R = D / 8;  // columns of a CTA; rows of a lane
  using B = Block<D, GATE, W>;
  __shared__ B blocks[2];
  __shared__ float partial[D / 32][SUMS], total[SUMS];
  __shared__ __align__(16) float norm[2 * C];  // of k, of q
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) & 3;
  const int cb = blockIdx.x % BLOCKS, bh = blockIdx.x / BLOCKS;
  const int b = bh / p.H, h = bh - b * p.H;
  int64_t slot;
  const int n = tokens_of(p, b, threadIdx.x == 0, slot), rounds = (n + C - 1) / C;

  if (threadIdx.x >= 128) {
    // ---- the warps that prepare: thread f has feature f of the eight tokens
    const int f = threadIdx.x - 128, at = (f / R) * B::SL + f % R;
    const bool has = f < D;
    T rk[C], rq[C], rv[CPL];
    float rg[C], rbeta = 0.f;
    const int vt = f >> 4, vc = (f & 15) * CPL;  // the value entries it brings
    auto load = [&](int round) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int64_t t = round * C + i;
        rk[i] = rq[i] = from_f<T>(0.f);
        rg[i] = 0.f;
        if (t >= n) continue;  // behind the row's last token: nothing, with a decay of 1
        if (has) {
          rk[i] = static_cast<const T*>(p.k)[b * p.ks[0] + t * p.ks[1] + h * p.ks[2] + f];
          rq[i] = static_cast<const T*>(p.q)[b * p.qs[0] + t * p.qs[1] + h * p.qs[2] + f];
        }
        const int64_t ga = b * p.gs[0] + t * p.gs[1] + h * p.gs[2];
        if (GATE == 2 && has) rg[i] = p.g[ga + f];
        if (GATE == 1) rg[i] = p.g[ga];
      }
      const int64_t t = round * C + vt;
#pragma unroll
      for (int e = 0; e < CPL; ++e)
        rv[e] = t < n ? static_cast<const T*>(p.v)[b * p.vs[0] + t * p.vs[1] + h * p.vs[2] + cb * W + vc + e] : from_f<T>(0.f);
      const int64_t tb = round * C + f;
      rbeta = f < C && tb < n ? beta_of<T>(p, b * p.bs[0] + tb * p.bs[1] + h * p.bs[2]) : 0.f;
    };
    auto prepare = [&](int round) {
      B& blk = blocks[round & 1];
      float k[C], q[C], c[C], ck[PAIRS];  // c: from the block's start; ck: c_ij k_j
#pragma unroll
      for (int i = 0; i < C; ++i) {
        k[i] = to_f(rk[i]);
        q[i] = to_f(rq[i]);
        const float a = GATE ? expf(rg[i]) : 1.f;
        c[i] = i && GATE ? c[i - 1] * a : a;
#pragma unroll
        for (int j = 0; j <= i; ++j) {
          const int e = i * (i + 1) / 2 + j;
          ck[e] = j == i ? k[i] : GATE ? ck[(i - 1) * i / 2 + j] * a : k[j];
        }
      }
#pragma unroll
      for (int e = 0; e < CPL; ++e) blk.v[vt][vc + e] = to_f(rv[e]);
      if (f < C) blk.beta[f] = rbeta;
      if (round + 1 < rounds) load(round + 1);
      if (has) {
        float x[32], y[32], z[16];
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = k[pair_i(e)] * ck[e];
        partial[warp][lane] = reduce_scatter<32>(x, lane);
#pragma unroll
        for (int e = 0; e < 32; ++e) y[e] = q[pair_i(e)] * ck[e];
        partial[warp][PAIRS + lane] = reduce_scatter<32>(y, lane);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          z[e] = e < 4 ? k[C - 1] * ck[32 + e] : e < 8 ? q[C - 1] * ck[28 + e] : q[e - 8] * q[e - 8];
        const float last = reduce_scatter<16>(z, lane);
        if (lane < 16) partial[warp][lane < 4 ? 32 + lane : lane < 8 ? PAIRS + 28 + lane : 2 * PAIRS + lane - 8] = last;
      }
      named_bar_sync(1, 128);
      auto sum = [&](int e) {
        float x = partial[0][e];
#pragma unroll
        for (int w = 1; w < D / 32; ++w) x += partial[w][e];
        return x;
      };
      if (f < SUMS) total[f] = sum(f);
      if (f >= 128 - 2 * C) {
        const int e = f - (128 - 2 * C);
        const float x = sum(e < C ? e * (e + 3) / 2 : 2 * PAIRS + e - C);
        norm[e] = (e < C ? 1.f : p.scale) * (p.l2norm ? 1.f / fmaxf(sqrtf(x), 1e-12f) : 1.f);
      }
      named_bar_sync(1, 128);
      if (f < C * C) {
        const int i = f / C, j = f % C, e = i * (i + 1) / 2 + j;
        blk.N[i][j] = j <= i ? total[PAIRS + e] * norm[C + i] * norm[j] : 0.f;
        if (j < i) blk.Mt[j][i] = total[e] * norm[i] * norm[j];
      }
      if (has) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
          blk.k[i][at] = k[i] * c[i] * norm[i];
          blk.q[i][at] = q[i] * c[i] * norm[C + i];
          blk.kc[i][at] = ck[(C - 1) * C / 2 + i] * norm[i];
        }
        if (GATE == 2) blk.c7[at] = c[C - 1];
        if (GATE == 1 && f == 0) blk.c7[0] = c[C - 1];
      }
    };
    if (rounds > 0) {
      load(0);
      prepare(0);
    }
    __syncthreads();
    for (int round = 0; round < rounds; ++round) {
      if (round + 1 < rounds) prepare(round + 1);
      __syncthreads();
    }
    return;
  }

  // ---- the warps that hold the state: lane (slice, lc) has rows slice R .. of columns col .. col + CPL - 1
  const int slice = lane >> 2, mine = CPL == 2 ? slice & 1 : 0;  // the one of its columns that it solves for
  const int local = warp * 4 * CPL + (lane & 3) * CPL, col = cb * W + local;
  float* sp = p.state + ((n ? slot : 0) * p.H + h) * D * D + static_cast<int64_t>(slice) * R * D + col;
  T* op = static_cast<T*>(p.o) + (static_cast<int64_t>(b) * p.T * p.H + h) * D + col + mine;
  const int64_t ostep = static_cast<int64_t>(p.H) * D;
  float2 S[CPL][R / 2];
  if (n > 0) {
#pragma unroll
    for (int r = 0; r < R / 2; ++r)
#pragma unroll
      for (int e = 0; e < CPL; ++e) S[e][r] = make_float2(sp[2 * r * D + e], sp[(2 * r + 1) * D + e]);
  }
  __syncthreads();
  for (int round = 0; round < rounds; ++round) {
    const B& blk = blocks[round & 1];
    // products of the state with eight vectors, over this lane's rows
    auto products = [&](const float (&vec)[C][B::ROW], float (&x)[CPL][C]) {
      float2 acc[CPL][C];
#pragma unroll
      for (int e = 0; e < CPL; ++e)
#pragma unroll
        for (int i = 0; i < C; ++i) acc[e][i] = make_float2(0.f, 0.f);
#pragma unroll
      for (int r = 0; r < R / 4; ++r)
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const float4 w = *reinterpret_cast<const float4*>(&vec[i][slice * B::SL + r * 4]);
#pragma unroll
          for (int e = 0; e < CPL; ++e) {
            acc[e][i] = fma2(S[e][2 * r], make_float2(w.x, w.y), acc[e][i]);
            acc[e][i] = fma2(S[e][2 * r + 1], make_float2(w.z, w.w), acc[e][i]);
          }
        }
#pragma unroll
      for (int e = 0; e < CPL; ++e)
#pragma unroll
        for (int i = 0; i < C; ++i) x[e][i] = acc[e][i].x + acc[e][i].y;
    };
    float x[CPL][C], y[CPL][C], u[CPL][C];
    products(blk.k, x);
    products(blk.q, y);
    // the column's own sums, over the eight slices
    float own[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      if (CPL == 2) own[i] = (mine ? x[CPL - 1][i] : x[0][i]) + __shfl_xor_sync(0xffffffffu, mine ? x[0][i] : x[CPL - 1][i], 4);
      else own[i] = x[0][i] + __shfl_xor_sync(0xffffffffu, x[0][i], 4);
      own[i] += __shfl_xor_sync(0xffffffffu, own[i], 8);
      own[i] += __shfl_xor_sync(0xffffffffu, own[i], 16);
      own[i] = blk.v[i][local + mine] - own[i];
    }
#pragma unroll
    for (int j = 0; j < C; ++j) {
      own[j] *= blk.beta[j];
#pragma unroll
      for (int i = j + 1; i < C; ++i) own[i] = fmaf(-blk.Mt[j][i], own[j], own[i]);
    }
    // q sums: a lane keeps CPL tokens of its own column
    const bool b0 = slice & 1, b1 = slice & 2, b2 = slice & 4;
    float qs[C];
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (CPL == 2) qs[i] = (mine ? y[CPL - 1][i] : y[0][i]) + __shfl_xor_sync(0xffffffffu, mine ? y[0][i] : y[CPL - 1][i], 4);
      else qs[i] = y[0][i];
    int token = 0;
    auto halve = [&](int keep, bool upper, int lanes) {
#pragma unroll
      for (int i = 0; i < C / 2; ++i)
        if (i < keep) {
          const float other = __shfl_xor_sync(0xffffffffu, upper ? qs[i] : qs[i + keep], lanes);
          qs[i] = (upper ? qs[i + keep] : qs[i]) + other;
        }
      token += upper ? keep : 0;
    };
    halve(4, b1, 8);
    halve(2, b2, 16);
    if (CPL == 1) halve(1, b0, 4);
#pragma unroll
    for (int e = 0; e < CPL; ++e) {
      const int i = token + e;
      float o = qs[e];
#pragma unroll
      for (int j = 0; j < C; ++j) o = fmaf(blk.N[i][j], own[j], o);
      if (round * C + i < n) op[(round * C + i) * ostep] = from_f<T>(o);
    }
#pragma unroll
    for (int j = 0; j < C; ++j) {
      if (CPL == 2) {
        const float other = __shfl_xor_sync(0xffffffffu, own[j], 4);
        u[0][j] = mine ? other : own[j];
        u[CPL - 1][j] = mine ? own[j] : other;
      } else {
        u[0][j] = own[j];
      }
    }
#pragma unroll
    for (int r = 0; r < R / 4; ++r) {
      if (GATE) {
        const float4 c4 = GATE == 2 ? *reinterpret_cast<const float4*>(&blk.c7[slice * B::SL + r * 4])
                                    : make_float4(blk.c7[0], blk.c7[0], blk.c7[0], blk.c7[0]);
#pragma unroll
        for (int e = 0; e < CPL; ++e) {
          S[e][2 * r] = mul2(S[e][2 * r], make_float2(c4.x, c4.y));
          S[e][2 * r + 1] = mul2(S[e][2 * r + 1], make_float2(c4.z, c4.w));
        }
      }
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const float4 w = *reinterpret_cast<const float4*>(&blk.kc[j][slice * B::SL + r * 4]);
#pragma unroll
        for (int e = 0; e < CPL; ++e) {
          const float2 u2 = make_float2(u[e][j], u[e][j]);
          S[e][2 * r] = fma2(make_float2(w.x, w.y), u2, S[e][2 * r]);
          S[e][2 * r + 1] = fma2(make_float2(w.z, w.w), u2, S[e][2 * r + 1]);
        }
      }
    }
    __syncthreads();
  }
  if (n > 0) {
#pragma unroll
    for (int r = 0; r < R / 2; ++r)
#pragma unroll
      for (int e = 0; e < CPL; ++e) {
        sp[2 * r * D + e] = S[e][r].x;
        sp[(2 * r + 1) * D + e] = S[e][r].y;
      }
  }
  if (slice < CPL)
    for (int t = n; t < p.T; ++t) op[t * ostep] = from_f<T>(0.f);
}

template <class T, int D, int GATE>
static void launch(const DeltaStepArgs& a, cudaStream_t s) {
  if (a.T == 1) step_kernel<T, D, GATE><<<static_cast<unsigned>(a.B * a.H * (D / COLS)), 128, 0, s>>>(a);
  else block_kernel<T, D, GATE, 2><<<static_cast<unsigned>(a.B * a.H * (D / 32)), 256, 0, s>>>(a);
}
template <class T, int D>
static void by_gate(const DeltaStepArgs& a, cudaStream_t s) {
  if (a.gate == 0) launch<T, D, 0>(a, s);
  else if (a.gate == 1) launch<T, D, 1>(a, s);
  else launch<T, D, 2>(a, s);
}
template <class T>
static int by_width(const DeltaStepArgs& a, cudaStream_t s) {
  if (a.D == 128) by_gate<T, 128>(a, s);
  else if (a.D == 64) by_gate<T, 64>(a, s);
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
