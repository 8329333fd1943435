// K10c: the gated delta rule with a carried state, for decoding and short prompts:
//
//   S <- diag(a) S,   u = beta (v - k^T S),   S <- S + k u^T,   o = q^T S,     a = e^g (per head or per feature)
//
// The columns of S do not meet, so a CTA takes 32 of them and one row of 12 heads already loads 48 SMs.  With
// k^T (a S) and q^T (a S) taken in one pass,  o = q^T (a S) + (q . k) u  needs no second one.
//
// step_kernel (one token): the state's 8 D D bytes a head bound it.  A lane holds a column and a warp a quarter
// of its rows, so that every access is a full line; a thread's loads of the state are all in flight before the
// first is used, and the quarters, the norms of q and k included, meet at one barrier.  160 rows of 12 heads of 128
// (KDA): 47 us for 255 MB, 5.4 TB/s of the 6.46 that a copy reaches; with warps on 8 columns, each access four quarter
// lines, it took 70.  One row: 3 us.
//
// More tokens: eight at a time.  With c_i the decay from the block's start through token i and c_ij that behind token j
// through token i,
//   u_i = beta_i (v_i - (k_i c_i)^T S - sum_{j<i} M_ij u_j),     M_ij = k_i^T c_ij k_j
//   o_i = (q_i c_i)^T S + sum_{j<=i} N_ij u_j,                   N_ij = q_i^T c_ij k_j
//   S  <- c_7 S + sum_j (c_7j k_j) u_j^T
// so the chain through S, its reduction and its update is walked once for eight tokens.  Decays are products of a
// (never quotients or differences of sums), so none overflows and a decay of 0 is one.
// prepare_kernel forms what does not depend on S, for all blocks at once; block_kernel walks a row's blocks in order:
// its warps hold the columns in registers (a lane: CPL columns, an eighth of their rows) and read the block's vectors
// from shared memory, each 16 bytes for 4 CPL products, while bulk copies bring the next blocks.  The state is read
// and written once a call (once for each segment of a long one).  The chain of a block bounds it: 1.3 us, of which
// the two passes over S take half, at one warp a scheduler.  4 rows of up to 389 tokens, 12 heads of 128 (GDN): 78 us;
// token by token it took 147, with the blocks' own products formed beside the walk instead of before it 103.
#include "delta_step.h"
#include "common.cuh"

#include <cuda_fp16.h>

#include <algorithm>

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
  if (slot >= p.states && report) record_error(2, b);
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

// What block_kernel reads of eight tokens of a head.  The eighths of a vector lie in different banks.
template <int D>
struct Block {
  static constexpr int R = D / 8, SL = R + 4, ROW = 8 * SL;
  float k[C][ROW];    // c_i k_i
  float q[C][ROW];    // c_i q_i
  float kc[C][ROW];   // c_7j k_j
  float c7[ROW];
  float Mt[C][C];     // Mt[j][i] = M_ij
  float N[C][C];      // 0 above the diagonal
  float beta[C];
};
template <int D>
struct Image {        // as it lies in the workspace
  Block<D> block;
  float v[D / 16][C][16];
};
static_assert(sizeof(Block<128>) % 16 == 0 && sizeof(Block<64>) % 16 == 0, "bulk copies take multiples of 16 bytes");

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

// Block `blockIdx.x % rounds` of the segment for one (row, head): thread f has feature f of its eight tokens.
template <class T, int D, int GATE>
__global__ void __launch_bounds__(D) prepare_kernel(const DeltaStepArgs p, const int t0, const int rounds, Image<D>* images) {
  constexpr int WARPS = D / 32;
  __shared__ float partial[WARPS][SUMS], total[SUMS];
  __shared__ float norm[2 * C];  // of k, of q
  const int f = threadIdx.x, lane = f & 31, warp = f >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int bh = blockIdx.x / rounds, b = bh / p.H, h = bh - b * p.H, first = t0 + (blockIdx.x - bh * rounds) * C;
  int64_t slot;
  const int n = tokens_of(p, b, f == 0, slot);
  if (first >= n) return;
  Image<D>& im = images[blockIdx.x];
  Block<D>& blk = im.block;
  float k[C], q[C], c[C], ck[PAIRS];  // c: from the block's start; ck: c_ij k_j
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int64_t t = first + i;
    float a = 1.f, v = 0.f;
    k[i] = q[i] = 0.f;
    if (t < n) {  // behind the row's last token: nothing, with a decay of 1
      k[i] = to_f(static_cast<const T*>(p.k)[b * p.ks[0] + t * p.ks[1] + h * p.ks[2] + f]);
      q[i] = to_f(static_cast<const T*>(p.q)[b * p.qs[0] + t * p.qs[1] + h * p.qs[2] + f]);
      v = to_f(static_cast<const T*>(p.v)[b * p.vs[0] + t * p.vs[1] + h * p.vs[2] + f]);
      if (GATE) a = expf(p.g[b * p.gs[0] + t * p.gs[1] + h * p.gs[2] + (GATE == 2 ? f : 0)]);
    }
    im.v[f >> 4][i][f & 15] = v;
    c[i] = i && GATE ? c[i - 1] * a : a;
#pragma unroll
    for (int j = 0; j <= i; ++j) {
      const int e = i * (i + 1) / 2 + j;
      ck[e] = j == i ? k[i] : GATE ? ck[(i - 1) * i / 2 + j] * a : k[j];
    }
  }
  if (f < C) blk.beta[f] = first + f < n ? beta_of<T>(p, b * p.bs[0] + (first + f) * p.bs[1] + h * p.bs[2]) : 0.f;
  {
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
  __syncthreads();
  for (int e = f; e < SUMS; e += D) {
    float x = partial[0][e];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) x += partial[w][e];
    total[e] = x;
  }
  __syncthreads();
  if (f < 2 * C) {
    const float x = total[f < C ? f * (f + 3) / 2 : 2 * PAIRS + f - C];
    norm[f] = (f < C ? 1.f : p.scale) * (p.l2norm ? 1.f / fmaxf(sqrtf(x), 1e-12f) : 1.f);
  }
  __syncthreads();
  if (f < C * C) {
    const int i = f / C, j = f % C, e = i * (i + 1) / 2 + j;
    blk.N[i][j] = j <= i ? total[PAIRS + e] * norm[C + i] * norm[j] : 0.f;
    blk.Mt[j][i] = j < i ? total[e] * norm[i] * norm[j] : 0.f;
  }
  constexpr int R = Block<D>::R, SL = Block<D>::SL;
  const int at = (f / R) * SL + f % R;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    blk.k[i][at] = k[i] * c[i] * norm[i];
    blk.q[i][at] = q[i] * c[i] * norm[C + i];
    blk.kc[i][at] = ck[(C - 1) * C / 2 + i] * norm[i];
  }
  blk.c7[at] = c[C - 1];
}

NT_DEVICE void bulk_load(void* dst, const void* src, int bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

constexpr int BUFFERS = 4;
template <int D, int CPL>
struct Buffer {
  Block<D> block;
  float v[CPL][C][16];
};

// Tokens t0 .. t0 + tokens - 1 of one (row, head), 16 CPL columns a CTA.
template <class T, int D, bool DECAY, int CPL>
__global__ void __launch_bounds__(160) block_kernel(const DeltaStepArgs p, const int t0, const int tokens, const int rounds_all,
                                                    const Image<D>* images) {
  constexpr int W = 16 * CPL, BLOCKS = D / W, R = D / 8;  // columns of a CTA; rows of a lane
  using B = Block<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  Buffer<D, CPL>* buffers = reinterpret_cast<Buffer<D, CPL>*>(smem);
  __shared__ uint64_t full[BUFFERS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cb = blockIdx.x % BLOCKS, bh = blockIdx.x / BLOCKS;
  const int b = bh / p.H, h = bh - b * p.H;
  int64_t slot;
  const int n = min(max(tokens_of(p, b, false, slot) - t0, 0), tokens), rounds = (n + C - 1) / C;
  const Image<D>* im = images + static_cast<int64_t>(bh) * rounds_all;
  auto bring = [&](int round) {
    Buffer<D, CPL>& buf = buffers[round % BUFFERS];
    uint64_t* bar = full + round % BUFFERS;
    mbar_expect_tx(bar, sizeof(B) + sizeof(buf.v));
    bulk_load(&buf.block, &im[round].block, sizeof(B), bar);
    bulk_load(buf.v, im[round].v[cb * CPL], sizeof(buf.v), bar);
  };
  if (tid == 128) {
    for (int i = 0; i < BUFFERS; ++i) mbar_init(full + i, 1);
    fence_barrier_init();
  }

  if (warp == 4) {
    // It only brings blocks (by a warp that also computes: 87 instead of 78 us for the longest listed run).  It may
    // start while prepare_kernel runs, of which nothing was read up to here.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (lane == 0)
      for (int r = 0; r < min(rounds, BUFFERS); ++r) bring(r);
    __syncthreads();
    int round = 0;
    for (; round < rounds; ++round) {
      if (__syncthreads_or(0)) break;
      if (lane == 0 && round + BUFFERS < rounds) bring(round + BUFFERS);
      __syncwarp();
    }
    return;
  }
  // lane (slice, lc) has rows slice R .. of columns col .. col + CPL - 1, and solves for column col + mine
  const int slice = lane >> 2, mine = CPL == 2 ? slice & 1 : 0;
  const int local = warp * 4 * CPL + (lane & 3) * CPL, col = cb * W + local, vg = (local + mine) >> 4, vc = (local + mine) & 15;
  float* sp = p.state + ((n ? slot : 0) * p.H + h) * D * D + static_cast<int64_t>(slice) * R * D + col;
  T* op = static_cast<T*>(p.o) + ((static_cast<int64_t>(b) * p.T + t0) * p.H + h) * D + col + mine;
  const int64_t ostep = static_cast<int64_t>(p.H) * D;
  float2 S[CPL][R / 2];
  if (n > 0) {
#pragma unroll
    for (int r = 0; r < R / 2; ++r)
#pragma unroll
      for (int e = 0; e < CPL; ++e) S[e][r] = make_float2(sp[2 * r * D + e], sp[(2 * r + 1) * D + e]);
  }
  __syncthreads();
  bool fine = true;
  int round = 0;
  for (; round < rounds; ++round) {
    fine = mbar_wait(full + round % BUFFERS, (round / BUFFERS) & 1, 0xD50u);
    __syncwarp();
    const Buffer<D, CPL>& buf = buffers[round % BUFFERS];
    const B& blk = buf.block;
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
    // the column's own sums, over the eight slices
    float own[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      if (CPL == 2) own[i] = (mine ? x[CPL - 1][i] : x[0][i]) + __shfl_xor_sync(0xffffffffu, mine ? x[0][i] : x[CPL - 1][i], 4);
      else own[i] = x[0][i] + __shfl_xor_sync(0xffffffffu, x[0][i], 4);
      own[i] += __shfl_xor_sync(0xffffffffu, own[i], 8);
      own[i] += __shfl_xor_sync(0xffffffffu, own[i], 16);
      own[i] = buf.v[vg][i][vc] - own[i];
    }
    products(blk.q, y);  // independent of the solution: fills its waits
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const float4 m0 = *reinterpret_cast<const float4*>(&blk.Mt[j][0]), m1 = *reinterpret_cast<const float4*>(&blk.Mt[j][4]);
      const float m[C] = {m0.x, m0.y, m0.z, m0.w, m1.x, m1.y, m1.z, m1.w};
      own[j] *= blk.beta[j];
#pragma unroll
      for (int i = j + 1; i < C; ++i) own[i] = fmaf(-m[i], own[j], own[i]);
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
      const float4 n0 = *reinterpret_cast<const float4*>(&blk.N[i][0]), n1 = *reinterpret_cast<const float4*>(&blk.N[i][4]);
      float o = qs[e];
      o = fmaf(n0.x, own[0], o); o = fmaf(n0.y, own[1], o); o = fmaf(n0.z, own[2], o); o = fmaf(n0.w, own[3], o);
      o = fmaf(n1.x, own[4], o); o = fmaf(n1.y, own[5], o); o = fmaf(n1.z, own[6], o); o = fmaf(n1.w, own[7], o);
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
      if (DECAY) {
        const float4 c4 = *reinterpret_cast<const float4*>(&blk.c7[slice * B::SL + r * 4]);
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
    if (__syncthreads_or(!fine)) break;  // a wait that ran out ends the CTA
  }
  if (round < rounds) {  // copies in flight land before the CTA's shared memory is given away
    for (int r = round; r < min(round + BUFFERS, rounds); ++r) mbar_wait(full + r % BUFFERS, (r / BUFFERS) & 1, 0xD51u);
    return;
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
    for (int t = n; t < tokens; ++t) op[t * ostep] = from_f<T>(0.f);
}

template <class T, int D, bool DECAY, int CPL>
static int launch_blocks(const DeltaStepArgs& a, int t0, int tokens, int rounds, const Image<D>* images, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  constexpr int SMEM = BUFFERS * sizeof(Buffer<D, CPL>);
  if (smem_limit(done, block_kernel<T, D, DECAY, CPL>, SMEM) != cudaSuccess) return -1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.B * a.H * (D / (16 * CPL))));
  cfg.blockDim = dim3(160);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  // Launched early, the CTAs crowd on the SMs that prepare_kernel leaves first: 17 -> 14 us for 8 rows of 4 tokens,
  // but 85 -> 142 us for one row of 389, where the walk through the blocks is all.
  cfg.numAttrs = tokens <= 4 * C ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, block_kernel<T, D, DECAY, CPL>, a, t0, tokens, rounds, images) == cudaSuccess ? 0 : -1;
}
// Tokens of a segment: blocks that the workspace holds (64 MB, or one block of every head).
static int64_t segment_rounds(const DeltaStepArgs& a) {
  const int64_t image = a.D == 128 ? sizeof(Image<128>) : sizeof(Image<64>), heads = static_cast<int64_t>(a.B) * a.H;
  return std::max<int64_t>(1, std::min<int64_t>((a.T + C - 1) / C, (int64_t{64} << 20) / (image * heads)));
}

template <class T, int D, int GATE>
static int launch(const DeltaStepArgs& a, cudaStream_t s) {
  if (a.T == 1) {
    step_kernel<T, D, GATE><<<static_cast<unsigned>(a.B * a.H * (D / COLS)), 128, 0, s>>>(a);
    return 0;
  }
  Image<D>* images = static_cast<Image<D>*>(a.workspace);
  const int rounds = static_cast<int>(segment_rounds(a));
  for (int t0 = 0; t0 < a.T; t0 += rounds * C) {
    const int tokens = std::min(rounds * C, a.T - t0);
    prepare_kernel<T, D, GATE><<<static_cast<unsigned>(a.B * a.H * rounds), D, 0, s>>>(a, t0, rounds, images);
    // 32 columns a CTA use a vector twice as often as 16, which reach twice as many SMs
    const int rc = a.B * a.H * (D / 32) < a.sms ? launch_blocks<T, D, GATE != 0, 1>(a, t0, tokens, rounds, images, s)
                                                : launch_blocks<T, D, GATE != 0, 2>(a, t0, tokens, rounds, images, s);
    if (rc) return rc;
  }
  return 0;
}
template <class T, int D>
static int by_gate(const DeltaStepArgs& a, cudaStream_t s) {
  return a.gate == 0 ? launch<T, D, 0>(a, s) : a.gate == 1 ? launch<T, D, 1>(a, s) : launch<T, D, 2>(a, s);
}
template <class T>
static int by_width(const DeltaStepArgs& a, cudaStream_t s) {
  return a.D == 128 ? by_gate<T, 128>(a, s) : a.D == 64 ? by_gate<T, 64>(a, s) : -1;
}

}  // namespace dstep
}  // namespace nt

using namespace nt::dstep;

size_t nt_delta_step_workspace(const DeltaStepArgs& a) {
  if (a.T <= 1 || (a.D != 64 && a.D != 128)) return 0;
  return static_cast<size_t>(a.B) * a.H * segment_rounds(a) * (a.D == 128 ? sizeof(Image<128>) : sizeof(Image<64>));
}

int nt_delta_step(const DeltaStepArgs& a, cudaStream_t s) {
  if (a.B == 0 || a.T == 0 || a.H == 0) return 0;
  if (static_cast<int64_t>(a.B) * a.H * std::max<int64_t>(8, segment_rounds(a)) > INT32_MAX || a.gate < 0 || a.gate > 2) return -1;
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
