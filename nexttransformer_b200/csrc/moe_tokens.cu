// K26: a mixture-of-experts layer for up to 64 tokens (decoding): what it reads is the chosen experts' weights, once.
//
//   l = W_r x, p = softmax(l); the k experts with the largest p + bias (ties to the lower one); c = p / sum of the chosen p
//   y = sum over the chosen of c W2 relu(W1 x)^2 + W2' relu(W1' x)^2 (the shared expert)
//
// Three kernels, each started while the one before it ends:
//   route  a cluster of 8 CTAs for one or two tokens: logits in fp32, the choice, and x in the order of a matrix operand
//   fc     h = c relu(W1 x)^2, a warp (or a few) for 32 rows of an expert's W1
//   proj   y, a cluster for 32 (or 16) rows of every expert's W2, by parts of the sum
//
// With few tokens an expert meets one or two of them, so weights are the 16-row side of a 16 x 8 x 16 matrix instruction and
// tokens the narrow side; 2 to 16 operations a byte are far below the ratio at which tensor memory would matter.  The work is to
// keep loads in flight: each warp owns a ring of stages (16 or 32 rows of 128 bytes) that asynchronous copies fill across the
// borders of tiles and experts, and waits for nobody else until its sums are done.  An expert's tokens stand beside each other in
// the operands (gathered where they are read), so an expert costs a block of 8 columns whoever wants it.
//
// 12 tokens, d 2048, 64 experts of 1024, 8 a token and a shared one: 91 to 93 us for 438 MB (68 at 6.46 TB/s): fc and proj stream at about 5 TB/s once
// they run, the rest is three launches' ways to their first tile.  One token: 29 us for 76 MB (11.8), those ways alone.
// 64 tokens, 256 experts of 320: 100 us for 368 MB (57), where proj's pieces are five stages long and a third of its 182 instructions a
// stage begin and end them (19.7 million instructions and 113 us with tokens found in masks, a third walk through the pieces and one sum).
// Tried and not kept: stages of 128 columns (12 tokens 97 -> 128 us), fc with 16 rows at three CTAs an SM (93 -> 106), L2 prefetches of 256 bytes
// (1 %), x kept out of shared memory in route (28.7 -> 29.9), weights fetched into L2 while route runs (0 to 2 %) or while fc ends (64 tokens: +10 %),
// 32 rows and two CTAs an SM for proj of more than 16 tokens (104 -> 112).
#include "moe_tokens.h"
#include "warp_mma.cuh"

#include <algorithm>

namespace nt {
namespace moe_tokens {

constexpr int ROUTE_WARPS = 8, ROUTE_THREADS = ROUTE_WARPS * 32;
constexpr int WARPS = 4, THREADS = WARPS * 32, RESIDENT = 3;  // of the products: three CTAs an SM
constexpr int TILE = 16 * 128;  // bytes of 16 rows of 64 elements
constexpr int MOST = NT_MOE_TOKENS_MOST, EXPERTS = NT_MOE_TOKENS_EXPERTS, CHOICES = NT_MOE_TOKENS_CHOICES;
// Hidden values are held in the weights' type, as two numbers: the value rounded, and what that left.  fp16 ends at 65504, which a
// square passes where its root is 256: they are held as 2^-6 of themselves there (up to 4.2e6), and the sums are raised again.  Its smallest step, 2^-24,
// would then leave 2^-19 of any value out, however small, where outputs are rounded by as little as 2^-25.  So the second number
// is 2^11 times what is left (at most 16, half a unit of the largest, so 2^15), and has sums of its own: a hidden value is off by 2^-22 of itself or
// 2^-30, and a row of W2 would need a norm of 32 before that showed in an output.
template <class T> constexpr float LOWER = 1.f;
template <> constexpr float LOWER<__half> = 1.f / 64;
template <class T> constexpr float FINER = 1.f;
template <> constexpr float FINER<__half> = 2048.f;

struct Workspace {
  int* choice;    // [T, k]
  float* share;   // [T, E], set where chosen
  uint2* x;       // [groups of d, blocks of 8 tokens, 32]: a lane's part of a 16 x 8 operand
  uint4* h;       // [pairs of an expert and a block of 8 of its tokens, groups of F, 32]: the same of a value's two numbers
  int pairs;      // of routed experts; the shared expert's blocks, of groups of Fs each, come behind them
};
// 16 inner elements each, a whole number of stages; what lies behind the inner dimension is zero.
__host__ __device__ static int groups_of(int n) { return (n + 63) / 64 * 4; }
static int blocks_of(int n, int by) { return (n + by - 1) / by; }
static size_t layout(const MoeTokensArgs& a, Workspace& w) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t from = at;
    at += (bytes + 255) / 256 * 256;
    return static_cast<char*>(a.workspace) + from;
  };
  const int nb = blocks_of(a.T, 8);
  // every (expert, token) pair may start a block; an expert has at most nb blocks
  w.pairs = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(a.T) * a.k, static_cast<int64_t>(a.E) * nb));
  w.choice = reinterpret_cast<int*>(take(static_cast<size_t>(a.T) * a.k * 4));
  w.share = reinterpret_cast<float*>(take(static_cast<size_t>(a.T) * a.E * 4));
  w.x = reinterpret_cast<uint2*>(take(static_cast<size_t>(groups_of(a.d)) * nb * 256));
  w.h = reinterpret_cast<uint4*>(take((static_cast<size_t>(w.pairs) * groups_of(a.F) + static_cast<size_t>(nb) * groups_of(a.Fs)) * 512));
  return at;
}

NT_DEVICE void dependents_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
NT_DEVICE void wait_for_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ------------------------------------------------------------------------------------ route
// A cluster of ROUTE_RANKS CTAs has TOKENS tokens, a part of the experts each; the j-th CTA then chooses for the j-th token.  Several
// tokens share a reading of the router: 64 tokens on 256 experts of width 1280
// took 29 us with one token a cluster and 19 with four; the whole layer takes 104 us with four and 100 with two (16 warps a CTA: no less).
constexpr int ROUTE_RANKS = 8;
template <class T, int PER, int TOKENS>  // PER: experts a lane
__global__ void __launch_bounds__(ROUTE_THREADS) route_kernel(const MoeTokensArgs a, const Workspace w) {
  extern __shared__ __align__(16) float x[];  // [TOKENS, d]
  __shared__ float logits[EXPERTS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, t0 = blockIdx.x / ROUTE_RANKS * TOKENS, rank = blockIdx.x % ROUTE_RANKS;
  const int tokens = min(TOKENS, a.T - t0);
  dependents_may_start();
  // the router's rows are on their way while x comes
  for (int e = rank * ROUTE_WARPS + warp; e < a.E; e += ROUTE_RANKS * ROUTE_WARPS)
    for (int i = lane * 32; i < a.d; i += 1024) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.router + static_cast<int64_t>(e) * a.d + i));
  for (int i = tid * 8; i < a.d; i += ROUTE_THREADS * 8) {
    uint4 u[TOKENS];
#pragma unroll
    for (int j = 0; j < TOKENS; ++j)
      u[j] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + (t0 + min(j, tokens - 1)) * a.x_stride + i);
#pragma unroll
    for (int j = 0; j < TOKENS; ++j) {
      const uint32_t v[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) *reinterpret_cast<float2*>(x + j * a.d + i + 2 * e) = Num<T>::unpack(v[e]);
    }
  }
#pragma unroll
  for (int j = 0; j < TOKENS; ++j) {
    const T* src = static_cast<const T*>(a.x) + (t0 + min(j, tokens - 1)) * a.x_stride;
    // x as an operand: lane 4 n + c of a 16 x 8 tile has token n's channels 2 c, 2 c + 1 and 2 c + 8, 2 c + 9
    const int t = t0 + j, nb = (a.T + 7) / 8, groups = groups_of(a.d);
    if (j < tokens)
      for (int i = rank * ROUTE_THREADS + tid; i < groups * 4; i += ROUTE_RANKS * ROUTE_THREADS) {
        const int g = i >> 2, at = g * 16 + (i & 3) * 2;
        const uint32_t lo = at < a.d ? *reinterpret_cast<const uint32_t*>(src + at) : 0u;
        const uint32_t hi = at + 8 < a.d ? *reinterpret_cast<const uint32_t*>(src + at + 8) : 0u;
        w.x[(static_cast<int64_t>(g) * nb + t / 8) * 32 + (t % 8) * 4 + (i & 3)] = make_uint2(lo, hi);
      }
  }
  cluster_sync();  // x is there, and so are the CTAs that get the logits
  constexpr int ROWS = 2, BY = ROUTE_RANKS * ROUTE_WARPS;  // experts at once
  for (int e0 = rank * ROUTE_WARPS + warp; e0 < a.E; e0 += ROWS * BY) {
    float4 sum[ROWS][TOKENS];  // four chains of d / 128 products a lane
    const float4* row[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      row[k] = reinterpret_cast<const float4*>(a.router + static_cast<int64_t>(min(e0 + k * BY, a.E - 1)) * a.d);
#pragma unroll
      for (int j = 0; j < TOKENS; ++j) sum[k][j] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll 8
    for (int i = lane; i < a.d / 4; i += 32) {
      float4 u[ROWS];
#pragma unroll
      for (int k = 0; k < ROWS; ++k) u[k] = row[k][i];
#pragma unroll
      for (int j = 0; j < TOKENS; ++j) {
        const float4 v = reinterpret_cast<const float4*>(x + j * a.d)[i];
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
          sum[k][j].x = fmaf(u[k].x, v.x, sum[k][j].x);
          sum[k][j].y = fmaf(u[k].y, v.y, sum[k][j].y);
          sum[k][j].z = fmaf(u[k].z, v.z, sum[k][j].z);
          sum[k][j].w = fmaf(u[k].w, v.w, sum[k][j].w);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k)
#pragma unroll
      for (int j = 0; j < TOKENS; ++j) {
        const float v = warp_sum((sum[k][j].x + sum[k][j].y) + (sum[k][j].z + sum[k][j].w));
        if (lane == 0 && e0 + k * BY < a.E) {
          uint32_t remote;
          asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(logits + e0 + k * BY)), "r"(j));
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
        }
      }
  }
  cluster_sync();
  if (rank >= tokens || warp != 0) return;
  const int t = t0 + rank;
  float p[PER], score[PER], top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    p[i] = e < a.E ? logits[e] : -INFINITY;
    top = fmaxf(top, p[i]);
  }
  top = warp_max(top);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    p[i] = lane + 32 * i < a.E ? expf(p[i] - top) : 0.f;
    sum += p[i];
  }
  sum = warp_sum(sum);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    p[i] /= sum;
    score[i] = -INFINITY;
    if (e < a.E) score[i] = fmaxf(p[i] + (a.bias ? a.bias[e] : 0.f), -3.4028235e38f);  // NaN, too: it can still be chosen
  }
  float chosen_p = 0.f;  // lane j: the j-th choice's
  int chosen = 0;
#pragma unroll 1
  for (int j = 0; j < a.k; ++j) {
    float best = -INFINITY, its = 0.f;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (score[i] > best) {
        best = score[i];
        its = p[i];
        at = lane + 32 * i;
      }
    // the largest as a whole number in the order of the floats, then the lowest expert that has it
    const uint32_t u = __float_as_uint(best + 0.f), key = u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
    const uint32_t most = __reduce_max_sync(0xffffffffu, key);
    const int winner = __reduce_min_sync(0xffffffffu, key == most ? at : 0x7fffffff);
    const float winners = __shfl_sync(0xffffffffu, its, winner & 31);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 32 * i == winner) score[i] = -INFINITY;
    if (lane == j) {
      chosen = winner;
      chosen_p = winners;
    }
  }
  const float all = warp_sum(lane < a.k ? chosen_p : 0.f);
  if (lane < a.k) {
    w.choice[t * a.k + lane] = chosen;
    w.share[static_cast<int64_t>(t) * a.E + chosen] = chosen_p / all;
  }
}

// ------------------------------------------------------------------------------------ the experts
// What the products run over: entries of an expert and up to 16 of its tokens, experts in order and the shared one (E) last.
constexpr int ENTRIES = EXPERTS + MOST * CHOICES / 16 + MOST / 16;
struct Lists {
  unsigned long long mask[EXPERTS + 1];  // an expert's tokens; [E]: the shared expert's, all
  uint16_t expert[ENTRIES], block[ENTRIES];  // an entry's expert, and its first block of 8 tokens in h
  uint8_t first[ENTRIES];                // the first of its tokens, counted among the expert's
  uint8_t blocks[ENTRIES];               // of 8 of its tokens: 1 or 2
  int routed, entries;
  uint4 tokens[ENTRIES];                 // its tokens, a byte each, and -1
};
template <bool TOKENS>
NT_DEVICE void make_lists(const MoeTokensArgs& a, const Workspace& w, Lists& l) {
  const int tid = threadIdx.x, lane = tid & 31;
  for (int e = tid; e <= a.E; e += THREADS) l.mask[e] = 0;
  __syncthreads();
  for (int i = tid; i < a.T * a.k; i += THREADS) atomicOr(&l.mask[__ldcg(w.choice + i)], 1ull << quotient(i, a.k));
  __syncthreads();
  if (tid < 32) {
    int n = 0, blocks = 0;
    for (int e0 = 0; e0 < a.E; e0 += 32) {
      const int e = e0 + lane, tokens = e < a.E ? __popcll(l.mask[e]) : 0;
      const int own = ((tokens + 15) >> 4) | (((tokens + 7) >> 3) << 16);  // entries, blocks
      int upto = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      for (int i = 0; i < (own & 0xffff); ++i) {
        const int at = n + ((upto - own) & 0xffff) + i;
        l.expert[at] = static_cast<uint16_t>(e);
        l.block[at] = static_cast<uint16_t>(blocks + ((upto - own) >> 16) + 2 * i);
        l.first[at] = static_cast<uint8_t>(16 * i);
        l.blocks[at] = static_cast<uint8_t>(tokens - 16 * i > 8 ? 2 : 1);
      }
      const int all = __shfl_sync(0xffffffffu, upto, 31);
      n += all & 0xffff;
      blocks += all >> 16;
    }
    const int own = a.Fs ? (a.T + 15) >> 4 : 0;
    if (lane < own) {
      l.expert[n + lane] = static_cast<uint16_t>(a.E);
      l.block[n + lane] = static_cast<uint16_t>(2 * lane);
      l.first[n + lane] = static_cast<uint8_t>(16 * lane);
      l.blocks[n + lane] = static_cast<uint8_t>(a.T - 16 * lane > 8 ? 2 : 1);
    }
    if (lane == 0) {
      l.mask[a.E] = a.T == 64 ? ~0ull : (1ull << a.T) - 1;
      l.routed = n;
      l.entries = n + own;
    }
  }
  __syncthreads();
  if constexpr (TOKENS) {
    for (int i = tid; i < l.entries; i += THREADS) {
      unsigned long long m = l.mask[l.expert[i]];
      for (int skip = l.first[i]; skip; --skip) m &= m - 1;
      uint32_t u[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        u[j / 4] |= static_cast<uint32_t>((__ffsll(static_cast<long long>(m)) - 1) & 0xff) << (j % 4 * 8);
        m &= m - 1;
      }
      l.tokens[i] = make_uint4(u[0], u[1], u[2], u[3]);
    }
    __syncthreads();
  }
}
// The n-th token (from 0) of an entry, or -1.
NT_DEVICE int nth_token(const Lists& l, int entry, int n) { return reinterpret_cast<const int8_t*>(l.tokens + entry)[n]; }

// A warp's ring: STAGES stages of 16 MT rows of 64 elements, chunk c (16 bytes) of row r at c ^ (r & 7).
struct Ring {
  uint32_t base, in, out;  // addresses of the ring, of the stage that is filled next and of the one that is read next
  uint32_t to[2];          // this lane's place in a stage for rows r and r + 4 (r < 4); 1024 further on for each 8 rows
  uint32_t at[4];          // this lane's matrix row of the four 16-column tiles; 2048 further on for each 16 rows
};
template <int BYTES>
NT_DEVICE Ring make_ring(const void* smem) {
  Ring r;
  const int lane = threadIdx.x & 31, row = lane >> 3, chunk = lane & 7;
  r.base = r.in = r.out = smem_u32(smem) + (threadIdx.x >> 5) * BYTES;
  r.to[0] = row * 128 + ((chunk ^ row) << 4);
  r.to[1] = (row + 4) * 128 + ((chunk ^ (row + 4)) << 4);
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int m = lane & 15;
    r.at[s] = m * 128 + (((2 * s + (lane >> 4)) ^ (m & 7)) << 4);
  }
  return r;
}

// A row tile of an entry: what a warp goes through, a stage of 64 inner elements after the other.
struct Piece {
  int entry, expert, tile;
  int inner, rows;    // elements of a weight row; rows of the tile (16 MT, or fewer at the end)
  unsigned blocks;    // bit b: it has tokens in its b-th block of 8
  int stage, stages;  // the next one; the first behind the piece
  int behind;         // what comes after it: an item, or a stage of all
};

struct Brief {  // what the products need of a piece
  int entry, expert, tile;
  unsigned blocks;
  bool last, more;  // this stage is the piece's last; there is one
};

// Goes through a warp's pieces: weights come `STAGES - 1` stages ahead, the other operand one.
//   first(piece) / next(piece) set a piece and say whether there is one (the copies, the operand and the products each go through them);
//   base(piece): the tile's first weight; operand(piece, pointers): this lane's part of the 16 x 8 tile of the piece's next stage, of
//   each block of 8 tokens (KEEP: null for zeros), `step` apart from tile to tile (a Frag of 16 bytes holds two numbers for each value);
//   ready(): what has to be waited for before the operand is read; done(piece, sums): a piece's products are complete.
// MT tiles of 16 rows share an operand's reading and the way through the loop: a warp's instructions wait for each other, and with 8
// warps an SM, 16 rows and 187 instructions a stage the first product took 60 us for 12 tokens, with 16 warps and 137 it took 44.
template <class T, int MT, int NB, int STAGES, class Frag, bool KEEP, class First, class Next, class Base, class Operand, class Ready, class Done>
NT_DEVICE void stream(const MoeTokensArgs& a, const void* smem, const int step, First first, Next next, Base base, Operand operand, Ready ready,
                      Done done) {
  float acc[MT][NB][4];
  constexpr bool TWO = sizeof(Frag) == 16;
  constexpr int STAGE = MT * TILE;
  Ring r = make_ring<STAGES * STAGE>(smem);
  auto turn = [&](uint32_t& stage) { stage = stage == r.base + (STAGES - 1) * STAGE ? r.base : stage + STAGE; };
  const int lane = threadIdx.x & 31, row = lane >> 3, chunk = lane & 7;
  Piece f, o;  // where the copies and the operand stand
  Brief c, n;  // the piece of the stage that is multiplied, and of the next one
  bool f_more = first(f);
  const char* f_at = nullptr;
  int64_t f_step = 0;  // four rows
  auto enter = [&]() {
    if (!f_more) return;
    f_at = reinterpret_cast<const char*>(static_cast<const T*>(base(f)) + static_cast<int64_t>(row) * f.inner + f.stage * 64 + chunk * 8);
    f_step = static_cast<int64_t>(f.inner) * (4 * sizeof(T));
  };
  enter();
  auto fetch = [&]() {
    if (f_more) {
      if (f.rows == 16 * MT && (f.stage + 1) * 64 <= f.inner) {
        const char* p = f_at;
#pragma unroll
        for (int e = 0; e < 4 * MT; ++e, p += f_step) cp_async16(r.in + r.to[e & 1] + (e >> 1) * 1024, p);
      } else {  // what is not there becomes zero
        const bool inside = f.stage * 64 + chunk * 8 < f.inner;
#pragma unroll
        for (int e = 0; e < 4 * MT; ++e) {
          const bool valid = inside && row + 4 * e < f.rows;
          cp_async16_or_zero(r.in + r.to[e & 1] + (e >> 1) * 1024, valid ? f_at + e * f_step : static_cast<const char*>(a.x), valid);
        }
      }
      turn(r.in);
      f_at += 128;
      if (++f.stage == f.stages) {
        f_more = next(f);
        enter();
      }
    }
    cp_commit();
  };
#pragma unroll 1
  for (int i = 0; i < STAGES - 1; ++i) fetch();
  ready();

  bool o_more = first(o);
  const Frag* at[NB];
  if (o_more) operand(o, at);
  auto load = [&](Frag (&b)[4][NB]) {
    n.more = o_more;
    if (!o_more) return;
    n.entry = o.entry;
    n.expert = o.expert;
    n.tile = o.tile;
    n.blocks = o.blocks;
    n.last = o.stage + 1 == o.stages;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      if ((o.blocks >> nb) & 1u) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          b[s][nb] = Frag{};
          if (!KEEP || at[nb]) b[s][nb] = TWO ? __ldcg(at[nb] + s * step) : at[nb][s * step];
        }
        if (!KEEP || at[nb]) at[nb] += 4 * step;
      }
    if (++o.stage == o.stages) {
      o_more = next(o);
      if (o_more) operand(o, at);
    }
  };
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][nb][e] = 0.f;
  // second numbers add up beside the first, where registers allow it (products on one sum wait for each other) or they are finer
  constexpr bool APART = TWO && (MT * NB <= 2 || FINER<T> != 1.f);
  float low[MT][NB][4] = {};
  auto together = [&]() {
    if constexpr (APART) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            acc[m][nb][e] += low[m][nb][e] * (1.f / FINER<T>);
            low[m][nb][e] = 0.f;
          }
    }
  };
  auto multiply = [&](const Frag (&b)[4][NB], Frag (&ahead)[4][NB]) {
    c = n;
    load(ahead);
    cp_wait<STAGES - 2>();
    __syncwarp();  // this stage has landed for every lane, and the stage before it is read by none
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      uint32_t w[4][4];
#pragma unroll
      for (int s = 0; s < 4; ++s) ldsm4(w[s], r.out + r.at[s] + m * TILE);
      if (m == MT - 1) {
        turn(r.out);
        fetch();
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        if ((c.blocks >> nb) & 1u)
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            Num<T>::mma(acc[m][nb], w[s], b[s][nb].x, b[s][nb].y);
            if constexpr (TWO) Num<T>::mma(APART ? low[m][nb] : acc[m][nb], w[s], b[s][nb].z, b[s][nb].w);
          }
    }
    if (c.last) {
      together();
      done(c, acc);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[m][nb][e] = 0.f;
    }
  };
  Frag even[4][NB], odd[4][NB];
  load(even);
#pragma unroll 1
  while (n.more) {
    multiply(even, odd);
    if (!n.more) break;
    multiply(odd, even);
  }
  cp_wait<0>();
}

// NB blocks of 8 tokens an entry: 1 where there are no more than 8 tokens, else 2.  `wide`
// warps share a tile, a part of its stages each, where tiles are few or their last round would leave many warps without one: one token
// on experts of 1024 x 2048 has 288 tiles for 1776 warps.
constexpr int FC_MT = 2, FC_STAGES = 3;
template <class T, int NB>
__global__ void __launch_bounds__(THREADS, RESIDENT) fc_kernel(const MoeTokensArgs a, const Workspace w) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Lists l;
  __shared__ float4 parts[WARPS][FC_MT][NB][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  wait_for_predecessor();
  dependents_may_start();
  make_lists<true>(a, w, l);
  constexpr int ROWS = 16 * FC_MT;
  const int tiles = (a.F + ROWS - 1) / ROWS, shared_tiles = (a.Fs + ROWS - 1) / ROWS, groups = groups_of(a.F), shared_groups = groups_of(a.Fs);
  const int routed = l.routed * tiles, items = routed + (l.entries - l.routed) * shared_tiles;
  const int stages = (a.d + 63) / 64, slots = gridDim.x * WARPS;
  // rounds of tiles times what a warp does for one: its part of the stages, and about three stages' time for beginning and ending it
  auto cost = [&](int n) { return static_cast<float>((items * n + slots - 1) / slots) * (static_cast<float>(stages) / n + 3.f); };
  int wide = 1;
  for (int n = 2; n <= WARPS && n <= stages; n *= 2)
    if (cost(n) < cost(wide)) wide = n;
  const int group = warp / wide, part = warp % wide, by = gridDim.x * (WARPS / wide);
  // (the first items go to different SMs)
  auto set = [&](Piece& p, int item) {
    if (item >= items) return false;
    const bool shared = item >= routed;
    const int i = shared ? item - routed : item, per = shared ? shared_tiles : tiles, n = quotient(i, per);
    p.entry = (shared ? l.routed : 0) + n;
    p.tile = i - n * per;
    p.expert = l.expert[p.entry];
    p.inner = a.d;
    p.rows = min(ROWS, (shared ? a.Fs : a.F) - p.tile * ROWS);
    p.blocks = (1u << l.blocks[p.entry]) - 1u;
    p.stage = stages * part / wide;
    p.stages = stages * (part + 1) / wide;
    p.behind = item + by;
    return true;
  };
  stream<T, FC_MT, NB, FC_STAGES, uint2, false>(
      a, smem, (a.T + 7) / 8 * 32, [&](Piece& p) { return set(p, group * gridDim.x + blockIdx.x); }, [&](Piece& p) { return set(p, p.behind); },
      [&](const Piece& p) -> const void* {
        const T* e = p.expert == a.E ? static_cast<const T*>(a.shared_fc) : static_cast<const T*>(a.w_fc) + static_cast<int64_t>(p.expert) * a.F * a.d;
        return e + static_cast<int64_t>(p.tile) * ROWS * a.d;
      },
      [&](const Piece& p, const uint2* (&at)[NB]) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          // columns without a token may be anyone's: they are dropped
          const int t = max(0, nth_token(l, p.entry, nb * 8 + (lane >> 2)));
          at[nb] = w.x + (t >> 3) * 32 + (t & 7) * 4 + (lane & 3) + p.stage * 4 * ((a.T + 7) / 8 * 32);
        }
      },
      [] {},
      [&](const Brief& p, float (&acc)[FC_MT][NB][4]) {
        if (wide > 1) {  // the first warp adds up
#pragma unroll
          for (int m = 0; m < FC_MT; ++m)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) parts[warp][m][nb][lane] = make_float4(acc[m][nb][0], acc[m][nb][1], acc[m][nb][2], acc[m][nb][3]);
          named_bar_sync(1 + group, wide * 32);
          if (part == 0)
            for (int k = 1; k < wide; ++k)
#pragma unroll
              for (int m = 0; m < FC_MT; ++m)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                  const float4 v = parts[warp + k][m][nb][lane];
                  acc[m][nb][0] += v.x; acc[m][nb][1] += v.y; acc[m][nb][2] += v.z; acc[m][nb][3] += v.w;
                }
          named_bar_sync(1 + group, wide * 32);
          if (part) return;
        }
        // h, in the order in which it is an operand: rows of the tile become the products' inner dimension.  It is held as two
        // numbers of its type, so that little but the output's rounding shows.
        const bool shared = p.expert == a.E;
        const int inner = shared ? shared_groups : groups;
        uint4* h = w.h + (shared ? static_cast<int64_t>(w.pairs) * groups : 0ll) * 32;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          if (!((p.blocks >> nb) & 1u)) break;
          int t[2];
          float share[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            t[e] = nth_token(l, p.entry, nb * 8 + (lane & 3) * 2 + e);
            share[e] = t[e] < 0 ? 0.f : shared ? LOWER<T> : LOWER<T> * __ldcg(w.share + static_cast<int64_t>(t[e]) * a.E + p.expert);
          }
          uint4* to = h + ((static_cast<int64_t>(l.block[p.entry]) + nb) * inner + p.tile * FC_MT) * 32 + lane;
#pragma unroll
          for (int m = 0; m < FC_MT; ++m, to += 32) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float u = acc[m][nb][k] < 0.f ? 0.f : acc[m][nb][k];  // a NaN stays one
              v[k] = t[k & 1] < 0 ? 0.f : share[k & 1] * (u * u);
            }
            const uint32_t hi0 = Num<T>::pack(v[0], v[1]), hi1 = Num<T>::pack(v[2], v[3]);
            const float2 f0 = Num<T>::unpack(hi0), f1 = Num<T>::unpack(hi1);
            // (of an infinite value the rest is NaN, and so would the sum be)
            auto rest = [](float value, float held) { return isinf(held) ? 0.f : (value - held) * FINER<T>; };
            const uint32_t lo0 = Num<T>::pack(rest(v[0], f0.x), rest(v[1], f0.y)), lo1 = Num<T>::pack(rest(v[2], f1.x), rest(v[3], f1.y));
            *to = make_uint4(transpose8x8(hi0), transpose8x8(hi1), transpose8x8(lo0), transpose8x8(lo1));
          }
          if (p.tile == (shared ? shared_tiles : tiles) - 1)  // the groups behind the last
            for (int g = (p.tile + 1) * FC_MT; g < inner; ++g, to += 32) *to = make_uint4(0, 0, 0, 0);
        }
      });
}

// Up to 16 tokens are the columns of every entry, and the sums stay in registers (KEEP; a piece's are added to those of the tokens that
// it is for); of more, an entry's own are, and its sums are added to the tokens' in shared memory.
template <class T, int MT, int NB, int STAGES, bool KEEP>
__global__ void __launch_bounds__(THREADS, RESIDENT) proj_kernel(const MoeTokensArgs a, const Workspace w, const int parts) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Lists l;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, part = blockIdx.x % parts, tile = blockIdx.x / parts;
  constexpr int ROWS = 16 * MT, PITCH = ROWS + 1;
  float* const sums = reinterpret_cast<float*>(smem + (KEEP ? 0 : WARPS * STAGES * MT * TILE));  // [warp][token][PITCH]
  if (!KEEP)
    for (int i = tid; i < WARPS * a.T * PITCH; i += THREADS) sums[i] = 0.f;
  make_lists<!KEEP>(a, w, l);  // (the route kernel ended before the one before this began its work)
  const int per = (a.F + 63) / 64, shared_per = (a.Fs + 63) / 64, groups = groups_of(a.F), shared_groups = groups_of(a.Fs);
  // an equal run of the stages of all entries
  const int routed = l.routed * per, all = routed + (l.entries - l.routed) * shared_per;
  const int runs = parts * WARPS, run = part * WARPS + warp, few = all / runs, more = all % runs;
  const int first = run * few + min(run, more), last = first + few + (run < more ? 1 : 0);
  auto enter = [&](Piece& p, int at) {  // at stage p.stage of p.entry, which is stage `at` of all
    const bool shared = p.entry >= l.routed;
    p.tile = tile;
    p.expert = l.expert[p.entry];
    p.inner = shared ? a.Fs : a.F;
    p.rows = min(ROWS, a.d - tile * ROWS);
    if (KEEP) {
      const unsigned mask = static_cast<unsigned>(l.mask[p.expert]);
      p.blocks = (mask & 0xffu ? 1u : 0u) | (mask >> 8 ? 2u : 0u);
    } else {
      p.blocks = (1u << l.blocks[p.entry]) - 1u;
    }
    p.stages = min(shared ? shared_per : per, p.stage + last - at);
    p.behind = at + p.stages - p.stage;
  };
  auto set = [&](Piece& p) {
    if (first >= last) return false;
    const bool shared = first >= routed;
    const int i = shared ? first - routed : first, n = quotient(i, shared ? shared_per : per);
    p.entry = (shared ? l.routed : 0) + n;
    p.stage = i - n * (shared ? shared_per : per);
    enter(p, first);
    return true;
  };
  auto next = [&](Piece& p) {
    if (p.behind >= last) return false;
    ++p.entry;
    p.stage = 0;
    enter(p, p.behind);
    return true;
  };
  float kept[MT][NB][4] = {};
  stream<T, MT, NB, STAGES, uint4, KEEP>(
      a, smem, 32, set, next,
      [&](const Piece& p) -> const void* {
        const T* e = p.expert == a.E ? static_cast<const T*>(a.shared_proj) : static_cast<const T*>(a.w_proj) + static_cast<int64_t>(p.expert) * a.d * a.F;
        return e + static_cast<int64_t>(tile) * ROWS * p.inner;
      },
      [&](const Piece& p, const uint4* (&at)[NB]) {
        const bool shared = p.expert == a.E;
        const int inner = shared ? shared_groups : groups;
        const uint4* h = w.h + (shared ? static_cast<int64_t>(w.pairs) * groups : 0ll) * 32;
        const unsigned mask = static_cast<unsigned>(l.mask[p.expert]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          if (KEEP) {  // column t is token t, which is the expert's `place`-th
            const int t = nb * 8 + (lane >> 2), place = __popc(mask & ((1u << t) - 1u));
            at[nb] = (mask >> t) & 1u
                         ? h + ((static_cast<int64_t>(l.block[p.entry]) + (place >> 3)) * inner + p.stage * 4) * 32 + (place & 7) * 4 + (lane & 3)
                         : nullptr;
          } else {
            at[nb] = h + ((static_cast<int64_t>(l.block[p.entry]) + nb) * inner + p.stage * 4) * 32 + lane;
          }
        }
      },
      [] { wait_for_predecessor(); },  // weights may come before, h may not
      [&](const Brief& p, const float (&own)[MT][NB][4]) {
        if constexpr (KEEP) {
          // A token has the sums of its own experts alone: another's weights times its zeros need not be 0 (infinities)
          const unsigned mask = static_cast<unsigned>(l.mask[p.expert]) >> ((lane & 3) * 2);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if ((mask >> (nb * 8 + e)) & 1u)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                  kept[m][nb][e] += own[m][nb][e];
                  kept[m][nb][e + 2] += own[m][nb][e + 2];
                }
          return;
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          if (!((p.blocks >> nb) & 1u)) break;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int t = nth_token(l, p.entry, nb * 8 + (lane & 3) * 2 + e);
            if (t < 0) continue;
            float* to = sums + (warp * a.T + t) * PITCH + (lane >> 2);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              to[16 * m] += own[m][nb][e];
              to[16 * m + 8] += own[m][nb][e + 2];
            }
          }
        }
        __syncwarp();  // the next entry's lanes may hold this one's tokens elsewhere
      });
  if (KEEP) {
    __syncthreads();  // the rings are done with
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = nb * 8 + (lane & 3) * 2 + e;
        if (t >= a.T) continue;
        float* to = sums + (warp * a.T + t) * PITCH + (lane >> 2);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          to[16 * m] = kept[m][nb][e];
          to[16 * m + 8] = kept[m][nb][e + 2];
        }
      }
  }

  // ---- the warps' sums, then the parts', in their order
  __syncthreads();
  float* const whole = sums;
  for (int i = tid; i < a.T * ROWS; i += THREADS) {
    const int at = i / ROWS * PITCH + i % ROWS;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) v += sums[k * a.T * PITCH + at];
    whole[at] = v;
  }
  if (parts > 1) cluster_sync();
  else __syncthreads();
  if (part == 0) {
    for (int i = tid; i < a.T * ROWS / 2; i += THREADS) {  // a pair of channels of a token
      const int t = i / (ROWS / 2), ch = i % (ROWS / 2) * 2;
      const float* own = whole + t * PITCH + ch;
      float2 v = make_float2(own[0], own[1]);
      for (int c = 1; c < parts; ++c) {
        uint32_t remote;
        float2 u;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(own)), "r"(c));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(u.x) : "r"(remote) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(u.y) : "r"(remote + 4) : "memory");
        v.x += u.x;
        v.y += u.y;
      }
      const float f = 1.f / LOWER<T>;
      if (tile * ROWS + ch < a.d)  // (d is even)
        *reinterpret_cast<uint32_t*>(static_cast<T*>(a.y) + static_cast<int64_t>(t) * a.d + tile * ROWS + ch) = Num<T>::pack(v.x * f, v.y * f);
    }
  }
  if (parts > 1) cluster_sync();  // nobody leaves while its sums are read
}

template <class Kernel, class... Args>
static int start(Kernel kern, int grid, int threads, size_t smem, int cluster, bool early, cudaStream_t s, Args... args) {
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (early) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? 0 : -1;
}
template <class T, int TOKENS>
static int route(const MoeTokensArgs& a, const Workspace& w, cudaStream_t s) {
  const auto kern = a.E <= 64 ? route_kernel<T, 2, TOKENS> : a.E <= 256 ? route_kernel<T, 8, TOKENS> : route_kernel<T, EXPERTS / 32, TOKENS>;
  return start(kern, (a.T + TOKENS - 1) / TOKENS * ROUTE_RANKS, ROUTE_THREADS, TOKENS * a.d * sizeof(float), ROUTE_RANKS, false, s, a, w);
}
template <class T>
static int route_for(const MoeTokensArgs& a, const Workspace& w, cudaStream_t s) {
  // as few tokens a cluster as keep the clusters on the SMs at once, and as 48 KB hold beside the logits
  if (a.T * ROUTE_RANKS <= a.sms || a.d * 8 > 48 * 1024 - static_cast<int>(sizeof(float)) * EXPERTS) return route<T, 1>(a, w, s);
  return route<T, 2>(a, w, s);
}
// Clusters of more than 8 CTAs have to be allowed for a kernel, on each device once.
template <class Kernel>
static cudaError_t larger_clusters(std::atomic<uint64_t>& done, Kernel kern) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  const uint64_t bit = dev < 64 ? (uint64_t(1) << dev) : 0;
  if (bit && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess && bit) done.fetch_or(bit, std::memory_order_acq_rel);
  return e;
}
template <class T, int MT, int NB, int STAGES, bool KEEP>
static int project(const MoeTokensArgs& a, const Workspace& w, cudaStream_t s) {
  static std::atomic<uint64_t> done{0}, wide_done{0};
  constexpr int RINGS = WARPS * STAGES * MT * TILE, SUM = WARPS * (16 * MT + 1) * static_cast<int>(sizeof(float));  // of a token
  static_assert(!KEEP || 16 * SUM <= RINGS, "sums lie in the rings");
  const auto kern = proj_kernel<T, MT, NB, STAGES, KEEP>;
  if (smem_limit(done, kern, RINGS + (KEEP ? 0 : MOST * SUM)) != cudaSuccess || larger_clusters(wide_done, kern) != cudaSuccess) return -1;
  // Parts of the sum as a cluster, as many as are resident at once; more than 8 where a warp still gets a dozen stages (few tiles of
  // wide experts: 6 tokens, 216 / 3424: 60 us with 8, 44 with 16; but 28 tokens, 424 / 216: 38 and 47).
  const int64_t stages = static_cast<int64_t>(std::min(a.E, a.T * a.k)) * blocks_of(a.F, 64) + blocks_of(a.Fs, 64);
  const int tiles = blocks_of(a.d, 16 * MT), most = stages >= 12 * WARPS * 16 ? 16 : 8, places = RESIDENT * a.sms;
  // Clusters that are placed beside the last CTAs of the kernel before leave gaps, so they take 13 of 15 places, or wait for its end where
  // the rest is worth it (80 clusters for 444 places, 64 tokens: 122 us with 4 CTAs each, 158 with 5, and 113 if these wait).
  const int spare = std::max(1, std::min(most, places * 13 / 15 / tiles)), full = std::max(1, std::min(most, places / tiles));
  const bool early = full * 4 < spare * 5;
  const int parts = early ? spare : full;
  return start(kern, tiles * parts, THREADS, RINGS + (KEEP ? 0 : a.T * SUM), parts, early, s, a, w, parts);
}
template <class T, int NB>
static int launch(const MoeTokensArgs& a, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  constexpr int RINGS = WARPS * FC_STAGES * FC_MT * TILE;
  if (smem_limit(done, fc_kernel<T, NB>, RINGS) != cudaSuccess) return -1;
  Workspace w;
  layout(a, w);
  if (route_for<T>(a, w, s)) return -1;
  if (start(fc_kernel<T, NB>, RESIDENT * a.sms, THREADS, RINGS, 1, true, s, a, w)) return -1;
  if (a.T > 16) return project<T, 1, 2, 5, false>(a, w, s);
  // narrow layers have too few tiles of 32 rows for the SMs
  return blocks_of(a.d, 32) * 8 * 3 >= RESIDENT * a.sms * 2 ? project<T, 2, NB, 3, true>(a, w, s) : project<T, 1, NB, 5, true>(a, w, s);
}

}  // namespace moe_tokens
}  // namespace nt

using namespace nt::moe_tokens;

size_t nt_moe_tokens_workspace(const MoeTokensArgs& a) {
  Workspace w;
  return layout(a, w);
}

int nt_moe_tokens(const MoeTokensArgs& a, cudaStream_t s) {
  if (a.T == 0) return 0;
  if (a.T > MOST || a.E < 1 || a.E > EXPERTS || a.k < 1 || a.k > CHOICES || a.k > a.E || a.d < 8 || a.d % 8 || a.d > NT_MOE_TOKENS_WIDTH ||
      a.F < 8 || a.F % 8 || a.Fs % 8 || static_cast<int64_t>(a.E) * ((a.F + 15) / 16) + a.Fs > INT32_MAX / 2)
    return -1;
  if (a.fp16) return a.T <= 8 ? launch<__half, 1>(a, s) : launch<__half, 2>(a, s);
  return a.T <= 8 ? launch<__nv_bfloat16, 1>(a, s) : launch<__nv_bfloat16, 2>(a, s);
}
