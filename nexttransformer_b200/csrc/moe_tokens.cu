// K26: a mixture-of-experts layer for up to 64 tokens (decoding): what it reads is the chosen experts' weights, once.
//
//   l = W_r x, p = softmax(l); the k experts with the largest p + bias (ties to the lower one); c = p / sum of the chosen p
//   y = sum over the chosen of c W2 relu(W1 x)^2 + W2' relu(W1' x)^2 (the shared expert)
//
// Three kernels, each started while the one before it ends:
//   route  a cluster of CTAs a token: logits in fp32, the choice, and x in the order of a matrix operand
//   fc     h = c relu(W1 x)^2, a warp for 16 rows of an expert's W1
//   proj   y, a CTA (or a cluster, by parts of the sum) for 16 rows of every expert's W2, added up in registers
//
// With few tokens an expert meets one or two of them, so weights are the 16-row side of a 16 x 8 x 16 matrix instruction and
// tokens the narrow side; 2 to 16 operations a byte are far below the ratio at which tensor memory would matter.  The work is to
// keep loads in flight: each warp owns a ring of 2 KB stages (16 rows of 128 bytes) that asynchronous copies fill across the
// borders of tiles and experts, and waits for nobody else until its sums are done.
#include "moe_tokens.h"
#include "warp_mma.cuh"

#include <algorithm>

namespace nt {
namespace moe_tokens {

constexpr int ROUTE_WARPS = 8, ROUTE_THREADS = ROUTE_WARPS * 32;
constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int STAGE = 2048, STAGES = 12, RING = STAGE * STAGES;  // 24 KB a warp; two CTAs an SM
constexpr int SMEM = WARPS * RING;
constexpr int MOST = NT_MOE_TOKENS_MOST, EXPERTS = NT_MOE_TOKENS_EXPERTS, CHOICES = NT_MOE_TOKENS_CHOICES;
// Hidden values are held in the weights' type.  fp16 ends at 65504, which a square passes where its root is 256: they
// are held as 2^-6 of themselves there (up to 4.2e6), and the sums are raised again.
template <class T> constexpr float LOWER = 1.f;
template <> constexpr float LOWER<__half> = 1.f / 64;

struct Workspace {
  int* choice;    // [T, k]
  float* share;   // [T, E], set where chosen
  uint2* x;       // [ceil(d / 16), blocks of 8 tokens, 32]: a lane's part of a 16 x 8 operand
  uint2* h;       // [pairs of an expert and a block of 8 of its tokens, ceil(F / 16), 32]
  int pairs;      // of routed experts; the shared expert's blocks, of ceil(Fs / 16) each, come behind them
};
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
  w.x = reinterpret_cast<uint2*>(take(static_cast<size_t>(blocks_of(a.d, 16)) * nb * 256));
  w.h = reinterpret_cast<uint2*>(take(static_cast<size_t>(w.pairs) * blocks_of(a.F, 16) * 256 + static_cast<size_t>(nb) * blocks_of(a.Fs, 16) * 256));
  return at;
}

NT_DEVICE void dependents_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
NT_DEVICE void wait_for_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ------------------------------------------------------------------------------------ route
template <class T>
__global__ void __launch_bounds__(ROUTE_THREADS) route_kernel(const MoeTokensArgs a, const Workspace w, const int ranks) {
  extern __shared__ __align__(16) float x[];
  __shared__ float logits[EXPERTS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, t = blockIdx.x / ranks, rank = blockIdx.x % ranks;
  dependents_may_start();
  const T* src = static_cast<const T*>(a.x) + t * a.x_stride;
  for (int i = tid * 8; i < a.d; i += ROUTE_THREADS * 8) {
    const uint4 u = *reinterpret_cast<const uint4*>(src + i);
    const uint32_t v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) *reinterpret_cast<float2*>(x + i + 2 * e) = Num<T>::unpack(v[e]);
  }
  // x as an operand: lane 4 n + c of a 16 x 8 tile has token n's channels 2 c, 2 c + 1 and 2 c + 8, 2 c + 9
  const int nb = (a.T + 7) / 8, groups = (a.d + 15) / 16;
  for (int i = rank * ROUTE_THREADS + tid; i < groups * 4; i += ranks * ROUTE_THREADS) {
    const int g = i >> 2, at = g * 16 + (i & 3) * 2;
    const uint32_t lo = *reinterpret_cast<const uint32_t*>(src + at), hi = at + 8 < a.d ? *reinterpret_cast<const uint32_t*>(src + at + 8) : 0u;
    w.x[(static_cast<int64_t>(g) * nb + t / 8) * 32 + (t % 8) * 4 + (i & 3)] = make_uint2(lo, hi);
  }
  cluster_sync();  // x is there, and the first CTA, which gets the logits
  for (int e = rank * ROUTE_WARPS + warp; e < a.E; e += ranks * ROUTE_WARPS) {
    const float4* row = reinterpret_cast<const float4*>(a.router + static_cast<int64_t>(e) * a.d);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);  // four chains of d / 128 products a lane
#pragma unroll 8
    for (int i = lane; i < a.d / 4; i += 32) {
      const float4 u = row[i], v = reinterpret_cast<const float4*>(x)[i];
      sum.x = fmaf(u.x, v.x, sum.x);
      sum.y = fmaf(u.y, v.y, sum.y);
      sum.z = fmaf(u.z, v.z, sum.z);
      sum.w = fmaf(u.w, v.w, sum.w);
    }
    const float l = warp_sum((sum.x + sum.y) + (sum.z + sum.w));
    if (lane == 0) {
      uint32_t to = smem_u32(logits + e), remote;
      asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(to));
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(l) : "memory");
    }
  }
  cluster_sync();
  if (rank != 0 || warp != 0) return;
  constexpr int PER = EXPERTS / 32;
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
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, best, o), theirs = __shfl_xor_sync(0xffffffffu, its, o);
      const int where = __shfl_xor_sync(0xffffffffu, at, o);
      if (other > best || (other == best && where < at)) {
        best = other;
        its = theirs;
        at = where;
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 32 * i == at) score[i] = -INFINITY;
    if (lane == j) {
      chosen = at;
      chosen_p = its;
    }
  }
  const float all = warp_sum(lane < a.k ? chosen_p : 0.f);
  if (lane < a.k) {
    w.choice[t * a.k + lane] = chosen;
    w.share[static_cast<int64_t>(t) * a.E + chosen] = chosen_p / all;
  }
}

// ------------------------------------------------------------------------------------ the experts
// Who wants which expert, from the choices: one bit a token, the wanted experts in order, and their first block of 8 tokens.
struct Lists {
  unsigned long long mask[EXPERTS + 1];  // [E]: the shared expert's, all tokens
  uint16_t expert[EXPERTS + 1];          // wanted ones; the shared expert (E) comes last
  uint16_t block[EXPERTS + 1];           // their first block
  int wanted;
};
NT_DEVICE void make_lists(const MoeTokensArgs& a, const Workspace& w, Lists& l) {
  const int tid = threadIdx.x, lane = tid & 31;
  for (int e = tid; e <= a.E; e += THREADS) l.mask[e] = 0;
  __syncthreads();
  for (int i = tid; i < a.T * a.k; i += THREADS) atomicOr(&l.mask[__ldcg(w.choice + i)], 1ull << (i / a.k));
  __syncthreads();
  if (tid < 32) {
    int n = 0, blocks = 0;
    for (int e0 = 0; e0 < a.E; e0 += 32) {
      const int e = e0 + lane;
      const int own = e < a.E ? (__popcll(l.mask[e]) + 7) >> 3 : 0;
      const unsigned who = __ballot_sync(0xffffffffu, own > 0);
      int upto = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      if (own) {
        const int at = n + __popc(who & ((1u << lane) - 1u));
        l.expert[at] = static_cast<uint16_t>(e);
        l.block[at] = static_cast<uint16_t>(blocks + upto - own);
      }
      n += __popc(who);
      blocks += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) {
      if (a.Fs) {
        l.mask[a.E] = a.T == 64 ? ~0ull : (1ull << a.T) - 1;
        l.expert[n] = static_cast<uint16_t>(a.E);
        l.block[n] = 0;
        ++n;
      }
      l.wanted = n;
    }
  }
  __syncthreads();
}
// The n-th token (from 0) of a mask, or -1.
NT_DEVICE int nth_token(unsigned long long m, int n) {
  for (int i = 0; i < n && m; ++i) m &= m - 1;
  return m ? __ffsll(static_cast<long long>(m)) - 1 : -1;
}

// A warp's ring: 16 rows of 64 elements a stage, chunk c of row r at c ^ (r & 7).
struct Ring {
  uint32_t base, to;     // of the ring; this lane's first place in a stage
  int stage_in, stage_out;
  uint32_t at[4];        // this lane's matrix row of the four 16-column tiles
};
NT_DEVICE Ring make_ring(const void* smem) {
  Ring r;
  const int lane = threadIdx.x & 31, row = lane >> 3, chunk = lane & 7;
  r.base = smem_u32(smem) + (threadIdx.x >> 5) * RING;
  r.to = row * 128 + ((chunk ^ row) << 4);  // rows row + 4 e have the chunk at the same place, or across (chunk ^ 4)
  r.stage_in = r.stage_out = 0;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int m = lane & 15;
    r.at[s] = m * 128 + (((2 * s + (lane >> 4)) ^ (m & 7)) << 4);
  }
  return r;
}
// Rows [0, rows) of a tile at p (this lane's row and chunk), stride bytes apart; `inside`: the lane's chunk is.  What is not
// there becomes zero (and names an address that is).
NT_DEVICE void copy_stage(Ring& r, const char* p, int64_t stride, int rows, bool inside, const void* there) {
  const uint32_t dst = r.base + r.stage_in * STAGE + r.to;
  const int row = (threadIdx.x & 31) >> 3;
  if (rows == 16 && inside) {
#pragma unroll
    for (int e = 0; e < 4; ++e) cp_async16((dst + e * 512) ^ ((e & 1) << 6), p + e * 4 * stride);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool valid = inside && row + 4 * e < rows;
      cp_async16_or_zero((dst + e * 512) ^ ((e & 1) << 6), valid ? p + e * 4 * stride : there, valid);
    }
  }
  if (++r.stage_in == STAGES) r.stage_in = 0;
}

template <class T, int NB>
__global__ void __launch_bounds__(THREADS, 2) fc_kernel(const MoeTokensArgs a, const Workspace w) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Lists l;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  wait_for_predecessor();
  dependents_may_start();
  make_lists(a, w, l);
  const int tiles = (a.F + 15) / 16, shared_tiles = (a.Fs + 15) / 16, stages = (a.d + 63) / 64, groups = (a.d + 15) / 16, nb_x = (a.T + 7) / 8;
  const int routed = l.wanted - (a.Fs ? 1 : 0), items = routed * tiles + shared_tiles;
  const int first = warp * gridDim.x + blockIdx.x, step = gridDim.x * WARPS;
  if (first >= items) return;
  Ring r = make_ring(smem);
  const int row = lane >> 3, chunk = lane & 7, width = a.d;

  struct Item {
    int e, at, tile, hidden;  // expert, its place in the list, row tile, rows in all
  };
  auto item_of = [&](int i) {
    Item it;
    if (i < routed * tiles) {
      it.at = quotient(i, tiles);
      it.tile = i - it.at * tiles;
      it.hidden = a.F;
    } else {
      it.at = routed;
      it.tile = i - routed * tiles;
      it.hidden = a.Fs;
    }
    it.e = l.expert[it.at];
    return it;
  };
  // ---- the copies' place
  int f_item = first, f_stage = 0, f_rows = 0;
  const char* f_at = nullptr;
  auto enter = [&]() {
    const Item it = item_of(f_item);
    const T* base = it.e == a.E ? static_cast<const T*>(a.shared_fc) : static_cast<const T*>(a.w_fc) + static_cast<int64_t>(it.e) * a.F * a.d;
    f_at = reinterpret_cast<const char*>(base + (static_cast<int64_t>(it.tile) * 16 + row) * a.d + chunk * 8);
    f_rows = min(16, it.hidden - it.tile * 16);
  };
  enter();
  auto fetch = [&]() {
    if (f_item < items) {
      copy_stage(r, f_at, static_cast<int64_t>(a.d) * sizeof(T), f_rows, f_stage * 64 + chunk * 8 < width, a.x);
      f_at += 128;
      if (++f_stage == stages) {
        f_stage = 0;
        f_item += step;
        if (f_item < items) enter();
      }
    }
    cp_commit();
  };
#pragma unroll 1
  for (int i = 0; i < STAGES - 1; ++i) fetch();

#pragma unroll 1
  for (int item = first; item < items; item += step) {
    const Item it = item_of(item);
    const unsigned long long mask = l.mask[it.e];
    const int blocks = (__popcll(mask) + 7) >> 3;  // of 8 of the expert's tokens
    const uint2* xs[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int t = nb < blocks ? max(0, nth_token(mask, nb * 8 + (lane >> 2))) : 0;
      xs[nb] = w.x + (t >> 3) * 32 + (t & 7) * 4 + (lane & 3);
    }
    float acc[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[nb][e] = 0.f;
#pragma unroll 1
    for (int st = 0; st < stages; ++st) {
      uint2 b[4][NB];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int g = st * 4 + s;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          b[s][nb] = make_uint2(0u, 0u);
          if (nb < blocks && g < groups) b[s][nb] = xs[nb][static_cast<int64_t>(g) * nb_x * 32];
        }
      }
      cp_wait<STAGES - 2>();
      __syncwarp();  // this stage has landed for every lane, and the stage before it is read by none
      const uint32_t base = r.base + r.stage_out * STAGE;
      if (++r.stage_out == STAGES) r.stage_out = 0;
      uint32_t wf[4][4];
#pragma unroll
      for (int s = 0; s < 4; ++s) ldsm4(wf[s], base + r.at[s]);
      fetch();
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          if (nb < blocks) Num<T>::mma(acc[nb], wf[s], b[s][nb].x, b[s][nb].y);
    }
    // ---- h, in the order in which it is an operand: rows of the tile become the products' inner dimension
    const int inner = it.e == a.E ? shared_tiles : tiles;
    uint2* h = w.h + (it.e == a.E ? static_cast<int64_t>(w.pairs) * tiles : static_cast<int64_t>(l.block[it.at]) * tiles) * 32;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      if (nb >= blocks) break;
      float v[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = nth_token(mask, nb * 8 + (lane & 3) * 2 + e);
        const float c = t < 0 ? 0.f : it.e == a.E ? LOWER<T> : LOWER<T> * w.share[static_cast<int64_t>(t) * a.E + it.e];
        const float u = fmaxf(acc[nb][e], 0.f), z = fmaxf(acc[nb][e + 2], 0.f);
        // a NaN has to stay one; columns that are no token's give zero
        v[e] = t < 0 ? 0.f : c * (isnan(acc[nb][e]) ? acc[nb][e] : u * u);
        v[e + 2] = t < 0 ? 0.f : c * (isnan(acc[nb][e + 2]) ? acc[nb][e + 2] : z * z);
      }
      h[(static_cast<int64_t>(nb) * inner + it.tile) * 32 + lane] =
          make_uint2(transpose8x8(Num<T>::pack(v[0], v[1])), transpose8x8(Num<T>::pack(v[2], v[3])));
    }
  }
  cp_wait<0>();
}

template <class T, int NB>
__global__ void __launch_bounds__(THREADS, 2) proj_kernel(const MoeTokensArgs a, const Workspace w, const int parts) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Lists l;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, part = blockIdx.x % parts, tile = blockIdx.x / parts;
  make_lists(a, w, l);  // (the route kernel ended before the one before this began its work)
  const int per = (a.F + 63) / 64, shared_per = (a.Fs + 63) / 64, tiles = (a.F + 15) / 16, shared_tiles = (a.Fs + 15) / 16;
  const int routed = l.wanted - (a.Fs ? 1 : 0), all = routed * per + shared_per;
  // an equal run of the stages of all wanted experts
  const int runs = parts * WARPS, run = part * WARPS + warp, few = all / runs, more = all % runs;
  const int first = run * few + min(run, more), last = first + few + (run < more ? 1 : 0);
  Ring r = make_ring(smem);
  const int row = lane >> 3, chunk = lane & 7, rows = min(16, a.d - tile * 16);
  float acc[NB][4];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[nb][e] = 0.f;

  struct Place {
    int at, stage, stages, hidden;
  };
  auto place_of = [&](int i) {
    Place p;
    if (i < routed * per) {
      p.at = quotient(i, per);
      p.stage = i - p.at * per;
      p.stages = per;
      p.hidden = a.F;
    } else {
      p.at = routed;
      p.stage = i - routed * per;
      p.stages = shared_per;
      p.hidden = a.Fs;
    }
    return p;
  };
  if (first < last) {
    Place f = place_of(first);
    const char* f_at = nullptr;
    int f_left = last - first;
    auto enter = [&]() {
      const int e = l.expert[f.at];
      const T* base = e == a.E ? static_cast<const T*>(a.shared_proj) : static_cast<const T*>(a.w_proj) + static_cast<int64_t>(e) * a.d * a.F;
      f_at = reinterpret_cast<const char*>(base + (static_cast<int64_t>(tile) * 16 + row) * f.hidden + f.stage * 64 + chunk * 8);
    };
    enter();
    auto fetch = [&]() {
      if (f_left > 0) {
        copy_stage(r, f_at, static_cast<int64_t>(f.hidden) * sizeof(T), rows, f.stage * 64 + chunk * 8 < f.hidden, a.x);
        f_at += 128;
        --f_left;
        if (++f.stage == f.stages) {
          f.stage = 0;
          ++f.at;
          if (f_left > 0) {
            f.stages = f.at < routed ? per : shared_per;
            f.hidden = f.at < routed ? a.F : a.Fs;
            enter();
          }
        }
      }
      cp_commit();
    };
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; ++i) fetch();
    wait_for_predecessor();  // weights may come before, h may not

    Place c = place_of(first);
    int left = last - first;
#pragma unroll 1
    while (left > 0) {
      const int e = l.expert[c.at], n = min(left, c.stages - c.stage), inner = e == a.E ? shared_tiles : tiles;
      const unsigned long long mask = l.mask[e];
      const uint2* h = w.h + (e == a.E ? static_cast<int64_t>(w.pairs) * tiles : static_cast<int64_t>(l.block[c.at]) * tiles) * 32;
      // columns are tokens here, which an expert's blocks hold one after another
      const uint2* hs[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int t = nb * 8 + (lane >> 2);
        const bool is = (mask >> t) & 1ull;
        const int place = __popcll(mask & ((1ull << t) - 1ull));
        hs[nb] = is ? h + static_cast<int64_t>(place >> 3) * inner * 32 + (place & 7) * 4 + (lane & 3) : nullptr;
      }
#pragma unroll 1
      for (int st = c.stage; st < c.stage + n; ++st) {
        uint2 b[4][NB];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const int g = st * 4 + s;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            b[s][nb] = make_uint2(0u, 0u);
            if (hs[nb] && g < inner) b[s][nb] = __ldcg(hs[nb] + g * 32);
          }
        }
        cp_wait<STAGES - 2>();
        __syncwarp();
        const uint32_t base = r.base + r.stage_out * STAGE;
        if (++r.stage_out == STAGES) r.stage_out = 0;
        uint32_t wf[4][4];
#pragma unroll
        for (int s = 0; s < 4; ++s) ldsm4(wf[s], base + r.at[s]);
        fetch();
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            if ((mask >> (nb * 8)) & 0xffull) Num<T>::mma(acc[nb], wf[s], b[s][nb].x, b[s][nb].y);
      }
      left -= n;
      c.stage += n;
      if (c.stage == c.stages) {
        c.stage = 0;
        ++c.at;
        c.stages = c.at < routed ? per : shared_per;
        c.hidden = c.at < routed ? a.F : a.Fs;
      }
    }
    cp_wait<0>();
  } else {
    wait_for_predecessor();
  }

  // ---- the warps' sums, then the parts', in their order
  __syncthreads();
  float4* sums = reinterpret_cast<float4*>(smem);  // [warp][nb][lane]
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) sums[(warp * NB + nb) * 32 + lane] = make_float4(acc[nb][0], acc[nb][1], acc[nb][2], acc[nb][3]);
  __syncthreads();
  float4* whole = sums + WARPS * NB * 32;
  for (int i = tid; i < NB * 32; i += THREADS) {
    float4 v = sums[i];
#pragma unroll
    for (int k = 1; k < WARPS; ++k) {
      const float4 u = sums[k * NB * 32 + i];
      v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
    }
    whole[i] = v;
  }
  if (parts > 1) cluster_sync();
  else __syncthreads();
  if (part == 0) {
    for (int i = tid; i < NB * 32; i += THREADS) {
      float4 v = whole[i];
      for (int c = 1; c < parts; ++c) {
        uint32_t remote;
        float4 u;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(whole + i)), "r"(c));
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(u.x), "=f"(u.y), "=f"(u.z), "=f"(u.w) : "r"(remote) : "memory");
        v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
      }
      // a lane has channels g and g + 8 of tokens 2 c and 2 c + 1
      const int t = (i >> 5) * 8 + (i & 3) * 2, ch = tile * 16 + ((i & 31) >> 2);
      T* y = static_cast<T*>(a.y);
      const float f = 1.f / LOWER<T>;
      const uint32_t lo = Num<T>::pack(v.x * f, v.z * f), hi = Num<T>::pack(v.y * f, v.w * f);
      auto put = [&](int token, int at, uint32_t u) {
        if (token < a.T && at < a.d) reinterpret_cast<uint16_t*>(y)[static_cast<int64_t>(token) * a.d + at] = static_cast<uint16_t>(u);
      };
      put(t, ch, lo);
      put(t, ch + 8, lo >> 16);
      put(t + 1, ch, hi);
      put(t + 1, ch + 8, hi >> 16);
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
template <class T, int NB>
static int launch(const MoeTokensArgs& a, cudaStream_t s) {
  static std::atomic<uint64_t> fc_done{0}, proj_done{0};
  if (smem_limit(fc_done, fc_kernel<T, NB>, SMEM) != cudaSuccess || smem_limit(proj_done, proj_kernel<T, NB>, SMEM) != cudaSuccess) return -1;
  Workspace w;
  layout(a, w);
  int ranks = 8;
  while (ranks > 1 && a.T * ranks > 2 * a.sms) ranks /= 2;
  if (start(route_kernel<T>, a.T * ranks, ROUTE_THREADS, a.d * sizeof(float), ranks, false, s, a, w, ranks)) return -1;
  if (start(fc_kernel<T, NB>, 2 * a.sms, THREADS, SMEM, 1, true, s, a, w)) return -1;
  const int tiles = (a.d + 15) / 16, parts = std::max(1, std::min(8, 2 * a.sms / tiles));
  return start(proj_kernel<T, NB>, tiles * parts, THREADS, SMEM, parts, true, s, a, w, parts);
}
template <class T>
static int by_tokens(const MoeTokensArgs& a, cudaStream_t s) {
  if (a.T <= 8) return launch<T, 1>(a, s);
  if (a.T <= 16) return launch<T, 2>(a, s);
  if (a.T <= 32) return launch<T, 4>(a, s);
  return launch<T, 8>(a, s);
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
  return a.fp16 ? by_tokens<__half>(a, s) : by_tokens<__nv_bfloat16>(a, s);
}
