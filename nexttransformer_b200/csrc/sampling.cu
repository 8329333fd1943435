// K25: one token for each row of logits, from a number u in [0, 1) that the caller draws.
//
//   w_i = exp((x_i - max x) / T); order: x falling, index rising among equals
//   top-k: the first k.  top-p: those before which less than p of (the first k's) mass lies.  min-p: w_i >= min_p
//   token = the smallest index up to which more than u of the kept mass lies (in the order of indices)
//
// Weights are whole numbers, 2^S w rounded (S = 62 - log2 V), from a 64-bit exp: sums are exact in any order, so atomics and
// the split of a row change nothing, and a token differs from the one that real numbers give only when u lies within
// about V 2^-S of a border.
//
// A row lies in the shared memory of a cluster of CTAs and is read from memory once (longer ones are read again, from L2).  A
// selection's border (the k-th, or the one at which p is reached) is found by a histogram of 2048 bins of T / 32 below the
// maximum, whose bins the CTAs add up through distributed shared memory.  What can be kept, where it is few, goes to one CTA, which
// ranks the border's bin and draws; where it is many, the masses before the border's bin are summed by runs of indices.  A bin of
// more than 1024 is split by the numbers' bits, and equal logits by their indices.
//
// Bound by latency and by 64-bit arithmetic: 1 x 32768, top-k and top-p: 14 us, of which (clock stamps) loads take 0.5, the maximum 1.3, the
// histogram 1.1, its crossing and the list 3.4, the gathering 1.8, the two borders 3.1, the draw 2.4.  224 x 65536 with a setting for each row: 80 to 83 us
// for 59 MB (9 at the copy rate): two CTAs an SM, so three to four rounds, each CTA 17 us (top-k) to 40 (top-p alone), with 8 or 9
// for each pass that takes the exp of every logit in 64 bits.
// Tried and not kept: a sort of the kept ones (5 us and more), every CTA reading all bins' masses of all (15 us instead of 4).
#include "sampling.h"
#include "common.cuh"

#include <cuda_fp16.h>
#include <math.h>

namespace nt {
namespace sampling {

constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 2048;
constexpr int FEW = 2048, EACH = FEW / THREADS;  // a list that one CTA takes; its entries a thread
constexpr int CAP = FEW / 2;                     // entries of one bin that are ranked among each other
constexpr int SEGMENT_MOST = 16384;  // logits that a CTA holds in shared memory, 64 KB, so that two CTAs fit an SM
constexpr int VOCABULARY_MOST = 1 << 19;
constexpr int CLUSTER_MOST = 8;
using u64 = unsigned long long;

template <class T> NT_DEVICE float to_float(T v);
template <> NT_DEVICE float to_float(float v) { return v; }
template <> NT_DEVICE float to_float(__half v) { return __half2float(v); }
template <> NT_DEVICE float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Whole numbers in the order of the floats (which have no -0 here).
NT_DEVICE uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
}

NT_DEVICE float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

// An entry of a list: its number grows along the order.
NT_DEVICE u64 entry_of(uint32_t key, int index) { return (static_cast<u64>(~key) << 32) | static_cast<uint32_t>(index); }
NT_DEVICE float value_in(u64 entry) { return value_of(~static_cast<uint32_t>(entry >> 32)); }

struct Border {     // kept: keys above it, and those equal to it up to its index
  uint32_t key;
  int index;
};
struct Note {       // what a CTA tells the others
  u64 mass;
  uint32_t count, low, high;
  int index;
};

struct Shared {
  union {
    u64 mass[BINS];
    uint32_t count[BINS];
    u64 sorted[FEW];  // entries that are ranked (and their shares)
  };
  union {
    u64 list[FEW];    // this CTA's candidates
    u64 by_index[FEW / 2];
  };
  Note note[2];
  u64 scan[WARPS + 1], own[WARPS];
  float top[WARPS];
  double table[64];
  int nan;
  uint32_t listed, low, high;
  int found;
  u64 found_before, found_own;
};

// The same address in CTA `rank` of the cluster.
template <class P>
NT_DEVICE P* peer(P* p, int rank) {
  uint64_t r;
  asm("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
  return reinterpret_cast<P*>(r);
}

constexpr int TABLE = 64;  // 2^(i / 64)

// A CTA's part of a row: in shared memory, or read again at each pass.
template <class T, bool HELD>
struct Row {
  float* held;
  const T* in;
  int n, first, V;   // how many, index of the first
  int ranks, rank;
  float top;         // the row's largest
  float none;        // smaller ones have no weight
  bool infinite;     // the largest are inf: they count as 0, the others as -inf
  double factor, peak;  // 64 log2(e) / T; top
  const double* table;
  float half_top, per_bin;  // half the largest; bins for half a logit's distance from it
  int shift;         // S

  NT_DEVICE float operator[](int i) const {
    if (HELD) return held[i];
    const float x = to_float(in[i]) + 0.f;  // -0 becomes 0
    return infinite ? (x == INFINITY ? 0.f : -INFINITY) : x;
  }
  // f(x, i) for the CTA's logits; several are asked for at once.
  template <class F>
  NT_DEVICE void each(F f) const {
    constexpr int U = HELD ? 4 : 8;
    for (int i0 = threadIdx.x; i0 < n; i0 += THREADS * U) {
      float x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = i0 + u * THREADS < n ? (*this)[i0 + u * THREADS] : 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * THREADS < n) f(x[u], i0 + u * THREADS);
    }
  }
};

// 2^shift exp((x - top) / T), to 1e-13 of it; 0 from 2^(shift - 70) down.  64 (x - top) log2(e) / T is n and a rest; 2^(n mod 64 / 64) stands
// in a table, and the rest's power is its series: with z = rest ln 2 / 64, |z| <= 0.0054, the first term left out is z^5 / 120 = 4e-14.
template <class R>
NT_DEVICE double power(const R& r, float x, int shift) {
  constexpr double LN = 0.69314718055994530942 / TABLE, MAGIC = 6755399441055744.0;  // 1.5 2^52: adding it rounds to a whole number
  const double t = (static_cast<double>(fmaxf(x, r.none)) - r.peak) * r.factor;  // 0 for the top whatever T is: of two products a rest would stay
  const double whole = t + MAGIC, z = t - (whole - MAGIC);
  double p = LN * LN * LN * LN / 24;
  p = fma(p, z, LN * LN * LN / 6);
  p = fma(p, z, LN * LN / 2);
  p = fma(p, z, LN);
  p = fma(p, z, 1.0);
  const int n = __double2loint(whole);
  p *= r.table[n & (TABLE - 1)];
  // p 2^e; never below 2^-140 (48 T may be rounded to twice that), so that only the exponent's bits change
  const double v = __hiloint2double(__double2hiint(p) + (((n >> 6) + shift) << 20), __double2loint(p));
  return x < r.none ? 0.0 : v;
}
template <class R>
NT_DEVICE u64 weight_of(const R& r, float x) {
  const double v = power(r, x, r.shift) + 4503599627370496.0;  // 2^52: the whole number is in the lower bits
  return static_cast<u64>(__double_as_longlong(v)) & 0xfffffffffffffull;
}
// Bins keep the order of the logits; the last, from 64 T on, has no weight (-inf and NaN, of inf 0, go there).  Adding 2^23 rounds
// to a whole number, which is the sum's lower bits: a conversion would take an instruction of a quarter of the rate.  (Half the distance: the
// whole passes fp32's range where logits of 3e38 stand on both sides of 0.)
template <class R>
NT_DEVICE float bin_sum(const R& r, float x) { return fminf(fmaf(x, -0.5f, r.half_top) * r.per_bin, static_cast<float>(BINS - 1)) + 8388608.f; }
template <class R>
NT_DEVICE int bin_of(const R& r, float x) { return __float_as_int(bin_sum(r, x)) & (BINS - 1); }
NT_DEVICE bool within(const Border& b, float x, int index) {
  const uint32_t k = key_of(x);
  return k > b.key || (k == b.key && index <= b.index);
}

template <class V>
NT_DEVICE V warp_scan(V v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V w = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += w;
  }
  return v;
}
// Exclusive sum over the CTA's threads; `total` gets the whole.  Two barriers.
NT_DEVICE u64 block_scan(u64 v, Shared& s, u64& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const u64 upto = warp_scan(v, lane);
  __syncthreads();
  if (lane == 31) s.scan[warp] = upto;
  __syncthreads();
  u64 before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const u64 x = s.scan[w];
    if (w < warp) before += x;
    total += x;
  }
  return before + upto - v;
}

NT_DEVICE u64 share_of(float p, u64 total, bool up) {  // p total, 0 <= p < 1, to a whole number
  const u64 f = static_cast<u64>(static_cast<double>(p) * 18446744073709551616.0);
  return __umul64hi(f, total) + (up && f * total != 0 ? 1 : 0);
}

// Adds to a 64-bit sum in shared memory by its halves: the upper one is rarely touched.
NT_DEVICE void add_to(u64* p, u64 w) {
  uint32_t* half = reinterpret_cast<uint32_t*>(p);
  const uint32_t lo = static_cast<uint32_t>(w), before = atomicAdd(half, lo);
  const uint32_t hi = static_cast<uint32_t>(w >> 32) + (before + lo < lo ? 1u : 0u);
  if (hi) atomicAdd(half + 1, hi);
}
template <bool MASS>
NT_DEVICE void clear_bins(Shared& s) {
  uint4* p = reinterpret_cast<uint4*>(s.mass);
  for (int i = threadIdx.x; i < BINS * (MASS ? 8 : 4) / 16; i += THREADS) p[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
}
template <bool MASS, class R>
NT_DEVICE void add_to_bin(const R& r, Shared& s, int bin, float x) {
  if (MASS) add_to(&s.mass[bin], weight_of(r, x));
  else atomicAdd(&s.count[bin], 1u);
}
// The bin in which the sum over the cluster's bins (`alone`: this CTA's) reaches the target, or -1; `before`: the sum over those
// before it.  A target of 0 is set to `share` of the whole first.  Counts of up to four
// CTAs are read by all of them; else each adds up its part of the bins and tells the others (all masses of eight CTAs read by all took 15 us
// instead of 4).  Where all read all, others may still be at this CTA's bins when it returns: `s.count` and what shares its memory may be
// written again only behind a cluster barrier.
template <bool MASS, class R>
NT_DEVICE int crossing(const R& r, Shared& s, int& round, u64& target, float share, u64& before, bool alone = false) {
  constexpr int MOST = BINS / THREADS;
  const int tid = threadIdx.x, lane = tid & 31, ranks = alone ? 1 : r.ranks;
  const bool apart = ranks > 4 || (MASS && ranks > 1);
  const int part = apart ? BINS / ranks : BINS, per = max(1, part / THREADS), from = (apart ? r.rank * part : 0) + tid * per;
  u64 sum[MOST] = {}, all = 0;
  if (ranks == 1) {
#pragma unroll
    for (int e = 0; e < MOST; ++e) sum[e] = MASS ? s.mass[from + e] : s.count[from + e];
  } else if (!apart) {
    uint4 u[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) u[c] = c < ranks ? reinterpret_cast<const uint4*>(peer(s.count, c))[tid] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      sum[0] += u[c].x; sum[1] += u[c].y; sum[2] += u[c].z; sum[3] += u[c].w;
    }
  } else if (tid * per < part) {
#pragma unroll
    for (int e = 0; e < MOST; ++e)
      if (e < per) {
        u64 v[CLUSTER_MOST];
#pragma unroll
        for (int c = 0; c < CLUSTER_MOST; ++c) {
          v[c] = 0;
          if (c < ranks) v[c] = MASS ? peer(s.mass, c)[from + e] : peer(s.count, c)[from + e];
        }
#pragma unroll
        for (int c = 0; c < CLUSTER_MOST; ++c) sum[e] += v[c];
      }
  }
#pragma unroll
  for (int e = 0; e < MOST; ++e) all += sum[e];
  if (tid == 0) s.found = -1;
  u64 total;
  u64 at = block_scan(all, s, total);
  if (apart) {
    if (tid == 0) s.note[round & 1].mass = total;
    cluster_sync();
    const u64 upto = warp_scan(lane < ranks ? peer(&s.note[round & 1], lane)->mass : 0ull, lane);
    if (r.rank) at += __shfl_sync(0xffffffffu, upto, r.rank - 1);
    total = __shfl_sync(0xffffffffu, upto, 31);
    ++round;
  }
  if (MASS && target == 0) target = share > 0.f ? max(share_of(share, total, true), 1ull) : 1ull;
#pragma unroll
  for (int e = 0; e < MOST; ++e) {
    if (at < target && target <= at + sum[e])
      for (int c = 0; c < (apart ? ranks : 1); ++c) {
        Shared* to = apart ? peer(&s, c) : &s;
        to->found = from + e;
        to->found_before = at;
      }
    at += sum[e];
  }
  if (apart) cluster_sync();
  else __syncthreads();
  before = s.found_before;
  return s.found;
}
// A histogram of the elements within `outer` by their distance from the top, and its crossing.
template <bool MASS, class R>
NT_DEVICE int first_crossing(const R& r, Shared& s, int& round, const Border& outer, u64& target, float share, u64& before) {
  clear_bins<MASS>(s);
  const bool any = outer.key == 0;
  r.each([&](float x, int i) {
    const int bin = bin_of(r, x);
    if (bin < BINS - 1 && (any || within(outer, x, r.first + i))) add_to_bin<MASS>(r, s, bin, x);
  });
  cluster_sync();
  return crossing<MASS>(r, s, round, target, share, before);
}

// Of m entries in any order and their shares: the one at which the sum over the order reaches the target.  As many lanes as
// there are for it add up each entry's predecessors.
NT_DEVICE u64 ranked(const u64* entry, const u64* share, int m, u64 target, u64 done, Shared& s) {
  const int tid = threadIdx.x;
  int lanes = 1;
  while (lanes < 32 && 2 * lanes * m <= THREADS && 32 * lanes <= m) lanes *= 2;
  const int part = tid & (lanes - 1);
  for (int i0 = 0; i0 < m; i0 += THREADS / lanes) {
    const int i = i0 + tid / lanes;
    const u64 own = i < m ? entry[i] : 0ull;
    u64 sum = 0;
#pragma unroll 4
    for (int j = part; j < m; j += lanes) {
      const u64 v = share[j];
      sum += entry[j] < own ? v : 0ull;
    }
    for (int o = lanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    sum += done;
    if (i < m && sum < target && target <= sum + share[i]) s.found_own = own;
  }
  __syncthreads();
  return s.found_own;
}

// Lists the elements that `is(x, index)` names, up to FEW of them, and counts all; ends with a barrier.  A thread looks at 32 before it asks
// for room.
template <class R, class Is>
NT_DEVICE void list_elements(const R& r, Shared& s, Is is) {
  const int tid = threadIdx.x, lane = tid & 31;
  if (tid == 0) s.listed = 0;
  __syncthreads();
  for (int i0 = 0; i0 < r.n; i0 += THREADS * 32) {
    unsigned mine = 0;
#pragma unroll 1
    for (int e = 0; e < 32 && i0 + e * THREADS < r.n; e += 8) {
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + (e + u) * THREADS + tid;
        x[u] = i < r.n ? r[i] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + (e + u) * THREADS + tid;
        if (i < r.n && is(x[u], r.first + i)) mine |= 1u << (e + u);
      }
    }
    if (!__any_sync(0xffffffffu, mine)) continue;
    const uint32_t upto = warp_scan(static_cast<uint32_t>(__popc(mine)), lane);
    uint32_t at = 0;
    if (lane == 31) at = atomicAdd(&s.listed, upto);
    at = __shfl_sync(0xffffffffu, at, 31) + upto - __popc(mine);
    for (; mine; mine &= mine - 1, ++at) {
      const int i = i0 + (__ffs(mine) - 1) * THREADS + tid;
      if (at < FEW) s.list[at] = entry_of(key_of(r[i]), r.first + i);
    }
  }
  __syncthreads();
}

// The border of a selection: the element at which the sum (of weights, or of ones) over the order reaches `target`, which lies in
// bin `chosen`, behind a sum of `done`.  Only elements within `outer` count.
template <bool MASS, class R>
NT_DEVICE Border find_border(const R& r, Shared& s, int& round, const Border& outer, u64 target, int chosen, u64 done) {
  const int tid = threadIdx.x, lane = tid & 31;
  uint32_t low = 0, high = 0xffffffffu;  // of the candidates' keys, after the first list
  bool first = true;
  auto candidate = [&](float x, int index) {
    if (first) return bin_of(r, x) == chosen && within(outer, x, index);
    const uint32_t k = key_of(x);
    return k >= low && k <= high && within(outer, x, index);
  };
#pragma unroll 1
  while (true) {
    // ---- this CTA's candidates: a list, their number, and, where they are many, their extremes
    if (tid == 0) {
      s.low = 0xffffffffu;
      s.high = 0;
    }
    list_elements(r, s, candidate);
    if (s.listed > CAP) {
      uint32_t least = 0xffffffffu, most = 0;
      r.each([&](float x, int i) {
        if (!candidate(x, r.first + i)) return;
        least = min(least, key_of(x));
        most = max(most, key_of(x));
      });
      least = __reduce_min_sync(0xffffffffu, least);
      most = __reduce_max_sync(0xffffffffu, most);
      if (lane == 0) {
        atomicMin(&s.low, least);
        atomicMax(&s.high, most);
      }
    } else {
      for (uint32_t i = tid; i < s.listed; i += THREADS) {
        const uint32_t k = ~static_cast<uint32_t>(s.list[i] >> 32);
        atomicMin(&s.low, k);
        atomicMax(&s.high, k);
      }
    }
    __syncthreads();
    if (tid == 0) {
      Note& n = s.note[round & 1];
      n.count = s.listed;
      n.low = s.low;
      n.high = s.high;
    }
    cluster_sync();
    const Note* theirs = peer(&s.note[round & 1], min(lane, r.ranks - 1));
    const uint32_t counts = lane < r.ranks ? theirs->count : 0u;  // lane c: CTA c's
    const uint32_t many = __reduce_add_sync(0xffffffffu, counts);
    low = __reduce_min_sync(0xffffffffu, theirs->low);
    high = __reduce_max_sync(0xffffffffu, theirs->high);
    ++round;
    first = false;
    if (many <= CAP) {
      // ---- rank them among each other (each CTA by itself)
      uint32_t at = 0;
      for (int c = 0; c < r.ranks; ++c) {
        const uint32_t n = __shfl_sync(0xffffffffu, counts, c);
        for (uint32_t i = tid; i < n; i += THREADS) {
          const u64 v = peer(s.list, c)[i];
          s.sorted[at + i] = v;
          s.sorted[CAP + at + i] = MASS ? weight_of(r, value_in(v)) : 1ull;
        }
        at += n;
      }
      __syncthreads();
      const u64 v = ranked(s.sorted, s.sorted + CAP, static_cast<int>(many), target, done, s);
      return {~static_cast<uint32_t>(v >> 32), static_cast<int>(static_cast<uint32_t>(v))};
    }
    if (low == high) {
      // ---- equal logits: the first of them by index.  The number of those that are kept:
      const u64 each = MASS ? weight_of(r, value_of(low)) : 1ull;
      u64 need = (target - done + each - 1) / each;  // at least 1
      for (int c = 0; c < r.rank; ++c) {
        const uint32_t n = __shfl_sync(0xffffffffu, counts, c);
        need = need > n ? need - n : 0;  // 0 from the CTA on that has the last
      }
      // every warp takes a run of indices
      const int run = (r.n + WARPS - 1) / WARPS, from = (tid >> 5) * run, to = min(r.n, from + run);
      u64 mine = 0, total;
      for (int i = from + lane; i < to; i += 32) mine += candidate(r[i], r.first + i) ? 1 : 0;
      u64 prior = block_scan(mine, s, total);
      prior = __shfl_sync(0xffffffffu, prior, 0);  // of the warps before
      if (tid == 0) s.note[round & 1].index = -1;
      __syncthreads();
      if (need && need <= total) {
        for (int i0 = from; i0 < to; i0 += 32) {
          const int i = i0 + lane;
          const bool is = i < to && candidate(r[i], r.first + i);
          const unsigned who = __ballot_sync(0xffffffffu, is);
          if (is && prior + __popc(who & ((2u << lane) - 1u)) == need) s.note[round & 1].index = r.first + i;
          prior += __popc(who);
        }
      }
      cluster_sync();
      const int index = lane < r.ranks ? peer(&s.note[round & 1], lane)->index : -1;
      ++round;
      return {low, __reduce_max_sync(0xffffffffu, index)};
    }
    // ---- many that differ: a histogram of their keys, the largest first
    const int shift = max(0, 32 - __clz(high - low) - 11);
    clear_bins<MASS>(s);
    r.each([&](float x, int i) {
      if (candidate(x, r.first + i)) add_to_bin<MASS>(r, s, (high - key_of(x)) >> shift, x);
    });
    cluster_sync();
    u64 rest = target - done, before;  // crossing() counts from the first bin
    const int bin = crossing<MASS>(r, s, round, rest, 0.f, before);
    done += before;
    high = high - (static_cast<uint32_t>(bin) << shift);
    low = max(low, shift ? high - ((1u << shift) - 1u) : high);
  }
}

struct Filters {
  int first;       // top-k (0x7fffffff: off)
  float share;     // top-p (1: off)
  double least;    // min-p
  float number;    // u
};
// min-p; the largest logits pass whatever their computed weight is
template <class R>
NT_DEVICE bool passes(const R& r, const Filters& f, float x) {
  return !(f.least > 0.0) || x == r.top || (f.least < 1.0 && power(r, x, 0) >= f.least);
}

// The entry of the list at which the sum (of weights, or of ones) over the order reaches `target`.  `chosen`, `done`: its bin, and the
// sum before that.  A thread has EACH entries; those up to `last` count.  Entries are ordered as their numbers are.
template <bool MASS, class R>
NT_DEVICE u64 border_of_few(const R& r, Shared& s, const u64 (&entry)[EACH], const u64 (&w)[EACH], u64 last, int chosen, u64 target,
                            u64 done) {
  const int tid = threadIdx.x;
  if (tid == 0) s.listed = 0;
  __syncthreads();
  int mine = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if (entry[e] <= last && bin_of(r, value_in(entry[e])) == chosen) mine |= 1 << e;
  uint32_t at = mine ? atomicAdd(&s.listed, __popc(mine)) : 0u;
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if ((mine >> e) & 1) {
      s.sorted[at] = entry[e];
      s.list[at++] = MASS ? w[e] : 1ull;
    }
  __syncthreads();
  return ranked(s.sorted, s.list, s.listed, target, done, s);
}

// Where few elements can be kept (the bins up to `chosen`, `done` before it): one CTA gathers them and draws.  MASS: target is the mass
// at which p is reached; else it is the k of top-k, and what p is reached at follows.  False: they are many.
template <bool MASS, class R>
NT_DEVICE bool draw_from_few(const SampleArgs& a, const R& r, Shared& s, int& round, const Border& outer, int chosen, u64 target, u64 done,
                             const Filters& f, int b) {
  const int tid = threadIdx.x, lane = tid & 31;
  const bool any = outer.key == 0;
  const float end = static_cast<float>(chosen) + 8388608.f;
  list_elements(r, s, [&](float x, int index) { return bin_sum(r, x) <= end && (any || within(outer, x, index)); });
  if (tid == 0) s.note[round & 1].count = s.listed;
  cluster_sync();
  const uint32_t counts = lane < r.ranks ? peer(&s.note[round & 1], lane)->count : 0u, upto = warp_scan(counts, lane);
  const int many = static_cast<int>(__shfl_sync(0xffffffffu, upto, 31));
  ++round;
  if (many > FEW) return false;
  // a thread's entries, straight from the lists (0xff..: none)
  u64 entry[EACH];
  if (r.rank == 0) {
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int at = e * THREADS + tid;
      entry[e] = ~0ull;
      int c = 0;
      uint32_t before = 0;
      for (int o = 0; o < r.ranks; ++o) {
        const uint32_t end = __shfl_sync(0xffffffffu, upto, o);
        if (static_cast<uint32_t>(at) >= end) {
          c = o + 1;
          before = end;
        }
      }
      if (at < many) entry[e] = peer(s.list, c)[at - before];
    }
  }
  cluster_sync();  // the lists are read: the other CTAs are done
  if (r.rank != 0) return true;

  u64 w[EACH], total, last = ~0ull - 1;
#pragma unroll
  for (int e = 0; e < EACH; ++e) w[e] = 0;
  if (!MASS) last = border_of_few<false>(r, s, entry, w, last, chosen, target, done);
  u64 sum = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if (entry[e] <= last) {
      w[e] = weight_of(r, value_in(entry[e]));
      sum += w[e];
    }
  if (MASS) {
    last = border_of_few<true>(r, s, entry, w, last, chosen, target, done);
  } else if (f.share < 1.f) {
    clear_bins<true>(s);
#pragma unroll
    for (int e = 0; e < EACH; ++e)
      if (w[e]) add_to(&s.mass[bin_of(r, value_in(entry[e]))], w[e]);
    __syncthreads();
    target = 0;
    const int bin = crossing<true>(r, s, round, target, f.share, done, true);
    __syncthreads();  // the bins are read
    last = border_of_few<true>(r, s, entry, w, last, bin, target, done);
  }
  uint32_t index[EACH];
  sum = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const float x = value_in(entry[e]);
    index[e] = static_cast<uint32_t>(entry[e]);
    if (entry[e] > last || !passes(r, f, x)) w[e] = 0;
    sum += w[e];
  }
  block_scan(sum, s, total);
  // ---- the draw goes by index: runs of indices first, then the indices of the run
  u64 aim = min(share_of(f.number, total, false), total - 1);
  const int low_bits = max(0, 32 - __clz(r.V - 1) - 9);  // V <= 2^19: at most 1024 indices a run
  s.by_index[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if (w[e]) add_to(&s.by_index[index[e] >> low_bits], w[e]);
  __syncthreads();
  u64 own = s.by_index[tid], ignored, at = block_scan(own, s, ignored);
  if (at <= aim && aim < at + own) {
    s.found = tid;
    s.found_before = at;
  }
  __syncthreads();
  const uint32_t run = s.found;
  aim -= s.found_before;
  for (int i = tid; i < (1 << low_bits); i += THREADS) s.by_index[i] = 0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if (w[e] && (index[e] >> low_bits) == run) s.by_index[index[e] & ((1u << low_bits) - 1u)] = w[e];
  __syncthreads();
  const u64 u = 2 * tid < (1 << low_bits) ? s.by_index[2 * tid] : 0, v = 2 * tid + 1 < (1 << low_bits) ? s.by_index[2 * tid + 1] : 0;
  at = block_scan(u + v, s, ignored);
  if (at <= aim && aim < at + u + v) {
    const bool second = aim >= at + u;
    a.tokens[b] = (static_cast<int64_t>(run) << low_bits) + 2 * tid + (second ? 1 : 0);
    a.logprobs[b] = static_cast<float>(log(static_cast<double>(second ? v : u) / static_cast<double>(total)));
  }
  return true;
}

struct Sums {        // of the kept mass
  u64 total, prior, own;  // of the row, of the CTAs before this one, of this one
};
// The runs of indices that warps sum up: warp w of a CTA has [w run, (w + 1) run).
template <class R>
NT_DEVICE int run_of(const R& r) { return (r.n + WARPS - 1) / WARPS; }

// Where many are kept up to bin `chosen`: one pass sums the masses of the bins before it (into s.own, a warp's run each) and lists that
// bin's elements, which are few as a rule; ranked, they give the border and their part of the masses.  False: the bin's are many.
template <class R>
NT_DEVICE bool sum_up_to(const R& r, Shared& s, int& round, const Border& outer, int chosen, u64 target, u64 done, const Filters& f, Border& border,
                         Sums& sums) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, run = run_of(r), from = min(r.n, warp * run), to = min(r.n, from + run);
  if (tid == 0) s.listed = 0;
  __syncthreads();
  const bool any = outer.key == 0;
  const float end = static_cast<float>(chosen) + 8388608.f;
  u64 mass = 0;
  for (int i0 = from; i0 < to; i0 += 1024) {  // a thread looks at 32 before it computes any weight: most are not kept
    unsigned below = 0, at = 0;
#pragma unroll 1
    for (int e = 0; e < 32 && i0 + 32 * e < to; e += 8) {
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = i0 + 32 * (e + k) + lane;
        x[k] = i < to ? r[i] : -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float v = bin_sum(r, x[k]);
        if (v <= end && (any || within(outer, x[k], r.first + i0 + 32 * (e + k) + lane))) (v == end ? at : below) |= 1u << (e + k);
      }
    }
    while (__any_sync(0xffffffffu, below)) {
      if (below) {
        const float x = r[i0 + 32 * (__ffs(below) - 1) + lane];
        if (passes(r, f, x)) mass += weight_of(r, x);
        below &= below - 1;
      }
    }
    if (!__any_sync(0xffffffffu, at)) continue;
    const uint32_t upto = warp_scan(static_cast<uint32_t>(__popc(at)), lane);
    uint32_t place = 0;
    if (lane == 31) place = atomicAdd(&s.listed, upto);
    place = __shfl_sync(0xffffffffu, place, 31) + upto - __popc(at);
    for (; at; at &= at - 1, ++place) {
      const int i = i0 + 32 * (__ffs(at) - 1) + lane;
      if (place < FEW) s.list[place] = entry_of(key_of(r[i]), r.first + i);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
  if (lane == 0) s.own[warp] = mass;
  __syncthreads();
  if (tid == 0) {
    Note& n = s.note[round & 1];
    n.count = s.listed;
    n.mass = 0;
    for (int w = 0; w < WARPS; ++w) n.mass += s.own[w];
  }
  cluster_sync();
  const Note* theirs = peer(&s.note[round & 1], min(lane, r.ranks - 1));
  const uint32_t counts = lane < r.ranks ? theirs->count : 0u;  // lane c: CTA c's
  u64 masses = lane < r.ranks ? theirs->mass : 0ull;
  ++round;
  if (__reduce_add_sync(0xffffffffu, counts) > CAP) return false;
  uint32_t many = 0;
  for (int c = 0; c < r.ranks; ++c) {
    const uint32_t n = __shfl_sync(0xffffffffu, counts, c);
    for (uint32_t i = tid; i < n; i += THREADS) {
      const u64 v = peer(s.list, c)[i];
      s.sorted[many + i] = v;
      s.sorted[CAP + many + i] = weight_of(r, value_in(v));
    }
    many += n;
  }
  __syncthreads();
  const u64 last = ranked(s.sorted, s.sorted + CAP, static_cast<int>(many), target, done, s);
  border = {~static_cast<uint32_t>(last >> 32), static_cast<int>(static_cast<uint32_t>(last))};
  // what the bin adds: to every CTA's mass (each knows them all), and to this CTA's runs
  uint32_t at = 0;
  for (int c = 0; c < r.ranks; ++c) {
    const uint32_t n = __shfl_sync(0xffffffffu, counts, c);
    u64 more = 0;
    for (uint32_t i = lane; i < n; i += 32) {
      const u64 v = s.sorted[at + i];
      if (v > last || !passes(r, f, value_in(v))) continue;
      const u64 w = s.sorted[CAP + at + i];
      more += w;
      if (c == r.rank && warp == 0) add_to(&s.own[(static_cast<int>(static_cast<uint32_t>(v)) - r.first) / run], w);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) more += __shfl_xor_sync(0xffffffffu, more, o);
    if (lane == c) masses += more;
    at += n;
  }
  const u64 upto = warp_scan(masses, lane);
  sums.total = __shfl_sync(0xffffffffu, upto, 31);
  sums.own = __shfl_sync(0xffffffffu, masses, r.rank);
  sums.prior = __shfl_sync(0xffffffffu, upto, r.rank) - sums.own;
  __syncthreads();
  return true;
}

template <class T, bool HELD, bool VECTORS>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const SampleArgs a, const int segment, const int ranks) {
  extern __shared__ __align__(16) float values[];
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x / ranks;
  auto value = [&](const RowValue& v) { return v.rows ? static_cast<const float*>(v.rows)[b] : static_cast<float>(v.all); };
  Row<T, HELD> r;
  r.held = values;
  r.ranks = ranks;
  r.rank = blockIdx.x % ranks;
  r.V = a.V;
  r.first = min(r.rank * segment, a.V);
  r.n = min(segment, a.V - r.first);
  r.in = static_cast<const T*>(a.logits) + b * a.row_stride + r.first;
  const float heat = value(a.temperature), u = a.uniform[b], top_p = value(a.top_p), min_p = value(a.min_p);
  const int top_k = a.top_k.rows ? static_cast<const int*>(a.top_k.rows)[b] : static_cast<int>(a.top_k.all);
  int round = 0;

  // ---- the row comes in; its largest logit
  float top = -INFINITY;
  bool nan = false;
  auto take = [&](int i, float x) {
    x += 0.f;  // -0 becomes 0
    if (HELD) values[i] = x;
    top = fmaxf(top, x);
    nan |= isnan(x);
  };
  const T* in = r.in;
  if (VECTORS) {
    constexpr int E = 16 / sizeof(T);
    struct alignas(16) Vec { T x[E]; };
    for (int i0 = 0; i0 < r.n; i0 += THREADS * E * 4) {
      Vec v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + (k * THREADS + tid) * E;
        if (i < r.n) v[k] = *reinterpret_cast<const Vec*>(in + i);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + (k * THREADS + tid) * E;
        if (i < r.n)
#pragma unroll
          for (int e = 0; e < E; ++e) take(i + e, to_float(v[k].x[e]));
      }
    }
  } else {
    for (int i0 = 0; i0 < r.n; i0 += THREADS * 8) {
      T v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = i0 + k * THREADS + tid;
        if (i < r.n) v[k] = in[i];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = i0 + k * THREADS + tid;
        if (i < r.n) take(i, to_float(v[k]));
      }
    }
  }
  if (tid == 0) s.nan = 0;
  if (tid < TABLE) s.table[tid] = exp2(static_cast<double>(tid) / TABLE);
  __syncthreads();
  if (nan) s.nan = 1;
  top = warp_max(top);
  if (lane == 0) s.top[warp] = top;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < WARPS; ++w) top = fmaxf(top, s.top[w]);
    s.note[0].low = __float_as_uint(top);
    s.note[0].index = s.nan;
  }
  cluster_sync();
  {
    const Note* n = peer(&s.note[0], min(lane, ranks - 1));  // lane c: CTA c's
    nan = __any_sync(0xffffffffu, n->index != 0);
    top = warp_max(__uint_as_float(n->low));
  }
  ++round;
  if (nan || top == -INFINITY) {
    if (r.rank == 0 && tid == 0) {
      a.tokens[b] = nan ? -2 : -1;
      a.logprobs[b] = nan ? NAN : -INFINITY;
    }
    cluster_sync();  // the others may still read this CTA's note
    return;
  }
  r.infinite = top == INFINITY;  // the infinite ones share the choice
  if (r.infinite) {
    if (HELD)
      for (int i = tid; i < r.n; i += THREADS) values[i] = values[i] == INFINITY ? 0.f : -INFINITY;
    top = 0.f;
    __syncthreads();
  }
  const bool greedy = !(heat > 0.f);
  r.top = top;
  r.factor = greedy ? 0.0 : TABLE * 1.4426950408889634074 / static_cast<double>(heat);
  r.peak = top;
  r.table = s.table;
  r.none = fmaxf(top - 48.f * heat, -3.4028235e38f);  // 2^-69
  r.half_top = 0.5f * top;
  r.per_bin = fminf(64.f / heat, 3e38f);
  r.shift = min(50, 30 + __clz(a.V));  // V 2^S <= 2^62

  const Filters f = {top_k > 0 && top_k < a.V ? top_k : 0x7fffffff, top_p < 1.f ? top_p : 1.f,
                     min_p > 0.f ? fmin(static_cast<double>(min_p), 1.0) : 0.0, u > 0.f ? fminf(u, 0.99999994f) : 0.f};

  // ---- the order's kept part
  bool summed = false;
  Sums sums;
  Border kept = {0u, 0x7fffffff};
  if (greedy) {
    kept.key = key_of(top);  // its first index is found below
  } else {
    u64 target = f.first, before;
    if (f.first < 0x7fffffff) {
      const int chosen = first_crossing<false>(r, s, round, kept, target, 0.f, before);
      if (chosen >= 0) {  // (else the k-th has no weight)
        if (draw_from_few<false>(a, r, s, round, kept, chosen, target, before, f, b)) return;
        kept = find_border<false>(r, s, round, kept, target, chosen, before);
      } else {
        cluster_sync();  // the bins are read by all, and may be cleared
      }
    }
    if (f.share < 1.f) {
      target = 0;
      const int chosen = first_crossing<true>(r, s, round, kept, target, f.share, before);
      // The mass over the weight of the bin's lower end bounds their number; real rows have an eighth of that, or less
      const bool few = target >> 3 <= static_cast<u64>(FEW) * weight_of(r, top - static_cast<float>(2 * chosen + 2) / r.per_bin);
      if (few && draw_from_few<true>(a, r, s, round, kept, chosen, target, before, f, b)) return;
      Border cut;
      summed = sum_up_to(r, s, round, kept, chosen, target, before, f, cut, sums);
      kept = summed ? cut : find_border<true>(r, s, round, kept, target, chosen, before);
    }
  }
  const bool all = kept.key == 0;
  auto mass_of = [&](int i) -> u64 {
    const float x = r[i];
    if (!all && !within(kept, x, r.first + i)) return 0ull;
    if (greedy) return 1ull;
    if (!passes(r, f, x)) return 0ull;
    return weight_of(r, x);
  };

  // ---- the draw: masses of the warps' runs of indices, the run that u falls into, the thread, the token
  const int run = run_of(r), from = min(r.n, warp * run), to = min(r.n, from + run);
  if (!summed) {
    u64 mine = 0;
    for (int i = from + lane; i < to; i += 32) mine += mass_of(i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) s.own[warp] = mine;
    __syncthreads();
    if (tid == 0) {
      u64 sum = 0;
      for (int w = 0; w < WARPS; ++w) sum += s.own[w];
      s.note[round & 1].mass = sum;
    }
    cluster_sync();
    const u64 theirs = lane < ranks ? peer(&s.note[round & 1], lane)->mass : 0ull, upto = warp_scan(theirs, lane);  // lane c: CTA c's
    sums.total = __shfl_sync(0xffffffffu, upto, 31);
    sums.own = __shfl_sync(0xffffffffu, theirs, r.rank);
    sums.prior = __shfl_sync(0xffffffffu, upto, r.rank) - sums.own;
  }
  const u64 total = sums.total, prior = sums.prior, own = sums.own;
  const u64 aim = greedy ? 0 : min(share_of(f.number, total, false), total - 1);
  if (prior <= aim && aim < prior + own) {
    int w = 0;
    u64 at = prior;
    while (w < WARPS - 1 && aim >= at + s.own[w]) at += s.own[w++];
    const int begin = min(r.n, w * run), end = min(r.n, begin + run), each = (end - begin + THREADS - 1) / THREADS;
    const int lo = min(end, begin + tid * each), hi = min(end, lo + each);
    u64 sum = 0, ignored;
    for (int i = lo; i < hi; ++i) sum += mass_of(i);
    at += block_scan(sum, s, ignored);
    if (at <= aim && aim < at + sum) {
      int i = lo;
      u64 m = mass_of(i);
      while (aim >= at + m) {
        at += m;
        m = mass_of(++i);
      }
      a.tokens[b] = r.first + i;
      a.logprobs[b] = greedy ? 0.f : static_cast<float>(log(static_cast<double>(m) / static_cast<double>(total)));
    }
  }
  cluster_sync();  // nobody leaves while its notes are read
}

template <class T, bool HELD, bool VECTORS>
static int launch(const SampleArgs& a, int segment, int ranks, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  auto kern = sample_kernel<T, HELD, VECTORS>;
  if (HELD && smem_limit(done, kern, SEGMENT_MOST * 4) != cudaSuccess) return -1;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.B) * ranks);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = HELD ? segment * 4 : 0;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a, segment, ranks) == cudaSuccess ? 0 : -1;
}
template <class T>
static int by_type(const SampleArgs& a, cudaStream_t s) {
  constexpr int E = 16 / sizeof(T);
  // As many CTAs as hold the row on chip; few rows are spread further.  224 x 65536, a filter or three in each row: one CTA a row
  // (read again at each pass) 163 us, two 116, four 84, eight 120; 1 x 32768: one 25 us, two 14.9, four 13.8, eight 14.5.
  int ranks = 1;
  while (ranks < CLUSTER_MOST && ((a.V + ranks - 1) / ranks > SEGMENT_MOST || (ranks < 4 && a.B * ranks * 2ll <= 2 * a.sms && a.V / ranks > 4096))) ranks *= 2;
  const int segment = ((a.V + ranks - 1) / ranks + E - 1) / E * E;
  const bool vectors = a.V % E == 0 && a.row_stride % E == 0 && reinterpret_cast<uintptr_t>(a.logits) % 16 == 0;
  if (segment <= SEGMENT_MOST) return vectors ? launch<T, true, true>(a, segment, ranks, s) : launch<T, true, false>(a, segment, ranks, s);
  return vectors ? launch<T, false, true>(a, segment, ranks, s) : launch<T, false, false>(a, segment, ranks, s);
}

}  // namespace sampling
}  // namespace nt

using namespace nt::sampling;

int nt_sample_most() { return VOCABULARY_MOST; }

int nt_sample_logits(const SampleArgs& a, cudaStream_t s) {
  if (a.B == 0) return 0;
  if (a.V < 1 || a.V > nt_sample_most() || a.B > INT32_MAX / CLUSTER_MOST) return -1;
  if (a.type == LOGITS_BF16) return by_type<__nv_bfloat16>(a, s);
  if (a.type == LOGITS_FP16) return by_type<__half>(a, s);
  if (a.type == LOGITS_FP32) return by_type<float>(a, s);
  return -1;
}
