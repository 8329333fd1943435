// K24: the paged key-value cache of the decoding engine.
//
// append     k' = s rope(k) / rms(rope(k)), v' = v + 3 sigmoid(gate) ve into the pages, q' = s rope(q) / rms(rope(q))
// attention  o = softmax(scale q K^T) V over the pages, a few new tokens per row, GQA, left window
//
// Both are bound by memory.  What each kernel does about it, and what it measured on one B200 (copies reach 6.46 TB/s
// there), stands beside it; times are the device's.
#include "paged.h"
#include "warp_mma.cuh"

#include <algorithm>
#include <type_traits>

namespace nt {
namespace paged {

constexpr float EPS = 1.1920929e-07f;  // FLT_EPSILON, as the shell's RMSNorm
// By how many powers of two probabilities are raised, see the softmax
template <class T> constexpr float RAISE_OF = 0.f;
template <> constexpr float RAISE_OF<__half> = 7.f;

// ------------------------------------------------------------------------------------ append
// D / 8 lanes hold one head of one token; lane j has channels 4 j to 4 j + 3 of each half, so that it holds
// both members of its rotated pairs.  They take PER heads of their token, whose loads are all in flight at once
// and which share the token's angles and place in the cache.  Blocks with small y turn queries and keys, the
// others mix values.  One pass: every input element is read once and every output element written once, and what is
// no token is not read.  8 prompts of up to 2048 tokens, 10 + 5 heads of 128: 27 us where its 117 MB (and 17 MB of
// zeros) would take 21 at the copy rate; instruction issue (0.7 a cycle and scheduler) is the next limit.  One token: 2.5 us,
// the chain from the row's length over its page to the store.
template <class T>
NT_DEVICE void load_halves(const T* p, int half, uint2& lo, uint2& hi) {
  lo = __ldcs(reinterpret_cast<const uint2*>(p));
  hi = __ldcs(reinterpret_cast<const uint2*>(p + half));
}
template <class T>
NT_DEVICE void unpack4(uint2 u, float2 (&x)[2]) {
  x[0] = Num<T>::unpack(u.x);
  x[1] = Num<T>::unpack(u.y);
}
template <class T>
NT_DEVICE uint2 pack4(const float2 (&x)[2]) {
  return make_uint2(Num<T>::pack(x[0].x, x[0].y), Num<T>::pack(x[1].x, x[1].y));
}
template <class T, int D, int PER>
__global__ void __launch_bounds__(256, 4) append_kernel(const PagedAppendArgs a, const int turning) {
  constexpr int L = D / 8, HALF = D / 2;
  const int lane = threadIdx.x % L, tok = blockIdx.x * (256 / L) + threadIdx.x / L;
  const bool live = tok < a.B * a.t;  // whole warps stay for the shuffles
  const int b = live ? (a.t == 1 ? tok : quotient(tok, a.t)) : 0, i = live ? tok - b * a.t : 0;
  const int start = a.start[b], n = a.count ? a.count[b] : a.t;
  bool real = live && i < n && start >= 0;
  if (real && start >= a.rope_rows - i) {
    if (lane == 0) record_error(3, b);
    real = false;
  }
  const int pos = real ? start + i : 0;
  // the token's place in the cache
  const PagedCacheArgs& m = a.cache;
  auto find_page = [&](int& slot) -> int64_t {
    const int column = quotient(pos, m.page);
    slot = pos - column * m.page;
    if (column >= m.columns) {
      if (lane == 0) record_error(1, b);
      return -1;
    }
    const int page = m.table[static_cast<int64_t>(b) * m.columns + column];
    if (page >= 0 && page < m.pages) return page;
    if (lane == 0) record_error(2, b);
    return -1;
  };

  if (static_cast<int>(blockIdx.y) >= turning) {
    // ---- values
    if (!real) return;
    const int h0 = (blockIdx.y - turning) * PER, heads = min(PER, a.Hk - h0);
    uint2 lo[PER], hi[PER], elo[PER], ehi[PER];
    T gate[PER];
    const T* src = static_cast<const T*>(a.vin) + b * a.vs[0] + i * a.vs[1] + h0 * a.vs[2] + lane * 4;
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (e < heads) {
        load_halves(src, HALF, lo[e], hi[e]);
        src += a.vs[2];
      }
    if (a.ve) {
      const T* es = static_cast<const T*>(a.ve) + b * a.es[0] + i * a.es[1] + h0 * a.es[2] + lane * 4;
      const T* gs = static_cast<const T*>(a.ve_gate) + b * a.gs[0] + i * a.gs[1] + h0 * a.gs[2];
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (e < heads) {
          load_halves(es, HALF, elo[e], ehi[e]);
          gate[e] = *gs;
          es += a.es[2];
          gs += a.gs[2];
        }
    }
    int slot;
    const int64_t page = find_page(slot);
    if (page < 0) return;
    T* dst = static_cast<T*>(m.v) + page * m.page_stride_v + slot * m.slot_stride_v + h0 * m.head_stride_v + lane * 4;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if (e >= heads) break;
      if (a.ve) {
        float2 x[2], y[2], u[2], w[2];
        const float f = 3.f / (1.f + __expf(-Num<T>::one(gate[e])));
        const float2 ff = make_float2(f, f);
        unpack4<T>(lo[e], x); unpack4<T>(elo[e], u);
        unpack4<T>(hi[e], y); unpack4<T>(ehi[e], w);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          x[j] = fma2(ff, u[j], x[j]);
          y[j] = fma2(ff, w[j], y[j]);
        }
        lo[e] = pack4<T>(x);
        hi[e] = pack4<T>(y);
      }
      *reinterpret_cast<uint2*>(dst) = lo[e];
      *reinterpret_cast<uint2*>(dst + HALF) = hi[e];
      dst += m.head_stride_v;
    }
    return;
  }

  // ---- queries and keys; h counts through both
  const int h0 = blockIdx.y * PER, heads = min(PER, a.H + a.Hk - h0);
  T* q_out = static_cast<T*>(a.q_out) + (static_cast<int64_t>(tok) * a.H + h0) * D + lane * 4;
  uint2 lo[PER], hi[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) lo[e] = hi[e] = make_uint2(0, 0);
  if (real) {
    const T* src = h0 < a.H ? static_cast<const T*>(a.q) + b * a.qs[0] + i * a.qs[1] + h0 * a.qs[2] + lane * 4 : nullptr;
    int64_t step = a.qs[2];
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (e < heads) {
        if (h0 + e == a.H || (e == 0 && h0 > a.H)) {
          src = static_cast<const T*>(a.kin) + b * a.ks[0] + i * a.ks[1] + (h0 + e - a.H) * a.ks[2] + lane * 4;
          step = a.ks[2];
        }
        load_halves(src, HALF, lo[e], hi[e]);
        src += step;
      }
  }
  T* k_out = nullptr;
  float2 c[2] = {}, s[2] = {}, ns[2];
  if (real) {
    if (h0 + heads > a.H) {
      int slot;
      const int64_t page = find_page(slot);
      if (page >= 0)
        k_out = static_cast<T*>(m.k) + page * m.page_stride_k + slot * m.slot_stride_k + max(h0 - a.H, 0) * m.head_stride_k + lane * 4;
    }
    unpack4<T>(*reinterpret_cast<const uint2*>(static_cast<const T*>(a.cos) + static_cast<int64_t>(pos) * HALF + lane * 4), c);
    unpack4<T>(*reinterpret_cast<const uint2*>(static_cast<const T*>(a.sin) + static_cast<int64_t>(pos) * HALF + lane * 4), s);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) ns[j] = make_float2(-s[j].x, -s[j].y);
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    if (e >= heads) break;
    float2 x[2], y[2], u[2], w[2];
    unpack4<T>(lo[e], x);
    unpack4<T>(hi[e], y);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      u[j] = fma2(y[j], s[j], mul2(x[j], c[j]));
      w[j] = fma2(x[j], ns[j], mul2(y[j], c[j]));
    }
    if (a.norm) {
      const float2 pair = fma2(w[1], w[1], fma2(u[1], u[1], fma2(w[0], w[0], mul2(u[0], u[0]))));
      float sum = pair.x + pair.y;
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float r = a.scale * rsqrtf(sum * (1.f / D) + EPS);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        u[j] = mul2(u[j], make_float2(r, r));
        w[j] = mul2(w[j], make_float2(r, r));
      }
    }
    T* dst;
    if (h0 + e < a.H) {  // tokens behind a row's count have zeros in, and give zeros
      dst = live ? q_out : nullptr;
      q_out += D;
    } else {
      dst = k_out;
      if (k_out) k_out += m.head_stride_k;
    }
    if (dst) {
      *reinterpret_cast<uint2*>(dst) = pack4<T>(u);
      *reinterpret_cast<uint2*>(dst + HALF) = pack4<T>(w);
    }
  }
}

template <class T, int D, int PER>
static int launch_append(const PagedAppendArgs& a, unsigned blocks, cudaStream_t s) {
  const int turning = (a.H + a.Hk + PER - 1) / PER, mixing = (a.Hk + PER - 1) / PER;
  if (turning + mixing > 65535) return -1;
  append_kernel<T, D, PER><<<dim3(blocks, turning + mixing), 256, 0, s>>>(a, turning);
  return 0;
}
template <class T, int D>
static int launch_append(const PagedAppendArgs& a, cudaStream_t s) {
  const int64_t tokens = static_cast<int64_t>(a.B) * a.t, per_block = 256 / (D / 8), blocks = (tokens + per_block - 1) / per_block;
  if (tokens > INT32_MAX - per_block) return -1;
  // Five heads a thread keep enough bytes in flight and share a token's address work; with few tokens, one head a thread
  // reaches more SMs.  Device times at 10 / 5, 16 / 1, 12 / 12, 8 / 2, 6 / 6 and 12 / 3 heads of 64 and 128: 8 prompts of 2048
  // tokens take 11 to 49 us with five, 22 to 34 % more with one, up to 8 % more with four (6 / 6: 4 to 6 % less, its last
  // group is half empty) and up to 19 % more with three; a prompt of 400 tokens takes 2.8 to 3.7 us with one and
  // 14 to 32 % more with five.  At two thirds of the limit five take 0 to 14 % more than one, just above it 0 to 14 % less.
  return blocks * ((a.H + 2 * a.Hk + 4) / 5) >= 2 * a.sms ? launch_append<T, D, 5>(a, static_cast<unsigned>(blocks), s)
                                                          : launch_append<T, D, 1>(a, static_cast<unsigned>(blocks), s);
}

// --------------------------------------------------------------------------------- attention
// The R = t (H / Hk) query rows that share a KV head are the columns of the products, 8 or 16 at a time
// (NQ blocks of 8):  S^T = K Q^T  and  O^T = V^T P^T, so that keys and head channels, of which there are
// many, fill the 16-row side of the 16 x 8 x 16 matrix instruction and one decoding row per head wastes
// the narrow side only.  The accumulator of S^T becomes the operand P^T through a transposing move between
// registers.  At 16 queries a key costs 4 D x 16 operations against 4 D bytes: 16 operations a byte, far
// below the ratio (263) at which tensor memory and wider instructions would matter; the kernel's work is to
// keep loads in flight, so each warp owns a ring of 16-key stages filled with 16-byte asynchronous copies
// and waits for nobody else.
//
// Work: a row's keys (window cut off) are tiles of 16.  The tiles of all rows and KV heads form one line, each CTA
// takes an equal piece of it and each warp an equal piece of that, so unequal rows load the SMs equally and one
// long row uses all of them; a boundary near a (row, KV head)'s end moves there, which saves a join and costs a few
// tiles of balance.  A warp that covers a whole (row, KV head) writes its result; other pieces are joined in the CTA,
// and what crosses CTAs by the CTA that arrives last, up to 16 pieces at a time.  Pieces are always joined in the
// order of the line, so results do not depend on timing.
//
// Measured: 16 rows of 32768 keys, 10 / 5 heads of 128: 208.8 us, 6.43 TB/s.  64 rows of 512 to 8192 keys, 16 / 1 heads:
// 28.5 us for 89 MB.  Clock stamps of a first warp a CTA, same case: the first tile is there after 4.1 us (length, page and
// key are a trip to memory each), the tiles are done after 16 us in half of the CTAs and 23 in all, the CTAs' joins
// after 18.7 and 25.9 us and those across CTAs after 27.  One row of 1001 keys: 11.5 us, few (row, KV head) pairs on few
// SMs; first tile 2.9, tiles 7.9, join 9.7 us.
// Tried and not kept: a second kernel for the join (10 us for one row, but two launches, 9 instead of 6 us on the
// host), joins spread over rows instead of accumulator blocks, smaller reaches for the boundaries (16
// tiles 1 %, 8 tiles 2 % slower over a set of calls), at least 4 tiles a warp (4 % slower over it; 1: 2 % faster).
// More than 16 query rows a KV head are row tiles that each read the keys again, by instructions made for 8 queries: 8
// prompts of 2048 tokens, 10 / 5 heads of 128, take 715 us, where the training attention on tcgen05 takes 146 for the same
// contiguous keys and the arithmetic 51; 4 prompts of 512 take 52 against 26.  248 rows of 5 tokens, 12 / 3 heads, 1709
// keys take 236 us where one reading takes 102.  Ways to read them once, in an earlier build (237 us): warps of a CTA side
// by side on the row tiles of the same keys: 179 us, but 5 % more for every call with one row tile and 12 % more over a set
// with several; row tiles outermost on the line: 183 us and 1 % less over the set, but 1039 instead of 700 us for 8
// prompts of 2048 tokens.  Neither was kept.
//
// Pages in 8 bits: codes become fp16 in registers, which holds them exactly, and so do queries (bf16 ones after a power of two a row).  A
// tile is a block, so its keys' scale goes into the scores' factor and its values' into the probabilities, relative to a unit that follows
// them, like the maximum.  A line's bytes suit the products as they lie: a lane's four neighbouring channels of a key are its share of a
// 16-column step, for keys and queries alike, and two keys' pairs of channels from a transposing load are two rows of V^T.
// 16 rows of 32768 keys, 10 / 5 heads of 128: 122 us, 5.5 TB/s (209 in 16 bits): a tile is 324 instructions, and two warps
// a scheduler wait for their own (4.6 cycles each).  64 rows of 512 to 8192 keys, 16 / 1 heads: 27.0 us, 24 x 4 tokens with a window of 1023: 23.5,
// 1 x 1001: 12.6, no less than in 16 bits: the way to the first tile and the joins.  Tried and not kept: two tiles at once
// (122 -> 127 us, 23.5 -> 22.8), addresses of neighbouring tokens without additions (no difference).
constexpr float LAZY = 8.f;  // see the softmax
constexpr int WARPS = 8, TILE = 16, MIN_TILES = 2, CTA_SNAP = 32, WARP_SNAP = 2, FAN = 16;
// Rows of the batch whose tiles a CTA lines up in shared memory; a larger batch has CTAs enough and gives
// each (row, KV head) one.
constexpr int MAX_ITEMS = 2048;

struct E4M3 {  // a cache in 8 bits, with a scale for each 16 tokens and KV head
  uint8_t code;
};

template <class C, int D, int NQ>
struct Shape {
  static constexpr bool F8 = sizeof(C) == 1;
  static constexpr int NR = NQ * 8;
  static constexpr int LINE = D * static_cast<int>(sizeof(C));  // bytes of a key
  static constexpr int HALF = TILE * LINE, STAGE = 2 * HALF + (F8 ? 16 : 0);  // bytes of K, of K and V (and their scales)
  static constexpr int STAGES = 24 * 1024 / (2 * HALF);        // 24 KB a warp, 192 KB an SM
  static constexpr int RING = STAGES * STAGE;
  // Floats of a piece, in the order of the accumulators: NQ x D / 16 blocks of 32 lanes x 4 sums, then for each
  // NQ and lane % 4 the maxima and totals of that lane's two queries
  static constexpr int BLOCKS = NQ * (D / 16), PART = BLOCKS * 128 + NQ * 16;
  static constexpr int SMEM = WARPS * RING;
  static_assert(PART * 4 <= RING, "a warp's last piece lies in its own ring");
  static_assert(SMEM + 12 * MAX_ITEMS + 1024 <= 227 * 1024, "shared memory of a CTA");
};
// Workspace: two pieces a CTA (1: a (row, KV head) that begins there, 0: one that began earlier), one piece
// a warp (its first, where that is not its last), and three counters a CTA.
static int64_t ws_floats(int64_t grid, int part) { return grid * (2 + WARPS) * part; }
constexpr int COUNTERS = 3;

struct Item {      // a row tile of one row of the batch
  int b, r0;       // row, first query row
  int start, n;    // tokens before the call, new tokens
  int first, end;  // keys [first, end) that one of the query rows sees
  int all_from, all_to;  // keys [all_from, all_to) that all of them see
  int tiles;       // from first rounded down to 16; at least 1, so that rows without keys are written
};

// r / group with the rounded-up reciprocal of the group (exact while r group < 2^32; 0 stands for a group of 1)
NT_DEVICE int token_of(int r, uint32_t inverse) { return inverse ? static_cast<int>(__umulhi(r, inverse)) : r; }

struct Geometry {
  int items, row_tiles, group, R, capacity;
  uint32_t inverse;
  bool direct;
};

// A row's tokens before the call, and its new ones.
NT_DEVICE int2 span_of(const PagedAttnArgs& a, const Geometry& g, int id) {
  const int b = g.row_tiles == 1 ? id : id / g.row_tiles, start = a.start[b], n = a.count ? min(a.count[b], a.t) : a.t;
  return make_int2(start, start < 0 ? 0 : n);
}
template <int NR>
NT_DEVICE Item get_item(const PagedAttnArgs& a, const Geometry& g, int id, int2 span) {
  Item it;
  it.b = g.row_tiles == 1 ? id : id / g.row_tiles;
  it.r0 = (id - it.b * g.row_tiles) * NR;
  it.start = span.x;
  it.n = span.y;
  const int i0 = token_of(it.r0, g.inverse), i1 = min(token_of(min(it.r0 + NR, g.R) - 1, g.inverse), it.n - 1);
  it.first = it.end = it.all_from = it.all_to = 0;
  if (i0 <= i1) {
    it.end = static_cast<int>(min(static_cast<int64_t>(it.start) + i1 + 1, static_cast<int64_t>(g.capacity)));
    it.all_to = min(it.start + i0 + 1, it.end);
    if (a.window >= 0) {
      it.first = max(0, min(it.start + i0 - a.window, it.end));
      it.all_from = max(0, it.start + i1 - a.window);
    }
  }
  it.tiles = max(1, (it.end - (it.first & ~(TILE - 1)) + TILE - 1) / TILE);
  return it;
}

// What a line's chunk numbers are turned by, so that eight lines' equal chunks lie in different banks.
template <int LINE>
NT_DEVICE int turned(int row) { return LINE == 64 ? (row >> 1) & 3 : row & 7; }
// Two e4m3 numbers (the lower or upper half of v) as two fp16 numbers, which hold them exactly.
NT_DEVICE uint32_t widen(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}
NT_DEVICE uint32_t widen_low(uint32_t v) { return widen(static_cast<uint16_t>(v)); }
NT_DEVICE uint32_t widen_high(uint32_t v) { return widen(static_cast<uint16_t>(v >> 16)); }
NT_DEVICE float power_of_two(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
NT_DEVICE float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Weight of a piece with maximum m in a sum with maximum top (both in powers of two; -inf: no keys).
NT_DEVICE float piece_weight(float m, float top) { return top == -INFINITY ? 0.f : exp2_fast(m - top); }
// A row without keys gives zeros; a total of NaN stays NaN.
NT_DEVICE float inverse_total(float l) { return l == 0.f ? 0.f : 1.f / l; }
NT_DEVICE float weighted(float w, float x) { return w == 0.f ? 0.f : w * x; }

// Where a warp's copies stand on the line.
struct Cursor {
  int id, hk, j;       // item, KV head, tile
  Item it;
  int column, slot;    // of the tile's first key
  int seen, pages;     // lane l holds the page of column seen + l
  bool there;          // the page lies in the cache
  const void *k, *v;   // this lane's first element of the tile
  const float *ks, *vs;  // the tile's scales (8 bits)
};

NT_DEVICE void load_pages(const PagedAttnArgs& a, Cursor& c, int lane) {
  c.seen = c.column;
  const int col = c.column + lane;
  c.pages = col < a.cache.columns ? a.cache.table[static_cast<int64_t>(c.it.b) * a.cache.columns + col] : -1;
}
NT_DEVICE void prefetch_l1(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }
template <class T, int NR>
NT_DEVICE void enter(const PagedAttnArgs& a, const Geometry& g, Cursor& c, int2 span, int lane) {
  c.it = get_item<NR>(a, g, c.id, span);
  // the queries are wanted when the products get here, a ring later
  const int r = c.it.r0 + (lane & (NR - 1)), i = token_of(r, g.inverse);
  if (r < g.R && i < c.it.n) {
    const T* q = static_cast<const T*>(a.q) + c.it.b * a.qs[0] + i * a.qs[1] + (c.hk * g.group + r - i * g.group) * a.qs[2];
    prefetch_l1(q);
    if (lane >= NR && a.D > 64) prefetch_l1(q + 64);
  }
  const int key = (c.it.first & ~(TILE - 1)) + c.j * TILE;
  c.column = quotient(key, a.cache.page);
  c.slot = key - c.column * a.cache.page;
  load_pages(a, c, lane);
}
// The tile's page is the next of the list (or the item's first).
template <class C>
NT_DEVICE void turn_page(const PagedAttnArgs& a, Cursor& c, const C* kc, const C* vc, int lane) {
  if (c.column - c.seen >= 32) load_pages(a, c, lane);
  const int page = __shfl_sync(0xffffffffu, c.pages, c.column - c.seen);
  c.there = page >= 0 && page < a.cache.pages;
  if (!c.there && c.it.first < c.it.end && lane == 0) record_error(2, c.it.b);
  const int64_t p = c.there ? page : 0;
  c.k = kc + p * a.cache.page_stride_k + c.hk * a.cache.head_stride_k + c.slot * a.cache.slot_stride_k;
  c.v = vc + p * a.cache.page_stride_v + c.hk * a.cache.head_stride_v + c.slot * a.cache.slot_stride_v;
  if (sizeof(C) == 1) {
    c.ks = a.cache.k_scale + p * a.cache.k_scale_strides[0] + c.hk * a.cache.k_scale_strides[1] + (c.slot / TILE) * a.cache.k_scale_strides[2];
    c.vs = a.cache.v_scale + p * a.cache.v_scale_strides[0] + c.hk * a.cache.v_scale_strides[1] + (c.slot / TILE) * a.cache.v_scale_strides[2];
  }
}

// Joins block blk of up to 16 pieces; piece(k) is the k-th, in the order of the line.  stat gets the maxima and
// totals of the lane's two queries.
template <class C, int D, int NQ, bool L2, class Piece>
NT_DEVICE float4 join_block(int n, int blk, int lane, Piece piece, float4& stat) {
  using S = Shape<C, D, NQ>;
  auto load = [](const float* p) {
    return L2 ? __ldcg(reinterpret_cast<const float4*>(p)) : *reinterpret_cast<const float4*>(p);
  };
  const int stats = S::BLOCKS * 128 + (blk / (D / 16)) * 16 + (lane & 3) * 4, sums = blk * 128 + lane * 4;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  stat = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
#pragma unroll 1
  for (int from = 0; from < n; from += 8) {
    float4 t[8], v[8];  // eight pieces are asked for at once
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      t[k] = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
      const float* p = from + k < n ? piece(from + k) : nullptr;
      if (p) {
        t[k] = load(p + stats);
        v[k] = load(p + sums);
      }
    }
    float top0 = stat.x, top1 = stat.z;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      top0 = fmaxf(top0, t[k].x);
      top1 = fmaxf(top1, t[k].z);
    }
    const float f0 = piece_weight(stat.x, top0), f1 = piece_weight(stat.z, top1);
    stat = make_float4(top0, f0 * stat.y, top1, f1 * stat.w);
    sum.x *= f0; sum.y *= f1; sum.z *= f0; sum.w *= f1;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float w0 = piece_weight(t[k].x, top0), w1 = piece_weight(t[k].z, top1);
      // Rows without keys count for nothing, whatever their sums are.  A total of NaN has a maximum that knows nothing of
      // it, so it goes on whatever its weight is.  (Tested here and not beside the tiles, where it cost 1.7 %.)
      if (w0 != 0.f || isnan(t[k].y)) {
        stat.y = fmaf(w0, t[k].y, stat.y);
        sum.x = fmaf(w0, v[k].x, sum.x);
        sum.z = fmaf(w0, v[k].z, sum.z);
      }
      if (w1 != 0.f || isnan(t[k].w)) {
        stat.w = fmaf(w1, t[k].w, stat.w);
        sum.y = fmaf(w1, v[k].y, sum.y);
        sum.w = fmaf(w1, v[k].w, sum.w);
      }
    }
  }
  return sum;
}
template <class C, int D, int NQ>
NT_DEVICE void store_block(float* piece, int blk, int lane, const float4& sum, const float4& stat) {
  using S = Shape<C, D, NQ>;
  *reinterpret_cast<float4*>(piece + blk * 128 + lane * 4) = sum;
  if (blk % (D / 16) == 0 && lane < 4)
    *reinterpret_cast<float4*>(piece + S::BLOCKS * 128 + (blk / (D / 16)) * 16 + lane * 4) = stat;
}
// The output rows of a block of 8 queries: to the row of the query that a lane holds after the transpose.
template <class T, class C, int D>
NT_DEVICE T* output_row(const PagedAttnArgs& a, const Geometry& g, int b, int r, int hk, int lane) {
  r = min(r, g.R - 1);
  const int i = token_of(r, g.inverse);
  return static_cast<T*>(a.out) +
         ((static_cast<int64_t>(b) * a.t + i) * a.H + hk * g.group + (r - i * g.group)) * D + (lane & 3) * (sizeof(C) == 1 ? 4 : 2);
}
template <class T, class C>
NT_DEVICE void write_block(T* row, bool live, int d, const float4& sum, float w0, float w1) {
  const uint32_t u0 = transpose8x8(Num<T>::pack(weighted(w0, sum.x), weighted(w1, sum.y)));
  const uint32_t u1 = transpose8x8(Num<T>::pack(weighted(w0, sum.z), weighted(w1, sum.w)));
  if (!live) return;
  if (sizeof(C) == 1) {  // the rows of the products are the even channels of the block, then the odd ones
    *reinterpret_cast<uint2*>(row + d * 16) = make_uint2(__byte_perm(u0, u1, 0x5410), __byte_perm(u0, u1, 0x7632));
  } else {
    *reinterpret_cast<uint32_t*>(row + d * 16) = u0;
    *reinterpret_cast<uint32_t*>(row + d * 16 + 8) = u1;
  }
}

template <class T, class C, int D, int NQ>
__global__ void __launch_bounds__(WARPS * 32, 1)
    attn_kernel(const PagedAttnArgs a, const Geometry g, float* ws, unsigned* counters) {
  using S = Shape<C, D, NQ>;
  using M = std::conditional_t<S::F8, __half, T>;  // what the products multiply
  constexpr bool F8 = S::F8, TWO = !F8 || std::is_same_v<T, M>;  // probabilities as two numbers, see below
  constexpr int NR = S::NR, LINE = S::LINE, CHUNKS = LINE / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int pre[MAX_ITEMS + 1];  // tiles of a KV head before each item
  __shared__ int2 spans[MAX_ITEMS];
  __shared__ int warp_total[WARPS];
  __shared__ int part_id[2 * WARPS], part_flag[2 * WARPS];
  __shared__ bool arrived_last;
  float4* joined = reinterpret_cast<float4*>(smem);  // the rings are done with when CTAs' pieces are joined
  float4* joined_stat = joined + S::BLOCKS * 32;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int Hk = a.Hk, me = blockIdx.x;
  float* ws_warp = ws + (static_cast<int64_t>(gridDim.x) * 2 + static_cast<int64_t>(me) * WARPS) * S::PART;

  // ---- this CTA's piece of the line: each of G has `each` tiles, the first `more` one more, but a boundary that
  // falls within CTA_SNAP tiles of a (row, KV head)'s start or end goes there, and between warps within WARP_SNAP
  int G = 1, each = 0, more = 0;
  int4 begin;  // of this warp's piece: place on the line, item, KV head, tile
  int left;    // its tiles
  if (tid < 2 * WARPS) part_id[tid] = -1;
  if (g.direct) {
    const int id = me / Hk;
    const int2 span = span_of(a, g, id);
    const Item it = get_item<NR>(a, g, id, span);
    if (tid == 0) {
      spans[0] = span;
      if (it.n > 0 && static_cast<int64_t>(it.start) + it.n > g.capacity) record_error(1, it.b);
    }
    const int few = it.tiles / WARPS, rest = it.tiles % WARPS, x = warp * few + min(warp, rest);
    begin = make_int4(x, id, me - id * Hk, x);
    left = few + (warp < rest ? 1 : 0);
    __syncthreads();
  } else {
    // thread t lines up items t per .. (t + 1) per - 1
    const int per = (g.items + WARPS * 32 - 1) / (WARPS * 32), from = tid * per, to = min(from + per, g.items);
    int sum = 0;
    for (int id = from; id < to; ++id) {
      const int2 span = span_of(a, g, id);
      const Item it = get_item<NR>(a, g, id, span);
      spans[id] = span;
      pre[id] = it.tiles;
      sum += it.tiles;
      if (me == 0 && it.n > 0 && static_cast<int64_t>(it.start) + it.n > g.capacity) record_error(1, it.b);
    }
    int scan = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += v;
    }
    if (lane == 31) warp_total[warp] = scan;
    __syncthreads();
    int before = scan - sum, W = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const int v = warp_total[w];
      if (w < warp) before += v;
      W += v;
    }
    for (int id = from; id < to; ++id) {
      const int n = pre[id];
      pre[id] = before;
      before += n;
    }
    if (tid == 0) pre[g.items] = W;
    W *= Hk;
    G = max(1, min(static_cast<int>(gridDim.x), max(W / (WARPS * MIN_TILES), (g.items * Hk + WARPS - 1) / WARPS)));
    if (me >= G) return;
    each = W / G;
    more = W - each * G;
    __syncthreads();
    auto snap = [&](int x, int reach) {
      if (x >= W) return make_int4(W, g.items, 0, 0);
      int id = 0, end = g.items;  // the last item whose tiles begin at or before x
      while (end - id > 1) {
        const int mid = (id + end) >> 1;
        if (pre[mid] * Hk <= x) id = mid; else end = mid;
      }
      const int rest = x - pre[id] * Hk, n = pre[id + 1] - pre[id], hk = Hk == 1 ? 0 : quotient(rest, n), j = rest - hk * n;
      if (j <= reach && j <= n - j) return make_int4(x - j, id, hk, 0);
      if (n - j <= reach) return hk + 1 < Hk ? make_int4(x + n - j, id, hk + 1, 0) : make_int4(x + n - j, id + 1, 0, 0);
      return make_int4(x, id, hk, j);
    };
    auto shfl4 = [](int4 v, int l) {
      return make_int4(__shfl_sync(0xffffffffu, v.x, l), __shfl_sync(0xffffffffu, v.y, l), __shfl_sync(0xffffffffu, v.z, l),
                       __shfl_sync(0xffffffffu, v.w, l));
    };
    // lanes 0 and 1 find the CTA's bounds, lanes 0 to 8 then the warps'
    const int c = me + (lane & 1);
    const int4 own = snap(c * each + min(c, more), CTA_SNAP), lo = shfl4(own, 0);
    const int hi = __shfl_sync(0xffffffffu, own.x, 1);
    if (lo.x == hi) return;
    const int few = (hi - lo.x) / WARPS, rest = (hi - lo.x) % WARPS;  // fewer tiles than warps: the last have none
    int4 at = snap(lo.x + lane * few + min(lane, rest), WARP_SNAP);
    if (lane == 0 || at.x < lo.x) at = lo;
    if (lane >= WARPS || at.x > hi) at.x = hi;
    begin = shfl4(at, warp);
    left = __shfl_sync(0xffffffffu, at.x, warp + 1) - begin.x;
  }
  auto span_at = [&](int id) { return spans[g.direct ? 0 : id]; };
  int fetch_left = left;

  if (left > 0) {
    Cursor f;
    f.id = begin.y;
    f.hk = begin.z;
    f.j = begin.w;
    enter<T, NR>(a, g, f, span_at(f.id), lane);
    Cursor c = f;  // where the products stand (its page fields are unused)

    uint8_t* ring = smem + warp * S::RING;
    const uint32_t ring_u = smem_u32(ring);
    const int lrow = lane / CHUNKS, lch = lane % CHUNKS;
    constexpr int ROWS = 32 / CHUNKS;       // rows of one copy instruction of the warp
    constexpr int PERIOD = 8 / ROWS;        // copies after which the swizzle repeats
    uint32_t to[PERIOD];
#pragma unroll
    for (int e = 0; e < PERIOD; ++e) to[e] = (e * ROWS + lrow) * LINE + ((lch ^ turned<LINE>(e * ROWS + lrow)) << 4);
    const C* kc = static_cast<const C*>(a.cache.k) + lrow * a.cache.slot_stride_k + lch * (16 / sizeof(C));
    const C* vc = static_cast<const C*>(a.cache.v) + lrow * a.cache.slot_stride_v + lch * (16 / sizeof(C));
    const int64_t kstep = ROWS * a.cache.slot_stride_k, vstep = ROWS * a.cache.slot_stride_v;

    bool turn = true;
    unsigned gone = 0;  // bit of a stage: its tile's page is not in the cache (0.8 % over a set of calls)
    auto fetch = [&](int stage) {
      if (fetch_left > 0) {
        if (turn) turn_page<C>(a, f, kc, vc, lane);
        gone = (gone & ~(1u << stage)) | (f.there ? 0u : 1u << stage);
        const int key = (f.it.first & ~(TILE - 1)) + f.j * TILE;
        const C *ks = static_cast<const C*>(f.k), *vs = static_cast<const C*>(f.v);
        const uint32_t dst = ring_u + stage * S::STAGE;
        if (f.there && key >= f.it.first && key + TILE <= f.it.end) {
#pragma unroll
          for (int e = 0; e < TILE / ROWS; ++e) {
            const uint32_t at = dst + to[e % PERIOD] + (e / PERIOD) * (8 * LINE);
            cp_async16(at, ks);
            cp_async16(at + S::HALF, vs);
            ks += kstep;
            vs += vstep;
          }
        } else {
          // keys outside [first, end) and without a page become zeros: whatever their memory holds never meets a product
#pragma unroll 1
          for (int e = 0; e < TILE / ROWS; ++e) {
            const int row = e * ROWS + lrow;
            const bool valid = f.there && key + row >= f.it.first && key + row < f.it.end;
            const uint32_t at = dst + row * LINE + ((lch ^ turned<LINE>(row)) << 4);
            cp_async16_or_zero(at, valid ? ks : kc, valid);
            cp_async16_or_zero(at + S::HALF, valid ? vs : vc, valid);
            ks += kstep;
            vs += vstep;
          }
        }
        if (F8 && lane < 2) cp_async4_or_zero(dst + 2 * S::HALF + lane * 4, lane ? f.vs : f.ks, f.there);
        --fetch_left;
        turn = false;
        if (++f.j == f.it.tiles) {
          f.j = 0;
          if (++f.hk == Hk) {
            f.hk = 0;
            ++f.id;
          }
          turn = true;
          if (fetch_left > 0) enter<T, NR>(a, g, f, span_at(f.id), lane);
        } else if ((f.slot += TILE) == a.cache.page) {
          f.slot = 0;
          ++f.column;
          turn = true;
        } else {
          f.k = static_cast<const C*>(f.k) + TILE * a.cache.slot_stride_k;
          f.v = static_cast<const C*>(f.v) + TILE * a.cache.slot_stride_v;
          if (F8) {
            f.ks += a.cache.k_scale_strides[2];
            f.vs += a.cache.v_scale_strides[2];
          }
        }
      }
      cp_commit();
    };

#pragma unroll 1
    for (int s = 0; s < S::STAGES - 1; ++s) fetch(s);
    int stage = 0;
    const float scale2 = a.scale * 1.4426950408889634f;
    const int qc = lane & 3, qr = lane >> 2;
    uint32_t kat[4], vat[4];  // this lane's matrix rows in a stage, for channel blocks 0 to 3
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int krow = lane & 15, vrow = (lane & 7) + ((lane >> 4) << 3);
      // 8 bits: both products take a line's 16-byte chunks in pairs, keys 0 to 7 before keys 8 to 15
      kat[e] = krow * LINE + (((e * 2 + (lane >> 4)) ^ turned<LINE>(krow)) << 4);
      vat[e] = F8 ? S::HALF + kat[e] : S::HALF + vrow * LINE + (((e * 2 + ((lane >> 3) & 1)) ^ turned<LINE>(vrow)) << 4);
    }

    while (left > 0) {
      // ---- one piece: tiles [c.j, c.j + n) of (c.id, c.hk)
      const int n = min(left, c.it.tiles - c.j), j0 = c.j;
      uint32_t qf[NQ][D / 16][2];
      float to_log[NQ][2];            // 8 bits: the factor of this lane's two queries' products
      float v_unit = 0.f, v_less = 0.f, v_most = 0.f;  // 8 bits: what sums are in units of, its inverse, and the largest it was
      int last[NQ][2], oldest[NQ][2];  // newest and oldest key that this lane's two queries see
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
        const int r = c.it.r0 + nq * 8 + qr, i = token_of(r, g.inverse);
        const bool live = r < g.R && i < c.it.n;
        const T* qp = static_cast<const T*>(a.q) + c.it.b * a.qs[0] + (live ? i : 0) * a.qs[1] +
                      (c.hk * g.group + (live ? r - i * g.group : 0)) * a.qs[2] + qc * (F8 ? 4 : 2);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          if (F8) {  // a lane's four neighbouring channels, as it finds them in a key's line
            const uint2 u = live ? *reinterpret_cast<const uint2*>(qp + kk * 16) : make_uint2(0u, 0u);
            qf[nq][kk][0] = u.x;
            qf[nq][kk][1] = u.y;
          } else {
            qf[nq][kk][0] = live ? *reinterpret_cast<const uint32_t*>(qp + kk * 16) : 0u;
            qf[nq][kk][1] = live ? *reinterpret_cast<const uint32_t*>(qp + kk * 16 + 8) : 0u;
          }
        }
        float own = scale2;  // what takes this lane's query row's products to powers of two
        if (F8 && !std::is_same_v<T, M>) {
          // bf16 queries become fp16: a power of two a row brings their largest to [2^12, 2^13), so that nothing is lost but
          // what lies 2^-37 below it
          float top = 0.f;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float2 x = Num<T>::unpack(qf[nq][kk][e]);
              top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
            }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // an infinite element stays one, and the finite beside it become small
          const int by = min(100, 139 - static_cast<int>(__float_as_uint(top) >> 23));
          const float f = power_of_two(by);
          own = scale2 * power_of_two(-by);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float2 x = Num<T>::unpack(qf[nq][kk][e]);
              qf[nq][kk][e] = Num<M>::pack(x.x * f, x.y * f);
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (F8) to_log[nq][e] = __shfl_sync(0xffffffffu, own, (qc * 2 + e) * 4);
          const int rc = c.it.r0 + nq * 8 + qc * 2 + e, ic = token_of(rc, g.inverse);
          const bool lc = rc < g.R && ic < c.it.n;
          last[nq][e] = lc ? min(c.it.start + ic, c.it.end - 1) : -1;
          oldest[nq][e] = lc && a.window >= 0 ? c.it.start + ic - a.window : 0;
        }
      }
      float o[NQ][D / 16][4], m[NQ][2], l[NQ][2];
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          m[nq][e] = -INFINITY;
          l[nq][e] = 0.f;
        }
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nq][d][e] = 0.f;
      }

      for (int tile = 0; tile < n; ++tile) {
        cp_wait<S::STAGES - 2>();
        __syncwarp();  // this stage has landed for every lane, and the stage before it is read by none
        int ahead = stage + S::STAGES - 1;
        if (ahead >= S::STAGES) ahead -= S::STAGES;
        const uint32_t base = ring_u + stage * S::STAGE;
        const bool lost = (gone >> stage) & 1u;
        if (++stage == S::STAGES) stage = 0;

        float s[NQ][4], s2[NQ][4];  // two chains of products
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nq][e] = s2[nq][e] = 0.f;
        float2 scales = make_float2(1.f, 1.f);
        if constexpr (F8) {
          scales = *reinterpret_cast<const float2*>(smem + (base - smem_u32(smem)) + 2 * S::HALF);
#pragma unroll
          for (int kk = 0; kk < D / 16; kk += 2) {
            uint32_t c4[4];  // chunk kk of keys 0 to 7, of keys 8 to 15, then chunk kk + 1
            ldsm4(c4, base + kat[kk >> 1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t kf[4] = {widen_low(c4[2 * e]), widen_low(c4[2 * e + 1]), widen_high(c4[2 * e]), widen_high(c4[2 * e + 1])};
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq) Num<M>::mma(e ? s2[nq] : s[nq], kf, qf[nq][kk + e][0], qf[nq][kk + e][1]);
            }
          }
        } else {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t kf[4];
            ldsm4(kf, base + kat[kk & 3] + (kk >> 2) * 128);
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) Num<M>::mma(kk & 1 ? s2[nq] : s[nq], kf, qf[nq][kk][0], qf[nq][kk][1]);
          }
        }
        fetch(ahead);  // issued while the products finish
        // a tile without a page lies behind every query
        const int key0 = lost ? INT32_MAX - 2 * TILE : (c.it.first & ~(TILE - 1)) + (j0 + tile) * TILE, key = key0 + qr;
        const bool edge = key0 < c.it.all_from || key0 + TILE > c.it.all_to;
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nq][e] = (s[nq][e] + s2[nq][e]) * (F8 ? to_log[nq][e & 1] * scales.x : scale2);
          if (edge) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (key > last[nq][e] || key < oldest[nq][e]) s[nq][e] = -INFINITY;
              if (key + 8 > last[nq][e] || key + 8 < oldest[nq][e]) s[nq][e + 2] = -INFINITY;
            }
          }
        }
        // The reference m follows the maximum only when a score passes it by more than 2^LAZY, so that most tiles
        // need neither a reduction over the lanes nor a rescaling; probabilities stay below 2^(RAISE + LAZY), inside the
        // types' limits, and sums and pieces are relative to m all the same.
        constexpr float RAISE = RAISE_OF<M>;
        bool passed = false;
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
          for (int e = 0; e < 4; ++e) passed |= s[nq][e] > m[nq][e & 1] + (RAISE + LAZY);
        if (__any_sync(0xffffffffu, passed)) {
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq) {
            float top[2] = {fmaxf(s[nq][0], s[nq][2]), fmaxf(s[nq][1], s[nq][3])};
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
              top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], d));
              top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], d));
            }
            float f[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              top[e] = fmaxf(m[nq][e], top[e] - RAISE);
              f[e] = piece_weight(m[nq][e], top[e]);
              m[nq][e] = top[e];
              l[nq][e] *= f[e];
            }
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              o[nq][d][0] *= f[0]; o[nq][d][1] *= f[1];
              o[nq][d][2] *= f[0]; o[nq][d][3] *= f[1];
            }
          }
        }
        // A probability is the sum of two numbers of the cache's type: 16 bits for bf16, 22 for fp16.  The error against 64
        // bits stays that of the output's rounding (1.66e-3 of the norm for 1 x 1001 bf16 keys, as with fp32 probabilities;
        // three bf16 numbers, which hold all 24 bits, change results by 1e-4 of the norm and cost 2.3 % over a set of
        // calls).  fp16 ends at 2^-24, where the second number of a probability below 2^-14 is lost, so its reference m lies
        // RAISE below the maximum that it follows: probabilities reach 2^(RAISE + LAZY) = 2^15, the type's top, in products and
        // totals alike, and what is then lost is 2^-32 of the largest a key.
        // 8 bits: one fp16 number (11 bits) is enough where the output has bf16's 8; fp16 queries keep both.
        uint32_t pf[NQ][2], pl[NQ][2];
        // Values' scales go into the probabilities relative to a unit, the power of two at or above the scale of a tile.  It stays while
        // scales are no larger, and no smaller than 2^-7 of it: a probability is held in full down to 2^-14 of the largest then, and what is lost below
        // is 2^-25 of the tile's own values.  Else it follows the tile (a block of values 2^20 times the others', which these queries may not
        // even see, would leave nothing of theirs), down to 2^-64 of the largest, so that sums stay in range.
        if (F8 && (scales.y > v_unit || scales.y * 128.f < v_unit) && scales.y > 0.f) {  // (the same for the whole warp)
          const float up = __uint_as_float(min((__float_as_uint(scales.y) + 0x7fffffu) & 0xff800000u, 0x7f000000u));
          v_most = fmaxf(v_most, up);
          const float unit = fmaxf(up, v_most * 0x1p-64f), f = v_unit / unit;  // (a power of two, so that nothing is rounded)
          v_unit = unit;
          v_less = 1.f / unit;
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nq][d][e] *= f;
        }
        const float weight = scales.y * v_less;
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
          const float r0 = m[nq][0] == -INFINITY ? 0.f : m[nq][0], r1 = m[nq][1] == -INFINITY ? 0.f : m[nq][1];
          s[nq][0] = exp2_fast(s[nq][0] - r0); s[nq][1] = exp2_fast(s[nq][1] - r1);
          s[nq][2] = exp2_fast(s[nq][2] - r0); s[nq][3] = exp2_fast(s[nq][3] - r1);
          l[nq][0] += s[nq][0] + s[nq][2];
          l[nq][1] += s[nq][1] + s[nq][3];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (F8) {
              s[nq][2 * e] *= weight;
              s[nq][2 * e + 1] *= weight;
            }
            const uint32_t high = Num<M>::pack(s[nq][2 * e], s[nq][2 * e + 1]);
            pf[nq][e] = transpose8x8(high);
            if constexpr (TWO) {
              const float2 h = Num<M>::unpack(high);
              pl[nq][e] = transpose8x8(Num<M>::pack(s[nq][2 * e] - h.x, s[nq][2 * e + 1] - h.y));
            }
          }
        }
        if constexpr (F8) {
#pragma unroll
          for (int d = 0; d < D / 16; d += 2) {
            uint32_t c4[4];  // a lane has two channels of two keys; chunk d of keys 0 to 7, of keys 8 to 15, then chunk d + 1
            ldsm4t(c4, base + vat[d >> 1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t x = __byte_perm(c4[2 * e], 0u, 0x3120), y = __byte_perm(c4[2 * e + 1], 0u, 0x3120);
              const uint32_t vf[4] = {widen_low(x), widen_high(x), widen_low(y), widen_high(y)};
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq) Num<M>::mma(o[nq][d + e], vf, pf[nq][0], pf[nq][1]);
              if constexpr (TWO)
#pragma unroll
                for (int nq = 0; nq < NQ; ++nq) Num<M>::mma(o[nq][d + e], vf, pl[nq][0], pl[nq][1]);
            }
          }
        } else {
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            uint32_t vf[4];
            ldsm4t(vf, base + vat[d & 3] + (d >> 2) * 128);
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) Num<M>::mma(o[nq][d], vf, pf[nq][0], pf[nq][1]);
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) Num<M>::mma(o[nq][d], vf, pl[nq][0], pl[nq][1]);
          }
        }
      }
      if (F8)
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nq][d][e] *= v_unit;

      // ---- the piece's end; rows that are no tokens have no keys
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[nq][e] += __shfl_xor_sync(0xffffffffu, l[nq][e], d);
          if (last[nq][e] < 0) {
            l[nq][e] = 0.f;
            m[nq][e] = -INFINITY;
          }
        }
      const bool begins = j0 == 0, ends = j0 + n == c.it.tiles;
      left -= n;
      if (begins && ends) {
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
          const int r = c.it.r0 + nq * 8 + qr;
          T* row = output_row<T, C, D>(a, g, c.it.b, r, c.hk, lane);
          const float w0 = inverse_total(l[nq][0]), w1 = inverse_total(l[nq][1]);
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
            write_block<T, C>(row, r < g.R, d, make_float4(o[nq][d][0], o[nq][d][1], o[nq][d][2], o[nq][d][3]), w0, w1);
        }
      } else {
        const bool final_piece = left == 0;
        float* part = final_piece ? reinterpret_cast<float*>(ring) : ws_warp + warp * S::PART;
        if (final_piece) {
          cp_wait<0>();
          __syncwarp();
        }
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
            store_block<C, D, NQ>(part, nq * (D / 16) + d, lane, make_float4(o[nq][d][0], o[nq][d][1], o[nq][d][2], o[nq][d][3]),
                               make_float4(m[nq][0], l[nq][0], m[nq][1], l[nq][1]));
        if (lane == 0) {
          const int slot = 2 * warp + (final_piece ? 1 : 0);
          part_id[slot] = c.id * Hk + c.hk;
          part_flag[slot] = (begins ? 1 : 0) | (ends ? 2 : 0);
        }
      }
      c.j += n;
      if (c.j == c.it.tiles) {
        c.j = 0;
        if (++c.hk == Hk) {
          c.hk = 0;
          ++c.id;
          if (left > 0) c.it = get_item<NR>(a, g, c.id, span_at(c.id));
        }
      }
    }
    cp_wait<0>();
  }
  __syncthreads();

  // ---- join the CTA's pieces, a warp a block of 8 queries and 16 channels at a time
  int open_id[2] = {-1, -1};  // what this CTA leaves open: 0 began in an earlier one, 1 begins here
  {
    // Slot 2 w is warp w's first piece where that is not its last, which is in slot 2 w + 1.  Places on the line
    // only grow, so a piece that does not follow one of the same (row, KV head) leads.
    const int part = lane & 15, id = part_id[part], flag = part_flag[part];
    int before = part ? part_id[part - 1] : -1;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, before, o, 16);
      if (part >= o) before = max(before, v);
    }
    const unsigned valid = __ballot_sync(0xffffffffu, id >= 0) & 0xffffu;
    unsigned leaders = __ballot_sync(0xffffffffu, id >= 0 && before < id) & 0xffffu;
    int blk = warp;
    while (leaders) {
      const int leader = __ffs(leaders) - 1;
      leaders &= leaders - 1;
      const unsigned mask = valid & ~((1u << leader) - 1u) & (leaders ? (1u << (__ffs(leaders) - 1)) - 1u : 0xffffu);
      const int end = 31 - __clz(mask), gid = __shfl_sync(0xffffffffu, id, leader);
      const bool begins = __shfl_sync(0xffffffffu, flag, leader) & 1, ends = __shfl_sync(0xffffffffu, flag, end) & 2;
      if (!(begins && ends)) open_id[begins ? 1 : 0] = gid;
      // warps leader / 2 to end / 2 have at most one piece each
      const int w0 = leader >> 1, n = (end >> 1) - w0 + 1;
      for (; blk < S::BLOCKS; blk += WARPS) {
        float4 stat;
        const float4 sum = join_block<C, D, NQ, false>(n, blk, lane, [&](int k) {
          const int w = w0 + k;
          if (!((mask >> (2 * w)) & 3u)) return static_cast<const float*>(nullptr);  // it has no tiles
          return (mask >> (2 * w)) & 1u ? static_cast<const float*>(ws_warp + w * S::PART) : reinterpret_cast<const float*>(smem + w * S::RING);
        }, stat);
        if (!(begins && ends)) {
          store_block<C, D, NQ>(ws + (static_cast<int64_t>(me) * 2 + (begins ? 1 : 0)) * S::PART, blk, lane, sum, stat);
        } else {
          const int item = quotient(gid, Hk), b = g.row_tiles == 1 ? item : item / g.row_tiles;
          const int r = (item - b * g.row_tiles) * NR + (blk / (D / 16)) * 8 + (lane >> 2);
          write_block<T, C>(output_row<T, C, D>(a, g, b, r, gid - item * Hk, lane), r < g.R, blk % (D / 16), sum, inverse_total(stat.y),
                         inverse_total(stat.w));
        }
      }
      blk -= S::BLOCKS;
    }
  }
  if (g.direct || (open_id[0] < 0 && open_id[1] < 0)) return;

  // ---- and what several CTAs hold: the last of up to 16 neighbours joins their pieces, the last of these the rest.
  // The pieces were written by the whole CTA: the barrier orders them before the arriving thread's release, and its
  // acquire before what the CTA reads behind the second barrier (past L1, which nothing invalidates).
  auto arrive = [&](unsigned* counter, int n) {  // n arrivals bring the counter back to 0
    unsigned before;
    asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;" : "=r"(before) : "l"(counter), "r"(n - 1) : "memory");
    return before == static_cast<unsigned>(n - 1);
  };
  auto cta_of = [&](int x) { return x < more * (each + 1) ? quotient(x, each + 1) : more + quotient(x - more * (each + 1), each); };
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    const int gid = open_id[side];
    if (gid < 0) continue;
    const int item = quotient(gid, Hk), hk = gid - item * Hk, tiles = pre[item + 1] - pre[item], x = pre[item] * Hk + hk * tiles;
    // boundaries within CTA_SNAP tiles of its ends went there
    const int c0 = cta_of(x + CTA_SNAP), c1 = cta_of(x + tiles - 1 - CTA_SNAP), lead = c0 + ((me - c0) & ~(FAN - 1)), groups = (c1 - c0) / FAN + 1;
    const int b = g.row_tiles == 1 ? item : item / g.row_tiles, r0 = (item - b * g.row_tiles) * NR;
    auto at = [&](int c) { return ws + (static_cast<int64_t>(c) * 2 + (c == c0 ? 1 : 0)) * S::PART; };
    int first = lead, step = 1, n = min(FAN, c1 - lead + 1);
    unsigned* counter = counters + lead * COUNTERS + (lead == c0 ? 1 : 0);
#pragma unroll 1
    for (int level = 0;; ++level) {
      __syncthreads();
      if (tid == 0) arrived_last = arrive(counter, n);
      __syncthreads();
      if (!arrived_last) break;
      const bool done = level == 1 || groups == 1;
      for (int blk = warp; blk < S::BLOCKS; blk += WARPS) {
        float4 stat;
        const float4 sum = join_block<C, D, NQ, true>(n, blk, lane, [&](int k) { return static_cast<const float*>(at(first + k * step)); }, stat);
        if (!done) {
          // into the leader's piece: its sums are read by this warp alone, its maxima and totals by all
          joined[blk * 32 + lane] = sum;
          if (blk % (D / 16) == 0 && lane < 4) joined_stat[(blk / (D / 16)) * 4 + lane] = stat;
        } else {
          const int r = r0 + (blk / (D / 16)) * 8 + (lane >> 2);
          write_block<T, C>(output_row<T, C, D>(a, g, b, r, hk, lane), r < g.R, blk % (D / 16), sum, inverse_total(stat.y), inverse_total(stat.w));
        }
      }
      if (done) break;
      __syncthreads();
      for (int blk = warp; blk < S::BLOCKS; blk += WARPS)
        store_block<C, D, NQ>(at(lead), blk, lane, joined[blk * 32 + lane], joined_stat[(blk / (D / 16)) * 4 + (lane & 3)]);
      first = c0;
      step = FAN;
      n = groups;
      counter = counters + c0 * COUNTERS + 2;
    }
  }
}

// ----------------------------------------------------------------------------- append, 8 bits
// x is held as the e4m3 number next to x / S, S a power of two for each block of 16 tokens of a row (by position) and KV
// head: the smallest whose 448-fold reaches the block's largest |x|.  A power of two moves no digits, so a block that
// gets a larger token is written again with a larger S at the loss of nothing but what falls under the smallest step.
// S never falls while a block is filled; a call that begins a block chooses it anew.  What is not finite becomes NaN
// and does not count for S.
//
// A block of one KV head, its keys or its values, is written by one group of lanes or warps, so that nobody else writes
// its scale: all of its new tokens are in registers before the scale is known, and are read once.  8 prompts of up to 2048 tokens, 10 + 5
// heads of 128: 31.1 us for 104 MB (16.1 at the copy rate): 80 registers a thread leave 24 warps an SM, which wait for their tokens longest
// (long scoreboard 2.3 cycles an issue, 0.54 of the slots used).  One token of a row by the same blocks took 5.2 us, and 11.7 for 192 rows; by groups of lanes they take 2.9 and 3.4.
NT_DEVICE uint32_t to_e4m3(const float (&x)[4]) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x[1]), "f"(x[0]));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x[3]), "f"(x[2]));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}
// The smallest power of two, 2^-100 to 2^120, whose 448-fold (1.75 2^8) reaches top >= 0.
NT_DEVICE float block_scale(float top) {
  const uint32_t u = __float_as_uint(top);
  const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return power_of_two(max(-100, min(120, e)));
}
// Where a block of a row and KV head lies: its codes and its scale.
struct BlockAt {
  uint8_t* codes;   // null: nowhere
  int64_t step;     // from token to token
  float* scale;
};
NT_DEVICE BlockAt find_block(const PagedAppendArgs& a, int b, int position, int hk, bool values, bool tells) {
  const PagedCacheArgs& m = a.cache;
  const int column = quotient(position, m.page), slot = position - column * m.page;
  int fault = 1;
  if (column < m.columns) {
    const int page = m.table[static_cast<int64_t>(b) * m.columns + column];
    fault = 2;
    if (page >= 0 && page < m.pages) {
      if (values)
        return {static_cast<uint8_t*>(m.v) + page * m.page_stride_v + hk * m.head_stride_v + slot * m.slot_stride_v, m.slot_stride_v,
                m.v_scale + page * m.v_scale_strides[0] + hk * m.v_scale_strides[1] + (slot / TILE) * m.v_scale_strides[2]};
      return {static_cast<uint8_t*>(m.k) + page * m.page_stride_k + hk * m.head_stride_k + slot * m.slot_stride_k, m.slot_stride_k,
              m.k_scale + page * m.k_scale_strides[0] + hk * m.k_scale_strides[1] + (slot / TILE) * m.k_scale_strides[2]};
    }
  }
  if (tells) record_error(fault, b);
  return {nullptr, 0, nullptr};
}
// D / 16 lanes hold a head of a token, lane j channels 8 j to 8 j + 7 of each half, so that it has both members of its
// rotated pairs.
enum Kind { QUERY, KEY, VALUE };
struct Raw {
  uint4 lo, hi;    // the head's halves
  uint4 lo2, hi2;  // cosines and sines; of a value the halves of its embedding
};
template <class T>
NT_DEVICE void load16(const T* p, int half, uint4& lo, uint4& hi) {
  lo = __ldcs(reinterpret_cast<const uint4*>(p));
  hi = __ldcs(reinterpret_cast<const uint4*>(p + half));
}
template <class T>
NT_DEVICE void load_angles(const PagedAppendArgs& a, int position, int half, int mine, Raw& r) {
  const int64_t at = static_cast<int64_t>(position) * half + mine * 8;
  r.lo2 = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.cos) + at);
  r.hi2 = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.sin) + at);
}
template <class T>
NT_DEVICE void unpack8(const uint4& u, float2 (&x)[4]) {
  x[0] = Num<T>::unpack(u.x);
  x[1] = Num<T>::unpack(u.y);
  x[2] = Num<T>::unpack(u.z);
  x[3] = Num<T>::unpack(u.w);
}
// Both halves of what becomes of a head; zeros stay zeros.  Whole warps call it for queries and keys.
template <class T, int D>
NT_DEVICE void turn_raw(const PagedAppendArgs& a, const Raw& r, float2 (&x)[8]) {
  float2 y[4], z[4], c[4], s[4];
  unpack8<T>(r.lo, y);
  unpack8<T>(r.hi, z);
  unpack8<T>(r.lo2, c);
  unpack8<T>(r.hi2, s);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x[k] = fma2(z[k], s[k], mul2(y[k], c[k]));
    x[k + 4] = fma2(y[k], make_float2(-s[k].x, -s[k].y), mul2(z[k], c[k]));
  }
  if (!a.norm) return;
  float2 pair = mul2(x[0], x[0]);
#pragma unroll
  for (int k = 1; k < 8; ++k) pair = fma2(x[k], x[k], pair);
  float sum = pair.x + pair.y;
#pragma unroll
  for (int o = D / 32; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float f = a.scale * rsqrtf(sum * (1.f / D) + EPS);
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = mul2(x[k], make_float2(f, f));
}
// gate: 3 sigmoid of it is the embedding's share
NT_DEVICE float share_of(float gate) { return __fdividef(3.f, 1.f + expf(-gate)); }
template <class T>
NT_DEVICE void mix_raw(const Raw& r, bool embedded, float share, float2 (&x)[8]) {
  float2 u[4], w[4], y[4], z[4];
  unpack8<T>(r.lo, u);
  unpack8<T>(r.hi, w);
  unpack8<T>(r.lo2, y);
  unpack8<T>(r.hi2, z);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x[k] = embedded ? fma2(make_float2(share, share), y[k], u[k]) : u[k];
    x[k + 4] = embedded ? fma2(make_float2(share, share), z[k], w[k]) : w[k];
  }
}
// The largest finite |x|; the others become NaN.
template <int N>
NT_DEVICE float finite_top(float2 (&x)[N][8]) {
  constexpr uint32_t INF = 0x7f800000u;
  uint32_t top = 0;  // magnitudes are ordered as their bits are
  auto bits = [](float v) { return __float_as_uint(v) & 0x7fffffffu; };
#pragma unroll
  for (int e = 0; e < N; ++e)
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, max(bits(x[e][k].x), bits(x[e][k].y)));
  if (top >= INF) {
    top = 0;
    auto mend = [&](float& v) {
      if (bits(v) < INF) top = max(top, bits(v));
      else v = NAN;
    };
#pragma unroll
    for (int e = 0; e < N; ++e)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        mend(x[e][k].x);
        mend(x[e][k].y);
      }
  }
  return __uint_as_float(top);
}
NT_DEVICE void write_codes(uint8_t* at, int half, const float2 (&x)[8], float by) {
  uint32_t u[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 y = mul2(x[2 * k], make_float2(by, by)), z = mul2(x[2 * k + 1], make_float2(by, by));
    const float four[4] = {y.x, y.y, z.x, z.y};
    u[k] = to_e4m3(four);
  }
  *reinterpret_cast<uint2*>(at) = make_uint2(u[0], u[1]);
  *reinterpret_cast<uint2*>(at + half) = make_uint2(u[2], u[3]);
}
NT_DEVICE void rescale_codes(uint8_t* at, int half, float by) {
  const uint2 lo = *reinterpret_cast<const uint2*>(at), hi = *reinterpret_cast<const uint2*>(at + half);
  const uint32_t u[4] = {lo.x, lo.y, hi.x, hi.y};
  float2 x[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x[2 * k] = Num<__half>::unpack(widen_low(u[k]));
    x[2 * k + 1] = Num<__half>::unpack(widen_high(u[k]));
  }
  write_codes(at, half, x, by);
}
template <class T, int D>
NT_DEVICE void store_query(const PagedAppendArgs& a, int tok, int head, int mine, const float2 (&x)[8]) {
  T* dst = static_cast<T*>(a.q_out) + (static_cast<int64_t>(tok) * a.H + head) * D + mine * 8;
  uint32_t u[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) u[k] = Num<T>::pack(x[k].x, x[k].y);
  *reinterpret_cast<uint4*>(dst) = make_uint4(u[0], u[1], u[2], u[3]);
  *reinterpret_cast<uint4*>(dst + D / 2) = make_uint4(u[4], u[5], u[6], u[7]);
}

// One token a row: D / 16 lanes a head, of the queries, keys and values in turn.
template <class T, int D>
__global__ void __launch_bounds__(256) append8_one_kernel(const PagedAppendArgs a) {
  constexpr int L = D / 16, HALF = D / 2;
  const int mine = threadIdx.x % L, at = blockIdx.x * (256 / L) + threadIdx.x / L, heads = a.H + 2 * a.Hk;
  const bool live = at < a.B * heads;  // whole warps stay for the shuffles
  const int b = live ? quotient(at, heads) : 0, h = live ? at - b * heads : 0;
  const Kind kind = h < a.H ? QUERY : h < a.H + a.Hk ? KEY : VALUE;
  const int head = h - (kind == QUERY ? 0 : kind == KEY ? a.H : a.H + a.Hk);
  const int start = a.start[b];
  bool real = live && start >= 0 && (!a.count || a.count[b] > 0);
  if (real && start >= a.rope_rows) {
    if (mine == 0) record_error(3, b);
    real = false;
  }
  Raw r = {};
  BlockAt block = {};
  float old = 0.f, gate = 0.f;
  const int before = start & (TILE - 1);
  if (real) {
    const T* src = kind == QUERY ? static_cast<const T*>(a.q) + b * a.qs[0] + head * a.qs[2]
                 : kind == KEY ? static_cast<const T*>(a.kin) + b * a.ks[0] + head * a.ks[2]
                               : static_cast<const T*>(a.vin) + b * a.vs[0] + head * a.vs[2];
    load16(src + mine * 8, HALF, r.lo, r.hi);
    if (kind != VALUE) {
      load_angles<T>(a, start, HALF, mine, r);
    } else if (a.ve) {
      load16(static_cast<const T*>(a.ve) + b * a.es[0] + head * a.es[2] + mine * 8, HALF, r.lo2, r.hi2);
      gate = Num<T>::one(static_cast<const T*>(a.ve_gate)[b * a.gs[0] + head * a.gs[2]]);
    }
    if (kind != QUERY) {
      block = find_block(a, b, start - before, head, kind == VALUE, mine == 0);
      if (block.codes && before) old = *block.scale;
    }
  }
  float2 x[1][8];
  turn_raw<T, D>(a, r, x[0]);  // lanes of a warp differ in their kind: all pass the shuffles
  if (kind == VALUE) mix_raw<T>(r, a.ve, share_of(gate), x[0]);
  float top = 0.f;
  if (kind != QUERY) top = finite_top(x);
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (kind == QUERY) {
    if (live) store_query<T, D>(a, b, head, mine, x[0]);  // what is no token has zeros in, and gives zeros
    return;
  }
  if (!block.codes) return;
  const float scale = fmaxf(old, block_scale(top)), by = 1.f / scale;
  if (before && scale != old)
#pragma unroll 1
    for (int e = 0; e < before; ++e) rescale_codes(block.codes + e * block.step + mine * 8, HALF, old * by);
  write_codes(block.codes + before * block.step + mine * 8, HALF, x[0], by);
  if (mine == 0) *block.scale = scale;
}

// More tokens: WIDE warps a block of a KV head's keys or values, so that a thread holds STEPS tokens' 16 channels; the CTAs
// behind these turn the queries, PER heads of a token a group of lanes.
template <class T, int D, int PER, int STEPS>
__global__ void __launch_bounds__(256) append8_kernel(const PagedAppendArgs a, const int blocks, const int writing) {
  constexpr int L = D / 16, HALF = D / 2, ABREAST = 32 / L, WIDE = TILE / (ABREAST * STEPS);
  __shared__ float tops[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = lane % L;

  if (static_cast<int>(blockIdx.x) >= writing) {
    const int groups = (a.H + PER - 1) / PER, at = (blockIdx.x - writing) * (256 / L) + threadIdx.x / L;
    const int tok = PER >= a.H ? at : quotient(at, groups), h0 = (at - tok * groups) * PER;
    const bool live = tok < a.B * a.t;
    const int b = live ? quotient(tok, a.t) : 0, i = live ? tok - b * a.t : 0;
    const int start = a.start[b], n = a.count ? a.count[b] : a.t;
    const bool real = live && i < n && start >= 0 && start < a.rope_rows - i;
    uint4 lo[PER], hi[PER];
    Raw r = {};
    const T* src = static_cast<const T*>(a.q) + b * a.qs[0] + i * a.qs[1] + h0 * a.qs[2] + mine * 8;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      lo[e] = hi[e] = make_uint4(0, 0, 0, 0);
      if (real && h0 + e < a.H) load16(src, HALF, lo[e], hi[e]);
      src += a.qs[2];
    }
    if (real) load_angles<T>(a, start + i, HALF, mine, r);
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      float2 x[8];
      r.lo = lo[e];
      r.hi = hi[e];
      turn_raw<T, D>(a, r, x);
      if (live && h0 + e < a.H) store_query<T, D>(a, tok, h0 + e, mine, x);
    }
    return;
  }

  // ---- a block; its warps go on or return together
  const int item = blockIdx.x * (8 / WIDE) + warp / WIDE, part = warp % WIDE;
  const bool values = item & 1;
  const int line = quotient(item >> 1, a.Hk), hk = (item >> 1) - line * a.Hk, b = quotient(line, blocks), j = line - b * blocks;
  if (b >= a.B) return;
  const int start = a.start[b];
  int n = a.count ? min(a.count[b], a.t) : a.t;
  const bool tells = lane == 0 && part == 0;
  if (start < 0 || n <= 0) return;
  if (start > a.rope_rows - n) {
    if (tells) record_error(3, b);
    n = a.rope_rows - start;
    if (n <= 0) return;
  }
  const int64_t first = (start & ~(TILE - 1)) + static_cast<int64_t>(j) * TILE;
  if (first >= start + n) return;
  const int p0 = static_cast<int>(first);
  const int slot0 = part * (ABREAST * STEPS) + lane / L, i0 = p0 + slot0 - start;  // this lane's first slot, as a token of the call
  Raw r[STEPS];
  float gate[STEPS] = {};
  const T* src = (values ? static_cast<const T*>(a.vin) + b * a.vs[0] + hk * a.vs[2] : static_cast<const T*>(a.kin) + b * a.ks[0] + hk * a.ks[2]) + mine * 8;
  const int64_t step = values ? a.vs[1] : a.ks[1];
#pragma unroll
  for (int e = 0; e < STEPS; ++e) {
    const int i = i0 + e * ABREAST;
    r[e] = {};
    if (i < 0 || i >= n) continue;
    load16(src + i * step, HALF, r[e].lo, r[e].hi);
    if (!values) {
      load_angles<T>(a, start + i, HALF, mine, r[e]);
    } else if (a.ve) {
      load16(static_cast<const T*>(a.ve) + b * a.es[0] + hk * a.es[2] + mine * 8 + i * a.es[1], HALF, r[e].lo2, r[e].hi2);
      gate[e] = Num<T>::one((static_cast<const T*>(a.ve_gate) + b * a.gs[0] + hk * a.gs[2])[i * a.gs[1]]);
    }
  }
  const BlockAt block = find_block(a, b, p0, hk, values, tells);
  if (!block.codes) return;
  const float old = start > p0 ? *block.scale : 0.f;
  float2 x[STEPS][8];
#pragma unroll
  for (int e = 0; e < STEPS; ++e) {
    if (values) mix_raw<T>(r[e], a.ve, share_of(gate[e]), x[e]);
    else turn_raw<T, D>(a, r[e], x[e]);
  }
  float top = finite_top(x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (WIDE > 1) {
    if (lane == 0) tops[warp] = top;
    named_bar_sync(1 + warp / WIDE, WIDE * 32);  // (the old scale is read by now, too)
#pragma unroll
    for (int w = 0; w < WIDE; ++w) top = fmaxf(top, tops[warp - part + w]);
  }
  const float scale = fmaxf(old, block_scale(top)), by = 1.f / scale;
#pragma unroll
  for (int e = 0; e < STEPS; ++e) {
    const int i = i0 + e * ABREAST;
    uint8_t* at = block.codes + (slot0 + e * ABREAST) * block.step + mine * 8;
    if (i < 0) {
      if (scale != old) rescale_codes(at, HALF, old * by);
    } else if (i < n) {
      write_codes(at, HALF, x[e], by);
    }
  }
  if (tells) *block.scale = scale;
}

template <class T, int D, int PER, int STEPS>
static int launch_append8(const PagedAppendArgs& a, cudaStream_t s) {
  constexpr int L = D / 16, PER_CTA = 8 * STEPS * (32 / L) / TILE;
  const int64_t tokens = static_cast<int64_t>(a.B) * a.t, blocks = (a.t + 2 * (TILE - 1)) / TILE;
  const int64_t writing = (a.B * blocks * a.Hk * 2 + PER_CTA - 1) / PER_CTA;
  const int64_t turning = (tokens * ((a.H + PER - 1) / PER) + 256 / L - 1) / (256 / L);
  if (writing * PER_CTA > INT32_MAX || turning * (256 / L) > INT32_MAX) return -1;
  append8_kernel<T, D, PER, STEPS><<<static_cast<unsigned>(writing + turning), 256, 0, s>>>(a, static_cast<int>(blocks), static_cast<int>(writing));
  return 0;
}
template <class T, int D>
static int launch_append8(const PagedAppendArgs& a, cudaStream_t s) {
  if (a.t == 1) {
    constexpr int PER_CTA = 256 / (D / 16);
    const int64_t items = static_cast<int64_t>(a.B) * (a.H + 2 * a.Hk);
    if (items > INT32_MAX - PER_CTA) return -1;
    append8_one_kernel<T, D><<<static_cast<unsigned>((items + PER_CTA - 1) / PER_CTA), 256, 0, s>>>(a);
    return 0;
  }
  // Many heads of tokens keep the SMs busy with three query heads a group of lanes and two tokens a thread, which take fewer instructions; few
  // are done sooner by twice the threads.  One head and one token / three and two, us: 10 / 5 heads of 128, one row of 512 tokens
  // 3.0 / 3.4, of 1024 3.9 / 3.7, 4 of 700 7.8 / 6.9, 8 of 2048 42 / 35; 16 / 1 of 128, one row of 1024 3.4 / 3.6; 12 / 12 of 64, 192 of 4 9.1 / 7.6.
  return static_cast<int64_t>(a.B) * a.t * a.H >= 10240 ? launch_append8<T, D, 3, 2>(a, s) : launch_append8<T, D, 1, 1>(a, s);
}

struct Plan {
  int NR, grid;
  Geometry g;
};
static Plan make_plan(const PagedAttnArgs& a) {
  Plan p;
  Geometry& g = p.g;
  const int64_t group = a.H / a.Hk, R = a.t * group;
  g.group = static_cast<int>(group);
  g.R = static_cast<int>(R);
  g.inverse = group == 1 ? 0u : static_cast<uint32_t>(((int64_t{1} << 32) + group - 1) / group);
  p.NR = R <= 8 ? 8 : 16;
  g.row_tiles = static_cast<int>((R + p.NR - 1) / p.NR);
  const int64_t items = static_cast<int64_t>(a.B) * g.row_tiles;
  const int64_t capacity = std::min<int64_t>(static_cast<int64_t>(a.cache.columns) * a.cache.page, INT32_MAX - TILE);
  g.items = static_cast<int>(std::min<int64_t>(items, INT32_MAX));
  g.capacity = static_cast<int>(capacity);
  g.direct = items > MAX_ITEMS || items * (capacity / TILE + 1) * a.Hk > INT32_MAX;  // places on the line are 32-bit
  int64_t tiles = (capacity + TILE - 1) / TILE;
  if (a.window >= 0) tiles = std::min<int64_t>(tiles, (static_cast<int64_t>(a.window) + a.t) / TILE + 2);
  tiles = std::max<int64_t>(tiles, 1) * items * a.Hk;
  p.grid = static_cast<int>(g.direct ? std::min<int64_t>(items * a.Hk, INT32_MAX)
                                     : std::max<int64_t>(1, std::min<int64_t>(std::min(a.sms, FAN * FAN), std::max(tiles / (WARPS * MIN_TILES), (items * a.Hk + WARPS - 1) / WARPS))));
  return p;
}

template <class T, class C, int D, int NQ>
static int launch_attn(const PagedAttnArgs& a, const Plan& p, cudaStream_t s) {
  using S = Shape<C, D, NQ>;
  static std::atomic<uint64_t> done{0};
  auto kern = attn_kernel<T, C, D, NQ>;
  if (smem_limit(done, kern, S::SMEM) != cudaSuccess) return -1;
  kern<<<p.grid, WARPS * 32, S::SMEM, s>>>(a, p.g, a.workspace, a.counters);
  return 0;
}

template <class T, class C>
static int launch_attn(const PagedAttnArgs& a, const Plan& p, cudaStream_t s) {
  if (a.D == 128) return p.NR == 8 ? launch_attn<T, C, 128, 1>(a, p, s) : launch_attn<T, C, 128, 2>(a, p, s);
  return p.NR == 8 ? launch_attn<T, C, 64, 1>(a, p, s) : launch_attn<T, C, 64, 2>(a, p, s);
}

}  // namespace paged
}  // namespace nt

using namespace nt::paged;

int nt_paged_append(const PagedAppendArgs& a, cudaStream_t s) {
  if (a.B == 0 || a.t == 0) return 0;
  if (a.cache.k_scale) {
    if (a.D == 128) return a.fp16 ? launch_append8<__half, 128>(a, s) : launch_append8<__nv_bfloat16, 128>(a, s);
    if (a.D == 64) return a.fp16 ? launch_append8<__half, 64>(a, s) : launch_append8<__nv_bfloat16, 64>(a, s);
    return -1;
  }
  if (a.D == 128) return a.fp16 ? launch_append<__half, 128>(a, s) : launch_append<__nv_bfloat16, 128>(a, s);
  if (a.D == 64) return a.fp16 ? launch_append<__half, 64>(a, s) : launch_append<__nv_bfloat16, 64>(a, s);
  return -1;
}

size_t nt_paged_attn_workspace(const PagedAttnArgs& a) {
  const Plan p = make_plan(a);
  return p.g.direct ? 0 : ws_floats(p.grid, p.NR * a.D + p.NR * 2) * sizeof(float);
}
int nt_paged_attn_counters(int sms) { return std::min(sms, FAN * FAN) * COUNTERS; }

int nt_paged_attn(const PagedAttnArgs& a, cudaStream_t s) {
  if (a.B == 0 || a.t == 0) return 0;
  if (a.D != 64 && a.D != 128) return -1;
  const Plan p = make_plan(a);
  if (static_cast<int64_t>(p.g.items) * a.Hk >= INT32_MAX ||
      static_cast<int64_t>(p.g.R) * p.g.group >= (int64_t{1} << 32) - 16 * p.g.group ||
      static_cast<int64_t>(a.t) * p.g.group > INT32_MAX / 2)
    return -1;
  if (a.fp16) return a.cache.k_scale ? launch_attn<__half, E4M3>(a, p, s) : launch_attn<__half, __half>(a, p, s);
  return a.cache.k_scale ? launch_attn<__nv_bfloat16, E4M3>(a, p, s) : launch_attn<__nv_bfloat16, __nv_bfloat16>(a, p, s);
}

int nt_paged_read_error(unsigned* where) {
  nt::ErrorWord e{};
  cudaMemcpyFromSymbol(&e, nt::g_nt_error, sizeof(e));
  if (where) *where = e.where;
  if (e.code) {
    const nt::ErrorWord z{};
    cudaMemcpyToSymbol(nt::g_nt_error, &z, sizeof(z));
  }
  return static_cast<int>(e.code);
}
