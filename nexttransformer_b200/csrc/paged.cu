// K22: the paged key-value cache of the decoding engine.
//
// append     k' = s rope(k) / rms(rope(k)), v' = v + 3 sigmoid(gate) ve into the pages, q' = s rope(q) / rms(rope(q))
// attention  o = softmax(scale q K^T) V over the pages, a few new tokens per row, GQA, left window
//
// Both are bound by memory.  What each kernel does about it, and what it measured, stands beside it.
#include "paged.h"
#include "common.cuh"

#include <cuda_fp16.h>

#include <algorithm>

namespace nt {
namespace paged {

constexpr float EPS = 1.1920929e-07f;  // FLT_EPSILON, as the shell's RMSNorm

template <class T> struct Num;
template <> struct Num<__nv_bfloat16> {
  static NT_DEVICE float2 unpack(uint32_t v) { return unpack_bf16x2(v); }
  static NT_DEVICE uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static NT_DEVICE float one(__nv_bfloat16 v) { return __bfloat162float(v); }
  static NT_DEVICE void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Num<__half> {
  static NT_DEVICE float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
  static NT_DEVICE uint32_t pack(float lo, float hi) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static NT_DEVICE float one(__half v) { return __half2float(v); }
  static NT_DEVICE void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

template <class T>
NT_DEVICE void unpack8(const uint4& u, float (&x)[8]) {
  const float2 a = Num<T>::unpack(u.x), b = Num<T>::unpack(u.y), c = Num<T>::unpack(u.z), d = Num<T>::unpack(u.w);
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
}
template <class T>
NT_DEVICE uint4 pack8(const float (&x)[8]) {
  return make_uint4(Num<T>::pack(x[0], x[1]), Num<T>::pack(x[2], x[3]), Num<T>::pack(x[4], x[5]), Num<T>::pack(x[6], x[7]));
}

// ------------------------------------------------------------------------------------ append
// D / 8 lanes hold one head of one token, 16 bytes each; the two halves of a rotated pair are D / 16
// lanes apart.  One pass: every input element is read once and every output element written once.
template <class T, int D>
__global__ void __launch_bounds__(256) append_kernel(const PagedAppendArgs a) {
  constexpr int L = D / 8;
  const int heads = a.H + 2 * a.Hk;
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / L;
  const int lane = threadIdx.x % L;
  const int64_t units = static_cast<int64_t>(a.B) * a.t * heads;
  const bool live = unit < units;  // whole warps stay for the shuffles
  const int64_t tok = live ? unit / heads : 0;
  const int h = live ? static_cast<int>(unit - tok * heads) : 0;
  const int b = static_cast<int>(tok / a.t), i = static_cast<int>(tok - static_cast<int64_t>(b) * a.t);
  const int kind = h < a.H ? 0 : h < a.H + a.Hk ? 1 : 2;  // q, k, v
  const int hh = kind == 0 ? h : kind == 1 ? h - a.H : h - a.H - a.Hk;

  const T* src = static_cast<const T*>(kind == 0 ? a.q : kind == 1 ? a.kin : a.vin);
  const int64_t* st = kind == 0 ? a.qs : kind == 1 ? a.ks : a.vs;
  const uint4 raw = live ? *reinterpret_cast<const uint4*>(src + b * st[0] + i * st[1] + hh * st[2] + lane * 8)
                         : make_uint4(0, 0, 0, 0);
  const int start = a.start[b], n = a.count ? a.count[b] : a.t;
  const bool real = live && i < n && start >= 0;
  const int64_t pos = static_cast<int64_t>(start) + i;

  const bool turned = kind < 2;
  const bool in = real && (!turned || pos < a.rope_rows);
  if (real && !in && lane == 0) record_error(3, b);
  float x[8], y[8], c[8], s[8];
  unpack8<T>(raw, x);
  uint4 cw = make_uint4(0, 0, 0, 0), sw = cw;
  if (turned && in) {
    const int64_t at = pos * (D / 2) + (lane % (L / 2)) * 8;
    cw = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.cos) + at);
    sw = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.sin) + at);
  }
  unpack8<T>(cw, c);
  unpack8<T>(sw, s);
  const float sign = lane < L / 2 ? 1.f : -1.f;
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float other = __shfl_xor_sync(0xffffffffu, x[e], L / 2);
    y[e] = fmaf(sign * other, s[e], x[e] * c[e]);
    sum = fmaf(y[e], y[e], sum);
  }
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (!live) return;
  if (turned) {
    const float r = a.norm ? a.scale * rsqrtf(sum * (1.f / D) + EPS) : 1.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = in ? y[e] * r : 0.f;
  } else if (a.ve && real) {
    float w[8];
    unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.ve) + b * a.es[0] + i * a.es[1] + hh * a.es[2] +
                                               lane * 8),
               w);
    const float gate = Num<T>::one(static_cast<const T*>(a.ve_gate)[b * a.gs[0] + i * a.gs[1] + hh * a.gs[2]]);
    const float f = 3.f / (1.f + __expf(-gate));
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf(f, w[e], x[e]);
  }
  const uint4 o = pack8<T>(x);
  if (kind == 0) {  // tokens behind a row's count give zeros
    *reinterpret_cast<uint4*>(static_cast<T*>(a.q_out) + (tok * a.H + hh) * D + lane * 8) = o;
    return;
  }
  if (!in) return;
  const PagedCacheArgs& m = a.cache;
  const int64_t column = pos / m.page;
  if (column >= m.columns) {
    if (lane == 0) record_error(1, b);
    return;
  }
  const int64_t page = m.table[static_cast<int64_t>(b) * m.columns + column];
  if (page < 0 || page >= m.pages) {
    if (lane == 0) record_error(2, b);
    return;
  }
  const int64_t slot = pos - column * m.page;
  T* dst = kind == 1 ? static_cast<T*>(m.k) + page * m.page_stride_k + hh * m.head_stride_k + slot * m.slot_stride_k
                     : static_cast<T*>(m.v) + page * m.page_stride_v + hh * m.head_stride_v + slot * m.slot_stride_v;
  *reinterpret_cast<uint4*>(dst + lane * 8) = o;
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
// Work: a row's keys (window cut off) are tiles of 16.  The tiles of all rows and KV heads form one line,
// each CTA takes an equal piece of it and each warp an equal piece of that, so unequal rows load the SMs
// equally and one long row uses all of them.  A warp that covers a whole (row, KV head) writes its result;
// pieces are joined in the CTA through shared memory, and what crosses CTAs by join_kernel, both in the
// order of the line, so results do not depend on timing.
constexpr int WARPS = 8, TILE = 16, MIN_TILES = 1;
// Rows of the batch whose tiles a CTA lines up in shared memory; a larger batch has CTAs enough and gives
// each (row, KV head) one.
constexpr int MAX_ITEMS = 384;

template <int D, int NQ>
struct Shape {
  static constexpr int NR = NQ * 8;
  static constexpr int HALF = TILE * D * 2, STAGE = 2 * HALF;              // bytes of K, of K and V
  static constexpr int STAGES = D == 128 ? (NQ == 1 ? 3 : 2) : (NQ == 1 ? 6 : 5);
  static constexpr int RING = STAGES * STAGE;                              // of one warp
  static constexpr int ROW = D + 4;                                        // floats: D sums, maximum, total, 2 unused
  static constexpr int PART = NR * ROW * 4;
  static constexpr int SMEM = WARPS * (RING + PART);
  static_assert(PART <= RING, "a warp's last piece lies in its own ring");
  static_assert(SMEM + 2048 <= 227 * 1024, "shared memory of an SM");
};

struct Item {      // a row tile of one row of the batch
  int b, r0;       // row, first query row
  int start, n;    // tokens before the call, new tokens
  int first, end;  // keys [first, end) that one of the query rows sees
  int tiles;       // from first rounded down to 16; at least 1, so that rows without keys are written
};

NT_DEVICE Item get_item(const PagedAttnArgs& a, int id, int row_tiles, int NR, int group, int capacity) {
  Item it;
  it.b = id / row_tiles;
  it.r0 = (id - it.b * row_tiles) * NR;
  it.start = a.start[it.b];
  it.n = a.count ? min(a.count[it.b], a.t) : a.t;
  if (it.start < 0) it.n = 0;
  const int i0 = it.r0 / group, i1 = min((it.r0 + NR - 1) / group, it.n - 1);
  it.first = it.end = 0;
  if (i0 <= i1) {
    it.end = static_cast<int>(min(static_cast<int64_t>(it.start) + i1 + 1, static_cast<int64_t>(capacity)));
    it.first = a.window >= 0 ? max(0, min(it.start + i0 - a.window, it.end)) : 0;
  }
  it.tiles = max(1, (it.end - (it.first & ~(TILE - 1)) + TILE - 1) / TILE);
  return it;
}

NT_DEVICE void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
NT_DEVICE void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
NT_DEVICE void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
NT_DEVICE void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
NT_DEVICE void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
NT_DEVICE uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
NT_DEVICE float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Weight of a piece with maximum m in a sum with maximum top (both in powers of two; -inf: no keys).
NT_DEVICE float piece_weight(float m, float top) { return top == -INFINITY ? 0.f : exp2_fast(m - top); }
// A row without keys gives zeros; a total of NaN stays NaN.
NT_DEVICE float inverse_total(float l) { return l == 0.f ? 0.f : 1.f / l; }

// Where a warp's copies stand on the line.
struct Cursor {
  int id, hk, j;   // item, KV head, tile
  Item it;
  int column, slot;            // of the tile's first key
  int seen, pages;             // lane l holds the page of column seen + l
};

NT_DEVICE void load_pages(const PagedAttnArgs& a, Cursor& c, int lane) {
  c.seen = c.column;
  const int col = c.column + lane;
  c.pages = col < a.cache.columns ? a.cache.table[static_cast<int64_t>(c.it.b) * a.cache.columns + col] : -1;
}
NT_DEVICE void enter(const PagedAttnArgs& a, Cursor& c, int row_tiles, int NR, int group, int capacity, int lane) {
  c.it = get_item(a, c.id, row_tiles, NR, group, capacity);
  const int key = (c.it.first & ~(TILE - 1)) + c.j * TILE;
  c.column = key / a.cache.page;
  c.slot = key - c.column * a.cache.page;
  load_pages(a, c, lane);
}

template <class T, int D, int NQ>
__global__ void __launch_bounds__(WARPS * 32, 1)
    attn_kernel(const PagedAttnArgs a, const int items, const int row_tiles, const bool direct, float* ws_part, int4* ws_desc) {
  using S = Shape<D, NQ>;
  constexpr int NR = S::NR, CHUNKS = D / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int pre[MAX_ITEMS + 1];
  __shared__ int warp_sum_[WARPS];
  __shared__ int part_id[2 * WARPS], part_flag[2 * WARPS];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = a.H / a.Hk, R = a.t * group, Hk = a.Hk;
  const int capacity = static_cast<int>(min(static_cast<int64_t>(a.cache.columns) * a.cache.page, static_cast<int64_t>(INT32_MAX)));
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this CTA's piece [lo, hi) of the line
  int64_t lo, hi, W = 0;
  int G = 1, base_id = 0, base_hk = 0;
  if (direct) {
    base_id = blockIdx.x / Hk;
    base_hk = blockIdx.x - base_id * Hk;
    lo = 0;
    const Item it = get_item(a, base_id, row_tiles, NR, group, capacity);
    hi = it.tiles;
    if (tid == 0 && it.n > 0 && static_cast<int64_t>(it.start) + it.n > capacity) record_error(1, it.b);
  } else {
    constexpr int EACH = (MAX_ITEMS + WARPS * 32 - 1) / (WARPS * 32);
    int own[EACH], sum = 0;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int id = tid * EACH + e;
      own[e] = 0;
      if (id < items) {
        const Item it = get_item(a, id, row_tiles, NR, group, capacity);
        own[e] = it.tiles;
        if (blockIdx.x == 0 && it.n > 0 && static_cast<int64_t>(it.start) + it.n > capacity) record_error(1, it.b);
      }
      sum += own[e];
    }
    int scan = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += v;
    }
    if (lane == 31) warp_sum_[warp] = scan;
    __syncthreads();
    int before = scan - sum;
    for (int w = 0; w < warp; ++w) before += warp_sum_[w];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int id = tid * EACH + e;
      if (id < items) {
        pre[id] = before;
        before += own[e];
        if (id == items - 1) pre[items] = before;
      }
    }
    __syncthreads();
    W = static_cast<int64_t>(pre[items]) * Hk;
    G = static_cast<int>(max(static_cast<int64_t>(1), min(static_cast<int64_t>(gridDim.x), W / (WARPS * MIN_TILES))));
    if (static_cast<int>(blockIdx.x) >= G) {
      if (tid == 0) ws_desc[blockIdx.x] = make_int4(-1, 0, 0, 0);
      return;
    }
    lo = blockIdx.x * W / G;
    hi = (blockIdx.x + 1) * W / G;
  }
  const int64_t x0 = lo + warp * (hi - lo) / WARPS, x1 = lo + (warp + 1) * (hi - lo) / WARPS;
  int fetch_left = static_cast<int>(x1 - x0), left = fetch_left;
  if (lane < 2) part_id[2 * warp + lane] = -1;

  if (left > 0) {
    Cursor f;
    if (direct) {
      f.id = base_id; f.hk = base_hk; f.j = static_cast<int>(x0);
    } else {
      int l = 0, r = items;  // the last item whose tiles begin at or before x0
      while (r - l > 1) {
        const int mid = (l + r) >> 1;
        if (static_cast<int64_t>(pre[mid]) * Hk <= x0) l = mid; else r = mid;
      }
      const int64_t rest = x0 - static_cast<int64_t>(pre[l]) * Hk;
      const int n = pre[l + 1] - pre[l];
      f.id = l;
      f.hk = static_cast<int>(rest / n);
      f.j = static_cast<int>(rest - static_cast<int64_t>(f.hk) * n);
    }
    enter(a, f, row_tiles, NR, group, capacity, lane);
    Cursor c = f;  // where the products stand (its page fields are unused)

    uint8_t* ring = smem + warp * S::RING;
    const uint32_t ring_u = smem_u32(ring);
    const int lrow = lane / CHUNKS, lch = lane % CHUNKS;
    constexpr int ROWS = 32 / CHUNKS;  // rows of one copy instruction of the warp
    const T* kc = static_cast<const T*>(a.cache.k);
    const T* vc = static_cast<const T*>(a.cache.v);

    auto fetch = [&](int stage) {
      if (fetch_left > 0) {
        if (f.column - f.seen >= 32) load_pages(a, f, lane);
        const int page = __shfl_sync(0xffffffffu, f.pages, f.column - f.seen);
        const int key = (f.it.first & ~(TILE - 1)) + f.j * TILE;
        const bool there = page >= 0 && page < a.cache.pages;
        if (!there && f.it.first < f.it.end && lane == 0) record_error(2, f.it.b);
        const int64_t p = there ? page : 0;
        const T* ks = kc + p * a.cache.page_stride_k + f.hk * a.cache.head_stride_k + f.slot * a.cache.slot_stride_k + lch * 8;
        const T* vs = vc + p * a.cache.page_stride_v + f.hk * a.cache.head_stride_v + f.slot * a.cache.slot_stride_v + lch * 8;
        const uint32_t dst = ring_u + stage * S::STAGE;
#pragma unroll
        for (int e = 0; e < TILE / ROWS; ++e) {
          // keys outside [first, end) become zeros: whatever their memory holds never meets a product
          const int row = e * ROWS + lrow;
          const bool valid = there && key + row >= f.it.first && key + row < f.it.end;
          const uint32_t to = dst + row * (D * 2) + ((lch ^ (row & 7)) << 4);
          cp_async16(to, ks + (valid ? row * a.cache.slot_stride_k : 0), valid ? 16 : 0);
          cp_async16(to + S::HALF, vs + (valid ? row * a.cache.slot_stride_v : 0), valid ? 16 : 0);
        }
        --fetch_left;
        if (++f.j == f.it.tiles) {
          f.j = 0;
          if (++f.hk == Hk) {
            f.hk = 0;
            ++f.id;
          }
          if (fetch_left > 0) enter(a, f, row_tiles, NR, group, capacity, lane);
        } else if ((f.slot += TILE) == a.cache.page) {
          f.slot = 0;
          ++f.column;
        }
      }
      cp_commit();
    };

#pragma unroll
    for (int s = 0; s < S::STAGES - 1; ++s) fetch(s);
    int stage = 0;
    const float scale2 = a.scale * 1.4426950408889634f;
    const int qc = lane & 3, qr = lane >> 2;

    while (left > 0) {
      // ---- one piece: tiles [c.j, c.j + n) of (c.id, c.hk)
      const int n = min(left, c.it.tiles - c.j), j0 = c.j;
      uint32_t qf[NQ][D / 16][2];
      int last[NQ][2], oldest[NQ][2];  // newest and oldest key that this lane's two queries see
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
        const int r = c.it.r0 + nq * 8 + qr, i = r / group;
        const bool live = r < R && i < c.it.n;
        const T* qp = static_cast<const T*>(a.q) + c.it.b * a.qs[0] + (live ? i : 0) * a.qs[1] +
                      (c.hk * group + (live ? r - i * group : 0)) * a.qs[2] + qc * 2;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          qf[nq][kk][0] = live ? *reinterpret_cast<const uint32_t*>(qp + kk * 16) : 0u;
          qf[nq][kk][1] = live ? *reinterpret_cast<const uint32_t*>(qp + kk * 16 + 8) : 0u;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int rc = c.it.r0 + nq * 8 + qc * 2 + e, ic = rc / group;
          const bool lc = rc < R && ic < c.it.n;
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
        fetch(ahead);
        const uint32_t kbase = ring_u + stage * S::STAGE, vbase = kbase + S::HALF;
        if (++stage == S::STAGES) stage = 0;

        float s[NQ][4];
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nq][e] = 0.f;
        {
          const int row = lane & 15;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t kf[4];
            ldsm4(kf, kbase + row * (D * 2) + (((kk * 2 + (lane >> 4)) ^ (row & 7)) << 4));
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) Num<T>::mma(s[nq], kf, qf[nq][kk][0], qf[nq][kk][1]);
          }
        }
        const int key = (c.it.first & ~(TILE - 1)) + (j0 + tile) * TILE + qr;
        uint32_t pf[NQ][2];
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const bool in0 = key <= last[nq][e] && key >= oldest[nq][e];
            const bool in1 = key + 8 <= last[nq][e] && key + 8 >= oldest[nq][e];
            s[nq][e] = in0 ? s[nq][e] * scale2 : -INFINITY;
            s[nq][e + 2] = in1 ? s[nq][e + 2] * scale2 : -INFINITY;
          }
          float top[2] = {fmaxf(s[nq][0], s[nq][2]), fmaxf(s[nq][1], s[nq][3])};
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], d));
            top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], d));
          }
          float fix[2];
          bool moved = false;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mn = fmaxf(m[nq][e], top[e]);
            moved |= mn != m[nq][e];
            fix[e] = piece_weight(m[nq][e], mn);
            m[nq][e] = mn;
            const float ref = mn == -INFINITY ? 0.f : mn;
            s[nq][e] = exp2_fast(s[nq][e] - ref);
            s[nq][e + 2] = exp2_fast(s[nq][e + 2] - ref);
            l[nq][e] = (mn == -INFINITY ? l[nq][e] : l[nq][e] * fix[e]) + s[nq][e] + s[nq][e + 2];
          }
          if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              o[nq][d][0] *= fix[0]; o[nq][d][1] *= fix[1];
              o[nq][d][2] *= fix[0]; o[nq][d][3] *= fix[1];
            }
          }
          // probabilities are at most 1; rounding them to the cache's type costs no more than the rounding of
          // V does (their sum stays in fp32)
          pf[nq][0] = transpose8x8(Num<T>::pack(s[nq][0], s[nq][1]));
          pf[nq][1] = transpose8x8(Num<T>::pack(s[nq][2], s[nq][3]));
        }
        {
          const int row = (lane & 7) + ((lane >> 4) << 3), ch = (lane >> 3) & 1;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            uint32_t vf[4];
            ldsm4t(vf, vbase + row * (D * 2) + (((d * 2 + ch) ^ (row & 7)) << 4));
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) Num<T>::mma(o[nq][d], vf, pf[nq][0], pf[nq][1]);
          }
        }
      }

      // ---- the piece's end
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          l[nq][0] += __shfl_xor_sync(0xffffffffu, l[nq][0], d);
          l[nq][1] += __shfl_xor_sync(0xffffffffu, l[nq][1], d);
        }
      const bool begins = j0 == 0, ends = j0 + n == c.it.tiles;
      left -= n;
      if (begins && ends) {
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
          const float w0 = inverse_total(l[nq][0]), w1 = inverse_total(l[nq][1]);
          const int r = c.it.r0 + nq * 8 + qr, i = r / group;  // after the transpose this lane holds query qr
          T* op = static_cast<T*>(a.out) +
                  ((static_cast<int64_t>(c.it.b) * a.t + i) * a.H + c.hk * group + (r - i * group)) * D + qc * 2;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            const uint32_t u0 = transpose8x8(Num<T>::pack(o[nq][d][0] * w0, o[nq][d][1] * w1));
            const uint32_t u1 = transpose8x8(Num<T>::pack(o[nq][d][2] * w0, o[nq][d][3] * w1));
            if (r < R) {
              *reinterpret_cast<uint32_t*>(op + d * 16) = u0;
              *reinterpret_cast<uint32_t*>(op + d * 16 + 8) = u1;
            }
          }
        }
      } else {
        const bool final_piece = left == 0;
        const int slot = 2 * warp + (final_piece ? 1 : 0);
        float* part = reinterpret_cast<float*>(final_piece ? ring : smem + WARPS * S::RING + warp * S::PART);
        if (final_piece) {
          cp_wait<0>();
          __syncwarp();
        }
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float* row = part + (nq * 8 + qc * 2 + e) * S::ROW;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              row[d * 16 + qr] = o[nq][d][e];
              row[d * 16 + 8 + qr] = o[nq][d][e + 2];
            }
            if (qr == 0) {
              row[D] = m[nq][e];
              row[D + 1] = l[nq][e];
            }
          }
        if (lane == 0) {
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
          if (left > 0) c.it = get_item(a, c.id, row_tiles, NR, group, capacity);
        }
      }
    }
    cp_wait<0>();
  }
  __syncthreads();

  // ---- join the CTA's pieces in their order
  if (!direct && tid == 0) ws_desc[blockIdx.x] = make_int4(-1, 0, 0, 0);
  auto piece = [&](int s) {
    return reinterpret_cast<const float*>((s & 1) ? smem + (s >> 1) * S::RING : smem + WARPS * S::RING + (s >> 1) * S::PART);
  };
  for (int s0 = 0; s0 < 2 * WARPS;) {
    const int id = part_id[s0];
    if (id < 0) {
      ++s0;
      continue;
    }
    int s1 = s0 + 1, tail = s0;
    while (s1 < 2 * WARPS && (part_id[s1] == id || part_id[s1] < 0)) {
      if (part_id[s1] == id) tail = s1;
      ++s1;
    }
    const bool begins = part_flag[s0] & 1, ends = part_flag[tail] & 2;
    const int item = id / Hk, hk = id - item * Hk;
    const int b = item / row_tiles, r0 = (item - b * row_tiles) * NR;
    for (int e = tid; e < NR * (D / 4); e += WARPS * 32) {
      const int q = e / (D / 4), d = (e - q * (D / 4)) * 4, r = r0 + q;
      if (r >= R) continue;
      float top = -INFINITY;
      for (int s = s0; s <= tail; ++s)
        if (part_id[s] == id) top = fmaxf(top, piece(s)[q * S::ROW + D]);
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      float total = 0.f;
      for (int s = s0; s <= tail; ++s) {
        if (part_id[s] != id) continue;
        const float* row = piece(s) + q * S::ROW;
        const float w = piece_weight(row[D], top);
        const float4 v = *reinterpret_cast<const float4*>(row + d);
        sum.x = fmaf(w, v.x, sum.x); sum.y = fmaf(w, v.y, sum.y);
        sum.z = fmaf(w, v.z, sum.z); sum.w = fmaf(w, v.w, sum.w);
        total = fmaf(w, row[D + 1], total);
      }
      if (begins && ends) {
        const float w = inverse_total(total);
        const int i = r / group;
        T* op = static_cast<T*>(a.out) + ((static_cast<int64_t>(b) * a.t + i) * a.H + hk * group + (r - i * group)) * D + d;
        *reinterpret_cast<uint2*>(op) = make_uint2(Num<T>::pack(sum.x * w, sum.y * w), Num<T>::pack(sum.z * w, sum.w * w));
      } else {
        // slot 1: the (row, KV head) begins in this CTA; slot 0: it began in an earlier one
        float* row = ws_part + ((static_cast<int64_t>(blockIdx.x) * 2 + (begins ? 1 : 0)) * NR + q) * S::ROW;
        *reinterpret_cast<float4*>(row + d) = sum;
        if (d == 0) *reinterpret_cast<float2*>(row + D) = make_float2(top, total);
      }
    }
    if (begins && !ends && tid == 0) {
      // the (row, KV head) ends with the CTA that holds its last tile
      const int64_t n = pre[item + 1] - pre[item];
      const int64_t x = static_cast<int64_t>(pre[item]) * Hk + (hk + 1) * n - 1;
      ws_desc[blockIdx.x] = make_int4(static_cast<int>(((x + 1) * G - 1) / W), b, r0, hk);
    }
    s0 = s1;
  }
}

// Joins the pieces of a (row, KV head) that several CTAs hold: block (c, q) for query row q of the one that
// begins in CTA c.  Eight (16 for heads of 64) groups of threads take every eighth piece, four channels a
// thread, then the groups' sums are joined in their order.
template <class T, int D, int NR>
__global__ void __launch_bounds__(256) join_kernel(const PagedAttnArgs a, const float* ws_part, const int4* ws_desc) {
  constexpr int LANES = D / 4, GROUPS = 256 / LANES, ROW = D + 4;
  __shared__ float part[GROUPS][ROW];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c0 = blockIdx.x, q = blockIdx.y;
  const int4 desc = ws_desc[c0];
  if (desc.x < 0) return;
  const int group = a.H / a.Hk, r = desc.z + q;
  if (r >= a.t * group) return;
  const int g = threadIdx.x / LANES, d = (threadIdx.x % LANES) * 4, n = desc.x - c0 + 1;
  float top = -INFINITY, total = 0.f;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int p = g; p < n; p += GROUPS) {
    const float* row = ws_part + ((static_cast<int64_t>(c0 + p) * 2 + (p == 0 ? 1 : 0)) * NR + q) * ROW;
    const float4 v = *reinterpret_cast<const float4*>(row + d);
    const float2 ml = *reinterpret_cast<const float2*>(row + D);
    const float up = fmaxf(top, ml.x);
    const float w0 = piece_weight(top, up), w1 = piece_weight(ml.x, up);
    sum.x = sum.x * w0 + v.x * w1; sum.y = sum.y * w0 + v.y * w1;
    sum.z = sum.z * w0 + v.z * w1; sum.w = sum.w * w0 + v.w * w1;
    total = total * w0 + ml.y * w1;
    top = up;
  }
  *reinterpret_cast<float4*>(&part[g][d]) = sum;
  if (d == 0) {
    part[g][D] = top;
    part[g][D + 1] = total;
  }
  __syncthreads();
  if (g != 0) return;
  top = -INFINITY;
#pragma unroll
  for (int p = 0; p < GROUPS; ++p) top = fmaxf(top, part[p][D]);
  sum = make_float4(0.f, 0.f, 0.f, 0.f);
  total = 0.f;
#pragma unroll
  for (int p = 0; p < GROUPS; ++p) {
    const float w = piece_weight(part[p][D], top);
    const float4 v = *reinterpret_cast<const float4*>(&part[p][d]);
    sum.x = fmaf(w, v.x, sum.x); sum.y = fmaf(w, v.y, sum.y);
    sum.z = fmaf(w, v.z, sum.z); sum.w = fmaf(w, v.w, sum.w);
    total = fmaf(w, part[p][D + 1], total);
  }
  const float w = inverse_total(total);
  const int i = r / group;
  T* op = static_cast<T*>(a.out) +
          ((static_cast<int64_t>(desc.y) * a.t + i) * a.H + desc.w * group + (r - i * group)) * D + d;
  *reinterpret_cast<uint2*>(op) = make_uint2(Num<T>::pack(sum.x * w, sum.y * w), Num<T>::pack(sum.z * w, sum.w * w));
}

struct Plan {
  int NR, row_tiles, grid;
  int64_t items;
  bool direct;
};
static Plan make_plan(const PagedAttnArgs& a) {
  Plan p;
  const int64_t R = static_cast<int64_t>(a.t) * (a.H / a.Hk);
  p.NR = R <= 8 ? 8 : 16;
  p.row_tiles = static_cast<int>((R + p.NR - 1) / p.NR);
  p.items = static_cast<int64_t>(a.B) * p.row_tiles;
  const int64_t capacity = static_cast<int64_t>(a.cache.columns) * a.cache.page;
  p.direct = p.items > MAX_ITEMS || p.items * (capacity / TILE + 1) > INT32_MAX;  // the line's prefix sums are 32-bit
  int64_t tiles = (capacity + TILE - 1) / TILE;
  if (a.window >= 0) tiles = std::min<int64_t>(tiles, (static_cast<int64_t>(a.window) + a.t) / TILE + 2);
  tiles = std::max<int64_t>(tiles, 1) * p.items * a.Hk;
  p.grid = static_cast<int>(p.direct ? p.items * a.Hk
                                     : std::max<int64_t>(1, std::min<int64_t>(a.sms, tiles / (WARPS * MIN_TILES))));
  return p;
}

template <class T, int D, int NQ>
static int launch_attn(const PagedAttnArgs& a, const Plan& p, cudaStream_t s) {
  using S = Shape<D, NQ>;
  static std::atomic<uint64_t> done{0};
  auto kern = attn_kernel<T, D, NQ>;
  if (smem_limit(done, kern, S::SMEM) != cudaSuccess) return -1;
  float* part = a.workspace;
  int4* desc = reinterpret_cast<int4*>(part + static_cast<int64_t>(p.grid) * 2 * S::NR * S::ROW);
  kern<<<p.grid, WARPS * 32, S::SMEM, s>>>(a, static_cast<int>(p.items), p.row_tiles, p.direct, part, desc);
  if (p.direct || p.grid == 1) return 0;
  // launched with the attention kernel still running: its blocks wait for the pieces on the device
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.grid - 1, static_cast<unsigned>(std::min<int64_t>(S::NR, static_cast<int64_t>(a.t) * (a.H / a.Hk))));
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, join_kernel<T, D, S::NR>, a, static_cast<const float*>(part),
                            static_cast<const int4*>(desc)) == cudaSuccess ? 0 : -1;
}

}  // namespace paged
}  // namespace nt

using namespace nt::paged;

int nt_paged_append(const PagedAppendArgs& a, cudaStream_t s) {
  const int64_t units = static_cast<int64_t>(a.B) * a.t * (a.H + 2 * a.Hk);
  if (units == 0) return 0;
  if (a.D != 64 && a.D != 128) return -1;
  const int64_t blocks = (units * (a.D / 8) + 255) / 256;
  if (blocks > INT32_MAX) return -1;
  const unsigned g = static_cast<unsigned>(blocks);
  if (a.fp16) {
    if (a.D == 128) append_kernel<__half, 128><<<g, 256, 0, s>>>(a);
    else append_kernel<__half, 64><<<g, 256, 0, s>>>(a);
  } else {
    if (a.D == 128) append_kernel<__nv_bfloat16, 128><<<g, 256, 0, s>>>(a);
    else append_kernel<__nv_bfloat16, 64><<<g, 256, 0, s>>>(a);
  }
  return 0;
}

size_t nt_paged_attn_workspace(const PagedAttnArgs& a) {
  const Plan p = make_plan(a);
  if (p.direct) return 0;
  return static_cast<size_t>(p.grid) * (2 * p.NR * (a.D + 4) * sizeof(float) + sizeof(int4));
}

int nt_paged_attn(const PagedAttnArgs& a, cudaStream_t s) {
  if (a.B == 0 || a.t == 0) return 0;
  if (a.D != 64 && a.D != 128) return -1;
  const Plan p = make_plan(a);
  if (p.items * a.Hk > INT32_MAX) return -1;
  if (a.fp16) {
    if (a.D == 128) return p.NR == 8 ? launch_attn<__half, 128, 1>(a, p, s) : launch_attn<__half, 128, 2>(a, p, s);
    return p.NR == 8 ? launch_attn<__half, 64, 1>(a, p, s) : launch_attn<__half, 64, 2>(a, p, s);
  }
  if (a.D == 128)
    return p.NR == 8 ? launch_attn<__nv_bfloat16, 128, 1>(a, p, s) : launch_attn<__nv_bfloat16, 128, 2>(a, p, s);
  return p.NR == 8 ? launch_attn<__nv_bfloat16, 64, 1>(a, p, s) : launch_attn<__nv_bfloat16, 64, 2>(a, p, s);
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
