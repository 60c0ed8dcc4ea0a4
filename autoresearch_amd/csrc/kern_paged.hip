// kern_paged.hip -- attention of ragged new tokens over a paged KV cache
// (fg_paged_attn of include/fgpt.h).
//
// Rows: the query rows of one key head are flattened, R = token * G + (query
// head within the group of G = n_head / n_kv_head), so that a tile of rows
// reads each key and value once for its whole group. A work item is a tile of
// one sequence and key head against a part of its keys; which sequence a tile
// belongs to is found on the device from q_start (find_tile), since lengths
// may change under a captured launch.
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "fgpt_internal.h"
#include "kern_common.h"
#include "kern_epi.h"
#include "paged_internal.h"

namespace fgpt {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4v_t __attribute__((ext_vector_type(4)));

namespace {

constexpr float LOG2E = 1.4426950408889634f;

struct PagedArgs {
  const void* k;
  const void* v;
  const void* q;
  PagedOut out;
  int64_t q_ld;
  const int32_t* q_start;
  const int32_t* kv_len;
  const int32_t* table;
  int n_seq, n_rows, max_q, max_kv, table_ld, n_pages, pshift;
  int KH, G;
  int window, sinks;
  bool one_tile;  // a row tile a sequence at most: tile i is sequence i's
  float cs;       // softmax scale * log2(e)
  int ntile;      // bound on the row tiles of all sequences
  int nsplit;     // key parts of a tile at most
  int cpt;        // 32-key tiles of a part
  float* part;    // [ntile * KH][nsplit][rows * HD, then rows * (max, sum)]
};

// A row tile: its sequence, its first flattened row, its rows and the keys that
// any of them sees: [0, sa) and [lo, hi).
struct RowTile {
  int seq, r0, rows;    // rows: flattened rows of the tile
  int row0;             // the sequence's first row
  int pos0;             // position of the sequence's first new token
  int sa, lo, hi, kv;
};

// Which sequence row tile `id` (of RT flattened rows) belongs to. Tiles are
// numbered sequence after sequence; with one tile a sequence at most (decoding)
// the number is the sequence, else the wavefront counts the sequences' tiles,
// 64 of them a step. False: no such tile (a launch may have more workgroups than
// the batch has tiles).
template <int RT>
__device__ __forceinline__ bool find_tile(const PagedArgs& p, int id, RowTile& t) {
  const int lane = threadIdx.x & 63;
  auto q_of = [&](int s) {  // new tokens of sequence s, kept inside the arrays
    const int a = p.q_start[s], n = p.q_start[s + 1] - a;
    return a < 0 ? 0 : max(0, min(min(n, p.max_q), p.n_rows - a));
  };
  int first = 0, nq;
  if (p.one_tile) {
    if (id >= p.n_seq) return false;
    t.seq = id;
    nq = q_of(id);
  } else {
    int base = 0;
    t.seq = -1;
    for (int s0 = 0; s0 < p.n_seq; s0 += 64) {
      const int s = s0 + lane;
      const int n = s < p.n_seq ? (q_of(s) * p.G + RT - 1) / RT : 0;
      int sum = n;  // tiles of this step's sequences up to this one
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(sum, o, 64);
        if (lane >= o) sum += up;
      }
      const uint64_t past = __ballot(base + sum > id);
      if (past) {
        const int l = __builtin_ctzll(past);
        t.seq = s0 + l;
        first = base + __shfl(sum - n, l, 64);
        break;
      }
      base += __shfl(sum, 63, 64);
    }
    if (t.seq < 0) return false;
    nq = q_of(t.seq);
  }
  t.seq = __builtin_amdgcn_readfirstlane(t.seq);
  first = __builtin_amdgcn_readfirstlane(first);
  nq = __builtin_amdgcn_readfirstlane(nq);
  const int tile = p.one_tile ? 0 : id - first;
  t.r0 = tile * RT;
  t.rows = min(RT, nq * p.G - t.r0);
  if (t.rows <= 0) return false;
  // (said to be uniform, or the compiler keeps masks and places per lane)
  t.row0 = __builtin_amdgcn_readfirstlane(p.q_start[t.seq]);
  t.kv = __builtin_amdgcn_readfirstlane(max(0, min(p.kv_len[t.seq], p.max_kv)));
  t.pos0 = t.kv - (__builtin_amdgcn_readfirstlane(p.q_start[t.seq + 1]) - t.row0);
  const int pf = t.pos0 + t.r0 / p.G, pl = t.pos0 + (t.r0 + t.rows - 1) / p.G;
  t.hi = max(0, min(pl + 1, t.kv));
  t.lo = p.window > 0 ? max(0, min(pf - p.window + 1, t.hi)) : 0;
  t.sa = p.window > 0 ? min(p.sinks, t.lo) : 0;
  return true;
}

// The n 32-key tiles of a row tile: na from key 0 on that hold the sinks, then
// those from key `from` on. Each has a key that some row sees.
struct KeyTiles {
  int na, from, n;
};
__device__ __forceinline__ KeyTiles key_tiles(const RowTile& t) {
  KeyTiles k;
  k.na = (t.sa + 31) / 32;
  k.from = max(t.lo & ~31, 32 * k.na);
  k.n = k.na + max(0, t.hi - k.from + 31) / 32;
  return k;
}

__device__ __forceinline__ int tile_base(const RowTile& t, const KeyTiles& k, int v) {
  return v < k.na ? 32 * v : k.from + 32 * (v - k.na);
}

// A tile's 16-key blocks, where their rows lie: pages hold 16 rows or a
// multiple, so a block lies in one. A wavefront looks up 64 blocks ahead, one a
// lane (PageList), and takes them by lane reads: the table's entries then cost
// no wait in the loop, and a block ten scalar instructions.
// Only rows that some query sees are read: in the place of another one the
// block's first such row, in the place of a block without any the tile's other
// block (its page may be gone, its memory hold anything).
struct PageList {
  uint32_t row;  // (page, key head)'s first row of the block, in rows of the pool
  uint32_t vis;  // which of its 16 rows are seen, and (above) the first that is
};
struct PageAsk {
  int e, page;  // first key, the table's entry
};
__device__ __forceinline__ PageAsk page_ask(const PagedArgs& p, const RowTile& t, const KeyTiles& kt,
                                            const int32_t* tab, int v, int kb) {
  PageAsk a;
  a.e = tile_base(t, kt, v) + 16 * kb;
  if (a.e >= t.sa && (a.e >= t.hi || a.e + 16 <= t.lo)) a.e += 16 - 32 * kb;
  a.page = tab[a.e >> p.pshift];
  return a;
}
__device__ __forceinline__ PageList page_place(const PagedArgs& p, const RowTile& t, int kvh,
                                               const PageAsk& a, bool& bad) {
  auto upto = [&](int j) { return (1u << max(0, min(j - a.e, 16))) - 1; };  // rows below key j
  const bool ok = (uint32_t)a.page < (uint32_t)p.n_pages;
  bad |= !ok;
  PageList l;
  l.row = (((uint32_t)(ok ? a.page : 0) * p.KH + kvh) << p.pshift) + (a.e & ((1 << p.pshift) - 1));
  const uint32_t seen = upto(t.sa) | (upto(t.hi) & ~upto(t.lo));
  l.vis = seen | ((uint32_t)__builtin_ctz(seen | 0x10000u) << 16);
  return l;
}
// The row of a block to read for its row x.
__device__ __forceinline__ int page_row(uint32_t vis, int x) {
  return (vis >> x) & 1 ? x : (int)(vis >> 16);
}
__device__ __forceinline__ uint32_t lane_u32(uint32_t v, int lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

__device__ __forceinline__ uint32_t bits(float f) { return __float_as_uint(f); }

// x as the sum of three bf16 terms: its leading 8 significant bits, the next 8,
// the last 8 (cut, not rounded, so the sum is x exactly).
__device__ __forceinline__ void split3(const float (&x)[8], bf16x8_t (&t)[3]) {
  uint32_t w[3][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      w[k][i] = __builtin_amdgcn_perm(bits(b), bits(a), 0x07060302u);
      if (k == 2) break;
      a -= __uint_as_float(bits(a) & 0xFFFF0000u);
      b -= __uint_as_float(bits(b) & 0xFFFF0000u);
    }
  }
#pragma unroll
  for (int k = 0; k < 3; ++k)
    t[k] = __builtin_bit_cast(bf16x8_t, u32x4v_t{w[k][0], w[k][1], w[k][2], w[k][3]});
}

// Values as the sum of N bf16 terms: three are exact, one is rounded (2^-8 of the
// value at most), two are rounded twice (2^-16).
template <int N>
struct Terms {
  bf16x8_t t[N];
  __device__ __forceinline__ void set(const float (&x)[8]) {
    if constexpr (N == 3) {
      split3(x, t);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        t[0][e] = (__bf16)x[e];
        if constexpr (N == 2) t[1][e] = (__bf16)(x[e] - (float)t[0][e]);
      }
    }
  }
};
// Of q and of the probabilities: fp32 rows three. bf16 rows one of q, exact, and
// of the probabilities two in k_paged_few, which waits for memory (32 windows of
// 2048 keys 36.3 us with one, 36.7 with two), one in k_paged_many, which its
// matrix instructions bound (387 GF of prompts 433 us with one, 597 with two).
// Error against 64 bits, relative: with one 0.0022, with two 0.0016, which is
// what rounding the exact result to bf16 gives.
template <bool QF>
using QTerms = Terms<QF ? 3 : 1>;
template <bool QF, bool MANY>
using PTerms = Terms<QF ? 3 : MANY ? 1 : 2>;

__device__ __forceinline__ f32x4_t mma16(const bf16x8_t& a, const bf16x8_t& b, const f32x4_t& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// c += a . b over b's terms, smallest first.
template <int N>
__device__ __forceinline__ f32x4_t mma_terms(const bf16x8_t& a, const Terms<N>& b, f32x4_t c) {
#pragma unroll
  for (int i = N - 1; i >= 0; --i) c = mma16(a, b.t[i], c);
  return c;
}

// One 32-key tile's pieces of the K and V rows, as a lane (row c = lane % 16,
// group g = lane / 16) loads them, the lane's query operand and the two
// products. Which head dims a K slot of S^T = K Q^T and row c of O^T's i-th
// block (vdim) stand for is chosen so that a lane's pieces are whole 16-byte (8
// for head dim 64) loads of adjacent lanes.
template <int HD, bool QF, bool KF>
struct KvTile;
// fp32 pages: v_mfma_f32_16x16x4_f32, whose operands are single values (K slot g
// of step (j, e) is head dim 16 j + 4 g + e; of the second product, key 4 g + r):
// exact products without cutting K and V into terms, which costs a wavefront
// more clocks than these MFMAs take, and registers (one token after 300
// positions, the cut ones 13.4 us, so 8.4).
template <int HD, bool QF>
struct KvTile<HD, QF, true> {
  static constexpr int NJ = HD / 16, VD = HD / 16;
  typedef float elem;
  static __device__ __forceinline__ int vdim(int c, int i) { return 64 * (i / 4) + 4 * c + i % 4; }
  float4 q[NJ], k[2][NJ], v[8][VD / 4];
  static __device__ __forceinline__ float at(const float4& f, int e) {
    return e == 0 ? f.x : e == 1 ? f.y : e == 2 ? f.z : f.w;
  }
  __device__ __forceinline__ void load_q(const void* base, int64_t row, int g) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) q[j] = *(const float4*)((const float*)base + row + 16 * j + 4 * g);
  }
  __device__ __forceinline__ void load_k(int kb, const float* row, int g) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) k[kb][j] = *(const float4*)(row + 16 * j + 4 * g);
  }
  __device__ __forceinline__ void load_v(int e, const float* row, int c) {
#pragma unroll
    for (int i = 0; i < VD / 4; ++i) v[e][i] = *(const float4*)(row + 64 * i + 4 * c);
  }
  __device__ __forceinline__ f32x4_t scores(int kb) const {
    f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s = __builtin_amdgcn_mfma_f32_16x16x4f32(at(k[kb][j], e), at(q[j], e), s, 0, 0, 0);
    return s;
  }
  __device__ __forceinline__ void add_values(const float (&p)[8], f32x4_t (&o)[VD]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int i = 0; i < VD; ++i)
        o[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(at(v[e][i / 4], i % 4), p[e], o[i], 0, 0, 0);
  }
};
// bf16 pages: v_mfma_f32_16x16x32_bf16, K and V exact in one term, q and
// probabilities in QTerms and PTerms.
template <int HD, bool QF>
struct KvTile<HD, QF, false> {
  static constexpr int NS = HD / 32, VD = HD / 16;
  typedef uint16_t elem;
  static __device__ __forceinline__ int vdim(int c, int i) { return VD * c + i; }
  typedef uint32_t vrow_t __attribute__((ext_vector_type(VD / 2)));
  QTerms<QF> q[NS];
  u32x4v_t k[2][NS];
  vrow_t v[8];
  __device__ __forceinline__ void load_q(const void* base, int64_t row, int g) {
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      if constexpr (QF) {
        const float* qp = (const float*)base + row + 32 * s + 8 * g;
        const float4 a = *(const float4*)qp, b = *(const float4*)(qp + 4);
        const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        q[s].set(x);
      } else {
        q[s].t[0] = __builtin_bit_cast(bf16x8_t, *(const u32x4v_t*)((const uint16_t*)base + row + 32 * s + 8 * g));
      }
    }
  }
  __device__ __forceinline__ void load_k(int kb, const uint16_t* row, int g) {
#pragma unroll
    for (int s = 0; s < NS; ++s) k[kb][s] = *(const u32x4v_t*)(row + 32 * s + 8 * g);
  }
  __device__ __forceinline__ void load_v(int e, const uint16_t* row, int c) {
    v[e] = *(const vrow_t*)(row + VD * c);
  }
  __device__ __forceinline__ f32x4_t scores(int kb) const {
    f32x4_t sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < NS; ++s) sc = mma_terms(__builtin_bit_cast(bf16x8_t, k[kb][s]), q[s], sc);
    return sc;
  }
  __device__ __forceinline__ void add_values(const float (&p)[8], f32x4_t (&o)[VD]) const {
    PTerms<QF, false> pt;
    pt.set(p);
#pragma unroll
    for (int i = 0; i < VD; ++i) {
      u32x4v_t w;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = __builtin_amdgcn_perm(v[2 * e + 1][i / 2], v[2 * e][i / 2],
                                     i & 1 ? 0x07060302u : 0x05040100u);
      o[i] = mma_terms(__builtin_bit_cast(bf16x8_t, w), pt, o[i]);
    }
  }
};

// Four consecutive head dims of one query row to their place.
template <bool QF>
__device__ __forceinline__ void store_row4(const PagedArgs& p, int64_t row, int col, const float (&v)[4]) {
  if constexpr (QF) {
    if (p.out.planes) {
      put4<false>(v, p.out.planes + tile_at(row, col, (int)p.out.ld), p.out.plane);
      return;
    }
    *(float4*)((float*)p.out.y + row * p.out.ld + col) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    const uint32_t a = (uint32_t)f32_to_bf16_rne(v[0]) | ((uint32_t)f32_to_bf16_rne(v[1]) << 16);
    const uint32_t b = (uint32_t)f32_to_bf16_rne(v[2]) | ((uint32_t)f32_to_bf16_rne(v[3]) << 16);
    *(uint2*)((uint16_t*)p.out.y + row * p.out.ld + col) = make_uint2(a, b);
  }
}

// Sum of a row's weights -> the factor of its output (no visible key: 0).
__device__ __forceinline__ float inv_sum(float l) { return l == 0.f ? 0.f : 1.0f / l; }

// ------------------------------------------------------------ few rows
// 16 flattened rows a tile, for decoding and short chunks: a workgroup's RWV
// wavefronts take every RWV-th 32-key tile of the item's part, keys and values
// from the pages straight to MFMA operands in registers, and meet in LDS.
// v_mfma_f32_16x16x32_bf16 with S^T = K Q^T: lane 16 g + c then holds query
// row c's scores of keys 4g .. 4g+3 of both 16-key blocks, which are the 8 K
// slots of its operand of O^T = V^T P^T. A block's page comes from the
// wavefront's list (PageList).
// Bound by the cache's bytes, every visible key and value being read once: 64
// tokens over bf16 caches of about 1000 positions, 6 heads of 128, 200 MB, 45 us
// (4.4 TB/s where a copy reaches 5.1); with rows too few for that by the way
// through table, page and products: one token after 300 positions 8.4 us, the
// merge 3.1.
constexpr int DR = 16, RWV = 4;

template <int HD>
constexpr int few_lds() { return RWV * DR * (HD + 4) * 4; }
template <int HD>
constexpr int64_t part_floats(int rows) { return (int64_t)rows * (HD + 2); }

template <int HD, bool QF, bool KF>
__global__ __launch_bounds__(64 * RWV, 2) void k_paged_few(PagedArgs p) {
  typedef KvTile<HD, QF, KF> Tile;
  typedef typename Tile::elem E;
  constexpr int VD = Tile::VD, OST = HD + 4;
  extern __shared__ __attribute__((aligned(16))) float xo[];  // [RWV][DR][OST]
  __shared__ float ml[RWV][DR][2];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % p.KH, rest = blockIdx.x / p.KH;
  const int id = rest % p.ntile, z = rest / p.ntile;
  RowTile t;
  if (!find_tile<DR>(p, id, t)) return;
  const KeyTiles kt = key_tiles(t);
  const int v0 = z * p.cpt, v1 = min(kt.n, v0 + p.cpt);
  if (z > 0 && v0 >= kt.n) return;

  // this lane's query row
  const int fr = t.r0 + min(c, t.rows - 1), tok = fr / p.G, h = kvh * p.G + fr % p.G;
  const int pos = t.pos0 + tok;
  const int klim = pos + 1, klo = p.window > 0 ? pos - p.window + 1 : 0;

  Tile kv;
  bool bad = false;
  const int32_t* tab = p.table + (int64_t)t.seq * p.table_ld;
  const int vw = v0 + wv;  // this wavefront's tiles: vw, vw + RWV, ..
  auto ask = [&](int it) {
    return page_ask(p, t, kt, tab, min(vw + RWV * (it + lane / 2), v1 - 1), lane & 1);
  };
  PageList pl = {};
  PageAsk next = {};
  // tile `it` of this wavefront
  auto load_k = [&](int it) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const int l = 2 * (it & 31) + kb;
      const E* base = (const E*)p.k + (uint64_t)lane_u32(pl.row, l) * HD;
      kv.load_k(kb, base + page_row(lane_u32(pl.vis, l), c) * HD, g);
    }
  };
  auto load_v = [&](int it) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const int l = 2 * (it & 31) + kb;
      const E* base = (const E*)p.v + (uint64_t)lane_u32(pl.row, l) * HD;
      const uint32_t vis = lane_u32(pl.vis, l);
#pragma unroll
      for (int r = 0; r < 4; ++r) kv.load_v(4 * kb + r, base + page_row(vis, 4 * g + r) * HD, c);
    }
  };
  if (vw < v1) {
    pl = page_place(p, t, kvh, ask(0), bad);
    load_k(0);
    load_v(0);
    next = ask(32);
  }
  kv.load_q(p.q, (int64_t)(t.row0 + tok) * p.q_ld + h * HD, g);
  f32x4_t o[VD];
#pragma unroll
  for (int i = 0; i < VD; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m_run = -FLT_MAX, l_run = 0.f;  // log2 domain; l_run: this lane's keys

  for (int it = 0, v = vw; v < v1; ++it, v += RWV) {
    const bool more = v + RWV < v1;
    const int b = tile_base(t, kt, v);
    if (more && (it & 31) == 31) {
      pl = page_place(p, t, kvh, next, bad);
      next = ask(it + 33);
    }
    f32x4_t sc[2] = {kv.scores(0), kv.scores(1)};
    if (more) load_k(it + 1);
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = b + 16 * (e >> 2) + 4 * g + (e & 3);
      const bool seen = j < klim && (j >= klo || j < p.sinks);
      sc[e >> 2][e & 3] = seen ? sc[e >> 2][e & 3] : -INFINITY;
      mx = fmaxf(mx, sc[e >> 2][e & 3]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * p.cs;
    // the running maximum moves only when a score passes it by 2^8, so that
    // most tiles leave O as it is; probabilities stay below 2^8
    if (__any(mx > m_run + 8.f)) {
      const float m_new = fmaxf(m_run, mx);
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < VD; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[i][r] *= alpha;
      m_run = m_new;
    }
    float pv[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      pv[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e >> 2][e & 3], p.cs, -m_run));
      l_run += pv[e];
    }
    kv.add_values(pv, o);
    if (more) load_v(it + 1);
  }

  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  if (__any(bad)) l_run = NAN;
  float* xr = xo + (wv * DR + c) * OST;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int i = 0; i < VD; i += 4)
      *(float4*)(xr + Tile::vdim(4 * g + r, i)) =
          make_float4(o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]);
  if (g == 0) {
    ml[wv][c][0] = m_run;
    ml[wv][c][1] = l_run;
  }
  __syncthreads();
  // a thread per row and four head dims, the wavefronts' sums in their order
  for (int w = tid; w < t.rows * (HD / 4); w += 64 * RWV) {
    const int r = w / (HD / 4), d = 4 * (w % (HD / 4));
    float m = -FLT_MAX, l = 0.f;
#pragma unroll
    for (int k = 0; k < RWV; ++k) m = fmaxf(m, ml[k][r][0]);
    float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < RWV; ++k) {
      const float f = exp2f(ml[k][r][0] - m);
      const float4 x = *(const float4*)(xo + (k * DR + r) * OST + d);
      l += f * ml[k][r][1];
      a[0] += f * x.x;
      a[1] += f * x.y;
      a[2] += f * x.z;
      a[3] += f * x.w;
    }
    if (kt.n > p.cpt) {  // several parts: left for k_paged_merge
      float* P0 = p.part + ((int64_t)(id * p.KH + kvh) * p.nsplit + z) * part_floats<HD>(DR);
      *(float4*)(P0 + r * HD + d) = make_float4(a[0], a[1], a[2], a[3]);
      if (d == 0) *(float2*)(P0 + DR * HD + 2 * r) = make_float2(m, l);
      continue;
    }
    const float inv = inv_sum(l);
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] *= inv;
    const int rr = t.r0 + r;
    store_row4<QF>(p, t.row0 + rr / p.G, (kvh * p.G + rr % p.G) * HD + d, a);
  }
}

// The parts of a row tile's keys joined in order: a thread per row and four
// head dims. Up to 8 parts take one round trip, issued before the lengths that
// say how many there are have come (the others' memory is there, unused).
template <int HD, bool QF, int RT>
__global__ __launch_bounds__(256) void k_paged_merge(PagedArgs p) {
  constexpr int PER = 1024 / HD;  // rows a workgroup takes
  constexpr int64_t PF = part_floats<HD>(RT);
  const int sub = blockIdx.x % (RT / PER), item = blockIdx.x / (RT / PER);
  const int kvh = item % p.KH, id = item / p.KH;
  const int r = sub * PER + threadIdx.x / (HD / 4), d = 4 * (threadIdx.x % (HD / 4));
  const float* P0 = p.part + (int64_t)item * p.nsplit * PF;
  float2 s[8];
  float4 x[8];
  auto load = [&](int k0) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k0 + k < p.nsplit) {
        s[k] = *(const float2*)(P0 + (k0 + k) * PF + RT * HD + 2 * r);
        x[k] = *(const float4*)(P0 + (k0 + k) * PF + r * HD + d);
      }
  };
  load(0);
  RowTile t;
  if (!find_tile<RT>(p, id, t)) return;
  const KeyTiles kt = key_tiles(t);
  if (kt.n <= p.cpt || r >= t.rows) return;  // (written by the attention kernel itself)
  const int n = (kt.n + p.cpt - 1) / p.cpt;
  float m = -FLT_MAX, l = 0.f;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < n; k0 += 8) {
    if (k0 > 0) load(k0);
    float top = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = k0 + k < n ? fmaxf(top, s[k].x) : top;
    const float f = exp2f(m - top);
    m = top;
    l *= f;
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] *= f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k0 + k >= n) break;
      const float w = exp2f(s[k].x - m);
      l += w * s[k].y;
      a[0] += w * x[k].x;
      a[1] += w * x[k].y;
      a[2] += w * x[k].z;
      a[3] += w * x[k].w;
    }
  }
  const float inv = inv_sum(l);
#pragma unroll
  for (int e = 0; e < 4; ++e) a[e] *= inv;
  const int rr = t.r0 + r;
  store_row4<QF>(p, t.row0 + rr / p.G, (kvh * p.G + rr % p.G) * HD + d, a);
}

// ------------------------------------------------------------ many rows
// For chunks of new tokens: 128 flattened rows a tile, 32 to each of four
// wavefronts, which all go through the same keys, a 32-key tile a step.
// v_mfma_f32_32x32x16_bf16 with S^T = K Q^T and O^T = V^T P^T: lane 32 g + c
// holds query row c of its wavefront. The key rows of a 32-key tile are taken
// with bits 2 and 3 of their number swapped, so that a lane's scores 8 s .. 8 s +
// 7 are keys 16 s + 8 g .., which are its K slots of the second product:
// probabilities never leave their registers. V^T's operand is read from the
// row-major value rows by the LDS's transposing reads (ds_read_b64_tr_b16).
//
// bf16 pages go memory -> LDS by DMA into two buffers, the next step's rows
// landing while this one's are used; fp32 ones through registers, cut into
// three bf16 terms once for the whole workgroup, into one buffer.
// Bound by a step's three chains, which take much the same time: 16 MFMAs, the
// softmax of 16 scores a lane, and 16 KB of LDS reads a wavefront (64 rows a
// wavefront would halve those: their scores and outputs do not fit the
// registers). bf16 prompts, 387 GF: 430 us, 900 TFLOP/s (a library matrix
// product 1360). fp32 rows and pages take six MFMAs a product, on bf16 pages
// three: one prompt of 2048 tokens on 6 heads of 128, 6.4 GF, 75 and 46 us; 5.2 GF
// of mixed fp32 chunks 70 us, and 7.5 for the merge.

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

template <int HD, bool QF, bool KF>
struct Many {
  static constexpr int RT = 128;  // rows of a tile, 32 a wavefront
  static constexpr int NA = KF ? 3 : 1;
  static constexpr int SK = 32;       // keys a step
  static constexpr int ROW = 2 * HD;  // bytes of a K or V row in LDS
  static constexpr int PLANE = SK * ROW;
  static constexpr int STAGE = 2 * NA * PLANE;  // K planes, V planes
  static constexpr int LDS = (KF ? 1 : 2) * STAGE;
  static constexpr int WAVES = QF ? 2 : 3;  // a SIMD
};

// key held by operand row i of a 32-key tile (bits 2 and 3 swapped)
__device__ __forceinline__ int tile_key(int i) { return (i & ~12) | ((i & 4) << 1) | ((i & 8) >> 1); }
// 16-byte slot of chunk c of row r: 16 rows read at one chunk lie in different
// banks (K), four rows read over 64 bytes too (V, the transposing reads)
template <int HD>
__device__ __forceinline__ int kslot(int r, int c) { return HD == 128 ? c ^ (r & 15) : c ^ ((r >> 1) & 7); }
template <int HD>
__device__ __forceinline__ int vslot(int r, int c) {
  return HD == 128 ? c ^ ((r & 3) << 2) : c ^ (((r >> 1) & 1) << 2);
}

__device__ __forceinline__ float swap_max(float v) {
  const uint32_t u = bits(v);
  const auto w = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
}
__device__ __forceinline__ float swap_sum(float v) {
  const uint32_t u = bits(v);
  const auto w = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(w[0]) + __uint_as_float(w[1]);
}

template <int NA, int N>
__device__ __forceinline__ f32x16_t mma32(const bf16x8_t (&a)[NA], const Terms<N>& b, f32x16_t c) {
#pragma unroll
  for (int o = 2; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (o - i >= 0 && o - i < N)
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b.t[o - i], c, 0, 0, 0);
  return c;
}

template <class T>
__device__ __forceinline__ T lds_at(uint32_t at) {
  return *(const __attribute__((address_space(3))) T*)(uintptr_t)at;
}
__device__ __forceinline__ s16x4_t lds_tr(uint32_t at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(uintptr_t)at);
}

template <int HD, bool QF, bool KF>
__global__ __launch_bounds__(256, (Many<HD, QF, KF>::WAVES)) void k_paged_many(PagedArgs p) {
  typedef Many<HD, QF, KF> C;
  constexpr int NS = HD / 16, ND = HD / 32, NA = C::NA, SK = C::SK, ROW = C::ROW,
                PLANE = C::PLANE, PER = 32;  // steps whose blocks a list holds
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, c = lane & 31;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % p.KH, rest = blockIdx.x / p.KH;
  const int id = p.ntile - 1 - rest % p.ntile, z = rest / p.ntile;  // longest tiles first
  RowTile t;
  if (!find_tile<C::RT>(p, id, t)) return;
  const KeyTiles kt = key_tiles(t);
  const int v0 = z * p.cpt, v1 = min(kt.n, v0 + p.cpt);
  if (z > 0 && v0 >= kt.n) return;
  const int nstep = v1 - v0;

  bool bad = false;
  const int32_t* tab = p.table + (int64_t)t.seq * p.table_ld;
  // block b of step st is lane 2 (st % PER) + b of the step's list
  auto ask = [&](int st) __attribute__((always_inline)) {
    return page_ask(p, t, kt, tab, min(v0 + st + lane / 2, v1 - 1), lane & 1);
  };
  PageList pl = {};  // of the step that is fetched next
  PageAsk next = {};
  auto turn = [&](int st) __attribute__((always_inline)) {  // pl for step st, in order
    if (st % PER == 0 && st > 0) {
      pl = page_place(p, t, kvh, next, bad);
      next = ask(st + PER);
    }
  };

  // ---- staging
  // bf16: rows of one 1 KB DMA group (RPG of them) lie in one block; this
  // wavefront fills groups wv, wv + 4, ..
  constexpr int RPG = 1024 / ROW, GPP = PLANE / 1024;  // rows a group, groups a plane
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_off(lds));
  auto fill = [&](int st, uint32_t to) __attribute__((always_inline)) {
    turn(st);
#pragma unroll
    for (int q = 0; q < GPP / 4; ++q) {
      const int grp = wv + 4 * q, r = grp * RPG + lane / (ROW / 16), slot = lane % (ROW / 16);
      const int at = 2 * (st % PER) + grp * RPG / 16;
      const uint64_t row = (uint64_t)lane_u32(pl.row, at) * HD;
      const int x = page_row(lane_u32(pl.vis, at), r & 15) * HD;
      dma16((const uint16_t*)p.k + row + (x + kslot<HD>(r, slot) * 8), lds0 + to + grp * 1024);
      dma16((const uint16_t*)p.v + row + (x + vslot<HD>(r, slot) * 8), lds0 + to + PLANE + grp * 1024);
    }
  };
  // fp32: this thread's 8-value chunks of both planes' rows, loaded a step ahead
  constexpr int CH = HD / 8, RPT = 256 / CH, NT = SK / RPT;  // chunks a row, rows at once, rounds
  float4 raw[KF ? NT : 1][4];
  auto fetch = [&](int st) __attribute__((always_inline)) {
    turn(st);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int r = i * RPT + tid / CH;
      // (a wavefront's rows lie in one block)
      const int at = 2 * (st % PER) + __builtin_amdgcn_readfirstlane(r / 16);
      const int off = page_row(lane_u32(pl.vis, at), r & 15) * HD + (tid % CH) * 8;
      const uint64_t row = (uint64_t)lane_u32(pl.row, at) * HD;
      const float* kp = (const float*)p.k + row + off;
      const float* vp = (const float*)p.v + row + off;
      raw[i][0] = *(const float4*)kp;
      raw[i][1] = *(const float4*)(kp + 4);
      raw[i][2] = *(const float4*)vp;
      raw[i][3] = *(const float4*)(vp + 4);
    }
  };
  auto put = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int r = i * RPT + tid / CH;
#pragma unroll
      for (int kvi = 0; kvi < 2; ++kvi) {
        const float4 a = raw[i][2 * kvi], b = raw[i][2 * kvi + 1];
        const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        bf16x8_t w[3];
        split3(x, w);
        const int slot = kvi ? vslot<HD>(r, tid % CH) : kslot<HD>(r, tid % CH);
#pragma unroll
        for (int k = 0; k < 3; ++k)
          *(bf16x8_t*)(lds + (3 * kvi + k) * PLANE + r * ROW + slot * 16) = w[k];
      }
    }
  };

  // ---- this lane's query row
  const int w0 = 32 * wv;  // the wavefront's first row of the tile
  const bool active = w0 < t.rows;
  const int fr = t.r0 + min(w0 + c, t.rows - 1), tok = fr / p.G, h = kvh * p.G + fr % p.G;
  const int klim = t.pos0 + tok + 1, klo = p.window > 0 ? klim - p.window : 0;
  QTerms<QF> q[NS];
  {
    const int64_t at = (int64_t)(t.row0 + tok) * p.q_ld + h * HD + 8 * g;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      if constexpr (QF) {
        const float* qp = (const float*)p.q + at + 16 * s;
        const float4 x0 = *(const float4*)qp, x1 = *(const float4*)(qp + 4);
        const float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
        q[s].set(x);
      } else {
        q[s].t[0] = __builtin_bit_cast(bf16x8_t, *(const u32x4v_t*)((const uint16_t*)p.q + at + 16 * s));
      }
    }
  }
  // positions of the wavefront's first and last row: which tiles need no mask
  const int wp0 = t.pos0 + (t.r0 + min(w0, t.rows - 1)) / p.G;
  const int wp1 = t.pos0 + (t.r0 + min(w0 + 32, t.rows) - 1) / p.G;

  // ---- operand places in LDS (of buffer 0; a step's buffer and rows are
  // added as constants). K: row tile_key(c), chunk 2 s + g. V: row 8 g + r3 of
  // each 16, dims 32 i + 16 (lane / 16 % 2) + 4 (lane % 4).
  uint32_t ka[NS], va[ND];
#pragma unroll
  for (int s = 0; s < NS; ++s) ka[s] = lds0 + tile_key(c) * ROW + kslot<HD>(tile_key(c), 2 * s + g) * 16;
  const int vr = 8 * g + ((lane >> 2) & 3);
#pragma unroll
  for (int i = 0; i < ND; ++i)
    va[i] = lds0 + NA * PLANE + vr * ROW +
            vslot<HD>(vr, 4 * i + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) * 16 + 8 * (lane & 1);

  f32x16_t o[ND];
  float m_run = -FLT_MAX, l_run = 0.f;
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.f;

  // S^T of the step's keys in K buffer `to`
  auto scores = [&](uint32_t to, f32x16_t& sc) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 16; ++r) sc[r] = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      bf16x8_t a[NA];
#pragma unroll
      for (int k = 0; k < NA; ++k) a[k] = lds_at<bf16x8_t>(ka[s] + to + k * PLANE);
      sc = mma32(a, q[s], sc);
    }
  };
  // masks where some row does not see the whole of step st's tile, and moves
  // the running maximum (only past a score 2^8 above it, as in k_paged_few)
  auto settle = [&](int st, f32x16_t& sc) __attribute__((always_inline)) {
    const int b = tile_base(t, kt, v0 + st);  // the tile's first key
    if (b + 31 > wp0 || (p.window > 0 && b <= wp1 - p.window)) {
      const int first = b + 8 * g;  // (this lane's keys are first + 0 .. 7 and 16 .. 23)
      int end = klim - first, from = klo - first, sink = p.sinks - first;
      // (keeps the compares in the branch: most steps are seen whole)
      asm volatile("" : "+v"(end), "+v"(from), "+v"(sink));
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int x = 16 * (r >> 3) + (r & 7);
        const bool seen = x < end && (x >= from || x < sink);
        sc[r] = seen ? sc[r] : -INFINITY;
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[r]);
    mx = swap_max(mx) * p.cs;
    if (__any(mx > m_run + 8.f)) {
      const float m_new = fmaxf(m_run, mx);
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
      m_run = m_new;
    }
  };
  // the probabilities' operands of the tile's two 16-key halves, and their sum
  auto weigh = [&](const f32x16_t& sc, PTerms<QF, true> (&pt)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * s + e], p.cs, -m_run));
      pt[s].set(x);
#pragma unroll
      for (int e = 0; e < 8; ++e) l_run += x[e];
    }
  };
  // O^T += V^T P^T from V buffer `to`
  auto add_values = [&](uint32_t to, const PTerms<QF, true> (&pt)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        bf16x8_t a[NA];
#pragma unroll
        for (int k = 0; k < NA; ++k)
          a[k] = __builtin_bit_cast(
              bf16x8_t, __builtin_shufflevector(lds_tr(va[i] + to + k * PLANE + 16 * s * ROW),
                                                lds_tr(va[i] + to + k * PLANE + (16 * s + 4) * ROW), 0, 1, 2,
                                                3, 4, 5, 6, 7));
        o[i] = mma32(a, pt[s], o[i]);
      }
  };

  if (nstep > 0) {
    pl = page_place(p, t, kvh, ask(0), bad);
    if constexpr (KF) fetch(0);
    else fill(0, 0);
    next = ask(PER);
  }
  auto step = [&](auto buf, int st) __attribute__((always_inline)) {
    constexpr uint32_t here = decltype(buf)::value * C::STAGE;
    if constexpr (KF) {
      if (st > 0) __syncthreads();  // (every wavefront is done with the last step)
      put();
      __syncthreads();
      if (st + 1 < nstep) fetch(st + 1);
    } else {
      stage_sync<0>();  // this step has landed, and nobody reads the other buffer
      if (st + 1 < nstep) fill(st + 1, C::STAGE - here);
    }
    if (!active || tile_base(t, kt, v0 + st) > wp1) return;  // (behind the wavefront's rows)
    f32x16_t sc;
    scores(here, sc);
    settle(st, sc);
    PTerms<QF, true> pt[2];
    weigh(sc, pt);
    add_values(here, pt);
  };
  for (int st = 0; st < nstep; st += 2) {
    step(std::integral_constant<int, 0>(), st);
    if (st + 1 < nstep) step(std::integral_constant<int, KF ? 0 : 1>(), st + 1);
  }
  if (!active) return;

  const bool whole = kt.n <= p.cpt;
  float* P0 = p.part + ((int64_t)(id * p.KH + kvh) * p.nsplit + z) * part_floats<HD>(C::RT);
  const int r = w0 + c;
  float l = swap_sum(l_run);
  if (__any(bad)) l = NAN;
  if (r >= t.rows) return;
  const float f = whole ? inv_sum(l) : 1.f;
  const int64_t row = t.row0 + tok;
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = o[i][4 * r4 + e] * f;
      const int d = 32 * i + 8 * r4 + 4 * g;
      if (whole) store_row4<QF>(p, row, h * HD + d, v);
      else *(float4*)(P0 + r * HD + d) = make_float4(v[0], v[1], v[2], v[3]);
    }
  if (!whole && g == 0) *(float2*)(P0 + C::RT * HD + 2 * r) = make_float2(m_run, l);
}

// ------------------------------------------------------------ host side

// (a constant, not the current device's: a workspace asked for with one device
// current serves a launch on another)
constexpr int64_t CUS = 256;

struct Plan {
  bool many;
  bool one_tile;
  int rt;      // rows of a tile
  int ntile, nsplit, cpt;
  int64_t floats;
};

// The tiles of a launch and the parts its keys are cut into, from the bounds
// alone (lengths may differ under a captured launch).
//
// Which kernel: 16-row tiles keep a wavefront a 32-key tile, and read the keys
// once for each tile; 128-row tiles read them (fp32 ones: cut them) once for eight
// of those, but keep a whole workgroup where that has one. The latter take over
// past 32 rows a sequence from MANY_WORK (16-row tile, 32-key tile) pairs on. us,
// 16 rows -> 128: fp32 rows and pages, 6 heads, 64 tokens after 936 (768 pairs)
// 14.9 -> 22.2, 8 x 96 after 1404 (13.5k) 90 -> 53, 500 tokens (3k) 18.6 -> 25.7,
// 2048 (49k) 118 -> 75, on bf16 pages 50 -> 47; bf16 rows, 32 heads on 4, 8 x 8
// tokens after 1490 (6k) 17.9 -> 17.7, 256 after 7744 (128k) 146 -> 56. At 32
// rows, 32 sequences of a 2048-key window on 32 heads (17k) 36.5 -> 42.3.
// Parts: as many as fill the CUs once with 16-row tiles (twice: 500 fp32 tokens
// 18.6 -> 24.6, those 32 windows 36.5 -> 40.6), of at least a tile a wavefront
// (two: one token on 6 fp32 heads after 300 positions 10.8 -> 13.9, on bf16 pages
// after 1000 9.5 -> 10.2, after 4000 13.0 -> 12.1); twice with 128-row ones (once:
// chunks and tokens of 9 sequences, 10 heads on 2, 92 -> 123, one fp32 prompt of
// 2048 75 -> 95).
constexpr int64_t MANY_WORK = 6000;
Plan plan_of(const fg_pages& pg, const fg_ragged& b, const fg_attn_cfg& c) {
  Plan pl;
  const int64_t G = c.n_head / pg.n_kv_head;
  // (no sequence has more new tokens than there are rows, whatever the caller's
  // bound; G of them per row stay far below 2^31)
  const int64_t max_q = std::min(b.max_q, b.n_rows);
  auto tiles = [&](int64_t rt) {
    return std::min((max_q * G + rt - 1) / rt * b.n_seq, b.n_rows * G / rt + b.n_seq);
  };
  auto key_tiles_most = [&](int64_t rt) {
    int64_t keys = std::max(1, b.max_kv);  // (a cache of no position still has its rows written)
    if (c.window > 0)  // (a tile's tokens see this many at most, and the tiles at both ends)
      keys = std::min<int64_t>(keys, (int64_t)c.window + rt / G + 1 + c.sinks + 96);
    return (keys + 31) / 32;
  };
  pl.many = max_q * G > 32 && tiles(DR) * pg.n_kv_head * key_tiles_most(DR) > MANY_WORK;
  pl.rt = pl.many ? Many<128, true, true>::RT : DR;
  pl.one_tile = max_q * G <= pl.rt;
  pl.ntile = (int)tiles(pl.rt);
  const int64_t nkt = key_tiles_most(pl.rt), items = (int64_t)pl.ntile * pg.n_kv_head;
  const int64_t want = pl.many ? (2 * CUS + items - 1) / items : CUS / items;
  const int64_t ns = std::max<int64_t>(1, std::min(want, (nkt + RWV - 1) / RWV));
  pl.cpt = (int)((nkt + ns - 1) / ns + RWV - 1) / RWV * RWV;
  pl.nsplit = (int)std::max<int64_t>(1, (nkt + pl.cpt - 1) / pl.cpt);
  pl.floats = pl.nsplit > 1 ? items * pl.nsplit * pl.rt * (pg.head_dim + 2) : 0;
  return pl;
}

template <int HD, bool QF, bool KF>
void launch_few(hipStream_t s, const PagedArgs& a) {
  constexpr int lds = few_lds<HD>();
  static std::atomic<uint64_t> lds_set{0};
  raise_lds_once((const void*)k_paged_few<HD, QF, KF>, lds, &lds_set);
  FG_LAUNCH((k_paged_few<HD, QF, KF>), dim3((unsigned)(a.ntile * a.KH * a.nsplit)), dim3(64 * RWV),
            lds, s, a);
  if (a.nsplit > 1)
    FG_LAUNCH((k_paged_merge<HD, QF, DR>), dim3((unsigned)(a.ntile * a.KH * (DR * HD / 1024))),
              dim3(256), 0, s, a);
}

template <int HD, bool QF, bool KF>
void launch_many(hipStream_t s, const PagedArgs& a) {
  typedef Many<HD, QF, KF> C;
  static std::atomic<uint64_t> lds_set{0};
  raise_lds_once((const void*)k_paged_many<HD, QF, KF>, C::LDS, &lds_set);
  FG_LAUNCH((k_paged_many<HD, QF, KF>), dim3((unsigned)(a.ntile * a.KH * a.nsplit)), dim3(256), C::LDS,
            s, a);
  if (a.nsplit > 1)
    FG_LAUNCH((k_paged_merge<HD, QF, C::RT>), dim3((unsigned)(a.ntile * a.KH * (C::RT * HD / 1024))),
              dim3(256), 0, s, a);
}

template <int HD, bool QF, bool KF>
void launch_t(hipStream_t s, const PagedArgs& a, bool many) {
  if (many) launch_many<HD, QF, KF>(s, a);
  else launch_few<HD, QF, KF>(s, a);
}

template <int HD>
void launch_hd(hipStream_t s, const PagedArgs& a, bool many, bool qf, bool kf) {
  if (kf) launch_t<HD, true, true>(s, a, many);
  else if (qf) launch_t<HD, true, false>(s, a, many);
  else launch_t<HD, false, false>(s, a, many);
}

}  // namespace

int64_t paged_attn_floats(const fg_pages& pg, const fg_ragged& b, const fg_attn_cfg& c) {
  return plan_of(pg, b, c).floats;
}

void launch_paged_attn(hipStream_t s, const fg_pages& pg, const fg_ragged& b, const fg_attn_cfg& c,
                       const void* q, const PagedOut& out, float* work) {
  const Plan pl = plan_of(pg, b, c);
  PagedArgs a;
  a.k = pg.k;
  a.v = pg.v;
  a.q = q;
  a.out = out;
  a.q_ld = c.q_ld ? c.q_ld : (int64_t)c.n_head * pg.head_dim;
  a.q_start = b.q_start;
  a.kv_len = b.kv_len;
  a.table = b.table;
  a.n_seq = b.n_seq;
  a.n_rows = b.n_rows;
  a.max_q = std::min(b.max_q, b.n_rows);
  a.one_tile = pl.one_tile;
  a.max_kv = b.max_kv;
  a.table_ld = b.table_ld;
  a.n_pages = pg.n_pages;
  a.pshift = __builtin_ctz(pg.page_size);
  a.KH = pg.n_kv_head;
  a.G = c.n_head / pg.n_kv_head;
  a.window = c.window;
  a.sinks = c.sinks;
  a.cs = (c.scale != 0.f ? c.scale : 1.0f / sqrtf((float)pg.head_dim)) * LOG2E;
  a.ntile = pl.ntile;
  a.nsplit = pl.nsplit;
  a.cpt = pl.cpt;
  a.part = work;
  if (pg.head_dim == 128)
    launch_hd<128>(s, a, pl.many, c.type == FG_F32, pg.type == FG_F32);
  else
    launch_hd<64>(s, a, pl.many, c.type == FG_F32, pg.type == FG_F32);
}

}  // namespace fgpt
