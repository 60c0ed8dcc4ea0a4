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
  int H, KH, G;
  int window, sinks;
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
// 64 of them a step. False: no such tile.
template <int RT>
__device__ __forceinline__ bool find_tile(const PagedArgs& p, int id, RowTile& t) {
  const int lane = threadIdx.x & 63;
  auto q_of = [&](int s) {  // new tokens of sequence s, kept inside the arrays
    const int a = p.q_start[s], n = p.q_start[s + 1] - a;
    return a < 0 ? 0 : max(0, min(min(n, p.max_q), p.n_rows - a));
  };
  int first = 0, nq;
  if (p.max_q * p.G <= RT) {
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
  const int tile = p.max_q * p.G <= RT ? 0 : id - first;
  t.r0 = tile * RT;
  t.rows = min(RT, nq * p.G - t.r0);
  if (t.rows <= 0) return false;
  t.row0 = p.q_start[t.seq];
  t.kv = max(0, min(p.kv_len[t.seq], p.max_kv));
  t.pos0 = t.kv - (p.q_start[t.seq + 1] - t.row0);
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

template <bool QF>
struct Terms {  // of q and of the probabilities
  static constexpr int N = QF ? 3 : 1;
  bf16x8_t t[N];
  __device__ __forceinline__ void set(const float (&x)[8]) {
    if constexpr (QF) {
      split3(x, t);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) t[0][e] = (__bf16)x[e];
    }
  }
};

__device__ __forceinline__ f32x4_t mma16(const bf16x8_t& a, const bf16x8_t& b, const f32x4_t& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// c += a . b over the term products that matter: all of those whose terms'
// places add up to 2 at most (the others are below 2^-24 of the product),
// smallest first.
template <int NA, int NB>
__device__ __forceinline__ f32x4_t mma_terms(const bf16x8_t (&a)[NA], const bf16x8_t (&b)[NB], f32x4_t c) {
#pragma unroll
  for (int o = 2; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (o - i >= 0 && o - i < NB) c = mma16(a[i], b[o - i], c);
  return c;
}

// One 32-key tile's pieces of the K and V rows, as a lane (row c = lane % 16,
// group g = lane / 16) loads them, and the operands made of them. K step s of
// S^T = K Q^T covers head dims 32 s + KD g + .. of the lane's key; row c of
// O^T's i-th block stands for head dim vdim(c, i): both are chosen so that a
// lane's pieces are whole 16-byte (8 for head dim 64) loads of adjacent lanes.
template <int HD, bool KF>
struct KvTile;
template <int HD>
struct KvTile<HD, true> {
  static constexpr int NS = HD / 32, VD = HD / 16, N = 3;
  typedef float elem;
  static __device__ __forceinline__ int vdim(int c, int i) { return 64 * (i / 4) + 4 * c + i % 4; }
  static __device__ __forceinline__ int qdim(int s, int g, int half) { return 32 * s + 16 * half + 4 * g; }
  float4 k[2][NS][2], v[8][VD / 4];
  __device__ __forceinline__ void load_k(int kb, const float* row, int g) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) k[kb][s][h] = *(const float4*)(row + qdim(s, g, h));
  }
  __device__ __forceinline__ void load_v(int e, const float* row, int c) {
#pragma unroll
    for (int i = 0; i < VD / 4; ++i) v[e][i] = *(const float4*)(row + 64 * i + 4 * c);
  }
  __device__ __forceinline__ void kop(int kb, int s, bf16x8_t (&t)[3]) const {
    const float4 a = k[kb][s][0], b = k[kb][s][1];
    const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    split3(x, t);
  }
  __device__ __forceinline__ void vop(int i, bf16x8_t (&t)[3]) const {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float4 w = v[e][i / 4];
      x[e] = i % 4 == 0 ? w.x : i % 4 == 1 ? w.y : i % 4 == 2 ? w.z : w.w;
    }
    split3(x, t);
  }
};
template <int HD>
struct KvTile<HD, false> {
  static constexpr int NS = HD / 32, VD = HD / 16, N = 1;
  typedef uint16_t elem;
  static __device__ __forceinline__ int vdim(int c, int i) { return VD * c + i; }
  static __device__ __forceinline__ int qdim(int s, int g, int half) { return 32 * s + 8 * g + 4 * half; }
  typedef uint32_t vrow_t __attribute__((ext_vector_type(VD / 2)));
  u32x4v_t k[2][NS];
  vrow_t v[8];
  __device__ __forceinline__ void load_k(int kb, const uint16_t* row, int g) {
#pragma unroll
    for (int s = 0; s < NS; ++s) k[kb][s] = *(const u32x4v_t*)(row + 32 * s + 8 * g);
  }
  __device__ __forceinline__ void load_v(int e, const uint16_t* row, int c) {
    v[e] = *(const vrow_t*)(row + VD * c);
  }
  __device__ __forceinline__ void kop(int kb, int s, bf16x8_t (&t)[1]) const {
    t[0] = __builtin_bit_cast(bf16x8_t, k[kb][s]);
  }
  __device__ __forceinline__ void vop(int i, bf16x8_t (&t)[1]) const {
    u32x4v_t w;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = __builtin_amdgcn_perm(v[2 * e + 1][i / 2], v[2 * e][i / 2],
                                   i & 1 ? 0x07060302u : 0x05040100u);
    t[0] = __builtin_bit_cast(bf16x8_t, w);
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
// slots of its operand of O^T = V^T P^T. Pages hold 16 rows or a multiple, so
// a block's page is one scalar load.
// Bound by the cache's bytes: every visible key and value is read once.
constexpr int DR = 16, RWV = 8;

template <int HD>
constexpr int few_lds() { return RWV * DR * (HD + 4) * 4; }
template <int HD>
constexpr int64_t part_floats(int rows) { return (int64_t)rows * (HD + 2); }

template <int HD, bool QF, bool KF>
__global__ __launch_bounds__(64 * RWV) void k_paged_few(PagedArgs p) {
  typedef KvTile<HD, KF> Tile;
  typedef typename Tile::elem E;
  constexpr int NS = Tile::NS, VD = Tile::VD, OST = HD + 4;
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
  const int P = 1 << p.pshift;
  const int32_t* tab = p.table + (int64_t)t.seq * p.table_ld;
  auto base_of = [&](int v) { return v < kt.na ? 32 * v : kt.from + 32 * (v - kt.na); };
  // A 16-key block of a tile: where its rows lie, and which row to read in the
  // place of one that no query sees (its page is only known to be there where
  // some query sees a key of the block; a block without one reads the other).
  struct Block {
    int64_t off;  // element offset of its first row
    int e, sub;   // first key, substitute row
  };
  auto block_of = [&](int v, int kb) {
    Block k;
    k.e = base_of(v) + 16 * kb;
    if (k.e >= t.sa && (k.e >= t.hi || k.e + 16 <= t.lo)) k.e += 16 - 32 * kb;
    const int pg = tab[k.e >> p.pshift];
    const bool ok = (uint32_t)pg < (uint32_t)p.n_pages;
    bad |= !ok;
    k.off = (((int64_t)(ok ? pg : 0) * p.KH + kvh) * P + (k.e & (P - 1))) * HD;
    k.sub = k.e < t.sa ? 0 : max(0, t.lo - k.e);
    return k;
  };
  auto row_of = [&](const Block& k, int x) {
    const int j = k.e + x;
    return j < t.sa || (j >= t.lo && j < t.hi) ? x : k.sub;
  };
  auto load_k = [&](const Block (&bl)[2]) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
      kv.load_k(kb, (const E*)p.k + bl[kb].off + row_of(bl[kb], c) * HD, g);
  };
  auto load_v = [&](const Block (&bl)[2]) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      kv.load_v(e, (const E*)p.v + bl[e >> 2].off + row_of(bl[e >> 2], 4 * g + (e & 3)) * HD, c);
  };
  int v = v0 + wv;
  if (v < v1) {
    const Block bl[2] = {block_of(v, 0), block_of(v, 1)};
    load_k(bl);
    load_v(bl);
  }
  Terms<QF> q[NS];
  {
    const int64_t at = (int64_t)(t.row0 + tok) * p.q_ld + h * HD;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      if constexpr (QF) {
        const float* qp = (const float*)p.q + at;
        const float4 a = *(const float4*)(qp + Tile::qdim(s, g, 0));
        const float4 b = *(const float4*)(qp + Tile::qdim(s, g, 1));
        const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        q[s].set(x);
      } else {  // (bf16 pages: a step's eight dims are consecutive)
        q[s].t[0] = __builtin_bit_cast(
            bf16x8_t, *(const u32x4v_t*)((const uint16_t*)p.q + at + Tile::qdim(s, g, 0)));
      }
    }
  }
  f32x4_t o[VD];
#pragma unroll
  for (int i = 0; i < VD; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m_run = -FLT_MAX, l_run = 0.f;  // log2 domain; l_run: this lane's keys

  for (; v < v1; v += RWV) {
    const bool more = v + RWV < v1;
    Block nb[2] = {};
    if (more) {
      nb[0] = block_of(v + RWV, 0);
      nb[1] = block_of(v + RWV, 1);
    }
    const int b = base_of(v);
    f32x4_t sc[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      sc[kb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        bf16x8_t a[Tile::N];
        kv.kop(kb, s, a);
        sc[kb] = mma_terms(a, q[s].t, sc[kb]);
      }
    }
    if (more) load_k(nb);
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
    Terms<QF> pt;
    pt.set(pv);
#pragma unroll
    for (int i = 0; i < VD; ++i) {
      bf16x8_t a[Tile::N];
      kv.vop(i, a);
      o[i] = mma_terms(a, pt.t, o[i]);
    }
    if (more) load_v(nb);
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
  const int r = tid / (HD / 4), d = 4 * (tid % (HD / 4));
  if (r >= t.rows) return;
  float m = -FLT_MAX, l = 0.f;
#pragma unroll
  for (int k = 0; k < RWV; ++k) m = fmaxf(m, ml[k][r][0]);
  float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < RWV; ++k) {
    const float w = exp2f(ml[k][r][0] - m);
    const float4 x = *(const float4*)(xo + (k * DR + r) * OST + d);
    l += w * ml[k][r][1];
    a[0] += w * x.x;
    a[1] += w * x.y;
    a[2] += w * x.z;
    a[3] += w * x.w;
  }
  if (kt.n > p.cpt) {  // several parts: left for k_paged_merge
    float* P0 = p.part + ((int64_t)(id * p.KH + kvh) * p.nsplit + z) * part_floats<HD>(DR);
    *(float4*)(P0 + r * HD + d) = make_float4(a[0], a[1], a[2], a[3]);
    if (d == 0) *(float2*)(P0 + DR * HD + 2 * r) = make_float2(m, l);
    return;
  }
  const float inv = inv_sum(l);
#pragma unroll
  for (int e = 0; e < 4; ++e) a[e] *= inv;
  const int rr = t.r0 + r;
  store_row4<QF>(p, t.row0 + rr / p.G, (kvh * p.G + rr % p.G) * HD + d, a);
}

// The parts of a row tile's keys joined in order: one workgroup an item, a
// thread per row and four head dims.
template <int HD, bool QF, int RT>
__global__ __launch_bounds__(256) void k_paged_merge(PagedArgs p) {
  constexpr int PER = 1024 / HD;  // rows a workgroup takes
  const int sub = blockIdx.x % (RT / PER), item = blockIdx.x / (RT / PER);
  const int kvh = item % p.KH, id = item / p.KH;
  RowTile t;
  if (!find_tile<RT>(p, id, t)) return;
  const KeyTiles kt = key_tiles(t);
  if (kt.n <= p.cpt) return;  // written by the attention kernel itself
  const int r = sub * PER + threadIdx.x / (HD / 4), d = 4 * (threadIdx.x % (HD / 4));
  if (r >= t.rows) return;
  const int n = (kt.n + p.cpt - 1) / p.cpt;
  const float* P0 = p.part + (int64_t)(id * p.KH + kvh) * p.nsplit * part_floats<HD>(RT);
  float m = -FLT_MAX, l = 0.f;
  for (int k = 0; k < n; ++k) m = fmaxf(m, P0[k * part_floats<HD>(RT) + RT * HD + 2 * r]);
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < n; ++k) {
    const float* P = P0 + k * part_floats<HD>(RT);
    const float2 s = *(const float2*)(P + RT * HD + 2 * r);
    const float4 x = *(const float4*)(P + r * HD + d);
    const float w = exp2f(s.x - m);
    l += w * s.y;
    a[0] += w * x.x;
    a[1] += w * x.y;
    a[2] += w * x.z;
    a[3] += w * x.w;
  }
  const float inv = inv_sum(l);
#pragma unroll
  for (int e = 0; e < 4; ++e) a[e] *= inv;
  const int rr = t.r0 + r;
  store_row4<QF>(p, t.row0 + rr / p.G, (kvh * p.G + rr % p.G) * HD + d, a);
}

// ------------------------------------------------------------ host side

// (a constant, not the current device's: a workspace asked for with one device
// current serves a launch on another)
constexpr int64_t CUS = 256;

struct Plan {
  int rt;      // rows of a tile
  int ntile, nsplit, cpt;
  int64_t floats;
};

// The tiles of a launch and the parts its keys are cut into, from the bounds
// alone (lengths may differ under a captured launch).
Plan plan_of(const fg_pages& pg, const fg_ragged& b, const fg_attn_cfg& c) {
  Plan pl;
  pl.rt = DR;
  const int64_t G = c.n_head / pg.n_kv_head;
  const int64_t per_seq = (b.max_q * G + pl.rt - 1) / pl.rt;
  pl.ntile = (int)std::min<int64_t>(per_seq * b.n_seq, b.n_rows * G / pl.rt + b.n_seq);
  int64_t keys = b.max_kv;
  if (c.window > 0)  // (a tile's tokens see this many at most, and the tiles at both ends)
    keys = std::min<int64_t>(keys, (int64_t)c.window + pl.rt / G + 1 + c.sinks + 96);
  const int64_t nkt = (keys + 31) / 32;
  // parts: enough workgroups for two a CU, each with a round of its
  // wavefronts' tiles at least
  const int64_t items = (int64_t)pl.ntile * pg.n_kv_head;
  const int64_t want = (2 * CUS + items - 1) / items;
  const int64_t most = (nkt + RWV - 1) / RWV;
  const int64_t ns = std::max<int64_t>(1, std::min(want, most));
  pl.cpt = (int)((nkt + ns - 1) / ns + RWV - 1) / RWV * RWV;
  pl.nsplit = (int)((nkt + pl.cpt - 1) / pl.cpt);
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

template <int HD>
void launch_hd(hipStream_t s, const PagedArgs& a, bool qf, bool kf) {
  if (kf)
    launch_few<HD, true, true>(s, a);
  else if (qf)
    launch_few<HD, true, false>(s, a);
  else
    launch_few<HD, false, false>(s, a);
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
  a.max_q = b.max_q;
  a.max_kv = b.max_kv;
  a.table_ld = b.table_ld;
  a.n_pages = pg.n_pages;
  a.pshift = __builtin_ctz(pg.page_size);
  a.H = c.n_head;
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
    launch_hd<128>(s, a, c.type == FG_F32, pg.type == FG_F32);
  else
    launch_hd<64>(s, a, c.type == FG_F32, pg.type == FG_F32);
}

}  // namespace fgpt
