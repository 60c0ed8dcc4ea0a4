// kern_draw.hip -- one id a row under temperature, top-k, top-p and min-p from
// given uniform numbers (fg_draw_rows of include/fgpt.h).
//
// No sort: each of the three filters keeps a prefix of the row in its order
// (descending logits, ties by ascending id), so top-k and top-p are a cut, the
// last id kept, and min-p is a bound on the masses. Where the cut lies is found
// from one histogram of counts and masses over bins of equal width in
// (max - x) / temp: the bin in which top_k's count or top_p's mass is reached,
// then the place within it by comparing its few ids with each other (a bin of
// more than LIST ids, as rows of many equal logits have, goes by digits
// instead). The kept mass is then summed by chunks of 64 ids, in id order, and
// the draw scans those.
//
// Masses are integers, e_i = exp((x_i - max) / temp) in steps of 2^-44 (sums of
// up to 2^18 of them fit 64 bits), so every sum is exact in any order: atomics
// may add them as they come, and an id next to a border of the cumulative mass
// comes out the same in every run. 32-bit sums would misplace about n 2^-24 of
// the draws of a row with n likely ids.
//
// A workgroup a row. Up to 8192 ids the row stays in registers and the time is
// that of the chain of block-wide steps (one row 15 us, 64 of 8192 ids 16.6);
// past that it is the exponentials'.
#include <algorithm>

#include "fgpt_internal.h"
#include "kern_common.h"
#include "paged_internal.h"

namespace fgpt {
namespace {

typedef unsigned long long u64;

constexpr int DT = 1024, DW = DT / 64;  // threads, wavefronts
constexpr int PER = 8;                  // ids a thread holds in registers
constexpr int BINS = 2 * DT;
constexpr float BIN_UNITS = 64.f;       // bins per unit of (max - x) / temp: 32 units in all
constexpr int LIST = 512;               // ids of one bin that are compared with each other
constexpr int TAB = 1024;
constexpr int MAX_CHUNKS = DRAW_MAX_V / 64;
constexpr int ID_BITS = 18;             // DRAW_MAX_V ids

struct DrawArgs {
  const float* x;
  int V;
  int64_t ld;
  fg_draw_cfg c;
  int32_t* ids;
  float* probs;
};

// Order-preserving integers of the logits (no NaN here; -0 counts as +0).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

// v of the lane that DPP control CTRL names, 0 where that is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_or_0(u64 v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
  return ((u64)hi << 32) | lo;
}
// Inclusive sums by lane: within rows of 16 lanes by row shifts, then the last
// lane of a row to the next row, of the first half to the second.
__device__ __forceinline__ u64 wave_scan(u64 v) {
  v += dpp_or_0<0x111, 0xF>(v);
  v += dpp_or_0<0x112, 0xF>(v);
  v += dpp_or_0<0x114, 0xF>(v);
  v += dpp_or_0<0x118, 0xF>(v);
  v += dpp_or_0<0x142, 0xA>(v);  // row_bcast15 into rows 1 and 3
  v += dpp_or_0<0x143, 0xC>(v);  // row_bcast31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ u64 lane_value(u64 v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
  return ((u64)hi << 32) | lo;
}

// The place of an id in the row's order: ascending (max key - key, id).
typedef u64 place_t;

struct Shared {
  unsigned int cnt[BINS];
  u64 mass[BINS];
  double tab[TAB];  // 2^(j / TAB)
  place_t list_at[LIST];
  u64 list_mass[LIST], list_sum[LIST];
  unsigned int list_rank[LIST];
  u64 red[2][DW];
  float redf[DW];
  int redi[DW];
  u64 found[4];
  int n_list;
};

struct Row {  // what a row's threads share
  const float* x;
  int V;
  float m;      // largest logit (may be +inf)
  uint32_t km;  // its key
  double unit;  // TAB / (ln 2 temp)
  float bin;    // BIN_UNITS / temp
  const double* tab;
  // exp((v - m) / temp) in steps of 2^-44: with y = (v - m) unit = n + f, |f| <=
  // 1/2, 2^(n / TAB) from the table times 2^(f / TAB), f's Taylor sum to degree 3
  // (the next term is below 6e-16). The addition of 2^52 rounds to an integer.
  __device__ __forceinline__ u64 mass(float v) const {
    if (v == m) return 1ull << 44;
    const double y = ((double)v - (double)m) * unit;
    if (!(y > -45.0 * TAB)) return 0;
    const double n = rint(y), f = y - n;
    constexpr double L = 0.69314718055994530942 / TAB;
    double s = fma(f, L * L * L / 6, L * L / 2);
    s = fma(f, s, L);
    s = fma(f, s, 1.0);
    const int k = (int)n;
    const double e = ldexp(s * tab[k & (TAB - 1)], 44 + (k >> 10));
    return (u64)__double_as_longlong(e + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
  }
  __device__ __forceinline__ int bin_of(float v) const {  // does not fall as v falls
    const float b = (m - v) * bin;
    return v == m ? 0 : b < (float)(BINS - 1) ? (int)b : BINS - 1;  // (NaN: the last)
  }
  __device__ __forceinline__ place_t place(float v, int i) const {
    return ((place_t)(km - key_of(v)) << ID_BITS) | (uint32_t)i;
  }
  __device__ __forceinline__ float value(place_t at) const {  // the logit at a place
    const uint32_t k = km - (uint32_t)(at >> ID_BITS);
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
  }
};

__device__ __forceinline__ bool drawable(float v) { return v > -INFINITY; }  // (false for NaN)

// f(v, i) for this thread's ids of [lo, hi) (lo a multiple of 64); HELD: of the
// whole row, from registers. Past the end it sees -inf, which is never drawn.
template <bool HELD, class F, int AHEAD = HELD ? PER : 16>
__device__ __forceinline__ void each(const Row& row, const float (&held)[PER], int lo, int hi, F&& f) {
  if constexpr (HELD) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      f(held[k], k * DT + (int)threadIdx.x);
    }
  } else {
    for (int i0 = lo + (int)threadIdx.x; i0 < hi; i0 += AHEAD * DT) {
      float v[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) v[k] = i0 + k * DT < hi ? row.x[i0 + k * DT] : -INFINITY;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) f(v[k], i0 + k * DT);
    }
  }
}

// Sums of the threads' a and b before this one, and of all threads.
__device__ void block_scan2(Shared& s, u64& a, u64& b, u64& all_a, u64& all_b) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const u64 ia = wave_scan(a), ib = wave_scan(b);
  if (lane == 63) {
    s.red[0][wv] = ia;
    s.red[1][wv] = ib;
  }
  __syncthreads();
  const u64 wa = wave_scan(lane < DW ? s.red[0][lane] : 0), wb = wave_scan(lane < DW ? s.red[1][lane] : 0);
  a = ia - a + (wv ? lane_value(wa, wv - 1) : 0);
  b = ib - b + (wv ? lane_value(wb, wv - 1) : 0);
  all_a = lane_value(wa, 63);
  all_b = lane_value(wb, 63);
}

// The n <= LIST places of s.list_at in ascending order, entry tid of them (past
// n: ~0): a bitonic network on as many wavefronts as they need, whose exchanges
// across 64 entries and more go through LDS. (k_draw_cut with lists of about
// 400: 11 us; 24 by comparing the entries with each other.)
__device__ place_t sort_list(Shared& s, unsigned n) {
  const int tid = threadIdx.x;
  place_t v = tid < (int)n ? s.list_at[tid] : ~0ull;
  int n2 = 64;
  while (n2 < (int)n) n2 <<= 1;
#pragma unroll 1
  for (int k = 2; k <= n2; k <<= 1) {
#pragma unroll 1
    for (int j = k >> 1; j > 0; j >>= 1) {
      place_t o = v;
      if (j >= 64) {
        __syncthreads();
        if (tid < n2) s.list_at[tid] = v;
        __syncthreads();
        if (tid < n2) o = s.list_at[tid ^ j];
      } else if (tid < n2) {
        o = __shfl_xor(v, j, 64);
      }
      v = (v < o) == (((tid & k) == 0) == ((tid & j) == 0)) ? v : o;
    }
  }
  return v;
}

// For entry tid of the n in the list: how many come before it in the row's order,
// and their mass. Each entry is compared with all others, by as many threads as
// there are for one (their shares meet in LDS). Sorting them as k_draw_cut does
// takes more steps of the workgroup than it saves where the row's lists are short
// (64 rows of 8192 ids 16.6 us so, 18.6 sorted).
__device__ __forceinline__ void rank_in_list(Shared& s, unsigned n, u64& rank, u64& mass) {
  const int tid = threadIdx.x;
  rank = mass = 0;
  if (n <= 64) {  // (not worth the meeting)
    if (tid < (int)n) {
      const place_t mine = s.list_at[tid];
#pragma unroll 4
      for (unsigned k = 0; k < n; ++k) {
        const bool first = s.list_at[k] < mine;
        rank += first ? 1 : 0;
        mass += first ? s.list_mass[k] : 0;
      }
    }
    return;
  }
  int n2 = 128;
  while (n2 < (int)n) n2 <<= 1;
  const int e = tid & (n2 - 1), part = tid / n2, parts = DT / n2;
  if (tid < LIST) {
    s.list_rank[tid] = 0;
    s.list_sum[tid] = 0;
  }
  __syncthreads();
  if (e < (int)n) {
    const place_t mine = s.list_at[e];
    unsigned r = 0;
    u64 w = 0;
#pragma unroll 8
    for (unsigned k = part; k < n; k += parts) {
      const bool first = s.list_at[k] < mine;
      r += first ? 1 : 0;
      w += first ? s.list_mass[k] : 0;
    }
    if (r) {
      atomicAdd(&s.list_rank[e], r);
      atomicAdd(&s.list_sum[e], w);
    }
  }
  __syncthreads();
  rank = tid < (int)n ? s.list_rank[tid] : 0;
  mass = tid < (int)n ? s.list_sum[tid] : 0;
}

// Where, in the row's order, the counts (or masses) first reach `want` >= 1:
// the place of that id, within the bin `b` before which `before` lies. mass_to
// gets the bin's mass up to and with it.
template <bool HELD>
__device__ place_t place_at(Shared& s, const Row& row, const float (&held)[PER], bool masses, u64 want,
                            int b, u64 before, u64* mass_to) {
  const int tid = threadIdx.x;
  const u64 left = want - before;
  const unsigned n = s.cnt[b];
  __syncthreads();  // (found and cnt are read)
  if (n <= LIST) {
    if (tid == 0) s.n_list = 0;
    __syncthreads();
    const float near = (float)b, far = b < BINS - 1 ? (float)(b + 1) : NAN;
    each<HELD>(row, held, 0, row.V, [&](float v, int i) {
      const float t = (row.m - v) * row.bin;
      if (t < near || t >= far) return;  // (most ids; what is left is looked at again)
      if (row.bin_of(v) != b || !drawable(v)) return;
      const int at = atomicAdd(&s.n_list, 1);
      s.list_at[at] = row.place(v, i);
      s.list_mass[at] = row.mass(v);
    });
    __syncthreads();
    u64 rank, mass;
    rank_in_list(s, n, rank, mass);
    if (tid < (int)n && (masses ? mass < left && left <= mass + s.list_mass[tid] : rank == left - 1)) {
      s.found[0] = s.list_at[tid];
      s.found[1] = mass + s.list_mass[tid];
    }
    __syncthreads();
    *mass_to = s.found[1];
    return s.found[0];
  }
  // by the digits of the places: 11, 11 and 10 bits of the key, 9 and 9 of the id
  constexpr int widths[5] = {11, 11, 10, 9, 9};
  place_t prefix = 0;
  u64 above_c = 0, above_m = 0;
  int shift = 32 + ID_BITS;
#pragma unroll 1
  for (int k = 0; k < 5; ++k) {
    const int width = widths[k];
    shift -= width;
    s.cnt[2 * tid] = s.cnt[2 * tid + 1] = 0;
    s.mass[2 * tid] = s.mass[2 * tid + 1] = 0;
    __syncthreads();
    each<HELD>(row, held, 0, row.V, [&](float v, int i) {
      if (!drawable(v) || row.bin_of(v) != b) return;
      const place_t p = row.place(v, i);
      if (k > 0 && (p >> (shift + width)) != prefix) return;
      const int d = (int)((p >> shift) & ((1u << width) - 1));
      atomicAdd(&s.cnt[d], 1u);
      atomicAdd(&s.mass[d], row.mass(v));
    });
    __syncthreads();
    const u64 c0 = s.cnt[2 * tid], m0 = s.mass[2 * tid];
    u64 pc = c0 + s.cnt[2 * tid + 1], pm = m0 + s.mass[2 * tid + 1], tc, tm;
    const u64 c1 = pc - c0, m1 = pm - m0;
    block_scan2(s, pc, pm, tc, tm);
    const u64 at0 = masses ? above_m + pm : above_c + pc, w0 = masses ? m0 : c0, w1 = masses ? m1 : c1;
    const bool h0 = at0 < left && left <= at0 + w0, h1 = at0 + w0 < left && left <= at0 + w0 + w1;
    if (h0 || h1) {
      s.found[0] = 2 * tid + (h1 ? 1 : 0);
      s.found[1] = above_m + pm + (h1 ? m0 : 0);
      s.found[2] = above_c + pc + (h1 ? c0 : 0);
      s.found[3] = h1 ? m1 : m0;
    }
    __syncthreads();
    prefix = (prefix << width) | s.found[0];
    above_m = s.found[1];
    above_c = s.found[2];
  }
  *mass_to = above_m + s.found[3];
  return prefix;
}

// ------------------------------------------------------------ the steps of a draw

// The largest of the threads' m and its first place (0x7fffffff: none).
__device__ __forceinline__ void block_top(Shared& s, float& m, int& at) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const float wm = wave_max(m);
  at = m == wm ? at : 0x7fffffff;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
  if (lane == 0) {
    s.redf[wv] = wm;
    s.redi[wv] = at;
  }
  __syncthreads();
  m = s.redf[0];
  at = s.redi[0];
#pragma unroll
  for (int k = 1; k < DW; ++k)
    if (s.redf[k] > m || (s.redf[k] == m && s.redi[k] < at)) {
      m = s.redf[k];
      at = s.redi[k];
    }
}

template <bool HELD>
__device__ __forceinline__ void top_of(const Row& row, const float (&held)[PER], int lo, int hi, float& m,
                                       int& at) {
  m = -INFINITY;
  at = 0x7fffffff;
  each<HELD>(row, held, lo, hi, [&](float v, int i) {
    if (v > m) {
      m = v;
      at = i;
    }
  });
}

struct Settings {
  float temp;
  int top_k;
  float top_p;
  bool by_k, by_p;
  u64 least;  // mass of an id that min_p keeps
};

__device__ __forceinline__ Settings settings_of(const DrawArgs& a, int r) {
  Settings c;
  c.temp = a.c.temp ? a.c.temp[r] : 1.f;
  const float min_p = a.c.min_p ? a.c.min_p[r] : 0.f;
  // (min_p above 1 keeps one id, also of several equal ones)
  c.top_k = min_p > 1.f ? 1 : a.c.top_k ? a.c.top_k[r] : 0;
  c.top_p = a.c.top_p ? a.c.top_p[r] : 1.f;
  c.by_k = c.top_k > 0 && c.top_k < a.V;
  c.by_p = c.top_p < 1.f;
  c.least = min_p > 0.f ? (min_p >= 1.f ? 1ull << 44 : (u64)ceil((double)min_p * 17592186044416.0)) : 0;
  return c;
}

// The row's units once its largest logit is known.
__device__ __forceinline__ void scale_by(Row& row, float m, float temp) {
  const float t = temp != temp ? 1.f : temp;
  row.m = m;
  row.km = key_of(m);
  row.unit = TAB * 1.44269504088896340736 / (double)t;
  row.bin = BIN_UNITS / t;
}

// A row without a draw: nothing to draw from (id -1), or temp <= 0.
__device__ __forceinline__ bool no_draw(const DrawArgs& a, int r, int at, float temp) {
  if (at != 0x7fffffff && !(temp <= 0.f)) return false;
  if (threadIdx.x == 0) {
    a.ids[r] = at == 0x7fffffff ? -1 : at;
    if (a.probs) a.probs[r] = at == 0x7fffffff ? 0.f : 1.f;
  }
  return true;
}

__device__ __forceinline__ void clear_bins(Shared& s) {
  s.cnt[2 * threadIdx.x] = s.cnt[2 * threadIdx.x + 1] = 0;
  s.mass[2 * threadIdx.x] = s.mass[2 * threadIdx.x + 1] = 0;
}

// Counts and (for top_p) masses of the ids of [lo, hi) by bin, into cleared bins.
template <bool HELD>
__device__ __forceinline__ void fill_bins(Shared& s, const Row& row, const float (&held)[PER], int lo, int hi,
                                          bool by_p) {
  each<HELD>(row, held, lo, hi, [&](float v, int) {
    if (!drawable(v)) return;
    const int b = row.bin_of(v);
    atomicAdd(&s.cnt[b], 1u);
    if (by_p) atomicAdd(&s.mass[b], row.mass(v));
  });
}

// The mass at which top_p of `all` is reached.
__device__ __forceinline__ u64 want_of(float top_p, u64 all) {
  const double w = ceil((double)(top_p > 0.f ? top_p : 0.f) * (double)all);
  return w < 1.0 ? 1ull : (u64)w;
}

// The last id that top_k and top_p keep, from the row's bins.
template <bool HELD>
__device__ place_t cut_of(Shared& s, const Row& row, const float (&held)[PER], const Settings& c) {
  const int tid = threadIdx.x;
  place_t cut = ~0ull;
  const u64 c0 = s.cnt[2 * tid], m0 = s.mass[2 * tid];
  u64 pc = c0 + s.cnt[2 * tid + 1], pm = m0 + s.mass[2 * tid + 1], all_c, all;
  const u64 c1 = pc - c0, m1 = pm - m0;
  block_scan2(s, pc, pm, all_c, all);
  // (place_at by digits uses the bins again: the masses before them stay in pm, m0, m1)
  auto find = [&](u64 want, u64 before, u64 w0, u64 w1) {
    if (before < want && want <= before + w0) {
      s.found[0] = 2 * tid;
      s.found[1] = before;
      s.found[2] = pm;
    } else if (before + w0 < want && want <= before + w0 + w1) {
      s.found[0] = 2 * tid + 1;
      s.found[1] = before + w0;
      s.found[2] = pm + m0;
    }
    __syncthreads();
  };
  if (c.by_k && (u64)c.top_k < all_c) {
    find(c.top_k, pc, c0, c1);
    const u64 above = s.found[2], before = s.found[1];
    u64 to;
    cut = place_at<HELD>(s, row, held, false, c.top_k, (int)s.found[0], before, &to);
    all = above + to;  // the mass that top_k leaves
    __syncthreads();
    s.cnt[2 * tid] = c0;
    s.cnt[2 * tid + 1] = c1;
    __syncthreads();
  }
  if (c.by_p) {
    const u64 want = want_of(c.top_p, all);
    find(want, pm, m0, m1);
    u64 to;
    const place_t c2 = place_at<HELD>(s, row, held, true, want, (int)s.found[0], s.found[1], &to);
    cut = c2 < cut ? c2 : cut;
  }
  return cut;
}

// Mass of id i if it is kept.
__device__ __forceinline__ u64 kept(const Row& row, place_t cut, u64 least, float v, int i) {
  if (!drawable(v) || row.place(v, i) > cut) return 0;
  const u64 w = row.mass(v);
  return w >= least ? w : 0;
}

// Kept mass of the chunks of 64 ids in [c_lo, c_hi); returns this lane's share
// of their sum (in lane 63).
__device__ __forceinline__ u64 chunk_masses(const Row& row, place_t cut, u64 least, int c_lo, int c_hi,
                                            u64* chunk_mass) {
  constexpr int AHEAD = 16;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  u64 all = 0;
  for (int c0 = c_lo + wv; c0 < c_hi; c0 += AHEAD * DW) {
    float v[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = 64 * (c0 + k * DW) + lane;
      v[k] = c0 + k * DW < c_hi && i < row.V ? row.x[i] : -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int c = c0 + k * DW;
      if (c >= c_hi) break;
      const u64 w = kept(row, cut, least, v[k], 64 * c + lane);
      const u64 sum = __any(w != 0) ? wave_scan(w) : 0;
      if (lane == 63) chunk_mass[c] = sum;
      all += sum;
    }
  }
  return all;
}

// The uniform number's place in a kept mass.
__device__ __forceinline__ u64 target_of(const DrawArgs& a, int r, u64 total) {
  const float u = a.c.u[r];
  const u64 t = (u64)((double)(u > 0.f ? (u < 1.f ? u : 1.f) : 0.f) * (double)total);
  return t < total ? t : total - 1;
}

// The draw, by one wavefront: the chunk of [c_lo, c_hi) that holds `target` of
// the kept mass (`before` of it lies in front of c_lo; WHOLE: nothing does, and
// target and total come from the chunks), then the id.
template <bool WHOLE>
__device__ __forceinline__ void pick(const DrawArgs& a, int r, const Row& row, place_t cut, u64 least,
                                     const u64* chunk_mass, int c_lo, int c_hi, u64 before, u64 target,
                                     u64 total) {
  const int lane = threadIdx.x & 63;
  const int per = (c_hi - c_lo + 63) / 64, q0 = c_lo + lane * per;
  u64 mine = 0;
#pragma unroll 8
  for (int q = 0; q < per; ++q) mine += q0 + q < c_hi ? chunk_mass[q0 + q] : 0;
  const u64 upto = before + wave_scan(mine);
  if constexpr (WHOLE) {
    total = lane_value(upto, 63);
    target = target_of(a, r, total);
  }
  const int l = __builtin_ctzll(__ballot(upto > target));
  before = lane_value(upto - mine, l);
  // that lane's chunks, a lane each (64 at most)
  const int cl = c_lo + l * per + lane;
  const u64 cm = lane < per && cl < c_hi ? chunk_mass[cl] : 0;
  const u64 cu = before + wave_scan(cm);
  const int lc = __builtin_ctzll(__ballot(cu > target));
  before = lane_value(cu - cm, lc);
  const int i = 64 * (c_lo + l * per + lc) + lane;
  const u64 w = kept(row, cut, least, i < a.V ? row.x[i] : -INFINITY, i);
  const u64 sum = before + wave_scan(w);
  if (lane == __builtin_ctzll(__ballot(sum > target))) {
    a.ids[r] = i;
    if (a.probs) a.probs[r] = (float)((double)w / (double)total);
  }
}

// ------------------------------------------------------------ a workgroup a row
template <bool HELD>
__global__ __launch_bounds__(DT) void k_draw_rows(DrawArgs a) {
  __shared__ Shared s;
  extern __shared__ __attribute__((aligned(16))) u64 chunk_mass[];  // [chunks]
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, r = blockIdx.x;
  const int chunks = (a.V + 63) / 64;
  Row row;
  row.x = a.x + (int64_t)r * a.ld;
  row.V = a.V;
  row.tab = s.tab;
  float held[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) held[k] = HELD && k * DT + tid < a.V ? row.x[k * DT + tid] : -INFINITY;
  s.tab[tid] = exp2(tid / (double)TAB);
  clear_bins(s);
  float m;
  int at;
  top_of<HELD>(row, held, 0, a.V, m, at);
  block_top(s, m, at);
  const Settings c = settings_of(a, r);
  if (no_draw(a, r, at, c.temp)) return;
  scale_by(row, m, c.temp);
  place_t cut = ~0ull;
  if (c.by_k || c.by_p) {
    fill_bins<HELD>(s, row, held, 0, a.V, c.by_p);
    __syncthreads();
    cut = cut_of<HELD>(s, row, held, c);
  }
  if constexpr (HELD) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int ch = k * DW + wv;
      if (ch >= chunks) break;
      const u64 sum = wave_scan(kept(row, cut, c.least, held[k], k * DT + tid));
      if (lane == 63) chunk_mass[ch] = sum;
    }
  } else {
    chunk_masses(row, cut, c.least, 0, chunks, chunk_mass);
  }
  __syncthreads();
  if (wv != 0) return;
  pick<true>(a, r, row, cut, c.least, chunk_mass, 0, chunks, 0, 0, 0);
}

// ------------------------------------------------------------ rows in slices
// Few rows of a large vocabulary leave most CUs without a row, and the
// exponentials of a whole row (one an id for the masses of the bins, one more
// for the chunks) to one of them. There the two passes that take them, and the
// maximum's, run on n_slice workgroups a row, in launches of their own, and the
// cut between them on one.
// 48 rows of 131073 ids, top-p: 165 us with a workgroup a row, 71 so (the
// maximum 8, the bins 13, which of them 8, their ids 10, the cut 11, the chunks
// 18, the draw 5). Adding up 256 ids in a lane before a wavefront's sum left the
// chunks at 18: the masses take it, not their sums.
struct Found {  // of a row's bins
  u64 count_before, mass_before, p_before, all;  // ahead of top_k's bin, of top_p's first; of the row
  int bk, p1, p2;    // top_k's bin, top_p's first and last (BINS: none)
  unsigned int n, listed;  // their ids, and how many of those the list has so far
};
struct SliceArgs {
  DrawArgs a;
  int n_slice, len;  // slices of a row (64 at most), ids of one (a multiple of 64)
  double* tab;       // [TAB]
  place_t* cut;      // [rows]
  Found* found;      // [rows]
  u64* mass;         // [rows][n_slice][BINS]
  u64* chunk_mass;   // [rows][chunks]
  u64* slice_mass;   // [rows][n_slice]: kept
  unsigned int* cnt; // as mass
  float* top;        // [rows][n_slice]
  int32_t* top_at;
  int32_t* list;     // [rows][LIST]: the ids that may be the cut
};

// A row as the later launches see it: its largest logit from its slices' (at:
// its first place, 0x7fffffff for none).
__device__ __forceinline__ Row slice_row(const SliceArgs& p, int r, const double* tab, const Settings& c,
                                         int& at) {
  const int lane = threadIdx.x & 63;
  float m = lane < p.n_slice ? p.top[r * p.n_slice + lane] : -INFINITY;
  at = lane < p.n_slice ? p.top_at[r * p.n_slice + lane] : 0x7fffffff;
  const float wm = wave_max(m);
  at = m == wm ? at : 0x7fffffff;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
  Row row;
  row.x = p.a.x + (int64_t)r * p.a.ld;
  row.V = p.a.V;
  row.tab = tab;
  scale_by(row, wm, c.temp);
  return row;
}

__global__ __launch_bounds__(DT) void k_draw_top(SliceArgs p) {
  __shared__ Shared s;
  const int r = blockIdx.x / p.n_slice, k = blockIdx.x % p.n_slice, lo = k * p.len;
  Row row;
  row.x = p.a.x + (int64_t)r * p.a.ld;
  row.V = p.a.V;
  const float held[PER] = {};
  float m;
  int at;
  top_of<false>(row, held, lo, min(p.a.V, lo + p.len), m, at);
  block_top(s, m, at);
  if (threadIdx.x == 0) {
    p.top[blockIdx.x] = m;
    p.top_at[blockIdx.x] = at;
  }
  if (blockIdx.x == 0) p.tab[threadIdx.x] = exp2(threadIdx.x / (double)TAB);
}

__global__ __launch_bounds__(DT) void k_draw_bins(SliceArgs p) {
  __shared__ Shared s;
  const int tid = threadIdx.x, r = blockIdx.x / p.n_slice, k = blockIdx.x % p.n_slice, lo = k * p.len;
  const Settings c = settings_of(p.a, r);
  if (!(c.by_k || c.by_p) || c.temp <= 0.f) return;
  s.tab[tid] = p.tab[tid];
  clear_bins(s);
  int at;
  const Row row = slice_row(p, r, s.tab, c, at);
  if (at == 0x7fffffff) return;
  __syncthreads();
  const float held[PER] = {};
  fill_bins<false>(s, row, held, lo, min(p.a.V, lo + p.len), c.by_p);
  __syncthreads();
  const int64_t to = (int64_t)blockIdx.x * BINS + 2 * tid;
  *(uint2*)(p.cnt + to) = make_uint2(s.cnt[2 * tid], s.cnt[2 * tid + 1]);
  p.mass[to] = s.mass[2 * tid];
  p.mass[to + 1] = s.mass[2 * tid + 1];
}

// The row's bins, from its slices'.
__device__ __forceinline__ void sum_bins(const SliceArgs& p, int r, Shared& s) {
  const int tid = threadIdx.x;
  uint2 n = make_uint2(0, 0);
  ulonglong2 w = make_ulonglong2(0, 0);
#pragma unroll 8
  for (int k = 0; k < p.n_slice; ++k) {
    const int64_t from = (int64_t)(r * p.n_slice + k) * BINS + 2 * tid;
    const uint2 x = *(const uint2*)(p.cnt + from);
    const ulonglong2 y = *(const ulonglong2*)(p.mass + from);
    n.x += x.x;
    n.y += x.y;
    w.x += y.x;
    w.y += y.y;
  }
  s.cnt[2 * tid] = n.x;
  s.cnt[2 * tid + 1] = n.y;
  s.mass[2 * tid] = w.x;
  s.mass[2 * tid + 1] = w.y;
}

// Which bins of the row can hold its cut: top_k's, and the ones that top_p's can
// be in for any mass that top_k may leave (the ids above its bin, with none or
// all of the bin's). Their ids are gathered by the slices; where they are more
// than LIST, k_draw_cut goes over the row itself.
__global__ __launch_bounds__(DT) void k_draw_find(SliceArgs p) {
  __shared__ Shared s;
  __shared__ u64 at[3][4];  // bin, counts before, mass before, mass with it
  __shared__ unsigned int sum;
  const int tid = threadIdx.x, r = blockIdx.x;
  const Settings c = settings_of(p.a, r);
  if (!(c.by_k || c.by_p) || c.temp <= 0.f) return;
  // (a row with nothing to draw has no bins: what comes of them is not used)
  sum_bins(p, r, s);
  if (tid == 0) {
    at[0][0] = BINS;  // (top_k takes all)
    sum = 0;
  }
  __syncthreads();
  const u64 cc[2] = {s.cnt[2 * tid], s.cnt[2 * tid + 1]}, mm[2] = {s.mass[2 * tid], s.mass[2 * tid + 1]};
  u64 pc = cc[0] + cc[1], pm = mm[0] + mm[1], all_c, all;
  block_scan2(s, pc, pm, all_c, all);
  auto mark = [&](int k, bool masses, u64 want) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const u64 c0 = pc + (j ? cc[0] : 0), m0 = pm + (j ? mm[0] : 0);
      const u64 b = masses ? m0 : c0, w = masses ? mm[j] : cc[j];
      if (b < want && want <= b + w) {
        at[k][0] = 2 * tid + j;
        at[k][1] = c0;
        at[k][2] = m0;
        at[k][3] = m0 + mm[j];
      }
    }
  };
  const bool cut_k = c.by_k && (u64)c.top_k < all_c;
  if (cut_k) mark(0, false, c.top_k);
  __syncthreads();
  const u64 low = cut_k ? at[0][2] : all, high = cut_k ? at[0][3] : all;
  if (c.by_p) {
    mark(1, true, want_of(c.top_p, low));
    mark(2, true, want_of(c.top_p, high));
  } else if (tid == 0) {
    at[1][0] = BINS;
    at[2][0] = 0;
  }
  __syncthreads();
  const int bk = (int)at[0][0], p1 = (int)at[1][0], p2 = (int)at[2][0];
  unsigned n = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int b = 2 * tid + j;
    n += b == bk || (b >= p1 && b <= p2) ? (unsigned)cc[j] : 0;
  }
  if (n) atomicAdd(&sum, n);
  __syncthreads();
  if (tid == 0) {
    Found f;
    f.bk = bk;
    f.p1 = p1;
    f.p2 = p2;
    f.count_before = cut_k ? at[0][1] : 0;
    f.mass_before = cut_k ? at[0][2] : 0;
    f.p_before = c.by_p ? at[1][2] : 0;
    f.all = all;
    f.n = sum;
    f.listed = 0;
    p.found[r] = f;
  }
}

__global__ __launch_bounds__(DT) void k_draw_gather(SliceArgs p) {
  const int r = blockIdx.x / p.n_slice, k = blockIdx.x % p.n_slice, lo = k * p.len;
  const Settings c = settings_of(p.a, r);
  if (!(c.by_k || c.by_p) || c.temp <= 0.f) return;
  int at;
  const Row row = slice_row(p, r, nullptr, c, at);
  if (at == 0x7fffffff) return;
  Found* f = p.found + r;
  if (f->n > LIST) return;
  const int bk = f->bk, p1 = f->p1, p2 = f->p2;
  const float held[PER] = {};
  each<false>(row, held, lo, min(p.a.V, lo + p.len), [&](float v, int i) {
    if (!drawable(v)) return;
    const int b = row.bin_of(v);
    if (b == bk || (b >= p1 && b <= p2)) p.list[(int64_t)r * LIST + atomicAdd(&f->listed, 1u)] = i;
  });
}

__global__ __launch_bounds__(DT) void k_draw_cut(SliceArgs p) {
  __shared__ Shared s;
  const int tid = threadIdx.x, r = blockIdx.x;
  const Settings c = settings_of(p.a, r);
  s.tab[tid] = p.tab[tid];
  int at;
  const Row row = slice_row(p, r, s.tab, c, at);
  if (no_draw(p.a, r, at, c.temp)) return;
  place_t cut = ~0ull;
  if (c.by_k || c.by_p) {
    const Found f = p.found[r];
    if (f.n > LIST) {
      sum_bins(p, r, s);
      __syncthreads();
      const float held[PER] = {};
      cut = cut_of<false>(s, row, held, c);
    } else {
      if (tid < (int)f.n) {
        const int i = p.list[(int64_t)r * LIST + tid];
        s.list_at[tid] = row.place(row.x[i], i);
      }
      if (tid == 0) s.n_list = 0;
      __syncthreads();
      const place_t mine = sort_list(s, f.n);
      int bin = -1;
      u64 w = 0, all = f.all;
      if (tid < (int)f.n) {
        const float v = row.value(mine);
        bin = row.bin_of(v);
        w = row.mass(v);
        if (bin < f.bk && f.bk < BINS) atomicAdd(&s.n_list, 1);
      }
      const bool in_k = bin == f.bk, in_p = bin >= f.p1 && bin <= f.p2;
      u64 mass_k = in_k ? w : 0, mass_p = in_p ? w : 0, all_k, all_p;
      block_scan2(s, mass_k, mass_p, all_k, all_p);
      if (f.bk < BINS) {  // (of the list, the ids in front of its bin are not counted)
        if (in_k && tid - s.n_list == (int)((u64)c.top_k - f.count_before) - 1) {
          s.found[0] = mine;
          s.found[1] = f.mass_before + mass_k + w;
        }
        __syncthreads();
        cut = s.found[0];
        all = s.found[1];
        __syncthreads();
      }
      if (c.by_p) {
        const u64 left = want_of(c.top_p, all) - f.p_before;
        if (in_p && mass_p < left && left <= mass_p + w) s.found[0] = mine;
        __syncthreads();
        cut = s.found[0] < cut ? s.found[0] : cut;
      }
    }
  }
  if (tid == 0) p.cut[r] = cut;
}

__global__ __launch_bounds__(DT) void k_draw_chunks(SliceArgs p) {
  __shared__ double tab[TAB];
  __shared__ u64 red[DW];
  const int r = blockIdx.x / p.n_slice, k = blockIdx.x % p.n_slice;
  const Settings c = settings_of(p.a, r);
  tab[threadIdx.x] = p.tab[threadIdx.x];
  int at;
  const Row row = slice_row(p, r, tab, c, at);
  if (at == 0x7fffffff || c.temp <= 0.f) return;
  __syncthreads();
  const int chunks = (p.a.V + 63) / 64, c0 = k * (p.len / 64);
  const u64 sum = chunk_masses(row, p.cut[r], c.least, c0, min(chunks, c0 + p.len / 64),
                               p.chunk_mass + (int64_t)r * chunks);
  if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    u64 t = 0;
#pragma unroll
    for (int w = 0; w < DW; ++w) t += red[w];
    p.slice_mass[blockIdx.x] = t;
  }
}

__global__ __launch_bounds__(64) void k_draw_pick(SliceArgs p) {
  const int r = blockIdx.x, lane = threadIdx.x;
  const Settings c = settings_of(p.a, r);
  int at;
  const Row row = slice_row(p, r, p.tab, c, at);
  if (at == 0x7fffffff || c.temp <= 0.f) return;
  const u64 mine = lane < p.n_slice ? p.slice_mass[r * p.n_slice + lane] : 0;
  const u64 upto = wave_scan(mine), total = lane_value(upto, 63), target = target_of(p.a, r, total);
  const int k = __builtin_ctzll(__ballot(upto > target));
  const int chunks = (p.a.V + 63) / 64, c0 = k * (p.len / 64);
  pick<false>(p.a, r, row, p.cut[r], c.least, p.chunk_mass + (int64_t)r * chunks, c0,
              min(chunks, c0 + p.len / 64), lane_value(upto - mine, k), target, total);
}

// Slices of a row: as many of 8192 ids as its vocabulary has, while all rows
// together have two a CU at most.
int slices_of(int32_t rows, int32_t V) {
  return V <= PER * DT ? 1 : std::max(1, std::min((V + PER * DT - 1) / (PER * DT), 512 / rows));
}

}  // namespace

int64_t draw_work_bytes(int32_t rows, int32_t V) {
  const int64_t n = rows > 0 ? slices_of(rows, V) : 1;
  if (n == 1) return 0;
  return TAB * 8 + rows * (8 + (int64_t)sizeof(Found) + LIST * 4 + n * 16 + n * BINS * 12 + ((V + 63) / 64 + 1) * 8);
}

void launch_draw_rows(hipStream_t s, const float* logits, int32_t rows, int32_t V, int64_t ld,
                      const fg_draw_cfg& c, int32_t* ids, float* probs, void* work) {
  const DrawArgs a{logits, V, ld, c, ids, probs};
  const int n = slices_of(rows, V), chunks = (V + 63) / 64;
  const unsigned lds = (unsigned)chunks * 8;
  if (V <= PER * DT) {
    FG_LAUNCH((k_draw_rows<true>), dim3((unsigned)rows), dim3(DT), lds, s, a);
    return;
  }
  if (n == 1) {
    static std::atomic<uint64_t> lds_set{0};
    raise_lds_once((const void*)k_draw_rows<false>, MAX_CHUNKS * 8, &lds_set);
    FG_LAUNCH((k_draw_rows<false>), dim3((unsigned)rows), dim3(DT), lds, s, a);
    return;
  }
  SliceArgs p;
  p.a = a;
  p.n_slice = n;
  p.len = (chunks + n - 1) / n * 64;
  const int64_t rn = (int64_t)rows * n;
  p.tab = (double*)work;
  p.mass = (u64*)(p.tab + TAB);
  p.chunk_mass = p.mass + rn * BINS;
  p.slice_mass = p.chunk_mass + (int64_t)rows * chunks;
  p.cut = (place_t*)(p.slice_mass + rn);
  p.found = (Found*)(p.cut + rows);
  p.cnt = (unsigned int*)(p.found + rows);
  p.list = (int32_t*)(p.cnt + rn * BINS);
  p.top = (float*)(p.list + (int64_t)rows * LIST);
  p.top_at = (int32_t*)(p.top + rn);
  const dim3 all((unsigned)rn), one((unsigned)rows);
  FG_LAUNCH(k_draw_top, all, dim3(DT), 0, s, p);
  FG_LAUNCH(k_draw_bins, all, dim3(DT), 0, s, p);
  FG_LAUNCH(k_draw_find, one, dim3(DT), 0, s, p);
  FG_LAUNCH(k_draw_gather, all, dim3(DT), 0, s, p);
  FG_LAUNCH(k_draw_cut, one, dim3(DT), 0, s, p);
  FG_LAUNCH(k_draw_chunks, all, dim3(DT), 0, s, p);
  FG_LAUNCH(k_draw_pick, one, dim3(64), 0, s, p);
}

}  // namespace fgpt
