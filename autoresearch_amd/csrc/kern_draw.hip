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
// that of the chain of block-wide steps; past that it is the exponentials'.
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
  u64 list_mass[LIST];
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
};

__device__ __forceinline__ bool drawable(float v) { return v > -INFINITY; }  // (false for NaN)

// f(v, i) for this thread's ids; HELD: from registers.
template <bool HELD, class F>
__device__ __forceinline__ void each(const Row& row, const float (&held)[PER], F&& f) {
  if constexpr (HELD) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = k * DT + (int)threadIdx.x;
      if (i < row.V) f(held[k], i);
    }
  } else {
    for (int i0 = threadIdx.x; i0 < row.V; i0 += PER * DT) {
      float v[PER];
#pragma unroll
      for (int k = 0; k < PER; ++k) v[k] = i0 + k * DT < row.V ? row.x[i0 + k * DT] : -INFINITY;
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (i0 + k * DT < row.V) f(v[k], i0 + k * DT);
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
    each<HELD>(row, held, [&](float v, int i) {
      if (!drawable(v) || row.bin_of(v) != b) return;
      const int at = atomicAdd(&s.n_list, 1);
      s.list_at[at] = row.place(v, i);
      s.list_mass[at] = row.mass(v);
    });
    __syncthreads();
    if (tid < (int)n) {
      const place_t mine = s.list_at[tid];
      const u64 w = s.list_mass[tid];
      u64 rank = 0, mass = 0;
#pragma unroll 4
      for (unsigned k = 0; k < n; ++k) {
        const bool first = s.list_at[k] < mine;
        rank += first ? 1 : 0;
        mass += first ? s.list_mass[k] : 0;
      }
      if (masses ? mass < left && left <= mass + w : rank == left - 1) {
        s.found[0] = mine;
        s.found[1] = mass + w;
      }
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
    each<HELD>(row, held, [&](float v, int i) {
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
  s.cnt[2 * tid] = s.cnt[2 * tid + 1] = 0;
  s.mass[2 * tid] = s.mass[2 * tid + 1] = 0;

  // the largest logit and its first id
  float m = -INFINITY;
  int at = 0x7fffffff;
  each<HELD>(row, held, [&](float v, int i) {
    if (v > m) {
      m = v;
      at = i;
    }
  });
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
  const float temp = a.c.temp ? a.c.temp[r] : 1.f;
  if (at == 0x7fffffff || temp <= 0.f) {
    if (tid == 0) {
      a.ids[r] = at == 0x7fffffff ? -1 : at;
      if (a.probs) a.probs[r] = at == 0x7fffffff ? 0.f : 1.f;
    }
    return;
  }
  const float t = temp != temp ? 1.f : temp;
  row.m = m;
  row.km = key_of(m);
  row.unit = TAB * 1.44269504088896340736 / (double)t;
  row.bin = BIN_UNITS / t;
  const int top_k = a.c.top_k ? a.c.top_k[r] : 0;
  const float top_p = a.c.top_p ? a.c.top_p[r] : 1.f, min_p = a.c.min_p ? a.c.min_p[r] : 0.f;
  const bool by_k = top_k > 0 && top_k < a.V, by_p = top_p < 1.f;

  place_t cut = ~0ull;  // the last id kept
  if (by_k || by_p) {
    each<HELD>(row, held, [&](float v, int) {
      if (!drawable(v)) return;
      const int b = row.bin_of(v);
      atomicAdd(&s.cnt[b], 1u);
      if (by_p) atomicAdd(&s.mass[b], row.mass(v));
    });
    __syncthreads();
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
        s.found[3] = s.cnt[2 * tid];
      } else if (before + w0 < want && want <= before + w0 + w1) {
        s.found[0] = 2 * tid + 1;
        s.found[1] = before + w0;
        s.found[2] = pm + m0;
      }
      __syncthreads();
    };
    if (by_k && (u64)top_k < all_c) {
      find(top_k, pc, c0, c1);
      const u64 above = s.found[2], before = s.found[1];
      u64 to;
      cut = place_at<HELD>(s, row, held, false, top_k, (int)s.found[0], before, &to);
      all = above + to;  // the mass that top_k leaves
      __syncthreads();
      s.cnt[2 * tid] = c0;
      s.cnt[2 * tid + 1] = c1;
      __syncthreads();
    }
    if (by_p) {
      const double w = ceil((double)(top_p > 0.f ? top_p : 0.f) * (double)all);
      const u64 want = w < 1.0 ? 1ull : (u64)w;
      find(want, pm, m0, m1);
      u64 to;
      const place_t c2 = place_at<HELD>(s, row, held, true, want, (int)s.found[0], s.found[1], &to);
      cut = c2 < cut ? c2 : cut;
    }
  }
  const u64 least =
      min_p > 0.f ? (min_p >= 1.f ? 1ull << 44 : (u64)ceil((double)min_p * 17592186044416.0)) : 0;

  // kept mass of each chunk of 64 ids (a wavefront's ids of one k)
  auto kept = [&](float v, int i) -> u64 {
    if (!drawable(v) || row.place(v, i) > cut) return 0;
    const u64 w = row.mass(v);
    return w >= least ? w : 0;
  };
  if constexpr (HELD) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int c = k * DW + wv;
      if (c >= chunks) break;
      const u64 sum = wave_scan(kept(held[k], k * DT + tid));
      if (lane == 63) chunk_mass[c] = sum;
    }
  } else {
    for (int c0 = wv; c0 < chunks; c0 += PER * DW) {
      float v[PER];
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = 64 * (c0 + k * DW) + lane;
        v[k] = i < a.V ? row.x[i] : -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int c = c0 + k * DW;
        if (c >= chunks) break;
        const u64 w = kept(v[k], 64 * c + lane);
        const u64 sum = __any(w != 0) ? wave_scan(w) : 0;
        if (lane == 63) chunk_mass[c] = sum;
      }
    }
  }
  __syncthreads();
  // the first wavefront finds the chunk, then the id
  if (wv != 0) return;
  const int per = (chunks + 63) / 64, q0 = lane * per;
  u64 mine = 0;
  for (int q = 0; q < per; ++q) mine += q0 + q < chunks ? chunk_mass[q0 + q] : 0;
  const u64 upto = wave_scan(mine), total = lane_value(upto, 63);
  const float u = a.c.u[r];
  u64 target = (u64)((double)(u > 0.f ? (u < 1.f ? u : 1.f) : 0.f) * (double)total);
  if (target >= total) target = total - 1;
  const int l = __builtin_ctzll(__ballot(upto > target));
  u64 before = lane_value(upto - mine, l);
  int c = l * per;
  while (before + chunk_mass[c] <= target) before += chunk_mass[c++];
  const int i = 64 * c + lane;
  const u64 w = kept(i < a.V ? row.x[i] : -INFINITY, i);
  const u64 sum = before + wave_scan(w);
  if (lane == __builtin_ctzll(__ballot(sum > target))) {
    a.ids[r] = i;
    if (a.probs) a.probs[r] = (float)((double)w / (double)total);
  }
}

}  // namespace

int64_t draw_work_bytes(int32_t, int32_t) { return 0; }

void launch_draw_rows(hipStream_t s, const float* logits, int32_t rows, int32_t V, int64_t ld,
                      const fg_draw_cfg& c, int32_t* ids, float* probs, void*) {
  const DrawArgs a{logits, V, ld, c, ids, probs};
  const unsigned lds = (unsigned)((V + 63) / 64 * 8);
  if (V <= PER * DT) {
    FG_LAUNCH((k_draw_rows<true>), dim3((unsigned)rows), dim3(DT), lds, s, a);
  } else {
    static std::atomic<uint64_t> lds_set{0};
    raise_lds_once((const void*)k_draw_rows<false>, MAX_CHUNKS * 8, &lds_set);
    FG_LAUNCH((k_draw_rows<false>), dim3((unsigned)rows), dim3(DT), lds, s, a);
  }
}

}  // namespace fgpt
