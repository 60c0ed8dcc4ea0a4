// kern_draw.hip -- one id a row under temperature, top-k, top-p and min-p from
// given uniform numbers (fg_draw_rows of include/fgpt.h).
//
// No sort: each of the three filters keeps a prefix of the row in descending
// order (ties by ascending id), so all of them together are one threshold: the
// ids whose key is above K, and the first `ties` ids of key K. K is found by
// histograms over the digits of the key (11, 11 and 10 bits): one pass over the
// row for the first digit of all ids, one each for the digits below within the
// bin where top_k's count or top_p's mass is reached. A last pass sums the kept
// mass by chunks of 64 ids, in id order, and the draw scans those.
//
// Masses are integers, e_i = exp((x_i - max) / temp) in steps of 2^-44 (sums of
// up to 2^18 of them fit 64 bits), so every sum is exact in any order: atomics
// may add them as they come, and an id next to a border of the cumulative mass
// comes out the same in every run. 32-bit sums would misplace about n 2^-24 of
// the draws of a row with n likely ids.
#include "fgpt_internal.h"
#include "kern_common.h"
#include "paged_internal.h"

namespace fgpt {
namespace {

typedef unsigned long long u64;

constexpr int DT = 1024, DW = DT / 64;   // threads, wavefronts
constexpr int BINS = 2048;               // of the widest digit
constexpr int MAX_CHUNKS = DRAW_MAX_V / 64;

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

// e^y in steps of 2^-44 for y <= 0: y = (n ln 2)/32 + r, |r| <= ln2 / 64, as
// 2^(n/32) (tab[j] = 2^(j/32)) times r's Taylor sum to degree 5 (the next term
// is below 2.3e-15). The addition of 2^52 rounds to an integer.
__device__ __forceinline__ u64 mass_of(double y, const double* tab) {
  if (!(y > -31.0)) return 0;  // (below half a step)
  const double n = rint(y * 46.166241308446828384);  // 32 / ln 2
  const double r = fma(-n, 0.021660849392498290, y);  // ln 2 / 32
  double s = fma(r, 1.0 / 120, 1.0 / 24);
  s = fma(r, s, 1.0 / 6);
  s = fma(r, s, 0.5);
  s = fma(r, s, 1.0);
  s = fma(r, s, 1.0);
  const int k = (int)n;
  const double e = ldexp(s * tab[k & 31], 44 + (k >> 5));
  return (u64)__double_as_longlong(e + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
}

struct Row {  // what a row's threads share
  const float* x;
  int V;
  float m;       // largest logit (may be +inf)
  uint32_t km;   // its key
  double inv_t;
  const double* tab;
  __device__ __forceinline__ bool drawable(float v) const { return v > -INFINITY; }  // (no NaN)
  __device__ __forceinline__ uint32_t down(float v) const { return km - key_of(v); }  // 0 at the top
  __device__ __forceinline__ u64 mass(float v) const {
    if (v == m) return 1ull << 44;
    return mass_of(((double)v - (double)m) * inv_t, tab);
  }
};

__device__ __forceinline__ u64 wave_scan(u64 v) {  // inclusive, by lane
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}

// Sum of the values of the threads before this one, and of all; red: [DW].
__device__ u64 block_scan(u64 v, u64* red, u64* total) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const u64 in = wave_scan(v);
  __syncthreads();
  if (lane == 63) red[wv] = in;
  __syncthreads();
  u64 before = 0, all = 0;
  for (int k = 0; k < DW; ++k) {
    const u64 r = red[k];
    before += k < wv ? r : 0;
    all += r;
  }
  *total = all;
  return before + in - v;
}

struct Hist {
  unsigned int cnt[BINS];
  u64 mass[BINS];
};

// Histogram of the digit (down >> shift) & mask over the ids whose digits above
// it are `prefix` (counts, and masses if wanted).
__device__ void fill(const Row& row, Hist& h, uint32_t prefix, int shift, int width, bool masses) {
  for (int i = threadIdx.x; i < BINS; i += DT) {
    h.cnt[i] = 0;
    h.mass[i] = 0;
  }
  __syncthreads();
  const uint32_t mask = (1u << width) - 1;
  for (int i = threadIdx.x; i < row.V; i += DT) {
    const float v = row.x[i];
    if (!row.drawable(v)) continue;
    const uint32_t d = row.down(v);
    if ((u64)d >> (shift + width) != prefix) continue;
    const uint32_t b = (d >> shift) & mask;
    atomicAdd(&h.cnt[b], 1u);
    if (masses) atomicAdd(&h.mass[b], row.mass(v));
  }
  __syncthreads();
}

// The first bin (from the top of the order) with which the counts (or masses)
// before it and its own reach `want` - that is before < want <= before + own;
// *before gets what lies above it. -1: all together stay below.
__device__ int find(const Hist& h, bool masses, u64 want, u64* before, u64* shared, u64* total) {
  const int i = 2 * threadIdx.x;
  const u64 a = masses ? h.mass[i] : h.cnt[i], b = masses ? h.mass[i + 1] : h.cnt[i + 1];
  u64 all;
  const u64 pre = block_scan(a + b, shared, &all);
  *total = all;
  if (threadIdx.x == 0) shared[DW] = (u64)-1;
  __syncthreads();
  if (pre < want && want <= pre + a) {
    shared[DW] = i;
    shared[DW + 1] = pre;
  } else if (pre + a < want && want <= pre + a + b) {
    shared[DW] = i + 1;
    shared[DW + 1] = pre + a;
  }
  __syncthreads();
  const int bin = (int)shared[DW];
  *before = shared[DW + 1];
  __syncthreads();
  return bin;
}

struct Cut {      // the kept ids: down < d, and the first `ties` ids of down == d
  uint32_t d;
  uint32_t ties;
};

// The cut at which the counts (masses) of the order reach `want` >= 1, given
// the histogram of the first digit; false where all of it stays below.
// before_mass (of counts): the mass above the cut, if asked for.
__device__ bool cut_at(const Row& row, Hist& h, bool masses, u64 want, Cut* cut, u64* shared) {
  u64 before, total, above = 0;
  int b = find(h, masses, want, &before, shared, &total);
  if (b < 0) return false;
  uint32_t prefix = b;
  above = before;
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const int shift = k == 0 ? 10 : 0, width = k == 0 ? 11 : 10;
    fill(row, h, prefix, shift, width, masses);
    b = find(h, masses, want - above, &before, shared, &total);
    above += before;
    prefix = (prefix << width) | (uint32_t)b;
  }
  cut->d = prefix;
  const u64 left = want - above;  // of the last digit's bin, all of one key
  if (masses) {
    const u64 each = h.mass[b] / h.cnt[b];
    cut->ties = (uint32_t)((left + each - 1) / each);
  } else {
    cut->ties = (uint32_t)left;
  }
  return true;
}

__global__ __launch_bounds__(DT) void k_draw_rows(DrawArgs a) {
  __shared__ Hist h;
  __shared__ u64 shared[DW + 2];
  __shared__ double tab[32];
  __shared__ float redf[DW];
  __shared__ int redi[DW];
  extern __shared__ __attribute__((aligned(16))) u64 chunk_mass[];  // [chunks], then their ties
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, r = blockIdx.x;
  const int chunks = (a.V + 63) / 64;
  unsigned int* chunk_ties = (unsigned int*)(chunk_mass + chunks);
  if (tid < 32) tab[tid] = exp2(tid / 32.0);
  Row row;
  row.x = a.x + (int64_t)r * a.ld;
  row.V = a.V;
  row.tab = tab;

  // the largest logit and its first id
  float m = -INFINITY;
  int at = 0x7fffffff;
  for (int i = tid; i < a.V; i += DT) {
    const float v = row.x[i];
    if (v > m) {
      m = v;
      at = i;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(m, o, 64);
    const int a2 = __shfl_xor(at, o, 64);
    if (m2 > m || (m2 == m && a2 < at)) {
      m = m2;
      at = a2;
    }
  }
  if (lane == 0) {
    redf[wv] = m;
    redi[wv] = at;
  }
  __syncthreads();
  m = redf[0];
  at = redi[0];
  for (int k = 1; k < DW; ++k)
    if (redf[k] > m || (redf[k] == m && redi[k] < at)) {
      m = redf[k];
      at = redi[k];
    }
  const float temp = a.c.temp ? a.c.temp[r] : 1.f;
  if (at == 0x7fffffff || temp <= 0.f) {
    if (tid == 0) {
      a.ids[r] = at == 0x7fffffff ? -1 : at;
      if (a.probs) a.probs[r] = at == 0x7fffffff ? 0.f : 1.f;
    }
    return;
  }
  row.m = m;
  row.km = key_of(m);
  row.inv_t = temp != temp ? 1.0 : 1.0 / (double)temp;
  const int top_k = a.c.top_k ? a.c.top_k[r] : 0;
  const float top_p = a.c.top_p ? a.c.top_p[r] : 1.f, min_p = a.c.min_p ? a.c.min_p[r] : 0.f;

  Cut cut{0xFFFFFFFFu, 0xFFFFFFFFu};  // everything
  const bool by_k = top_k > 0 && top_k < a.V, by_p = top_p < 1.f;
  if (by_k) {
    fill(row, h, 0, 21, 11, false);
    cut_at(row, h, false, (u64)top_k, &cut, shared);
  }
  if (by_p) {
    // the mass that top_k leaves, by id order of the ties as below
    u64 mass = 0, n = 0, all, ties;
    for (int i = tid; i < a.V; i += DT) {
      const float v = row.x[i];
      if (!row.drawable(v)) continue;
      const uint32_t d = row.down(v);
      if (d < cut.d || !by_k) mass += row.mass(v);
      if (by_k && d == cut.d) ++n;
    }
    block_scan(mass, shared, &all);
    __syncthreads();
    block_scan(n, shared, &ties);
    __syncthreads();
    if (by_k) {
      const u64 t = ties < cut.ties ? ties : cut.ties;
      // (a key's float: the inverse of key_of)
      const uint32_t k = row.km - cut.d;
      all += t * row.mass(__uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k));
    }
    const double want = ceil((double)(top_p > 0.f ? top_p : 0.f) * (double)all);
    fill(row, h, 0, 21, 11, true);
    Cut c2;
    if (cut_at(row, h, true, want < 1.0 ? 1ull : (u64)want, &c2, shared) &&
        (c2.d < cut.d || (c2.d == cut.d && c2.ties < cut.ties)))
      cut = c2;
  }
  const u64 floor_mass =
      min_p > 0.f ? (min_p >= 1.f ? 1ull << 44 : (u64)ceil((double)min_p * 17592186044416.0)) : 0;

  // kept mass and ties of each chunk of 64 ids
  auto kept = [&](float v, uint32_t d, u64* w) {  // above the cut, or one of its ties
    if (!row.drawable(v) || d > cut.d) return false;
    *w = row.mass(v);
    return *w >= floor_mass;
  };
  __syncthreads();
  for (int c = wv; c < chunks; c += DW) {
    const int i = 64 * c + lane;
    const float v = i < a.V ? row.x[i] : -INFINITY;
    u64 w = 0;
    const uint32_t d = row.drawable(v) ? row.down(v) : 0;
    const bool k = kept(v, d, &w);
    const uint64_t tie = __ballot(k && d == cut.d);
    const u64 s = wave_scan(k && d != cut.d ? w : 0);
    if (lane == 63) {
      chunk_mass[c] = s;
      chunk_ties[c] = __popcll(tie);
    }
  }
  __syncthreads();
  // the tied ids' own mass, and which of them stay: the first cut.ties
  u64 tie_mass = 0;
  {
    const uint32_t k = row.km - cut.d;
    if (cut.ties != 0xFFFFFFFFu && cut.d <= row.km)
      tie_mass = row.mass(__uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k));
  }
  const int per = (chunks + DT - 1) / DT, c0 = tid * per;
  u64 nt = 0, all, total;
  for (int q = 0; q < per; ++q)
    if (c0 + q < chunks) nt += chunk_ties[c0 + q];
  u64 tb = block_scan(nt, shared, &all);
  __syncthreads();
  u64 mine = 0;
  for (int q = 0; q < per; ++q)
    if (c0 + q < chunks) {
      const u64 n = chunk_ties[c0 + q];
      const u64 stay = tb >= cut.ties ? 0 : (n < cut.ties - tb ? n : cut.ties - tb);
      mine += chunk_mass[c0 + q] + stay * tie_mass;
      tb += n;
    }
  u64 before = block_scan(mine, shared, &total);
  const float u = a.c.u[r];
  double want = (double)(u > 0.f ? (u < 1.f ? u : 1.f) : 0.f) * (double)total;
  u64 target = (u64)want;
  if (target >= total) target = total - 1;
  __syncthreads();
  if (mine > 0 && before <= target && target < before + mine) {  // one thread
    tb -= nt;
    for (int q = 0; q < per && c0 + q < chunks; ++q) {
      const u64 n = chunk_ties[c0 + q];
      const u64 stay = tb >= cut.ties ? 0 : (n < cut.ties - tb ? n : cut.ties - tb);
      const u64 w = chunk_mass[c0 + q] + stay * tie_mass;
      if (target < before + w) {
        shared[DW] = c0 + q;
        shared[DW + 1] = target - before;
        shared[0] = stay;
        break;
      }
      before += w;
      tb += n;
    }
  }
  __syncthreads();
  if (wv != 0) return;
  const int c = (int)shared[DW], i = 64 * c + lane;
  const u64 stay = shared[0];
  const float v = i < a.V ? row.x[i] : -INFINITY;
  u64 w = 0;
  const uint32_t d = row.drawable(v) ? row.down(v) : 0;
  bool k = kept(v, d, &w);
  const uint64_t tie = __ballot(k && d == cut.d);
  if (d == cut.d && __popcll(tie & ((1ull << lane) - 1)) >= stay) k = false;
  const u64 s = wave_scan(k ? w : 0);
  const uint64_t hit = __ballot(k && s > shared[DW + 1]);
  if (lane == __builtin_ctzll(hit)) {
    a.ids[r] = i;
    if (a.probs) a.probs[r] = (float)((double)w / (double)total);
  }
}

}  // namespace

int64_t draw_work_bytes(int32_t, int32_t) { return 0; }

void launch_draw_rows(hipStream_t s, const float* logits, int32_t rows, int32_t V, int64_t ld,
                      const fg_draw_cfg& c, int32_t* ids, float* probs, void*) {
  const DrawArgs a{logits, V, ld, c, ids, probs};
  const unsigned lds = (unsigned)((V + 63) / 64 * 12 + 16);
  static std::atomic<uint64_t> lds_set{0};
  raise_lds_once((const void*)k_draw_rows, MAX_CHUNKS * 12 + 16, &lds_set);
  FG_LAUNCH(k_draw_rows, dim3((unsigned)rows), dim3(DT), lds, s, a);
}

}  // namespace fgpt
