// kern_adjust.hip -- penalties over each row's history, biases and grammar masks
// on rows of logits (fg_adjust_rows of include/fgpt.h).
//
// A workgroup takes a slice of a row: it counts the history's ids of its slice in
// LDS (integers: the order of the atomics does not matter), goes through its logits
// once and writes them once. Each slice reads the whole history, which is short
// beside the row and comes from the L2.
// Bound by a slice's round trips one after another (starts, history, counts, new
// values), then by bytes: 48 rows of 131073 ids, histories of up to 4000, 300 biases,
// masks, 51 MB, 16.7 us (9 without lists). One row of 8192 ids takes 4.2.
#include "fgpt_internal.h"
#include "kern_common.h"
#include "paged_internal.h"

namespace fgpt {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4u_t __attribute__((ext_vector_type(4), aligned(4)));  // rows start anywhere
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int AT = 256;                  // threads
constexpr uint32_t SEEN = 0x80000000u;   // in the history, before count_from

struct AdjustArgs {
  const float* x;
  float* out;
  int V, slices;
  int64_t ld, out_ld;
  fg_adjust_cfg c;
};

// A row's part [a, z) of a list of n entries, from its starts, kept inside it.
struct Part {
  int a, z;
};
__device__ __forceinline__ Part part_of(const int32_t* start, int row, int n) {
  Part p;
  p.a = max(0, min(start[row], n));
  p.z = max(p.a, min(start[row + 1], n));
  return p;
}

// (NaN: off)
__device__ __forceinline__ float setting(const float* p, int row, float off) {
  const float v = p ? p[row] : off;
  return v == v ? v : off;
}

// Few ids of a slice change: the history's are listed as they are first counted,
// and new values are made entry by entry, from logits read again, not id by id
// (a quotient for each of 16 ids a thread took as long as the row itself). They
// are kept where the counts were, for the thread that writes the id.
template <int QUADS>
__global__ __launch_bounds__(AT) void k_adjust(AdjustArgs a) {
#pragma clang fp contract(off)
  constexpr int SLICE = 4 * AT * QUADS, HU = 8;  // history ids of a thread in flight
  __shared__ __attribute__((aligned(16))) uint32_t cnt[SLICE];  // counts, then new values
  __shared__ uint16_t list[SLICE];                              // ids of the history
  // bits: ids with a new value; that a bias names; that several do
  __shared__ uint32_t fresh[SLICE / 32], named[SLICE / 32], again[SLICE / 32];
  __shared__ int n_list, twice;
  __shared__ int ids[AT], n_wave[AT / 64];
  __shared__ float vals[AT];
  const int tid = threadIdx.x, row = blockIdx.x / a.slices, lo = blockIdx.x % a.slices * SLICE;
  const fg_adjust_cfg& c = a.c;
  const float* x = a.x + row * a.ld;
  float* out = a.out + row * a.out_ld;

  // this thread's ids: four from lo + 4 (tid + AT j) on
  f32x4_t v[QUADS];
#pragma unroll
  for (int j = 0; j < QUADS; ++j) {
    const int i = lo + 4 * (tid + AT * j);
    if (i + 4 <= a.V) {
      v[j] = *(const f32x4u_t*)(x + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = i + e < a.V ? x[i + e] : 0.f;
    }
  }
  int mask = -1;
  if (c.mask) {
    mask = c.mask_row ? c.mask_row[row] : row;
    if (mask >= c.n_mask) mask = -1;
  }
  uint32_t word[QUADS];
#pragma unroll
  for (int j = 0; j < QUADS; ++j) {
    const int i = lo + 4 * (tid + AT * j);
    word[j] = mask >= 0 && i < a.V ? c.mask[mask * c.mask_ld + i / 32] >> (i % 32) : 15u;
  }

  Part h = {0, 0}, b = {0, 0};
  if (c.hist && (c.rep || c.pres || c.freq)) h = part_of(c.hist_start, row, c.n_hist);
  if (c.bias) b = part_of(c.bias_start, row, c.n_bias);
  const bool listed = h.z > h.a || b.z > b.a;
  if (listed) {
    const int end = min(SLICE, a.V - lo);
    // the place of an id in the slice, or SLICE
    auto place = [&](int id) {
      const uint32_t s = (uint32_t)id - (uint32_t)lo;
      return id >= 0 && s < (uint32_t)end ? (int)s : SLICE;
    };
    auto bit = [](const uint32_t* set, int s) { return (set[s / 32] >> (s % 32)) & 1; };
    auto put = [](uint32_t* set, int s) { return (atomicOr(set + s / 32, 1u << (s % 32)) >> (s % 32)) & 1; };
    int id[HU];
    auto load = [&](int k) {
#pragma unroll
      for (int u = 0; u < HU; ++u) id[u] = k + u * AT < h.z ? c.hist[k + u * AT] : -1;
    };
    load(h.a + tid);
    // this thread's entry of the bias list's first AT
    const int id0 = b.a + tid < b.z ? c.bias_id[b.a + tid] : -1;
    const float bias0 = b.a + tid < b.z ? c.bias[b.a + tid] : 0.f;
    const int from = h.a + (c.count_from ? max(0, min(c.count_from[row], h.z - h.a)) : 0);
    const float rep0 = setting(c.rep, row, 1.f), pres = setting(c.pres, row, 0.f), freq = setting(c.freq, row, 0.f);
    const float rep = rep0 > 0.f ? rep0 : 1.f;
#pragma unroll
    for (int j = 0; j < QUADS; ++j) *(u32x4_t*)(cnt + 4 * (tid + AT * j)) = u32x4_t{0, 0, 0, 0};
    if (tid < SLICE / 32) fresh[tid] = named[tid] = again[tid] = 0;
    if (tid == 0) n_list = twice = 0;
    lds_barrier();

    for (int k = h.a + tid; h.z > h.a;) {
#pragma unroll
      for (int u = 0; u < HU; ++u) {
        const int s = place(id[u]);
        if (s == SLICE) continue;
        const uint32_t was = k + u * AT >= from ? atomicAdd(cnt + s, 1u) : atomicOr(cnt + s, SEEN);
        if (was == 0) list[atomicAdd(&n_list, 1)] = (uint16_t)s;
      }
      k += HU * AT;
      if (k >= h.z) break;
      load(k);
    }
    auto name = [&](int i) {
      const int s = place(i);
      if (s < SLICE && put(named, s)) {
        put(again, s);
        twice = 1;
      }
    };
    name(id0);
    for (int k = b.a + tid + AT; k < b.z; k += AT) name(c.bias_id[k]);
    lds_barrier();

    for (int i = tid; i < n_list; i += AT) {
      const int s = list[i];
      const uint32_t times = cnt[s] & ~SEEN;
      float y = x[lo + s];
      if (times) y = (y - pres) - freq * (float)times;
      y = y > 0.f ? y / rep : y * rep;
      cnt[s] = __float_as_uint(y);
      put(fresh, s);
    }
    if (b.z > b.a) {
      lds_barrier();
      auto add = [&](int s, float y) {
        const float was = bit(fresh, s) ? __uint_as_float(cnt[s]) : x[lo + s];
        cnt[s] = __float_as_uint(was + y);
        put(fresh, s);
      };
      const int s0 = place(id0);
      if (s0 < SLICE && !bit(again, s0)) add(s0, bias0);
      for (int k = b.a + tid + AT; k < b.z; k += AT) {
        const int s = place(c.bias_id[k]);
        if (s < SLICE && !bit(again, s)) add(s, c.bias[k]);
      }
      // ids that several entries name: these entries in order, AT of the list at a
      // time; the first entry of an id among them adds all of the id's
      for (int k0 = b.a; twice && k0 < b.z; k0 += AT) {
        const int k = k0 + tid, mine = k < b.z ? c.bias_id[k] : -1, s = place(mine);
        const bool one = s < SLICE && bit(again, s);
        const uint64_t all = __ballot(one);
        __syncthreads();  // (the last AT entries' are used)
        if ((tid & 63) == 0) n_wave[tid >> 6] = __popcll(all);
        __syncthreads();
        int at = __popcll(all & ((1ull << (tid & 63)) - 1)), n = 0;
#pragma unroll
        for (int w = 0; w < AT / 64; ++w) {
          if (w < tid >> 6) at += n_wave[w];
          n += n_wave[w];
        }
        if (one) {
          ids[at] = mine;
          vals[at] = c.bias[k];
        }
        __syncthreads();
        if (tid >= n) continue;
        const int it = ids[tid];
        bool first = true;
        for (int u = 0; u < tid; ++u) first &= ids[u] != it;
        for (int u = tid; first && u < n; ++u)
          if (ids[u] == it) add(place(it), vals[u]);
      }
    }
    lds_barrier();
  }
#pragma unroll
  for (int j = 0; j < QUADS; ++j) {
    const int t = 4 * (tid + AT * j), i = lo + t;
    if (listed) {
      const uint32_t has = fresh[t / 32] >> (t % 32);
      if (has & 15) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((has >> e) & 1) v[j][e] = __uint_as_float(cnt[t + e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!((word[j] >> e) & 1)) v[j][e] = -INFINITY;
    if (i + 4 <= a.V) {
      *(f32x4u_t*)(out + i) = v[j];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < a.V) out[i + e] = v[j][e];
    }
  }
}

}  // namespace

void launch_adjust_rows(hipStream_t s, const float* x, int32_t rows, int32_t V, int64_t ld, const fg_adjust_cfg& c,
                        float* out, int64_t out_ld) {
  AdjustArgs a{x, out, V, 0, ld, out_ld, c};
  if (!a.c.mask_ld) a.c.mask_ld = (V + 31) / 32;
  // slices of 2048 ids, or 1024 where those are too few to fill the CUs twice (the rows
  // above with 4096: 18.5 us)
  a.slices = (V + 2047) / 2048;
  if ((int64_t)rows * a.slices >= 512) {
    FG_LAUNCH((k_adjust<2>), dim3((unsigned)(rows * a.slices)), dim3(AT), 0, s, a);
  } else {
    a.slices = (V + 1023) / 1024;
    FG_LAUNCH((k_adjust<1>), dim3((unsigned)(rows * a.slices)), dim3(AT), 0, s, a);
  }
}

}  // namespace fgpt
