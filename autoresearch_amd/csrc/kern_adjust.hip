// kern_adjust.hip -- penalties over each row's history, biases and grammar masks
// on rows of logits (fg_adjust_rows of include/fgpt.h).
//
// A workgroup takes a slice of a row: it counts the history's ids of its slice in
// LDS (integers: the order of the atomics does not matter), goes through its logits
// once and writes them once. Each slice reads the whole history, which is short
// beside the row and comes from the L2.
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

template <int QUADS>
__global__ __launch_bounds__(AT) void k_adjust(AdjustArgs a) {
#pragma clang fp contract(off)
  constexpr int SLICE = 4 * AT * QUADS;
  __shared__ __attribute__((aligned(16))) uint32_t cnt[SLICE];   // of the history
  __shared__ __attribute__((aligned(16))) uint32_t nb[SLICE];    // biases of an id
  __shared__ __attribute__((aligned(16))) float bias[SLICE];     // their sum
  __shared__ int ids[AT];
  __shared__ float vals[AT];
  __shared__ int twice;  // an id of the slice is named twice
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
  uint32_t word[QUADS];
  int mask = -1;
  if (c.mask) {
    mask = c.mask_row ? c.mask_row[row] : row;
    if (mask >= c.n_mask) mask = -1;
  }
#pragma unroll
  for (int j = 0; j < QUADS; ++j) {
    const int i = lo + 4 * (tid + AT * j);
    word[j] = mask >= 0 && i < a.V ? c.mask[mask * c.mask_ld + i / 32] >> (i % 32) : 15u;
  }

  Part h = {0, 0}, b = {0, 0};
  if (c.hist && (c.rep || c.pres || c.freq)) h = part_of(c.hist_start, row, c.n_hist);
  if (c.bias) b = part_of(c.bias_start, row, c.n_bias);
  if (h.z > h.a || b.z > b.a) {
#pragma unroll
    for (int j = 0; j < QUADS; ++j) {
      *(u32x4_t*)(cnt + 4 * (tid + AT * j)) = u32x4_t{0, 0, 0, 0};
      *(u32x4_t*)(nb + 4 * (tid + AT * j)) = u32x4_t{0, 0, 0, 0};
    }
    if (tid == 0) twice = 0;
    __syncthreads();
    const int end = min(SLICE, a.V - lo);
    const int from = h.a + (c.count_from ? max(0, min(c.count_from[row], h.z - h.a)) : 0);
    for (int k = h.a + tid; k < h.z; k += 4 * AT) {
      int id[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) id[u] = k + u * AT < h.z ? c.hist[k + u * AT] : -1;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t s = (uint32_t)id[u] - (uint32_t)lo;
        if (id[u] < 0 || s >= (uint32_t)end) continue;
        if (k + u * AT >= from) atomicAdd(cnt + s, 1u);
        else atomicOr(cnt + s, SEEN);
      }
    }
    for (int k = b.a + tid; k < b.z; k += AT) {
      const int id = c.bias_id[k];
      const uint32_t s = (uint32_t)id - (uint32_t)lo;
      if (id >= 0 && s < (uint32_t)end && atomicAdd(nb + s, 1u)) twice = 1;
    }
    __syncthreads();
    if (b.z > b.a) {
      if (!twice) {
        for (int k = b.a + tid; k < b.z; k += AT) {
          const int id = c.bias_id[k];
          const uint32_t s = (uint32_t)id - (uint32_t)lo;
          if (id >= 0 && s < (uint32_t)end) bias[s] = c.bias[k];
        }
      } else {
        // the list in order, AT entries at a time: the first entry of an id in them
        // adds up the id's, so that sums do not depend on who comes first
#pragma unroll
        for (int j = 0; j < QUADS; ++j) *(f32x4_t*)(bias + 4 * (tid + AT * j)) = f32x4_t{0.f, 0.f, 0.f, 0.f};
        for (int k0 = b.a; k0 < b.z; k0 += AT) {
          const int k = k0 + tid, id = k < b.z ? c.bias_id[k] : -1;
          __syncthreads();
          ids[tid] = id;
          vals[tid] = k < b.z ? c.bias[k] : 0.f;
          __syncthreads();
          const uint32_t s = (uint32_t)id - (uint32_t)lo;
          if (id < 0 || s >= (uint32_t)end) continue;
          bool first = true;
          float sum = bias[s];
          if (nb[s] == 1) {
            sum = vals[tid];
          } else {
            for (int u = 0; u < tid; ++u) first &= ids[u] != id;
            for (int u = tid; first && u < AT; ++u)
              if (ids[u] == id) sum += vals[u];
          }
          if (first) bias[s] = sum;
        }
      }
      __syncthreads();
    }
    const float rep0 = setting(c.rep, row, 1.f), pres = setting(c.pres, row, 0.f), freq = setting(c.freq, row, 0.f);
    const float rep = rep0 > 0.f ? rep0 : 1.f;
#pragma unroll
    for (int j = 0; j < QUADS; ++j) {
      const u32x4_t n = *(const u32x4_t*)(cnt + 4 * (tid + AT * j)), m = *(const u32x4_t*)(nb + 4 * (tid + AT * j));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (n[e]) {
          const uint32_t times = n[e] & ~SEEN;
          float y = v[j][e];
          if (times) y = (y - pres) - freq * (float)times;
          v[j][e] = y > 0.f ? y / rep : y * rep;
        }
        if (m[e]) v[j][e] += bias[4 * (tid + AT * j) + e];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < QUADS; ++j) {
    const int i = lo + 4 * (tid + AT * j);
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
  a.slices = (V + 4095) / 4096;
  if ((int64_t)rows * a.slices >= 512) {
    FG_LAUNCH((k_adjust<4>), dim3((unsigned)(rows * a.slices)), dim3(AT), 0, s, a);
  } else {
    a.slices = (V + 1023) / 1024;
    FG_LAUNCH((k_adjust<1>), dim3((unsigned)(rows * a.slices)), dim3(AT), 0, s, a);
  }
}

}  // namespace fgpt
