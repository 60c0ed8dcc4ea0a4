// kern_pages.hip -- what fills and moves the pages of a paged KV cache:
// k_qk_append (head norms, rotation, q out, k and v into their slots) and
// k_pages_copy (include/fgpt.h: fg_qk_append, fg_pages_copy).
#include <algorithm>

#include "fgpt_internal.h"
#include "kern_common.h"
#include "paged_internal.h"

namespace fgpt {
namespace {

typedef uint32_t u32x4v_t __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------ append
// A thread keeps to one token row and LPH-th of a head: VEC dims of the head's
// first half and the same of its second, so that a rotation pair lies in one
// lane, every access is a 16-byte one and its cos and sin are read once; it goes
// through the row's heads, HU of them in flight at a time. The mean square of a
// head is a sum over its LPH lanes. A workgroup takes RW rows: four from 2048
// rows on, where the head weights that a thread reads serve more heads (12k
// rows of 40 bf16 heads of 128 with weights, 271 MB: 118 us with one row, 62 with
// four; 11k of 24 heads of 64 without 25, 15), one below that (1024 rows of the
// former shape 7.0 us, with four rows 8.6).
// Bound by bytes: the row once in, once out.
struct AppendArgs {
  fg_pages pg;
  fg_ragged b;
  fg_append_cfg c;
  const void* qkv;
  void* q;
  int pshift;
};

template <int HD, bool F>
struct RowIO {
  static constexpr int VEC = F ? 4 : 8, LPH = HD / 2 / VEC;
  static __device__ __forceinline__ uint4 load(const void* base, int64_t i) {  // VEC values
    return *(const uint4*)((const char*)base + i * (F ? 4 : 2));
  }
  static __device__ __forceinline__ void values(const uint4& w, float (&v)[VEC]) {
    if constexpr (F) {
      v[0] = __uint_as_float(w.x);
      v[1] = __uint_as_float(w.y);
      v[2] = __uint_as_float(w.z);
      v[3] = __uint_as_float(w.w);
    } else {
      unpack8(w, v);
    }
  }
};

// Sum over aligned groups of N lanes (4, 8 or 16), in each of them: quad
// permutes, then half-row and row mirrors, which pair groups of equal values.
template <int N>
__device__ __forceinline__ float group_sum(float v) {
  v += dpp_f<0xB1>(v);
  v += dpp_f<0x4E>(v);
  if constexpr (N >= 8) v += dpp_f<0x141>(v);
  if constexpr (N >= 16) v += dpp_f<0x140>(v);
  return v;
}

template <int VEC, bool F>
__device__ __forceinline__ void store_vals(void* base, int64_t i, const float (&v)[VEC]) {
  if constexpr (F) {
#pragma unroll
    for (int k = 0; k < VEC; k += 4)
      *(float4*)((float*)base + i + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
  } else {
    uint32_t w[VEC / 2];
#pragma unroll
    for (int k = 0; k < VEC / 2; ++k)
      w[k] = (uint32_t)f32_to_bf16_rne(v[2 * k]) | ((uint32_t)f32_to_bf16_rne(v[2 * k + 1]) << 16);
    if constexpr (VEC == 8)
      *(uint4*)((uint16_t*)base + i) = make_uint4(w[0], w[1], w[2], w[3]);
    else
      *(uint2*)((uint16_t*)base + i) = make_uint2(w[0], w[1]);
  }
}

template <int HD, bool QF, bool KF, int RW>
__global__ __launch_bounds__(256) void k_qk_append(AppendArgs a) {
  typedef RowIO<HD, QF> IO;
  constexpr int VEC = IO::VEC, LPH = IO::LPH, HPT = 256 / (LPH * RW), HU = 4;  // heads at once
  static_assert(RW <= 4, "a wavefront finds a row");
  __shared__ int at[4][2];  // the rows' sequences and positions
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int r0 = blockIdx.x * RW;
  if (wv < RW) {
    // the row's sequence: the number of sequences that end at or before it
    const int row = r0 + wv;
    int seq = 0;
    for (int s0 = 0; s0 < a.b.n_seq; s0 += 64) {
      const bool before = s0 + lane < a.b.n_seq && a.b.q_start[s0 + lane + 1] <= row;
      seq += __popcll(__ballot(before));
    }
    if (lane == 0) {
      const bool real = row < a.b.n_rows && seq < a.b.n_seq;  // (else padding behind the last sequence)
      at[wv][0] = seq;
      at[wv][1] = real ? a.b.kv_len[seq] - (a.b.q_start[seq + 1] - row) : -1;
    }
  }
  __syncthreads();
  const int slot = threadIdx.x / LPH % RW, seq = at[slot][0], pos = at[slot][1];
  // (a whole group of LPH lanes has one row: the sums stay within it)
  if (pos < 0 || pos >= a.b.max_kv) return;
  const int64_t row = r0 + slot;
  const int P = 1 << a.pshift;
  const int page = a.b.table[(int64_t)seq * a.b.table_ld + (pos >> a.pshift)];
  const bool kept = (uint32_t)page < (uint32_t)a.pg.n_pages;
  const int H = a.c.n_head, KH = a.pg.n_kv_head, nh = H + 2 * KH;
  const int d = threadIdx.x % LPH * VEC;  // dims d.. and HD/2 + d..
  const int64_t in0 = row * a.c.qkv_ld, q0 = row * a.c.q_ld;
  float cs[VEC], sn[VEC];
  if (a.c.cos_buf) {
#pragma unroll
    for (int k = 0; k < VEC; k += 4) {
      const int64_t t = (int64_t)pos * (HD / 2) + d + k;
      const float4 x = *(const float4*)(a.c.cos_buf + t), y = *(const float4*)(a.c.sin_buf + t);
      cs[k] = x.x, cs[k + 1] = x.y, cs[k + 2] = x.z, cs[k + 3] = x.w;
      sn[k] = y.x, sn[k + 1] = y.y, sn[k + 2] = y.z, sn[k + 3] = y.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) cs[k] = 1.f, sn[k] = 0.f;
  }
  float wq[2 * VEC], wk[2 * VEC];
#pragma unroll
  for (int k = 0; k < 2 * VEC; ++k) {
    const int e = k < VEC ? d + k : HD / 2 + d + k - VEC;
    wq[k] = a.c.norm && a.c.wq ? a.c.wq[e] : 1.f;
    wk[k] = a.c.norm && a.c.wk ? a.c.wk[e] : 1.f;
  }
  // the two loads of a head: its halves' dims, or (interleaved) the pairs of d ..
  // and d + VEC/2 ..
  const int64_t l1 = a.c.interleaved ? 2 * d : d, l2 = a.c.interleaved ? 2 * d + VEC : HD / 2 + d;
  for (int h0 = threadIdx.x / (LPH * RW); h0 < nh; h0 += HU * HPT) {
    uint4 w1[HU], w2[HU];
#pragma unroll
    for (int u = 0; u < HU; ++u)
      if (h0 + u * HPT < nh) {
        const int64_t i = in0 + (int64_t)(h0 + u * HPT) * HD;
        w1[u] = IO::load(a.qkv, i + l1);
        w2[u] = IO::load(a.qkv, i + l2);
      }
#pragma unroll
    for (int u = 0; u < HU; ++u) {
      const int h = h0 + u * HPT;
      if (h >= nh) break;
      float x1[VEC], x2[VEC];
      if (a.c.interleaved) {
        float s[VEC], t[VEC];
        IO::values(w1[u], s);
        IO::values(w2[u], t);
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) {
          x1[k] = s[2 * k];
          x2[k] = s[2 * k + 1];
          x1[VEC / 2 + k] = t[2 * k];
          x2[VEC / 2 + k] = t[2 * k + 1];
        }
      } else {
        IO::values(w1[u], x1);
        IO::values(w2[u], x2);
      }
      if (h < H + KH) {
        if (a.c.norm) {
          float ss = 0.f;
#pragma unroll
          for (int k = 0; k < VEC; ++k) ss += x1[k] * x1[k] + x2[k] * x2[k];
          ss = group_sum<LPH>(ss);
          const float r = __builtin_amdgcn_rsqf(ss * (1.0f / HD) + a.c.eps);  // (off by an ulp at most)
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            x1[k] *= r * (h < H ? wq[k] : wk[k]);
            x2[k] *= r * (h < H ? wq[VEC + k] : wk[VEC + k]);
          }
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float s = x1[k], t = x2[k];
          x1[k] = s * cs[k] + t * sn[k];
          x2[k] = t * cs[k] - s * sn[k];
        }
      }
      if (h < H) {
        store_vals<VEC, QF>(a.q, q0 + (int64_t)h * HD + d, x1);
        store_vals<VEC, QF>(a.q, q0 + (int64_t)h * HD + HD / 2 + d, x2);
      } else if (kept) {
        const bool key = h < H + KH;
        const int kvh = h - H - (key ? 0 : KH);
        void* base = key ? a.pg.k : a.pg.v;
        const int64_t o = (((int64_t)page * KH + kvh) * P + (pos & (P - 1))) * HD + d;
        store_vals<VEC, KF>(base, o, x1);
        store_vals<VEC, KF>(base, o + HD / 2, x2);
      }
    }
  }
}

// ------------------------------------------------------------ page copies
// The list travels in the kernel's arguments (COPY_LIST pairs a launch, or 16
// where there are no more: less to write and to read), so the caller's arrays
// are free when the call returns and a captured launch holds its own list. A
// workgroup copies 16 KB of one page: four 16-byte loads a thread in flight
// before the first store. Bound by bytes: 701 pages of 40 planes, 1.84 GB moved,
// 368 us, 5.0 TB/s (a copy of 1 GB: 5.1).
constexpr int COPY_LIST = 440, COPY_FEW = 16, COPY_CHUNK = 16384;
template <int N>
struct CopyArgs {
  char* base;
  int64_t plane_bytes, page_bytes;
  int chunks;  // of a page
  int32_t src[N], dst[N];
};

template <int N>
__global__ __launch_bounds__(256) void k_pages_copy(CopyArgs<N> a) {
  const int chunk = blockIdx.x % a.chunks, i = blockIdx.x / a.chunks;
  const int64_t at = (int64_t)chunk * COPY_CHUNK + threadIdx.x * 16;
  char* plane = a.base + blockIdx.y * a.plane_bytes;
  const char* s = plane + a.src[i] * a.page_bytes;
  char* d = plane + a.dst[i] * a.page_bytes;
  u32x4v_t v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (at + k * 4096 < a.page_bytes) v[k] = *(const u32x4v_t*)(s + at + k * 4096);
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (at + k * 4096 < a.page_bytes) *(u32x4v_t*)(d + at + k * 4096) = v[k];
}

template <int N>
void copy_list(hipStream_t s, char* base, int32_t n_planes, int64_t plane_bytes, int64_t page_bytes,
               const int32_t* src, const int32_t* dst, int n) {
  CopyArgs<N> a;
  a.base = base;
  a.plane_bytes = plane_bytes;
  a.page_bytes = page_bytes;
  a.chunks = (int)((page_bytes + COPY_CHUNK - 1) / COPY_CHUNK);
  for (int i = 0; i < n; ++i) {
    a.src[i] = src[i];
    a.dst[i] = dst[i];
  }
  FG_LAUNCH((k_pages_copy<N>), dim3((unsigned)(n * a.chunks), (unsigned)n_planes), dim3(256), 0, s, a);
}

__global__ __launch_bounds__(256) void k_take_rows(const int32_t* __restrict__ rows,
                                                   const float* __restrict__ x, float* __restrict__ xo,
                                                   int nx, const float* __restrict__ q,
                                                   float* __restrict__ qo, int nq) {
  const int64_t from = rows[blockIdx.x], to = blockIdx.x;
  for (int k = threadIdx.x; k < nx; k += 256) xo[to * nx + k] = x[from * nx + k];
  for (int k = threadIdx.x; k < nq; k += 256) qo[to * nq + k] = q[from * nq + k];
}

template <int HD, bool QF, bool KF>
void append_t(hipStream_t s, const AppendArgs& a) {
  if (a.b.n_rows >= 2048)
    FG_LAUNCH((k_qk_append<HD, QF, KF, 4>), dim3((unsigned)((a.b.n_rows + 3) / 4)), dim3(256), 0, s, a);
  else
    FG_LAUNCH((k_qk_append<HD, QF, KF, 1>), dim3((unsigned)a.b.n_rows), dim3(256), 0, s, a);
}

template <int HD>
void append_hd(hipStream_t s, const AppendArgs& a) {
  if (a.pg.type == FG_F32 && a.c.type == FG_F32) append_t<HD, true, true>(s, a);
  else if (a.c.type == FG_F32) append_t<HD, true, false>(s, a);
  else if (a.pg.type == FG_F32) append_t<HD, false, true>(s, a);
  else append_t<HD, false, false>(s, a);
}

}  // namespace

void launch_qk_append(hipStream_t s, const fg_pages& pg, const fg_ragged& b, const fg_append_cfg& c,
                      const void* qkv, void* q_out) {
  AppendArgs a{pg, b, c, qkv, q_out, __builtin_ctz(pg.page_size)};
  if (!a.c.qkv_ld) a.c.qkv_ld = (int64_t)(c.n_head + 2 * pg.n_kv_head) * pg.head_dim;
  if (!a.c.q_ld) a.c.q_ld = (int64_t)c.n_head * pg.head_dim;
  if (pg.head_dim == 128)
    append_hd<128>(s, a);
  else
    append_hd<64>(s, a);
}

void launch_take_rows(hipStream_t s, const int32_t* rows, int n, const float* x, float* xo, int nx,
                      const float* q, float* qo, int nq) {
  FG_LAUNCH(k_take_rows, dim3((unsigned)n), dim3(256), 0, s, rows, x, xo, nx, q, qo, nq);
}

void launch_pages_copy(hipStream_t s, void* base, int32_t n_planes, int64_t plane_bytes,
                       int64_t page_bytes, const int32_t* src, const int32_t* dst, int32_t n) {
  // (a launch of at most 2^22 workgroups a plane)
  const int64_t chunks = (page_bytes + COPY_CHUNK - 1) / COPY_CHUNK;
  const int32_t most = (int32_t)std::min<int64_t>(COPY_LIST, (1 << 22) / chunks);
  for (int32_t i = 0; i < n; i += most) {
    const int32_t m = std::min(most, n - i);
    if (m <= COPY_FEW)
      copy_list<COPY_FEW>(s, (char*)base, n_planes, plane_bytes, page_bytes, src + i, dst + i, m);
    else
      copy_list<COPY_LIST>(s, (char*)base, n_planes, plane_bytes, page_bytes, src + i, dst + i, m);
  }
}

}  // namespace fgpt
