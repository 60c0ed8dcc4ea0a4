// kern_pages.hip -- what fills and moves the pages of a paged KV cache:
// k_qk_append (head norms, rotation, q out, k and v into their slots) and
// k_pages_copy (include/fgpt.h: fg_qk_append, fg_pages_copy).
#include "fgpt_internal.h"
#include "kern_common.h"
#include "paged_internal.h"

namespace fgpt {
namespace {

typedef uint32_t u32x4v_t __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------ append
// One workgroup a token row; LPH lanes a head, each with VEC dims of the
// head's first half and the same of its second, so that a rotation pair lies in
// one lane and every access is a 16-byte one. The mean square of a head is a
// sum over its LPH lanes. Bound by bytes: the row once in, once out.
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
  typedef float vals_t[VEC];
  static __device__ __forceinline__ void load(const void* base, int64_t i, vals_t& v) {
    if constexpr (F) {
      const float4 x = *(const float4*)((const float*)base + i);
      v[0] = x.x;
      v[1] = x.y;
      v[2] = x.z;
      v[3] = x.w;
    } else {
      unpack8(*(const uint4*)((const uint16_t*)base + i), v);
    }
  }
};

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

template <int HD, bool QF, bool KF>
__global__ __launch_bounds__(256) void k_qk_append(AppendArgs a) {
  typedef RowIO<HD, QF> IO;
  constexpr int VEC = IO::VEC, LPH = IO::LPH;
  const int row = blockIdx.x, lane = threadIdx.x & 63;
  // the row's sequence: the number of sequences that end at or before it
  int seq = 0;
  for (int s0 = 0; s0 < a.b.n_seq; s0 += 64) {
    const bool before = s0 + lane < a.b.n_seq && a.b.q_start[s0 + lane + 1] <= row;
    seq += __popcll(__ballot(before));
  }
  seq = __builtin_amdgcn_readfirstlane(seq);
  if (seq >= a.b.n_seq) return;  // padding behind the last sequence
  const int pos = a.b.kv_len[seq] - (a.b.q_start[seq + 1] - row);
  if (pos < 0 || pos >= a.b.max_kv) return;
  const int P = 1 << a.pshift;
  const int page = a.b.table[(int64_t)seq * a.b.table_ld + (pos >> a.pshift)];
  const bool kept = (uint32_t)page < (uint32_t)a.pg.n_pages;
  const int H = a.c.n_head, KH = a.pg.n_kv_head, nh = H + 2 * KH;
  const int sub = threadIdx.x % LPH, d = sub * VEC;  // dims d.. and HD/2 + d..
  const int64_t in0 = (int64_t)row * a.c.qkv_ld, q0 = (int64_t)row * a.c.q_ld;
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
  // (whole groups of LPH lanes leave the loop together: the sums stay within them)
  for (int h = threadIdx.x / LPH; h < nh; h += 256 / LPH) {
    float x1[VEC], x2[VEC];
    const int64_t at = in0 + (int64_t)h * HD;
    if (a.c.interleaved) {
      float u[VEC], w[VEC];
      IO::load(a.qkv, at + 2 * d, u);
      IO::load(a.qkv, at + 2 * d + VEC, w);
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) {
        x1[k] = u[2 * k];
        x2[k] = u[2 * k + 1];
        x1[VEC / 2 + k] = w[2 * k];
        x2[VEC / 2 + k] = w[2 * k + 1];
      }
    } else {
      IO::load(a.qkv, at + d, x1);
      IO::load(a.qkv, at + HD / 2 + d, x2);
    }
    if (h < H + KH) {
      if (a.c.norm) {
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < VEC; ++k) ss += x1[k] * x1[k] + x2[k] * x2[k];
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor(ss, o, 64);
        const float r = 1.0f / sqrtf(ss * (1.0f / HD) + a.c.eps);
        const float* w = h < H ? a.c.wq : a.c.wk;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          x1[k] *= r;
          x2[k] *= r;
          if (w) {
            x1[k] *= w[d + k];
            x2[k] *= w[HD / 2 + d + k];
          }
        }
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float u = x1[k], w = x2[k];
        x1[k] = u * cs[k] + w * sn[k];
        x2[k] = w * cs[k] - u * sn[k];
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

// ------------------------------------------------------------ page copies
// The list travels in the kernel's arguments (COPY_LIST pairs a launch), so the
// caller's arrays are free when the call returns and a captured launch holds
// its own list. A workgroup copies 16 KB of one page: four 16-byte loads a
// thread in flight before the first store. Bound by bytes.
constexpr int COPY_LIST = 440, COPY_CHUNK = 16384;
struct CopyArgs {
  char* base;
  int64_t plane_bytes, page_bytes;
  int n_planes, chunks;  // chunks of a page
  int32_t src[COPY_LIST], dst[COPY_LIST];
};

__global__ __launch_bounds__(256) void k_pages_copy(CopyArgs a) {
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

__global__ __launch_bounds__(256) void k_take_rows(const int32_t* __restrict__ rows,
                                                   const float* __restrict__ x, float* __restrict__ xo,
                                                   int nx, const float* __restrict__ q,
                                                   float* __restrict__ qo, int nq) {
  const int64_t from = rows[blockIdx.x], to = blockIdx.x;
  for (int k = threadIdx.x; k < nx; k += 256) xo[to * nx + k] = x[from * nx + k];
  for (int k = threadIdx.x; k < nq; k += 256) qo[to * nq + k] = q[from * nq + k];
}

template <int HD>
void append_hd(hipStream_t s, const AppendArgs& a) {
  const dim3 grid((unsigned)a.b.n_rows), block(256);
  if (a.pg.type == FG_F32 && a.c.type == FG_F32)
    FG_LAUNCH((k_qk_append<HD, true, true>), grid, block, 0, s, a);
  else if (a.c.type == FG_F32)
    FG_LAUNCH((k_qk_append<HD, true, false>), grid, block, 0, s, a);
  else if (a.pg.type == FG_F32)
    FG_LAUNCH((k_qk_append<HD, false, true>), grid, block, 0, s, a);
  else
    FG_LAUNCH((k_qk_append<HD, false, false>), grid, block, 0, s, a);
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
  CopyArgs a;
  a.base = (char*)base;
  a.plane_bytes = plane_bytes;
  a.page_bytes = page_bytes;
  a.n_planes = n_planes;
  a.chunks = (int)((page_bytes + COPY_CHUNK - 1) / COPY_CHUNK);
  for (int32_t i0 = 0; i0 < n; i0 += COPY_LIST) {
    const int m = n - i0 < COPY_LIST ? n - i0 : COPY_LIST;
    for (int i = 0; i < m; ++i) {
      a.src[i] = src[i0 + i];
      a.dst[i] = dst[i0 + i];
    }
    FG_LAUNCH(k_pages_copy, dim3((unsigned)(m * a.chunks), (unsigned)n_planes), dim3(256), 0, s, a);
  }
}

}  // namespace fgpt
