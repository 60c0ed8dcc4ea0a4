// kern_pages.hip -- what fills, reads and moves the pages of a paged KV cache:
// k_qk_append (head norms, rotation, q out, k and v into their slots),
// k_pages_read (tokens' rows back out of their slots) and k_pages_copy
// (include/fgpt.h: fg_qk_append, fg_pages_read, fg_pages_copy).
#include <algorithm>
#include <type_traits>

#include "fgpt_internal.h"
#include "kern_codes.h"
#include "kern_common.h"
#include "paged_internal.h"

namespace fgpt {
namespace {

typedef uint32_t u32x4v_t __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------ append
// A thread keeps to one token row and LPH-th of a head: VEC dims of the head's
// first half and the same of its second, so that a rotation pair lies in one
// lane, every access is a 16-byte one and its cos and sin are read once; it goes
// through the row's heads, HU of them in flight at a time. Five, since the rows of
// 40 heads of 128 in bf16 and of 18 in fp32 then take one round (12k rows of the
// former, 62 us with four, 59 with five, 61 with six). The mean square of a
// head is a sum over its LPH lanes. A workgroup takes RW rows: four from 2048
// rows on, where the head weights that a thread reads serve more heads (12k
// rows of 40 bf16 heads of 128 with weights, 271 MB: 118 us with one row, 59 with
// four; 11k of 24 heads of 64 without 25, 15), one below that (1024 rows of the
// former shape 7.0 us, with four rows 8.6).
// Bound by bytes: the row once in, once out. Into 8-bit pages a head's lanes find its
// largest value and write 8 codes each, and one the scale: 10k rows of 32 bf16 heads on
// 4, 203 MB, 49 us (4.2 TB/s). q is stored in the ordinary way: past the caches' order of
// use it takes 43, but the attention that reads it next 6 more.
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
__device__ __forceinline__ void load_vals(const void* base, int64_t i, float (&v)[VEC]) {
#pragma unroll
  for (int k = 0; k < VEC; k += 4) {
    if constexpr (F) {
      const float4 x = *(const float4*)((const float*)base + i + k);
      v[k] = x.x, v[k + 1] = x.y, v[k + 2] = x.z, v[k + 3] = x.w;
    } else {
      const uint2 x = *(const uint2*)((const uint16_t*)base + i + k);
      v[k] = __uint_as_float(x.x << 16), v[k + 1] = __uint_as_float(x.x & 0xFFFF0000u);
      v[k + 2] = __uint_as_float(x.y << 16), v[k + 3] = __uint_as_float(x.y & 0xFFFF0000u);
    }
  }
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

// Largest of the group's values, likewise.
template <int N>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  auto dpp = [](uint32_t u, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, decltype(ctrl)::value, 0xF, 0xF, false);
  };
  v = max(v, dpp(v, std::integral_constant<int, 0xB1>()));
  v = max(v, dpp(v, std::integral_constant<int, 0x4E>()));
  if constexpr (N >= 8) v = max(v, dpp(v, std::integral_constant<int, 0x141>()));
  if constexpr (N >= 16) v = max(v, dpp(v, std::integral_constant<int, 0x140>()));
  return v;
}

// A head's row (this lane's dims of both halves) as 8-bit codes, and its scale:
// max|x| / top, codes x / scale to the nearest (ties to even). The largest is
// taken over the values' bits, where infinities and NaN are above every finite
// one: such a row's scale is NaN.
template <int KT, int LPH, int VEC>
__device__ __forceinline__ void store_codes(uint8_t* codes, float* scale, int d, int half,
                                            const float (&x1)[VEC], const float (&x2)[VEC]) {
  constexpr float TOP = KT == FG_I8 ? 127.f : 448.f;
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < VEC; ++k)
    m = max(m, max(__float_as_uint(x1[k]) & 0x7FFFFFFFu, __float_as_uint(x2[k]) & 0x7FFFFFFFu));
  m = group_max<LPH>(m);
  const bool finite = m < 0x7F800000u;
  float s = __uint_as_float(m) / TOP;
  if (!(s >= __FLT_MIN__)) s = 0.f;  // (its inverse would be infinite)
  const bool live = finite && s > 0.f;  // (else codes of 0, not of -0 or NaN)
  const float inv = live ? 1.0f / s : 0.f;
  auto code4 = [&](const float* x) -> uint32_t {
    float y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = live ? __builtin_amdgcn_fmed3f(x[k] * inv, -TOP, TOP) : 0.f;
    if constexpr (KT == FG_E4M3) {
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
    } else {
      uint32_t w = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) w |= ((uint32_t)(int)__builtin_rintf(y[k]) & 255u) << (8 * k);
      return w;
    }
  };
  if constexpr (VEC == 8) {
    *(uint2*)(codes + d) = make_uint2(code4(x1), code4(x1 + 4));
    *(uint2*)(codes + half + d) = make_uint2(code4(x2), code4(x2 + 4));
  } else {
    *(uint32_t*)(codes + d) = code4(x1);
    *(uint32_t*)(codes + half + d) = code4(x2);
  }
  if (d == 0) *scale = finite ? s : NAN;
}

// The rows r0 .. r0 + RW-1 of a batch, a wavefront each: at[i] = the row's
// sequence (the number of sequences that end at or before it) and its position;
// below 0: padding behind the last sequence, or none.
template <int RW>
__device__ __forceinline__ void find_rows(const fg_ragged& b, int r0, int (&at)[4][2]) {
  static_assert(RW <= 4, "a wavefront finds a row");
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  if (wv < RW) {
    const int row = r0 + wv;
    int seq = 0;
    for (int s0 = 0; s0 < b.n_seq; s0 += 64) {
      const bool before = s0 + lane < b.n_seq && b.q_start[s0 + lane + 1] <= row;
      seq += __popcll(__ballot(before));
    }
    if (lane == 0) {
      const bool real = row < b.n_rows && seq < b.n_seq;
      at[wv][0] = seq;
      at[wv][1] = real ? b.kv_len[seq] - (b.q_start[seq + 1] - row) : -1;
    }
  }
  __syncthreads();
}

template <int HD, bool QF, int KT, int RW>
__global__ __launch_bounds__(256) void k_qk_append(AppendArgs a) {
  typedef RowIO<HD, QF> IO;
  constexpr int VEC = IO::VEC, LPH = IO::LPH, HPT = 256 / (LPH * RW), HU = 5;  // heads at once
  __shared__ int at[4][2];  // the rows' sequences and positions
  const int r0 = blockIdx.x * RW;
  find_rows<RW>(a.b, r0, at);
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
        const int64_t block = (int64_t)page * KH + kvh;
        const int slot = pos & (P - 1);
        if constexpr (KT == FG_F32 || KT == FG_BF16) {
          const int64_t o = (block * P + slot) * HD + d;
          store_vals<VEC, KT == FG_F32>(base, o, x1);
          store_vals<VEC, KT == FG_F32>(base, o + HD / 2, x2);
        } else {
          uint8_t* b = (uint8_t*)base + block * P * (HD + 4);
          store_codes<KT, LPH>(b + slot * HD, (float*)(b + P * HD) + slot, d, HD / 2, x1, x2);
        }
      }
    }
  }
}

// ------------------------------------------------------------ reading back
// A thread takes as many values of a row of k or v as a 16-byte store holds, so that
// a wavefront's stores are whole lines; rows are found as in the append, RW of them a
// workgroup. fp32 in, code times scale, one rounding. The rows go out past the
// caches' order of use (stores marked nontemporal): 12 sequences of 3000 to 9000
// positions, e4m3 to bf16, 256 MB, 40 us, with ordinary stores 61.
struct ReadArgs {
  fg_pages pg;
  fg_ragged b;
  void* out[2];
  int64_t ld;
  int pshift;
};

template <int HD, int KT, bool OF, int RW>
__global__ __launch_bounds__(256) void k_pages_read(ReadArgs a) {
  constexpr int VPT = OF ? 4 : 8;                 // values a thread
  constexpr int CPH = HD / VPT, CPR = 256 / RW;   // chunks of a head; threads of a row
  __shared__ int at[4][2];
  const int r0 = blockIdx.x * RW;
  find_rows<RW>(a.b, r0, at);
  const int i = threadIdx.x / CPR, seq = at[i][0], pos = at[i][1];
  if (pos < 0 || pos >= a.b.max_kv) return;
  const int64_t row = r0 + i;
  const int P = 1 << a.pshift, slot = pos & (P - 1), KH = a.pg.n_kv_head;
  const int page = a.b.table[(int64_t)seq * a.b.table_ld + (pos >> a.pshift)];
  const bool kept = (uint32_t)page < (uint32_t)a.pg.n_pages;
  for (int c = threadIdx.x % CPR; c < 2 * KH * CPH; c += CPR) {
    const int val = c >= KH * CPH, h = c / CPH - val * KH, d = c % CPH * VPT;
    if (!a.out[val]) continue;
    const void* base = val ? a.pg.v : a.pg.k;
    const int64_t block = (int64_t)(kept ? page : 0) * KH + h;
    float x[VPT];
    if constexpr (KT == FG_F32 || KT == FG_BF16) {
      load_vals<VPT, KT == FG_F32>(base, (block * P + slot) * HD + d, x);
    } else {
      const uint8_t* b = (const uint8_t*)base + block * P * (HD + 4);
      const float s = ((const float*)(b + P * HD))[slot];
      uint32_t w[VPT / 4];
      if constexpr (VPT == 8) {
        const uint2 u = *(const uint2*)(b + slot * HD + d);
        w[0] = u.x;
        w[1] = u.y;
      } else {
        w[0] = *(const uint32_t*)(b + slot * HD + d);
      }
#pragma unroll
      for (int k = 0; k < VPT / 4; ++k) code_values<KT>(w[k], x + 4 * k);
#pragma unroll
      for (int k = 0; k < VPT; ++k) x[k] *= s;
    }
    if (!kept)
#pragma unroll
      for (int k = 0; k < VPT; ++k) x[k] = NAN;
    u32x4v_t w;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = OF ? __float_as_uint(x[k])
                : (uint32_t)f32_to_bf16_rne(x[2 * k % VPT]) | ((uint32_t)f32_to_bf16_rne(x[(2 * k + 1) % VPT]) << 16);
    __builtin_nontemporal_store(w, (u32x4v_t*)((char*)a.out[val] + (row * a.ld + h * HD + d) * (OF ? 4 : 2)));
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

template <int HD, bool QF, int KT>
void append_t(hipStream_t s, const AppendArgs& a) {
  if (a.b.n_rows >= 2048)
    FG_LAUNCH((k_qk_append<HD, QF, KT, 4>), dim3((unsigned)((a.b.n_rows + 3) / 4)), dim3(256), 0, s, a);
  else
    FG_LAUNCH((k_qk_append<HD, QF, KT, 1>), dim3((unsigned)a.b.n_rows), dim3(256), 0, s, a);
}

template <int HD, bool QF>
void append_q(hipStream_t s, const AppendArgs& a) {
  if (a.pg.type == FG_F32) append_t<HD, QF, FG_F32>(s, a);
  else if (a.pg.type == FG_BF16) append_t<HD, QF, FG_BF16>(s, a);
  else if (a.pg.type == FG_I8) append_t<HD, QF, FG_I8>(s, a);
  else append_t<HD, QF, FG_E4M3>(s, a);
}

template <int HD>
void append_hd(hipStream_t s, const AppendArgs& a) {
  if (a.c.type == FG_F32) append_q<HD, true>(s, a);
  else append_q<HD, false>(s, a);
}

template <int HD, int KT, bool OF>
void read_t(hipStream_t s, const ReadArgs& a) {
  if (a.b.n_rows >= 2048)
    FG_LAUNCH((k_pages_read<HD, KT, OF, 4>), dim3((unsigned)((a.b.n_rows + 3) / 4)), dim3(256), 0, s, a);
  else
    FG_LAUNCH((k_pages_read<HD, KT, OF, 1>), dim3((unsigned)a.b.n_rows), dim3(256), 0, s, a);
}

template <int HD, bool OF>
void read_k(hipStream_t s, const ReadArgs& a) {
  if (a.pg.type == FG_F32) read_t<HD, FG_F32, OF>(s, a);
  else if (a.pg.type == FG_BF16) read_t<HD, FG_BF16, OF>(s, a);
  else if (a.pg.type == FG_I8) read_t<HD, FG_I8, OF>(s, a);
  else read_t<HD, FG_E4M3, OF>(s, a);
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

void launch_pages_read(hipStream_t s, const fg_pages& pg, const fg_ragged& b, int32_t type, int64_t ld,
                       void* k_out, void* v_out) {
  const ReadArgs a{pg, b, {k_out, v_out}, ld ? ld : (int64_t)pg.n_kv_head * pg.head_dim,
                   __builtin_ctz(pg.page_size)};
  if (pg.head_dim == 128 && type == FG_F32) read_k<128, true>(s, a);
  else if (pg.head_dim == 128) read_k<128, false>(s, a);
  else if (type == FG_F32) read_k<64, true>(s, a);
  else read_k<64, false>(s, a);
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
