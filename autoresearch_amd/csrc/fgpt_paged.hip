// fgpt_paged.hip -- the C entries of the paged cache's operators (include/fgpt.h):
// argument checks, the stream's device, the launches.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <vector>

#include "../../include/fgpt.h"
#include "fgpt_internal.h"
#include "paged_internal.h"

using namespace fgpt;

namespace {

int32_t err(int32_t code, const char* fmt, ...) {
  char msg[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof msg, fmt, ap);
  va_end(ap);
  return set_error(code, msg);
}

#define CHECK(cond, ...)                         \
  do {                                           \
    if (!(cond)) return err(FG_EARG, __VA_ARGS__); \
  } while (0)
#define RCCHK(x)                \
  do {                          \
    const int32_t r_ = (x);     \
    if (r_ != FG_OK) return r_; \
  } while (0)

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Makes the stream's device the current one for the call (NULL and the runtime's
// own streams are the current device's) and puts the caller's back afterwards.
class OnStream {
 public:
  int32_t enter(void* stream) {
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess || n < 1) {
      (void)hipGetLastError();
      return err(FG_ENODEV, "no HIP device visible");
    }
    int cur = 0, dev = 0;
    hipError_t e = hipGetDevice(&cur);
    dev = cur;
    const bool own = stream && stream != (void*)hipStreamLegacy && stream != (void*)hipStreamPerThread;
    if (e == hipSuccess && own) e = hipStreamGetDevice((hipStream_t)stream, &dev);
    if (e == hipSuccess && dev != cur) {
      e = hipSetDevice(dev);
      if (e == hipSuccess) back_ = cur;
    }
    if (e != hipSuccess) return err(FG_EHIP, "stream's device: %s", hipGetErrorString(e));
    return gfx950(dev);
  }
  ~OnStream() {
    if (back_ >= 0) (void)hipSetDevice(back_);
  }

 private:
  int back_ = -1;
  // (looked up once a device: the properties cost more than a launch)
  static int32_t gfx950(int dev) {
    static std::atomic<uint64_t> good{0};
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (good.load(std::memory_order_acquire) & bit) return FG_OK;
    hipDeviceProp_t p;
    const hipError_t e = hipGetDeviceProperties(&p, dev);
    if (e != hipSuccess) return err(FG_EHIP, "device properties: %s", hipGetErrorString(e));
    if (strncmp(p.gcnArchName, "gfx950", 6) != 0)
      return err(FG_ENODEV, "device %d is %s, this build targets gfx950", dev, p.gcnArchName);
    good.fetch_or(bit, std::memory_order_release);
    return FG_OK;
  }
};

int32_t launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FG_OK : err(FG_EHIP, "%s: %s", what, hipGetErrorString(e));
}

int32_t check_pages(const fg_pages* p) {
  CHECK(p && p->k && p->v, "pages: NULL argument");
  CHECK(p->head_dim == 64 || p->head_dim == 128, "head_dim %d unsupported (64 or 128)", p->head_dim);
  CHECK(p->page_size >= 16 && p->page_size <= 256 && (p->page_size & (p->page_size - 1)) == 0,
        "page_size %d is not a power of two in 16..256", p->page_size);
  CHECK(p->n_pages >= 1 && p->n_kv_head >= 1, "pages: n_pages and n_kv_head must be >= 1");
  CHECK(p->n_kv_head <= 1024, "n_kv_head %d above 1024", p->n_kv_head);
  CHECK((int64_t)p->n_pages * p->n_kv_head * p->page_size < (int64_t)1 << 32,
        "pages: %d x %d heads x %d rows above 2^32", p->n_pages, p->n_kv_head, p->page_size);
  CHECK(p->type == FG_F32 || p->type == FG_BF16, "pages: unknown type %d", p->type);
  CHECK(aligned(p->k) && aligned(p->v), "pages are not 16-byte aligned");
  return FG_OK;
}

int32_t check_batch(const fg_ragged* b, const fg_pages* p) {
  CHECK(b && b->q_start && b->kv_len && b->table, "batch: NULL argument");
  CHECK(b->n_seq >= 1, "batch: n_seq must be >= 1");
  CHECK(b->n_rows >= 0 && b->max_q >= 0, "batch: n_rows and max_q must be >= 0");
  CHECK(b->max_kv >= 0 && b->table_ld >= 1, "batch: max_kv must be >= 0, table_ld >= 1");
  CHECK((int64_t)b->max_kv <= (int64_t)b->table_ld * p->page_size,
        "batch: max_kv %d beyond table_ld %d pages of %d", b->max_kv, b->table_ld, p->page_size);
  // (launches of at most 2^23 workgroups)
  CHECK((int64_t)b->n_seq * p->n_kv_head <= 1 << 22 && b->n_rows <= 1 << 23,
        "batch: n_seq %d x %d heads above 2^22, or n_rows %d above 2^23", b->n_seq, p->n_kv_head, b->n_rows);
  CHECK(b->max_kv <= (1 << 30), "batch: max_kv %d above 2^30", b->max_kv);
  return FG_OK;
}

int32_t check_heads(int32_t n_head, const fg_pages* p, int32_t type, const fg_ragged* b) {
  CHECK(n_head >= 1 && n_head <= 1024 && n_head % p->n_kv_head == 0,
        "n_head %d is not a multiple of n_kv_head %d up to 1024", n_head, p->n_kv_head);
  CHECK(type == FG_F32 || type == FG_BF16, "unknown row type %d", type);
  CHECK((int64_t)b->n_rows * n_head <= 1 << 26, "batch: n_rows %d x %d heads above 2^26", b->n_rows,
        n_head);
  return FG_OK;
}

// Row distances: 0 = packed; else rows must not overlap and stay 16-byte aligned.
int32_t check_ld(int64_t ld, int64_t width, int32_t type, const char* what) {
  const int64_t step = type == FG_F32 ? 4 : 8;
  CHECK(ld == 0 || (ld >= width && ld % step == 0 && ld < ((int64_t)1 << 40)),
        "%s %lld: 0, or a multiple of %d from %lld on", what, (long long)ld, (int)step,
        (long long)width);
  return FG_OK;
}

int32_t check_attn(const fg_pages* pages, const fg_ragged* batch, const fg_attn_cfg* cfg) {
  RCCHK(check_pages(pages));
  RCCHK(check_batch(batch, pages));
  CHECK(cfg, "cfg is NULL");
  RCCHK(check_heads(cfg->n_head, pages, cfg->type, batch));
  CHECK(cfg->type == FG_F32 || pages->type == FG_BF16, "bf16 rows need bf16 pages");
  CHECK(cfg->window >= 0 && cfg->sinks >= 0, "window and sinks must be >= 0");
  CHECK(cfg->window <= (1 << 30) && cfg->sinks <= (1 << 30), "window or sinks above 2^30");
  CHECK(cfg->scale >= 0.f && cfg->scale <= 1e30f, "scale must be finite and >= 0");
  RCCHK(check_ld(cfg->q_ld, (int64_t)cfg->n_head * pages->head_dim, cfg->type, "q_ld"));
  RCCHK(check_ld(cfg->out_ld, (int64_t)cfg->n_head * pages->head_dim, cfg->type, "out_ld"));
  return FG_OK;
}

// The pages that a copy list has named, by hash: room for those alone, whatever
// the pool holds; on the stack up to SMALL pairs.
class Named {
 public:
  static constexpr int32_t SMALL = 64;
  explicit Named(int32_t n) {  // (may throw)
    while ((int64_t)1 << bits_ < 4 * (int64_t)n) ++bits_;
    if (n > SMALL) many_.assign((size_t)1 << bits_, 0);
    at_ = n > SMALL ? many_.data() : few_;
  }
  // 0: not named yet; else how (1 read, 2 written). It is named `how` from now on.
  int name(int32_t page, int how) {
    uint64_t& e = slot(page);
    const int was = (int)(e & 3);
    e = ((uint64_t)page << 2) | (uint64_t)how;
    return was;
  }

 private:
  uint64_t& slot(int32_t page) {
    uint64_t i = ((uint64_t)page * 0x9E3779B97F4A7C15ull) >> (64 - bits_);
    while (at_[i] && (at_[i] >> 2) != (uint64_t)page) i = (i + 1) & (((uint64_t)1 << bits_) - 1);
    return at_[i];
  }
  int bits_ = 4;
  uint64_t few_[4 * SMALL] = {};  // page << 2 | how; 0: free
  std::vector<uint64_t> many_;
  uint64_t* at_;
};

}  // namespace

// ------------------------------------------------------------ attention
extern "C" int32_t fg_paged_attn_work(const fg_pages* pages, const fg_ragged* batch,
                                      const fg_attn_cfg* cfg, int64_t* bytes) {
  CHECK(bytes, "bytes is NULL");
  RCCHK(check_attn(pages, batch, cfg));
  *bytes = batch->n_rows && batch->max_q ? 4 * paged_attn_floats(*pages, *batch, *cfg) : 0;
  return FG_OK;
}

extern "C" int32_t fg_paged_attn(const fg_pages* pages, const fg_ragged* batch,
                                 const fg_attn_cfg* cfg, const void* q, void* out, void* work,
                                 int64_t work_bytes, void* stream) {
  RCCHK(check_attn(pages, batch, cfg));
  if (batch->n_rows == 0 || batch->max_q == 0) return FG_OK;
  CHECK(q && out, "q or out is NULL");
  CHECK(aligned(q) && aligned(out) && aligned(work), "q, out or work is not 16-byte aligned");
  const int64_t packed = (int64_t)cfg->n_head * pages->head_dim;
  CHECK(out != q || batch->n_rows == 1 ||
            (cfg->q_ld ? cfg->q_ld : packed) == (cfg->out_ld ? cfg->out_ld : packed),
        "out is q with another row distance");
  const int64_t need = 4 * paged_attn_floats(*pages, *batch, *cfg);
  CHECK(need == 0 || (work && work_bytes >= need), "work: %lld bytes needed, %lld given",
        (long long)need, (long long)(work ? work_bytes : 0));
  OnStream on;
  RCCHK(on.enter(stream));
  PagedOut o;
  o.y = out;
  o.ld = cfg->out_ld ? cfg->out_ld : packed;
  launch_paged_attn((hipStream_t)stream, *pages, *batch, *cfg, q, o, (float*)work);
  return launched("paged attention");
}

// ------------------------------------------------------------ append
extern "C" int32_t fg_qk_append(const fg_pages* pages, const fg_ragged* batch,
                                const fg_append_cfg* cfg, const void* qkv, void* q_out,
                                void* stream) {
  RCCHK(check_pages(pages));
  RCCHK(check_batch(batch, pages));
  CHECK(cfg, "cfg is NULL");
  RCCHK(check_heads(cfg->n_head, pages, cfg->type, batch));
  const int64_t hd = pages->head_dim;
  RCCHK(check_ld(cfg->qkv_ld, (cfg->n_head + 2 * (int64_t)pages->n_kv_head) * hd, cfg->type, "qkv_ld"));
  RCCHK(check_ld(cfg->q_ld, cfg->n_head * hd, cfg->type, "q_ld"));
  CHECK(!cfg->norm || (cfg->eps >= 0.f && cfg->eps <= 1e30f), "eps must be finite and >= 0");
  CHECK(!cfg->cos_buf == !cfg->sin_buf, "cos_buf and sin_buf go together");
  CHECK(!cfg->cos_buf || cfg->rope_n >= batch->max_kv, "rope_n %d below max_kv %d", cfg->rope_n,
        batch->max_kv);
  CHECK(aligned(cfg->cos_buf) && aligned(cfg->sin_buf), "rope tables are not 16-byte aligned");
  if (batch->n_rows == 0) return FG_OK;
  CHECK(qkv && q_out, "qkv or q_out is NULL");
  CHECK(aligned(qkv) && aligned(q_out), "qkv or q_out is not 16-byte aligned");
  OnStream on;
  RCCHK(on.enter(stream));
  launch_qk_append((hipStream_t)stream, *pages, *batch, *cfg, qkv, q_out);
  return launched("append");
}

// ------------------------------------------------------------ page copies
extern "C" int32_t fg_pages_copy(void* base, int32_t n_planes, int64_t plane_bytes, int32_t n_pages,
                                 int64_t page_bytes, const int32_t* src, const int32_t* dst,
                                 int32_t n, void* stream) {
  CHECK(n >= 0 && n_planes >= 1 && n_pages >= 1, "n must be >= 0, n_planes and n_pages >= 1");
  CHECK(n_planes <= 65535, "n_planes %d above 65535", n_planes);
  CHECK(page_bytes >= 16 && page_bytes % 16 == 0 && page_bytes <= ((int64_t)1 << 30),
        "page_bytes %lld is not a multiple of 16 up to 2^30", (long long)page_bytes);
  CHECK(n_planes == 1 || (plane_bytes >= n_pages * page_bytes && plane_bytes % 16 == 0),
        "plane_bytes %lld: a multiple of 16, no less than %d pages", (long long)plane_bytes, n_pages);
  if (n == 0) return FG_OK;
  CHECK(base && src && dst, "NULL argument");
  CHECK(aligned(base), "base is not 16-byte aligned");
  try {
    CHECK(n <= n_pages, "%d copies among %d pages", n, n_pages);  // (some page would be written twice)
    Named pages(n);
    for (int32_t i = 0; i < n; ++i) {
      CHECK(src[i] >= 0 && src[i] < n_pages && dst[i] >= 0 && dst[i] < n_pages,
            "copy %d: page %d -> %d outside [0, %d)", i, src[i], dst[i], n_pages);
      CHECK(!pages.name(dst[i], 2), "copy %d: page %d is named before", i, dst[i]);
      CHECK(pages.name(src[i], 1) != 2, "copy %d: page %d is also written", i, src[i]);
    }
  } catch (const std::exception& e) {
    return err(FG_EARG, "page list: %s", e.what());
  }
  OnStream on;
  RCCHK(on.enter(stream));
  launch_pages_copy((hipStream_t)stream, base, n_planes, plane_bytes, page_bytes, src, dst, n);
  return launched("page copy");
}

// ------------------------------------------------------------ draws
extern "C" int32_t fg_draw_rows_work(int32_t rows, int32_t V, int64_t* bytes) {
  CHECK(bytes, "bytes is NULL");
  CHECK(rows >= 0, "rows must be >= 0");
  CHECK(V >= 1 && V <= DRAW_MAX_V, "V %d outside 1..%d", V, DRAW_MAX_V);
  *bytes = draw_work_bytes(rows, V);
  return FG_OK;
}

extern "C" int32_t fg_draw_rows(const float* logits, int32_t rows, int32_t V, int64_t ld,
                                const fg_draw_cfg* cfg, int32_t* ids, float* probs, void* work,
                                int64_t work_bytes, void* stream) {
  CHECK(rows >= 0, "rows must be >= 0");
  CHECK(V >= 1 && V <= DRAW_MAX_V, "V %d outside 1..%d", V, DRAW_MAX_V);
  CHECK(rows <= 1 << 21, "rows %d above 2^21", rows);
  CHECK(ld >= V && ld < ((int64_t)1 << 40), "ld %lld below V %d", (long long)ld, V);
  CHECK(cfg, "cfg is NULL");
  if (rows == 0) return FG_OK;
  CHECK(logits && ids && cfg->u, "logits, ids or u is NULL");
  const int64_t need = draw_work_bytes(rows, V);
  CHECK(need == 0 || (work && aligned(work) && work_bytes >= need),
        "work: %lld bytes needed, 16-byte aligned; %lld given", (long long)need,
        (long long)(work ? work_bytes : 0));
  OnStream on;
  RCCHK(on.enter(stream));
  launch_draw_rows((hipStream_t)stream, logits, rows, V, ld, *cfg, ids, probs, work);
  return launched("draw");
}
