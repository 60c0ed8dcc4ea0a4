// fgpt_pool.hip -- the bookkeeping of a paged cache's pages (fg_pool_* of
// include/fgpt.h): which pages a sequence holds, which of them sequences share,
// which are free. Host only. Every function either does all of its work or
// leaves the pool as it was.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <exception>
#include <functional>
#include <vector>

#include "../../include/fgpt.h"
#include "fgpt_internal.h"
#include "paged_internal.h"

using namespace fgpt;

struct fg_pool {
  struct Seq {
    int32_t len = 0;
    std::vector<int32_t> pages;  // -1: given back by fg_pool_slide
    // positions given back, and the widest window that no longer sees them
    int32_t gone_lo = 0, gone_hi = 0, window = 0;
  };
  int32_t n_pages, page_size;
  std::vector<int32_t> ref;      // sequences that hold a page
  std::vector<int32_t> free_pages;  // a heap, the lowest page on top
  std::vector<Seq> seqs;

  int32_t pages_of(int64_t len) const { return (int32_t)((len + page_size - 1) / page_size); }
  void give_back(int32_t page) {  // (free_pages has room for every page)
    if (page >= 0 && --ref[page] == 0) {
      free_pages.push_back(page);
      std::push_heap(free_pages.begin(), free_pages.end(), std::greater<int32_t>());
    }
  }
  int32_t take() {
    std::pop_heap(free_pages.begin(), free_pages.end(), std::greater<int32_t>());
    const int32_t p = free_pages.back();
    free_pages.pop_back();
    ref[p] = 1;
    return p;
  }
  // Whether the rows at positions 0..len-1 that a next token could see are held.
  bool whole(const Seq& s, int32_t len) const {
    return s.gone_hi == 0 || len <= s.gone_lo || (int64_t)len >= (int64_t)s.gone_hi + s.window - 1;
  }
};

namespace {

int32_t err(int32_t code, const char* fmt, ...) {
  char msg[300];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof msg, fmt, ap);
  va_end(ap);
  return set_error(code, msg);
}

#define CHECK(cond, ...)                           \
  do {                                             \
    if (!(cond)) return err(FG_EARG, __VA_ARGS__); \
  } while (0)

// No exception leaves a C entry.
template <class F>
int32_t entry(F&& f) {
  try {
    return f();
  } catch (const std::exception& e) {
    return err(FG_EARG, "page pool: %s", e.what());
  }
}

#define CHECK_SEQ(p, s)                                                               \
  do {                                                                                \
    CHECK(p, "pool is NULL");                                                         \
    CHECK((s) >= 0 && (s) < (int32_t)(p)->seqs.size(), "sequence %d outside [0, %d)", \
          (int)(s), (int)(p)->seqs.size());                                           \
  } while (0)

}  // namespace

int32_t fgpt::pool_last_page(const fg_pool* p, int32_t seq, int32_t* holders) {
  const fg_pool::Seq& s = p->seqs[seq];
  const int32_t page = s.pages.empty() ? -1 : s.pages.back();
  *holders = page < 0 ? 0 : p->ref[page];
  return page;
}

void fgpt::pool_share_again(fg_pool* p, int32_t seq, int32_t from) {
  fg_pool::Seq& s = p->seqs[seq];
  p->give_back(s.pages.back());
  s.pages.back() = from;
  ++p->ref[from];
}

extern "C" int32_t fg_pool_create(int32_t n_pages, int32_t page_size, int32_t max_seq, fg_pool** out) {
  CHECK(out, "out is NULL");
  *out = nullptr;
  CHECK(n_pages >= 1 && max_seq >= 1, "n_pages and max_seq must be >= 1");
  CHECK(page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
        "page_size %d is not a power of two in 16..256", page_size);
  CHECK((int64_t)n_pages * page_size <= (int64_t)1 << 40 && max_seq <= 1 << 24, "pool too large");
  return entry([&] {
    std::vector<int32_t> ref((size_t)n_pages, 0), free_pages((size_t)n_pages);
    std::vector<fg_pool::Seq> seqs((size_t)max_seq);
    for (int32_t i = 0; i < n_pages; ++i) free_pages[i] = i;  // (ascending: a heap already)
    fg_pool* p = new fg_pool();
    p->n_pages = n_pages;
    p->page_size = page_size;
    p->ref.swap(ref);
    p->free_pages.swap(free_pages);
    p->seqs.swap(seqs);
    *out = p;
    return FG_OK;
  });
}

extern "C" int32_t fg_pool_destroy(fg_pool* p) {
  delete p;
  return FG_OK;
}

extern "C" int32_t fg_pool_len(const fg_pool* p, int32_t seq, int32_t* len) {
  CHECK_SEQ(p, seq);
  CHECK(len, "len is NULL");
  *len = p->seqs[seq].len;
  return FG_OK;
}

extern "C" int32_t fg_pool_free(const fg_pool* p, int32_t* n) {
  CHECK(p && n, "NULL argument");
  *n = (int32_t)p->free_pages.size();
  return FG_OK;
}

extern "C" int32_t fg_pool_table(const fg_pool* p, int32_t seq, int32_t* pages, int32_t cap, int32_t* n) {
  CHECK_SEQ(p, seq);
  CHECK(n, "n is NULL");
  const fg_pool::Seq& s = p->seqs[seq];
  *n = (int32_t)s.pages.size();
  if (!pages) return FG_OK;
  CHECK(cap >= *n, "sequence %d holds %d pages, room for %d", seq, *n, cap);
  std::copy(s.pages.begin(), s.pages.end(), pages);
  return FG_OK;
}

extern "C" int32_t fg_pool_need(const fg_pool* p, int32_t seq, int32_t n, int32_t* pages) {
  CHECK_SEQ(p, seq);
  CHECK(pages, "pages is NULL");
  const fg_pool::Seq& s = p->seqs[seq];
  CHECK(n >= 0 && (int64_t)s.len + n <= 1 << 30, "%d tokens after %d: outside 0..2^30", n, s.len);
  *pages = n ? p->pages_of((int64_t)s.len + n) - (int32_t)s.pages.size() : 0;
  if (n && s.len % p->page_size && p->ref[s.pages.back()] > 1) ++*pages;  // its shared last page
  return FG_OK;
}

extern "C" int32_t fg_pool_extend(fg_pool* p, int32_t seq, int32_t n, int32_t* src, int32_t* dst) {
  int32_t need = 0;
  const int32_t rc = fg_pool_need(p, seq, n, &need);
  if (rc != FG_OK) return rc;
  CHECK(src && dst, "NULL argument");
  if (need > (int32_t)p->free_pages.size())
    return err(FG_EFULL, "page pool full: %d pages needed, %d free", need, (int)p->free_pages.size());
  return entry([&] {
    fg_pool::Seq& s = p->seqs[seq];
    s.pages.reserve((size_t)p->pages_of((int64_t)s.len + n));
    *src = *dst = -1;
    if (n && s.len % p->page_size && p->ref[s.pages.back()] > 1) {
      const int32_t fresh = p->take();
      *src = s.pages.back();
      *dst = fresh;
      --p->ref[*src];
      s.pages.back() = fresh;
    }
    s.len += n;
    while ((int32_t)s.pages.size() < p->pages_of(s.len)) s.pages.push_back(p->take());
    return FG_OK;
  });
}

extern "C" int32_t fg_pool_fork(fg_pool* p, int32_t from, int32_t to, int32_t len) {
  CHECK_SEQ(p, from);
  CHECK_SEQ(p, to);
  fg_pool::Seq &a = p->seqs[from], &b = p->seqs[to];
  CHECK(from != to, "sequence %d cannot be forked into itself", from);
  CHECK(b.len == 0 && b.pages.empty(), "sequence %d is not empty", to);
  CHECK(len >= 0 && len <= a.len, "len %d outside [0, %d]", len, a.len);
  CHECK(p->whole(a, len), "len %d: positions %d..%d of sequence %d were given back", len, a.gone_lo,
        a.gone_hi - 1, from);
  return entry([&] {
    std::vector<int32_t> pages(a.pages.begin(), a.pages.begin() + p->pages_of(len));
    for (int32_t g : pages)
      if (g >= 0) ++p->ref[g];
    b.pages.swap(pages);
    b.len = len;
    if (len > a.gone_lo && a.gone_hi > 0) {
      b.gone_lo = a.gone_lo;
      b.gone_hi = a.gone_hi;
      b.window = a.window;
    }
    return FG_OK;
  });
}

extern "C" int32_t fg_pool_trim(fg_pool* p, int32_t seq, int32_t len) {
  CHECK_SEQ(p, seq);
  fg_pool::Seq& s = p->seqs[seq];
  CHECK(len >= 0 && len <= s.len, "len %d outside [0, %d]", len, s.len);
  CHECK(p->whole(s, len), "len %d: positions %d..%d of sequence %d were given back", len, s.gone_lo,
        s.gone_hi - 1, seq);
  for (int32_t i = p->pages_of(len); i < (int32_t)s.pages.size(); ++i) p->give_back(s.pages[i]);
  s.pages.resize((size_t)p->pages_of(len));
  s.len = len;
  if (len <= s.gone_lo) s.gone_lo = s.gone_hi = s.window = 0;
  return FG_OK;
}

extern "C" int32_t fg_pool_slide(fg_pool* p, int32_t seq, int32_t window, int32_t sinks) {
  CHECK_SEQ(p, seq);
  CHECK(window >= 1 && sinks >= 0, "window must be >= 1, sinks >= 0");
  fg_pool::Seq& s = p->seqs[seq];
  // the next token, at position len, sees positions from len - window + 1 on
  const int64_t first = std::max<int64_t>(0, (int64_t)s.len - window + 1);
  const int32_t a = (int32_t)(((int64_t)sinks + p->page_size - 1) / p->page_size);
  const int32_t z = (int32_t)(first / p->page_size);  // pages a .. z-1 are behind it
  bool any = false;
  for (int32_t i = a; i < z; ++i)
    if (s.pages[i] >= 0) {
      p->give_back(s.pages[i]);
      s.pages[i] = -1;
      any = true;
    }
  if (any) {
    s.gone_lo = s.gone_hi ? std::min(s.gone_lo, a * p->page_size) : a * p->page_size;
    s.gone_hi = std::max(s.gone_hi, z * p->page_size);
    s.window = std::max(s.window, window);
  }
  return FG_OK;
}

// The pages in use past their own number move to the free ones below it.
void fgpt::pool_plan_moves(const fg_pool* p, PoolMoves* m) {
  const int32_t used = p->n_pages - (int32_t)p->free_pages.size();
  m->to.resize((size_t)p->n_pages);
  for (int32_t i = 0; i < p->n_pages; ++i) {
    m->to[i] = i;
    if (i < used && p->ref[i] == 0) m->dst.push_back(i);
    if (i >= used && p->ref[i] > 0) m->src.push_back(i);
  }
  for (size_t i = 0; i < m->src.size(); ++i) m->to[m->src[i]] = m->dst[i];
  m->free_pages.reserve((size_t)p->n_pages);  // (room for every page)
  for (int32_t i = used; i < p->n_pages; ++i) m->free_pages.push_back(i);
}

void fgpt::pool_apply_moves(fg_pool* p, PoolMoves* m) {
  for (size_t i = 0; i < m->src.size(); ++i) {
    p->ref[m->dst[i]] = p->ref[m->src[i]];
    p->ref[m->src[i]] = 0;
  }
  for (fg_pool::Seq& s : p->seqs)
    for (int32_t& g : s.pages)
      if (g >= 0) g = m->to[g];
  p->free_pages.swap(m->free_pages);
}

extern "C" int32_t fg_pool_compact(fg_pool* p, int32_t* src, int32_t* dst, int32_t cap, int32_t* n) {
  CHECK(p && n, "NULL argument");
  return entry([&] {
    PoolMoves m;
    pool_plan_moves(p, &m);
    *n = (int32_t)m.src.size();
    if (*n == 0) return (int32_t)FG_OK;
    if (!src || !dst || cap < *n) return err(FG_EARG, "%d pages move, room for %d", *n, src && dst ? cap : 0);
    std::copy(m.src.begin(), m.src.end(), src);
    std::copy(m.dst.begin(), m.dst.end(), dst);
    pool_apply_moves(p, &m);
    return (int32_t)FG_OK;
  });
}
