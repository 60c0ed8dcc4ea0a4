// paged_internal.h -- launchers of the paged cache's operators (kern_paged.hip,
// kern_pages.hip, kern_draw.hip). Arguments are checked by the C entries
// (fgpt_paged.hip); all launches go to `s`.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <vector>

#include "../../include/fgpt.h"

namespace fgpt {

// ---- attention
// Where the attention's output goes: rows of fp32 or bf16, or the split operand
// planes of the GEMM that follows (tile_at over n_head * head_dim columns).
struct PagedOut {
  void* y = nullptr;
  int64_t ld = 0;            // elements
  uint16_t* planes = nullptr;
  int64_t plane = 0;
};
// Workspace of an attention launch: floats (0: none needed).
int64_t paged_attn_floats(const fg_pages& pg, const fg_ragged& b, const fg_attn_cfg& c);
void launch_paged_attn(hipStream_t s, const fg_pages& pg, const fg_ragged& b, const fg_attn_cfg& c,
                       const void* q, const PagedOut& out, float* work);

// ---- append and page copies
void launch_qk_append(hipStream_t s, const fg_pages& pg, const fg_ragged& b, const fg_append_cfg& c,
                      const void* qkv, void* q_out);
void launch_pages_copy(hipStream_t s, void* base, int32_t n_planes, int64_t plane_bytes,
                       int64_t page_bytes, const int32_t* src, const int32_t* dst, int32_t n);

// xo[i] = x[rows[i]] (nx floats a row), qo likewise of q (nq), i < n.
void launch_take_rows(hipStream_t s, const int32_t* rows, int n, const float* x, float* xo, int nx,
                      const float* q, float* qo, int nq);

// ---- pages
// The last page of a pool's sequence (-1: none) and how many sequences hold it.
int32_t pool_last_page(const fg_pool* p, int32_t seq, int32_t* holders);
// The sequence shares page `from` again, which others hold, in the place of its
// last one (what fg_pool_extend changed, once its tokens are trimmed).
void pool_share_again(fg_pool* p, int32_t seq, int32_t from);
// The moves of a compaction, and their taking effect: between the two the caller
// copies the pages, or lets the moves go when that fails.
struct PoolMoves {
  std::vector<int32_t> src, dst;
  std::vector<int32_t> to, free_pages;  // each page's new place; the free ones afterwards
};
void pool_plan_moves(const fg_pool* p, PoolMoves* m);  // (may throw)
void pool_apply_moves(fg_pool* p, PoolMoves* m);       // (does not)

// ---- draws
constexpr int32_t DRAW_MAX_V = 1 << 18;
int64_t draw_work_bytes(int32_t rows, int32_t V);
void launch_draw_rows(hipStream_t s, const float* logits, int32_t rows, int32_t V, int64_t ld,
                      const fg_draw_cfg& c, int32_t* ids, float* probs, void* work);

}  // namespace fgpt
