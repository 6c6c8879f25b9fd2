// The paged KV caches' plans' work lists, the 8-bit one's layout, and the sizes
// that host and kernels agree on.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "oi2.h"

namespace oi2 {

constexpr int kPage = OI2_PAGE;
constexpr int kHeadD = 128;
constexpr int kHalfBlock = kPage * kHeadD;   // bytes of one page and head of k or of v
constexpr int kBlock = 2 * kHalfBlock;
constexpr float kCodeMax = 448.0f;
constexpr int kExpMin = -40, kExpMax = 60;

// Query rows (tokens times query heads per kv head) of a workgroup of the
// attention: up to 16 in the kernel for few rows, 128 in the one for many.
constexpr int kFewRows = 16, kManyRows = 128;
// Waves of a workgroup for few rows, each every fourth page.
constexpr int kFewWaves = 4;
// Workgroups that the attention's work is cut for, over all rows and kv heads.
constexpr int kFewWgs = 512, kManyWgs = 512;
// Tiles of up to so many pages are never cut: a round of four pages costs about
// 1.1 us, joining parts 3.5.
constexpr int kFewWhole = 16, kManyWhole = 16;

// Work lists of a plan.
struct AppendItem {           // one page that the step writes to
  int32_t page, token0;       // its first new token, in the packed order
  int32_t held, upto;         // places [held, upto) of the page are new
};
struct ItemHead {             // query tokens of one row over a range of its pages
  int32_t row, token0, n_tokens, pos0;    // pos0: position of token0
  int32_t page0, page1, kv_len;
  int32_t part, n_parts;                  // of the tokens' pages: which part, of how many
  int32_t slot0;                          // the parts' partial sums are at slot0 + part
  int32_t pad[2];
};
struct AttendItem : ItemHead {
  int32_t ids[4];                         // the first pages, so that they need no look-up
};
constexpr int kItemInts = sizeof(AttendItem) / 4;

struct PlanLayout {           // offsets in ints into oi2_page_plan.work
  int32_t cap_append, cap_few, cap_many, cap_parts_few, cap_parts_many;
  int32_t few_tokens, many_tokens;        // tokens of a workgroup
  int32_t parts_few, parts_many;          // parts per kv head that the work is cut for
  int64_t append, few, many, ints;
};
// counts at the head of the work lists
enum { kNAppend = 0, kNFew, kNMany, kHeadInts = 16 };

inline int64_t min64(int64_t a, int64_t b) { return a < b ? a : b; }

// Sizes for steps of at most n_tokens (<= max_tokens) tokens.
inline PlanLayout plan_layout(const oi2_paged& c, int32_t n_tokens, int32_t max_new) {
  PlanLayout l{};
  const int g = c.n_q / c.n_kv;
  const int64_t width = ((int64_t)c.max_len + kPage - 1) / kPage;
  const int64_t rows = min64(c.n_seqs, n_tokens);
  l.few_tokens = kFewRows / g;
  l.many_tokens = kManyRows / g;
  l.parts_many = (kManyWgs + c.n_kv - 1) / c.n_kv;
  // a row's n tokens touch at most n, and at most n / 64 + 2, pages
  l.cap_append = (int32_t)min64(min64(n_tokens, n_tokens / kPage + 2 * rows), c.n_pages);
  // where no row may have more than kFewRows, a rejected one still gets its zeros
  // from the kernel for few rows, in several tiles
  const bool few_only = (int64_t)max_new * g <= kFewRows;
  l.parts_few = (kFewWgs + c.n_kv - 1) / c.n_kv;
  const int64_t few = rows + (few_only ? n_tokens / l.few_tokens : 0), many = few_only ? 0 : rows + n_tokens / l.many_tokens;
  // parts are at least total / parts pages long, so there are tiles + parts of
  // them, and twice as many where only tiles with several count
  const bool cut_few = width > kFewWhole, cut_many = width > kManyWhole && many > 0;
  l.cap_few = (int32_t)(few + (cut_few ? l.parts_few : 0));
  l.cap_many = (int32_t)(many + (cut_many ? l.parts_many : 0));
  l.cap_parts_few = cut_few ? 2 * l.parts_few : 0;
  l.cap_parts_many = cut_many ? 2 * l.parts_many : 0;
  l.append = kHeadInts;
  l.few = l.append + 4 * (int64_t)l.cap_append;
  l.many = l.few + kItemInts * (int64_t)l.cap_few;
  l.ints = l.many + kItemInts * (int64_t)l.cap_many;
  return l;
}

// Checks of the arguments that the entry points share; OI2_OK or an error set.
int check_paged(const oi2_paged* c, int32_t layer, bool pool);
int check_plan(const oi2_paged* c, const oi2_page_plan* p);
int check_paged4(const oi2_paged* c, int32_t layer);     // of the 4-bit cache, which has no scales besides its pages

// The 4-bit cache's append and attention as one call's: the append clears the
// attention's counters, n_clear ints at `clear`, which then launches once
// (`cleared`).  kv4_counters: how many a workspace has, and where.
int kv4_append(const oi2_paged* c, const oi2_page_plan* p, int32_t layer, int32_t dtype, int32_t n_tokens, const oi2_heads* k,
               const oi2_heads* v, const oi2_rotary* r, const oi2_heads* q, void* q_out, int32_t* clear, int n_clear, void* stream);
int kv4_attend(const oi2_paged* c, const oi2_page_plan* p, int32_t layer, int32_t dtype, int32_t n_tokens, const oi2_heads* q, float scale,
               void* out, void* workspace, size_t workspace_bytes, bool cleared, void* stream);
int kv4_counters(const oi2_paged* c, const oi2_page_plan* p, void* workspace, int32_t** at);

int check_append(const oi2_paged* c, const oi2_page_plan* p, int32_t& dtype, bool& zero, int32_t n_tokens, const oi2_heads* k,
                 const oi2_heads* v, const oi2_rotary* r, const oi2_heads* q, const void* q_out);

}  // namespace oi2
