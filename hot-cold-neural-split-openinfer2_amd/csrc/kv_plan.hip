// Block tables, slot maps and work lists of the paged KV cache, built on the
// GPU from the rows' lengths.
//
// Everything is prefix sums over the rows (their tokens, pages needed, pages
// touched, attention tiles) and lists that those sums index: entry i of a list
// belongs to the row that a binary search in the sums (in LDS) finds, so the
// lists are written in parallel whatever the rows' sizes.  One workgroup does
// the sums and the lists; the positions and slots of the tokens are its own
// work for short steps and a launch of many workgroups for long ones.
//
// Bound by the chain of barriers and dependent loads, not by bytes: a few
// kilobytes for a decoding step.
#include "capi_util.h"
#include "kv_cache.h"
#include "oi2_device.h"

namespace oi2 {
namespace {

// Tokens up to which the one workgroup writes positions and slots itself.
constexpr int kOneLaunchTokens = 4096;

struct ExtendArgs {
  int n_seqs, max_len, width, n_pages, max_tokens, max_new, group;
  int few_only;               // no row is long enough for the kernel for many rows
  int fill;                   // positions and slots are written here
  const int32_t* new_lens;
  int32_t *table, *lens, *stack, *n_free;
  int32_t *cu, *positions, *slots, *kv_len, *rejected, *work;
  PlanLayout l;
};

__device__ __forceinline__ int pages_of(int n) { return (int)(((int64_t)n + kPage - 1) / kPage); }

// Inclusive prefix sum over the lanes of a wave: by row_shr 1, 2, 4, 8 within
// rows of 16, then row_bcast:15 and row_bcast:31 from row to row.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int64_t dpp_i64(int64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROW_MASK, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROW_MASK, 0xF, false);
  return (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
  v += dpp_i64<0x111, 0xF>(v);
  v += dpp_i64<0x112, 0xF>(v);
  v += dpp_i64<0x114, 0xF>(v);
  v += dpp_i64<0x118, 0xF>(v);
  v += dpp_i64<0x142, 0xA>(v);
  v += dpp_i64<0x143, 0xC>(v);
  return v;
}

// Exclusive prefix sum of one value per thread over the workgroup, and the
// total.  s: 16 words that no one else uses until the next call's first barrier.
__device__ __forceinline__ int64_t scan_excl(int64_t v, int64_t* s, int64_t& total) {
  const int lane = lane_id(), wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int64_t x = wave_scan(v);
  __syncthreads();
  if (lane == 63) s[wave] = x;
  __syncthreads();
  int64_t before = 0, all = 0;
  for (int w = 0; w < waves; ++w) {
    const int64_t t = s[w];
    if (w < wave) before += t;
    all += t;
  }
  total = all;
  return before + x - v;
}

// The last row r with sum[r] <= i, of n rows with ascending exclusive sums:
// the row that entry i belongs to (rows without entries share their sum with
// the next one, and are passed over).
__device__ __forceinline__ int row_of(const int32_t* sum, int n, int i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sum[mid] <= i) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int page_id(const ExtendArgs& a, int id) {
  return (unsigned)id < (unsigned)a.n_pages ? id : 0;   // a damaged table reads page 0
}

// Page p of row r: a new one is still on the stack, whose top n_free is the
// step's first; the others are in the table.
__device__ __forceinline__ int row_page(const ExtendArgs& a, int r, int p, int past, int need, int n_free) {
  const int fresh = p - pages_of(past);
  return page_id(a, fresh >= 0 ? a.stack[max(n_free - 1 - need - fresh, 0)] : a.table[(int64_t)r * a.width + p]);
}

// Packed pairs of sums, high and low 32 bits, neither past 2^31.
__device__ __forceinline__ int64_t pair(int64_t hi, int64_t lo) { return hi << 32 | lo; }

__global__ __launch_bounds__(1024) void k_page_extend(ExtendArgs a) {
  extern __shared__ int32_t lds[];
  __shared__ int64_t s_scan[16];
  __shared__ int s_taken;            // pages that rows take
  const int n = a.n_seqs, nt = blockDim.x, tid = threadIdx.x;
  if (tid == 0) s_taken = 0;
  int32_t* s_tok = lds;              // exclusive sums over the rows: tokens (capped at max_tokens + 1),
  int32_t* s_need = s_tok + n;       // pages needed,
  int32_t* s_touch = s_need + n;     // pages touched,
  int32_t* s_tile = s_touch + n;     // attention tiles
  int32_t* s_past = s_tile + n;
  int32_t* s_kv = s_past + n;
  int32_t* s_new = s_kv + n;         // tokens inside the buffer
  const int per = (n + nt - 1) / nt, r0 = min(tid * per, n), r1 = min(r0 + per, n);
  const int n_free = min(max(a.n_free[0], 0), a.n_pages);

  // tokens
  int64_t mine = 0, total;
  for (int r = r0; r < r1; ++r) {
    const int t = max(a.new_lens[r], 0);
    s_past[r] = min(max(a.lens[r], 0), a.max_len);
    s_new[r] = t;
    mine += t;
  }
  int64_t at = scan_excl(mine, s_scan, total);
  if (tid == 0) a.cu[n] = (int)min(total, (int64_t)0x7FFFFFFF);
  const int n_tokens = (int)min(total, (int64_t)a.max_tokens);
  // pages
  int64_t need = 0;
  for (int r = r0; r < r1; ++r) {
    const int t = s_new[r];
    a.cu[r] = (int)min(at, (int64_t)0x7FFFFFFF);
    s_tok[r] = (int)min(at, (int64_t)a.max_tokens + 1);
    at += t;
    const int64_t len = (int64_t)s_past[r] + t;
    const bool fits = len <= a.max_len && t <= a.max_new && at <= a.max_tokens;
    const int pages = fits ? pages_of((int)len) - pages_of(s_past[r]) : 0;
    s_kv[r] = fits ? (int)len : -1;
    s_need[r] = pages;
    need += pages;
  }
  int64_t all_need;
  int64_t before = scan_excl(need, s_scan, all_need);
  int64_t touch = 0, tiles = 0, pages_few = 0, pages_many = 0;
  for (int r = r0; r < r1; ++r) {
    const int pages = s_need[r], past = s_past[r], t = s_new[r];
    s_need[r] = (int)min(before, (int64_t)0x7FFFFFFF);
    before += pages;
    const bool taken = s_kv[r] >= 0 && (pages == 0 || before <= (int64_t)n_free);
    const int kv = taken ? s_kv[r] : 0;
    a.kv_len[r] = kv;
    a.rejected[r] = taken ? 0 : 1;
    if (taken) a.lens[r] = kv;
    // the rows that the pool serves are the first ones that need pages
    if (taken && pages > 0) atomicMax(&s_taken, (int)before);
    s_kv[r] = kv;
    const int in = max(0, min(t, a.max_tokens - s_tok[r]));
    s_new[r] = in;
    const int touched = taken && t > 0 ? pages_of(kv) - past / kPage : 0;
    const bool few = a.few_only || (int64_t)in * a.group <= kFewRows;
    const int tok = few ? a.l.few_tokens : a.l.many_tokens;
    const int tl = (in + tok - 1) / tok;
    const int64_t work = (int64_t)tl * pages_of(kv);
    pages_few += few ? work : 0;
    pages_many += few ? 0 : work;
    s_touch[r] = touched;
    s_tile[r] = tl;
    touch += touched;
    tiles += tl;
  }
  int64_t both, all_few, all_many;
  int64_t b = scan_excl(pair(touch, tiles), s_scan, both);
  scan_excl(pages_few, s_scan, all_few);
  scan_excl(pages_many, s_scan, all_many);
  int bt = (int)(b >> 32), bl = (int)(b & 0xFFFFFFFF);
  for (int r = r0; r < r1; ++r) {
    const int t = s_touch[r], l = s_tile[r];
    s_touch[r] = bt;
    s_tile[r] = bl;
    bt += t;
    bl += l;
  }
  const int n_touch = (int)(both >> 32), n_tile = (int)(both & 0xFFFFFFFF);
  // pages of a part: an equal share of all of them, in whole rounds of a
  // workgroup's four waves
  auto share = [](int64_t all, int parts) {
    return (int)min(max(((all + parts - 1) / parts + 3) / 4 * 4, (int64_t)4), (int64_t)1 << 26);
  };
  const int c_few = share(all_few, a.l.parts_few), c_many = share(all_many, a.l.parts_many);
  __syncthreads();

  const int taken = s_taken;
  for (int i = tid; i < taken; i += nt) {
    const int r = row_of(s_need, n, i), j = i - s_need[r];
    a.table[(int64_t)r * a.width + pages_of(s_past[r]) + j] = page_id(a, a.stack[n_free - 1 - i]);
  }
  if (tid == 0) {
    a.work[kNAppend] = n_touch;
    a.n_free[0] = n_free - taken;
  }

  AppendItem* ap = reinterpret_cast<AppendItem*>(a.work + a.l.append);
  for (int i = tid; i < n_touch; i += nt) {
    const int r = row_of(s_touch, n, i), past = s_past[r], p = past / kPage + i - s_touch[r];
    const int held = max(past - p * kPage, 0), upto = min(s_kv[r] - p * kPage, kPage);
    ap[i] = AppendItem{row_page(a, r, p, past, s_need[r], n_free), s_tok[r] + p * kPage + held - past, held, upto};
  }

  // attention tiles, cut into parts
  AttendItem* few_list = reinterpret_cast<AttendItem*>(a.work + a.l.few);
  AttendItem* many_list = reinterpret_cast<AttendItem*>(a.work + a.l.many);
  int64_t base_items = 0, base_slots = 0;
  for (int i0 = 0; i0 < n_tile; i0 += nt) {
    const int i = i0 + tid;
    bool few = false;
    int parts = 0, tok0 = 0, count = 0, r = 0, pages = 0, first = 0;
    if (i < n_tile) {
      r = row_of(s_tile, n, i);
      few = a.few_only || (int64_t)s_new[r] * a.group <= kFewRows;
      const int tok = few ? a.l.few_tokens : a.l.many_tokens;
      const int tl = (s_new[r] + tok - 1) / tok;
      const int j = tl - 1 - (i - s_tile[r]);        // the tiles that see most first
      first = j * tok;
      count = min(tok, s_new[r] - first);
      tok0 = s_tok[r] + first;
      pages = s_kv[r] ? pages_of(min(s_past[r] + first + count, s_kv[r])) : 0;
      const int c = few ? c_few : c_many;
      parts = pages <= (few ? kFewWhole : kManyWhole) ? 1 : (pages + c - 1) / c;
    }
    const int slots = parts > 1 ? parts : 0;
    int64_t t_items, t_slots;
    const int64_t x_items = scan_excl(few ? pair(0, parts) : pair(parts, 0), s_scan, t_items) + base_items;
    const int64_t x_slots = scan_excl(few ? pair(0, slots) : pair(slots, 0), s_scan, t_slots) + base_slots;
    base_items += t_items;
    base_slots += t_slots;
    if (i < n_tile) {
      const int item = (int)(few ? x_items & 0xFFFFFFFF : x_items >> 32);
      const int slot = (int)(few ? x_slots & 0xFFFFFFFF : x_slots >> 32);
      AttendItem* list = few ? few_list : many_list;
      const int each = parts > 1 ? ((pages + parts - 1) / parts + 3) / 4 * 4 : pages;   // at most c: as many parts, alike
      for (int k = 0; k < parts; ++k) {
        AttendItem x{{r, tok0, count, s_past[r] + first, min(k * each, pages), min((k + 1) * each, pages),
                      s_kv[r], k, parts, slot, {0, 0}}, {}};
#pragma unroll
        for (int e = 0; e < kFewWaves; ++e)
          if (few || e < 2) x.ids[e] = x.page0 + e < x.page1 ? row_page(a, r, x.page0 + e, s_past[r], s_need[r], n_free) : 0;
        list[item + k] = x;
      }
    }
  }
  if (tid == 0) {
    a.work[kNFew] = (int)(base_items & 0xFFFFFFFF);
    a.work[kNMany] = (int)(base_items >> 32);
  }
  if (a.fill)
    for (int t = tid; t < a.max_tokens; t += nt) {
      int pos = -1, slot = -1;
      if (t < n_tokens) {
        const int r = row_of(s_tok, n, t);
        if (s_kv[r]) {
          pos = s_past[r] + t - s_tok[r];
          slot = row_page(a, r, pos / kPage, s_past[r], s_need[r], n_free) * kPage + pos % kPage;
        }
      }
      a.positions[t] = pos;
      a.slots[t] = slot;
    }
}

// Positions and slots of a long step, from the plan's sums.
__global__ __launch_bounds__(256) void k_page_tokens(ExtendArgs a) {
  extern __shared__ int32_t s_cu[];
  const int n = a.n_seqs;
  for (int r = threadIdx.x; r < n; r += 256) s_cu[r] = a.cu[r];
  const int total = a.cu[n];
  __syncthreads();
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= a.max_tokens) return;
  int pos = -1, slot = -1;
  if (t < total) {
    const int r = row_of(s_cu, n, t), kv = a.kv_len[r];
    if (kv) {
      const int t1 = r + 1 < n ? s_cu[r + 1] : total;
      pos = kv - (t1 - t);
      slot = page_id(a, a.table[(int64_t)r * a.width + pos / kPage]) * kPage + pos % kPage;
    }
  }
  a.positions[t] = pos;
  a.slots[t] = slot;
}

struct RewindArgs {
  int n_seqs, max_len, width, n_pages;
  const int32_t* to;
  int32_t *table, *lens, *stack, *n_free;
};

__global__ __launch_bounds__(1024) void k_page_rewind(RewindArgs a) {
  extern __shared__ int32_t lds[];
  __shared__ int64_t s_scan[16];
  const int n = a.n_seqs, nt = blockDim.x, tid = threadIdx.x;
  int32_t* s_sum = lds;
  int32_t* s_keep = lds + n;
  const int per = (n + nt - 1) / nt, r0 = min(tid * per, n), r1 = min(r0 + per, n);
  const int n_free = min(max(a.n_free[0], 0), a.n_pages);
  int64_t mine = 0, all;
  for (int r = r0; r < r1; ++r) {
    const int len = min(max(a.lens[r], 0), a.max_len), to = a.to[r], keep = to < 0 || to > len ? len : to;
    if (keep != len) a.lens[r] = keep;
    s_keep[r] = pages_of(keep);
    s_sum[r] = pages_of(len) - pages_of(keep);
    mine += s_sum[r];
  }
  int64_t at = scan_excl(mine, s_scan, all);
  for (int r = r0; r < r1; ++r) {
    const int f = s_sum[r];
    s_sum[r] = (int)at;
    at += f;
  }
  const int freed = (int)min(all, (int64_t)(a.n_pages - n_free));   // more than the pool has room for: damaged
  __syncthreads();
  for (int i = tid; i < freed; i += nt) {
    const int r = row_of(s_sum, n, i);
    int32_t* e = a.table + (int64_t)r * a.width + s_keep[r] + i - s_sum[r];
    a.stack[n_free + freed - 1 - i] = *e;
    *e = -1;
  }
  if (tid == 0) a.n_free[0] = n_free + freed;
}

ExtendArgs extend_args(const oi2_paged* c, const oi2_page_plan* p, const int32_t* new_lens) {
  ExtendArgs a{};
  a.n_seqs = c->n_seqs;
  a.max_len = c->max_len;
  a.width = (c->max_len + kPage - 1) / kPage;
  a.n_pages = c->n_pages;
  a.max_tokens = p->max_tokens;
  a.max_new = p->max_new;
  a.group = c->n_q / c->n_kv;
  a.few_only = (int64_t)p->max_new * a.group <= kFewRows;
  a.fill = p->max_tokens <= kOneLaunchTokens;
  a.new_lens = new_lens;
  a.table = c->block_table;
  a.lens = c->lens;
  a.stack = c->free_pages;
  a.n_free = c->n_free;
  a.cu = p->cu;
  a.positions = p->positions;
  a.slots = p->slots;
  a.kv_len = p->kv_len;
  a.rejected = p->rejected;
  a.work = p->work;
  a.l = plan_layout(*c, p->max_tokens, p->max_new);
  return a;
}

bool sizes_ok(const oi2_paged* c) {
  if (c->n_kv < 1 || c->n_q < 1 || c->n_q > 1024 || c->n_q % c->n_kv) return false;
  const int g = c->n_q / c->n_kv;
  return (g == 1 || g == 2 || g == 4 || g == 8) && c->n_seqs >= 1 && c->n_seqs <= OI2_MAX_SEQS && c->max_len >= 1 &&
         c->max_len <= 0x7FFFFFFF - 2 * kPage && c->n_pages >= 1 && c->n_pages < 1 << 25 && c->n_layers >= 0;
}

}  // namespace

int check_paged(const oi2_paged* c, int32_t layer, bool pool) {
  OI2_CHECK_ARG(c, "null cache");
  OI2_CHECK_ARG(sizes_ok(c),
                "cache of %d rows of %d positions, %d pages, %d query and %d kv heads: 1 to %d rows, 1 to 2^25 - 1 pages, "
                "1, 2, 4 or 8 query heads per kv head",
                c->n_seqs, c->max_len, c->n_pages, c->n_q, c->n_kv, OI2_MAX_SEQS);
  OI2_CHECK_ARG(c->block_table && c->lens && c->free_pages && c->n_free, "null cache table");
  if (pool) {
    OI2_CHECK_ARG(layer >= 0 && layer < c->n_layers, "layer %d of a cache of %d", layer, c->n_layers);
    OI2_CHECK_ARG(c->pages && (uintptr_t)c->pages % 16 == 0, "pages must be non-null and 16-byte aligned");
    OI2_CHECK_ARG(c->scales && (uintptr_t)c->scales % 8 == 0, "scales must be non-null and 8-byte aligned");
  }
  return OI2_OK;
}

int check_plan(const oi2_paged* c, const oi2_page_plan* p) {
  OI2_CHECK_ARG(p, "null plan");
  OI2_CHECK_ARG(p->max_tokens >= 1 && p->max_tokens <= 1 << 28 && p->max_new >= 1, "plan of %d tokens, %d a row",
                p->max_tokens, p->max_new);
  OI2_CHECK_ARG(p->cu && p->positions && p->slots && p->kv_len && p->rejected, "null plan array");
  OI2_CHECK_ARG(p->work && (uintptr_t)p->work % 16 == 0, "plan work lists must be non-null and 16-byte aligned");
  return OI2_OK;
}

}  // namespace oi2

using namespace oi2;

extern "C" {

size_t oi2_page_plan_bytes(const oi2_paged* c, int32_t max_tokens, int32_t max_new) {
  if (!c || !sizes_ok(c) || max_tokens < 1 || max_tokens > 1 << 28 || max_new < 1) return 0;
  return (size_t)plan_layout(*c, max_tokens, max_new).ints * 4;
}

int oi2_page_extend(const oi2_paged* c, const oi2_page_plan* p, const int32_t* new_lens, void* stream) {
  clear_error();
  if (int rc = check_paged(c, 0, false)) return rc;
  if (int rc = check_plan(c, p)) return rc;
  OI2_CHECK_ARG(new_lens, "null lengths");
  const ExtendArgs a = extend_args(c, p, new_lens);
  hipStream_t st = (hipStream_t)stream;
  // short steps: fewer waves have less to wait for at each barrier
  const int threads = a.n_seqs <= 64 && p->max_tokens <= 128 ? 64 : a.n_seqs <= 256 && p->max_tokens <= 1024 ? 256 : 1024;
  hipLaunchKernelGGL(k_page_extend, dim3(1), dim3(threads), (size_t)a.n_seqs * 7 * 4, st, a);
  OI2_CHECK_LAUNCH();
  if (!a.fill) {
    hipLaunchKernelGGL(k_page_tokens, dim3((a.max_tokens + 255) / 256), dim3(256), (size_t)a.n_seqs * 4, st, a);
    OI2_CHECK_LAUNCH();
  }
  return OI2_OK;
}

int oi2_page_rewind(const oi2_paged* c, const int32_t* lens, void* stream) {
  clear_error();
  if (int rc = check_paged(c, 0, false)) return rc;
  OI2_CHECK_ARG(lens, "null lengths");
  RewindArgs a{};
  a.n_seqs = c->n_seqs;
  a.max_len = c->max_len;
  a.width = (c->max_len + kPage - 1) / kPage;
  a.n_pages = c->n_pages;
  a.to = lens;
  a.table = c->block_table;
  a.lens = c->lens;
  a.stack = c->free_pages;
  a.n_free = c->n_free;
  hipLaunchKernelGGL(k_page_rewind, dim3(1), dim3(a.n_seqs <= 64 ? 64 : a.n_seqs <= 256 ? 256 : 1024), (size_t)a.n_seqs * 2 * 4,
                     (hipStream_t)stream, a);
  OI2_CHECK_LAUNCH();
  return OI2_OK;
}

}  // extern "C"
