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
// Bound by the chain of barriers, dependent loads and fetches of its own code
// (which every launch fetches anew), not by bytes: a few kilobytes for a
// decoding step.  So counts are 32-bit and saturate, shares are products and
// groups shifts, and plans of short rows leave out the lists for long ones:
// 6 KB of code instead of 11, eight rows of a step 11.1 -> 7.2 us.  700 prompts
// of 115 thousand tokens: 28 us and 5 for the positions and slots.
#include "capi_util.h"
#include "kv_cache.h"
#include "oi2_device.h"

namespace oi2 {
namespace {

// Tokens up to which the one workgroup writes positions and slots itself.
constexpr int kOneLaunchTokens = 4096;
constexpr int kLogFew = 4, kLogMany = 7;
static_assert(1 << kLogFew == kFewRows && 1 << kLogMany == kManyRows);

struct ExtendArgs {
  int n_seqs, max_len, width, n_pages, max_tokens, max_new, log2_group;
  int fill;                   // positions and slots are written here
  const int32_t* new_lens;
  int32_t *table, *lens, *stack, *n_free;
  int32_t *cu, *positions, *slots, *kv_len, *rejected, *work;
  double per_part_few, per_part_many;   // 1 / parts
  PlanLayout l;
};

__device__ __forceinline__ int pages_of(int n) { return (int)(((int64_t)n + kPage - 1) / kPage); }

// Counts saturate at kMost, so that sums of any lengths compare rightly with
// the sizes that they are checked against, all of them below it.
constexpr uint32_t kMost = 0x7FFFFFFF;
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return min(a + b, kMost); }

// Inclusive prefix sum over the lanes of a wave: by row_shr 1, 2, 4, 8 within
// rows of 16, then row_bcast:15 and row_bcast:31 from row to row.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROW_MASK, 0xF, false);
}
__device__ __forceinline__ uint32_t row_scan(uint32_t v) {
  v = add_sat(v, dpp_u32<0x111, 0xF>(v));
  v = add_sat(v, dpp_u32<0x112, 0xF>(v));
  v = add_sat(v, dpp_u32<0x114, 0xF>(v));
  return add_sat(v, dpp_u32<0x118, 0xF>(v));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v = row_scan(v);
  v = add_sat(v, dpp_u32<0x142, 0xA>(v));
  v = add_sat(v, dpp_u32<0x143, 0xC>(v));
  return v;
}

// Exclusive prefix sums of N values per thread over the workgroup, and the
// totals.  s: N * 16 words that no one else uses until the next call's first
// barrier.
template <int N>
__device__ __forceinline__ void scan_excl(uint32_t (&v)[N], uint32_t (&total)[N], uint32_t* s) {
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), waves = blockDim.x >> 6;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    v[k] = wave_scan(v[k]);
    if (lane == 63) s[wave * N + k] = v[k];
    v[k] = dpp_u32<0x138, 0xF>(v[k]);      // wave_shr:1, 0 in lane 0
  }
  __syncthreads();
  // the waves' sums, up to 16, by the lanes of one row
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const uint32_t t = row_scan(lane < waves ? s[lane * N + k] : 0);
    total[k] = (uint32_t)__builtin_amdgcn_readlane((int)t, 15);
    if (wave > 0) v[k] = add_sat(v[k], (uint32_t)__builtin_amdgcn_readlane((int)t, wave - 1));
  }
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
// step's first; the others are in the table.  One load, by a chosen address: in
// a short step the fetches of the code cost as much as the rest.
__device__ __forceinline__ int row_page(const ExtendArgs& a, int r, int p, int past, int need, int n_free) {
  const int fresh = p - pages_of(past);
  const int32_t* at = fresh >= 0 ? a.stack + max(n_free - 1 - need - fresh, 0) : a.table + (int64_t)r * a.width + p;
  return page_id(a, *at);
}

// LONG: rows may be long enough for the attention's kernel for many rows.
template <bool LONG>
__global__ __launch_bounds__(1024) void k_page_extend(ExtendArgs a) {
  extern __shared__ int32_t lds[];
  __shared__ uint32_t s_scan[4 * 16];
  __shared__ unsigned long long s_work[2];   // pages that tiles of few and of many rows see
  __shared__ int s_halves;                   // tiles of many rows, twice those that are not cut
  __shared__ int s_taken;                    // pages that rows take
  const int n = a.n_seqs, nt = blockDim.x, tid = threadIdx.x;
  if (tid == 0) {
    s_taken = 0;
    s_work[0] = s_work[1] = 0;
    s_halves = 0;
  }
  int32_t* s_tok = lds;              // exclusive sums over the rows: tokens (capped at max_tokens + 1),
  int32_t* s_need = s_tok + n;       // pages needed,
  int32_t* s_touch = s_need + n;     // pages touched,
  int32_t* s_tile = s_touch + n;     // attention tiles
  int32_t* s_past = s_tile + n;
  int32_t* s_kv = s_past + n;
  int32_t* s_new = s_kv + n;         // tokens inside the buffer
  const int per = (n + nt - 1) >> (31 - __builtin_clz(nt));   // nt is a power of two
  const int r0 = min(tid * per, n), r1 = min(r0 + per, n);
  const int n_free = min(max(a.n_free[0], 0), a.n_pages);
  auto few_rows = [&](int tokens) { return !LONG || tokens <= kFewRows >> a.log2_group; };

  // tokens
  uint32_t at[1] = {0}, total[1];
#pragma unroll 1
  for (int r = r0; r < r1; ++r) {
    const int t = max(a.new_lens[r], 0);
    s_past[r] = min(max(a.lens[r], 0), a.max_len);
    s_new[r] = t;
    at[0] = add_sat(at[0], t);
  }
  scan_excl<1>(at, total, s_scan);
  if (tid == 0) a.cu[n] = (int)total[0];
  const int n_tokens = min((int)total[0], a.max_tokens);
  // pages
  uint32_t need[1] = {0}, all_need[1];
#pragma unroll 1
  for (int r = r0; r < r1; ++r) {
    const int t = s_new[r];
    a.cu[r] = (int)at[0];
    s_tok[r] = (int)min(at[0], (uint32_t)a.max_tokens + 1);
    at[0] = add_sat(at[0], t);
    const uint32_t len = add_sat(s_past[r], t);
    const bool fits = len <= (uint32_t)a.max_len && t <= a.max_new && at[0] <= (uint32_t)a.max_tokens;
    const int pages = fits ? pages_of((int)len) - pages_of(s_past[r]) : 0;
    s_kv[r] = fits ? (int)len : -1;
    s_need[r] = pages;
    need[0] = add_sat(need[0], pages);
  }
  scan_excl<1>(need, all_need, s_scan);
  uint32_t lists[2] = {0, 0}, in_lists[2];      // pages touched, tiles
#pragma unroll 1
  for (int r = r0; r < r1; ++r) {
    const int pages = s_need[r], past = s_past[r], t = s_new[r];
    s_need[r] = (int)need[0];
    need[0] = add_sat(need[0], pages);
    const bool taken = s_kv[r] >= 0 && (pages == 0 || need[0] <= (uint32_t)n_free);
    const int kv = taken ? s_kv[r] : 0;
    a.kv_len[r] = kv;
    a.rejected[r] = taken ? 0 : 1;
    if (taken) a.lens[r] = kv;
    // the rows that the pool serves are the first ones that need pages
    if (taken && pages > 0) atomicMax(&s_taken, (int)need[0]);
    s_kv[r] = kv;
    const int in = max(0, min(t, a.max_tokens - s_tok[r]));
    s_new[r] = in;
    const int touched = taken && t > 0 ? pages_of(kv) - past / kPage : 0;
    const bool few = few_rows(in);
    const int shift = (few ? kLogFew : kLogMany) - a.log2_group, tl = (in + (1 << shift) - 1) >> shift;
    const uint64_t work = (uint64_t)tl * pages_of(kv);
    if (work) atomicAdd(&s_work[LONG && !few], (unsigned long long)work);
    if (LONG && !few && work) atomicAdd(&s_halves, pages_of(kv) > kManyWhole ? tl : 2 * tl);
    s_touch[r] = touched;
    s_tile[r] = tl;
    lists[0] += touched;
    lists[1] += tl;
  }
  scan_excl<2>(lists, in_lists, s_scan);
#pragma unroll 1
  for (int r = r0; r < r1; ++r) {
    const int t = s_touch[r], l = s_tile[r];
    s_touch[r] = (int)lists[0];
    s_tile[r] = (int)lists[1];
    lists[0] += t;
    lists[1] += l;
  }
  const int n_touch = min((int)in_lists[0], a.l.cap_append), n_tile = (int)in_lists[1];
  __syncthreads();

  // Attention tiles in the order of their tokens, so that those of a call with
  // fewer tokens come first, cut into parts.  Pages of a part: an equal share of
  // all of them, rounded up (the product's error is far below 1 / parts), in
  // whole rounds of a workgroup's four waves.  A tile ends in half a part more on
  // average; those of many rows take that into the share while half a round of
  // parts is left, so that all of them run at once: 33 tiles of 11 to 68 pages
  // beside three of single tokens took 0.85 of the time.  Few rows, bound by their bytes,
  // lose by it (56 of 5 to 218 pages 71.8 -> 74).
  auto share = [](uint64_t pages, double per_part) {
    return ((int)min(max(ceil((double)pages * per_part), 1.0), 0x1p26) + 3) / 4 * 4;
  };
  const int c_few = share(s_work[0], a.per_part_few);
  int c_many = 0;
  if (LONG) {
    const int parts = a.l.parts_many, halves = s_halves;
    c_many = share(s_work[1], halves <= parts ? 2.0 / (2 * parts - halves) : a.per_part_many);
  }
  constexpr int kSums = LONG ? 4 : 2;        // items and partial sums, of few and of many rows
  uint32_t base[kSums] = {};
#pragma unroll 1
  for (int i0 = 0; i0 < n_tile; i0 += nt) {
    const int i = i0 + tid;
    bool few = true;
    int parts = 0, tok0 = 0, count = 0, r = 0, pages = 0, first = 0;
    if (i < n_tile) {
      r = row_of(s_tile, n, i);
      few = few_rows(s_new[r]);
      const int shift = (few ? kLogFew : kLogMany) - a.log2_group;
      first = (i - s_tile[r]) << shift;
      count = min(1 << shift, s_new[r] - first);
      tok0 = s_tok[r] + first;
      pages = s_kv[r] ? pages_of(min(s_past[r] + first + count, s_kv[r])) : 0;
      const int c = few ? c_few : c_many;
      parts = pages <= (few ? kFewWhole : kManyWhole) ? 1 : (int)((uint32_t)(pages + c - 1) / (uint32_t)c);
    }
    const uint32_t slots = parts > 1 ? parts : 0;
    uint32_t x[kSums] = {few ? (uint32_t)parts : 0, few ? slots : 0}, in_all[kSums];
    if constexpr (LONG) {
      x[2] = few ? 0 : parts;
      x[3] = few ? 0 : slots;
    }
    scan_excl<kSums>(x, in_all, s_scan);
    if (i < n_tile) {
      uint32_t item = base[0] + x[0], slot = base[1] + x[1];
      AttendItem* list = reinterpret_cast<AttendItem*>(a.work + a.l.few);
      if constexpr (LONG)
        if (!few) {
          item = base[2] + x[2];
          slot = base[3] + x[3];
          list = reinterpret_cast<AttendItem*>(a.work + a.l.many);
        }
      // at most c: as many parts, alike
      const int each = parts > 1 ? (int)(((uint32_t)(pages + parts - 1) / (uint32_t)parts + 3) / 4 * 4) : pages;
#pragma unroll 1
      for (int k = 0; k < parts; ++k) {
        AttendItem y{{r, tok0, count, s_past[r] + first, min(k * each, pages), min((k + 1) * each, pages),
                      s_kv[r], k, parts, (int)slot, {0, 0}}, {}};
        // pages past the part's are loaded like its last one
#pragma unroll
        for (int e = 0; e < kFewWaves; ++e)
          y.ids[e] = row_page(a, r, max(min(y.page0 + e, y.page1 - 1), 0), s_past[r], s_need[r], n_free);
        list[item + k] = y;
      }
    }
#pragma unroll
    for (int k = 0; k < kSums; ++k) base[k] += in_all[k];
  }
  if (tid == 0) {
    a.work[kNAppend] = n_touch;
    a.work[kNFew] = (int)base[0];
    a.work[kNMany] = LONG ? (int)base[kSums - 2] : 0;
    a.n_free[0] = n_free - s_taken;
  }

  // The other lists start at another wave each, so that in a short step their
  // loads are under way together.
  auto turned = [&](int k) { return (tid - 64 * k) & (nt - 1); };
  const int taken = s_taken;
#pragma unroll 1
  for (int i = turned(1); i < taken; i += nt) {
    const int r = row_of(s_need, n, i), j = i - s_need[r];
    a.table[(int64_t)r * a.width + pages_of(s_past[r]) + j] = page_id(a, a.stack[n_free - 1 - i]);
  }

  AppendItem* ap = reinterpret_cast<AppendItem*>(a.work + a.l.append);
#pragma unroll 1
  for (int i = turned(2); i < n_touch; i += nt) {
    const int r = row_of(s_touch, n, i), past = s_past[r], p = past / kPage + i - s_touch[r];
    const int held = max(past - p * kPage, 0), upto = min(s_kv[r] - p * kPage, kPage);
    ap[i] = AppendItem{row_page(a, r, p, past, s_need[r], n_free), s_tok[r] + p * kPage + held - past, held, upto};
  }

  if (a.fill)
#pragma unroll 1
    for (int t = turned(3); t < a.max_tokens; t += nt) {
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
  __shared__ uint32_t s_scan[16];
  const int n = a.n_seqs, nt = blockDim.x, tid = threadIdx.x;
  int32_t* s_sum = lds;
  int32_t* s_keep = lds + n;
  const int per = (n + nt - 1) >> (31 - __builtin_clz(nt)), r0 = min(tid * per, n), r1 = min(r0 + per, n);
  const int n_free = min(max(a.n_free[0], 0), a.n_pages);
  uint32_t mine[1] = {0}, all[1];
  for (int r = r0; r < r1; ++r) {
    const int len = min(max(a.lens[r], 0), a.max_len), to = a.to[r], keep = to < 0 || to > len ? len : to;
    if (keep != len) a.lens[r] = keep;
    s_keep[r] = pages_of(keep);
    s_sum[r] = pages_of(len) - pages_of(keep);
    mine[0] = add_sat(mine[0], s_sum[r]);
  }
  scan_excl<1>(mine, all, s_scan);
  for (int r = r0; r < r1; ++r) {
    const int f = s_sum[r];
    s_sum[r] = (int)mine[0];
    mine[0] = add_sat(mine[0], f);
  }
  const int freed = (int)min(all[0], (uint32_t)(a.n_pages - n_free));   // more than the pool has room for: damaged
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
  a.log2_group = __builtin_ctz((unsigned)(c->n_q / c->n_kv));
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
  a.per_part_few = 1.0 / a.l.parts_few;
  a.per_part_many = 1.0 / a.l.parts_many;
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
  const int threads = a.n_seqs <= 256 && p->max_tokens <= 1024 ? 256 : 1024;
  const bool few_only = (int64_t)p->max_new << a.log2_group <= kFewRows;
  hipLaunchKernelGGL(few_only ? k_page_extend<false> : k_page_extend<true>, dim3(1), dim3(threads), (size_t)a.n_seqs * 7 * 4, st, a);
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
