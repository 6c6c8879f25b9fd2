// Attention of a step's query tokens over the paged 8-bit KV cache.
//
//   attend_few   up to 16 query rows (tokens times query heads of a kv head)
//                over a range of a row's pages
//   attend_many  up to 128 query rows over a range of a row's pages
// in one launch.  Where a row's pages were cut into parts, a part leaves its
// sums in the workspace, and the one that arrives last joins them, in the order
// of the parts: the result does not depend on who that is.
//
// A page's k and v codes are widened exactly to fp16 (e4m3 has 4 significant
// bits) and multiplied on the matrix cores; the page's scales, powers of two,
// are applied to the scores (k) and inside the exponential (v):
//   p = exp2(score + ev - m),  out = sum p code_v,  l = sum p 2^-ev
// with m the running maximum of score + ev, so that out, whose parts a row of
// pages with different scales would otherwise have to rescale, is a plain sum,
// and p is large exactly where p times v's scale is.
//
// A lane of the scores' product S^T = K Q^T holds scores of one query row, and
// in the order in which the product out^T = V^T P^T takes them: the cache
// stores a page's k rows and v columns so that 16-byte loads of consecutive
// addresses are the operands of both.
#include "capi_util.h"
#include "kv_cache.h"
#include "rotary.h"

namespace oi2 {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896341f;
// p comes out times 2^kLift, and the running maximum follows the row's once that
// is 2^kSlack above it: p stays below fp16's 2^16, few pages rescale the sums,
// and a p's two parts end at 2^-24, 2^-30 of the largest p at most.  That cut is
// felt where a wave's pages hold many weights that small: 2^17 of them are 2^-13
// together, half of half a step of fp16, but with 2 and 13 2^-9.  With 8 and 7
// the same times; with 2 and 13 a prompt of 5000 tokens is 0.5 % faster and 56
// bf16 tokens over long contexts 3 %.
constexpr float kLift = 6.0f, kSlack = 9.0f;

struct PartArgs {             // of one of the two kernels
  const AttendItem* items;
  int groups;                 // workgroups of the launch
  int32_t* count;             // (slot, kv head) arrivals, zero before the launch
  float* o;                   // (slot, kv head, rows, 128)
  float* ml;                  // (slot, kv head, rows, 2)
};

struct AttendArgs {
  const int32_t* work;        // the plan's
  PartArgs few, many;
  const int32_t* table;
  const uint8_t* pages;       // of the layer
  const float* scales;
  int n_q, n_kv, group_log, width, n_pages, n_tokens;
  const uint16_t* q;
  int64_t token_stride, head_stride;
  int wide;                   // 16-byte loads of q
  float scale;                // of the scores, times log2 e
  uint16_t* out;
  const int32_t* total;       // tokens of the step
  int zero_groups;            // workgroups for the rows past them, or none
};

__device__ __forceinline__ h8 widen8(uint32_t d0, uint32_t d1) {
  const h4 lo = __builtin_shufflevector(fp8x2_to_f16x2(d0, false), fp8x2_to_f16x2(d0, true), 0, 1, 2, 3);
  const h4 hi = __builtin_shufflevector(fp8x2_to_f16x2(d1, false), fp8x2_to_f16x2(d1, true), 0, 1, 2, 3);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ __forceinline__ f32x4 mfma16(h8 a, h8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Loads at uniform addresses of what no kernel writes meanwhile (tables, scales,
// items), through the constant address space: scalar loads.  As vector loads
// they return in order behind the codes on their way, and waiting for a page's
// number then waits for those.
template <typename T>
__device__ __forceinline__ T scalar_load(const T* p) {
  static_assert(sizeof(T) % 4 == 0, "dwords");
  typedef const int32_t __attribute__((address_space(4))) cint;
  cint* c = (cint*)(uintptr_t)p;
  int32_t w[sizeof(T) / 4];
#pragma unroll
  for (unsigned i = 0; i < sizeof(T) / 4; ++i) w[i] = c[i];
  T v;
  __builtin_memcpy(&v, w, sizeof(T));
  return v;
}

// Bytes [0, n) of a dword's four kept, the rest zero.
__device__ __forceinline__ uint32_t first_bytes(uint32_t d, int n) {
  return n >= 4 ? d : n <= 0 ? 0u : d & ((1u << (8 * n)) - 1);
}

// A NaN among v must not reach rows that do not see its position (their p is 0,
// and 0 times it NaN).  Pages that hold one are marked; their NaN codes go into
// the products as 0, and the first position of a NaN is noted for each dim: a
// row that sees it has NaN there.
constexpr int kNoNan = 0x7FFFFFFF;
__device__ __forceinline__ void take_nans(u32x4& x, int pos, int* first) {   // 16 positions of a dim
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t is = ((x[k] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;   // the top bits of NaN codes' bytes
    if (is) {
      x[k] &= ~((is >> 7) * 0xFFu);
      atomicMin(first, pos + 4 * k + (__builtin_ctz(is) >> 3));
    }
  }
}

__device__ __forceinline__ float ldexp2(float x, int e) { return __builtin_ldexpf(x, e); }

// Eight consecutive q values as fp16 times 2^-e (bf16; fp16 comes as it is).
// The largest of a bf16 row is put at the top of fp16's range, at 2^15: every
// value down to 2^-29 of it is exact, smaller ones are off by 2^-40 of it.
constexpr int kTopExp = 15;
template <bool BF16>
__device__ __forceinline__ h8 q_frag(const uint16_t (&v)[8], int e, bool negate) {
  h8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    r[i] = BF16 ? (_Float16)ldexp2(bf16_bits_to_float(v[i]), -e) : __builtin_bit_cast(_Float16, v[i]);
  return negate ? -r : r;
}

// Eight probabilities, times 2^kLift, as the operand of out^T = V^T P^T: two fp16
// parts (hi truncated, lo the rest), 21 bits at least.  One part, to nearest,
// is off by 2^-12 of a probability, as much as an fp16 output's own rounding
// and an eighth of a bf16 one's: where values cancel that is most of the result,
// and a token would get other bits in a prompt than in a step of its own.  It
// would save a third of the products of many rows (a call of 5000 tokens 220 us
// instead of 292) and nothing of few ones, which the pages' loads bound.
struct Probs {
  h8 hi, lo;
};
__device__ __forceinline__ Probs to_probs(const float (&e)[8]) {
  u32x4 uh, ul;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(e[2 * k], e[2 * k + 1]));
    uh[k] = hi;
    ul[k] = __builtin_bit_cast(
        uint32_t, __builtin_amdgcn_cvt_pkrtz(fmaf(half_lo(hi), -1.0f, e[2 * k]), fmaf(half_hi(hi), -1.0f, e[2 * k + 1])));
  }
  return {__builtin_bit_cast(h8, uh), __builtin_bit_cast(h8, ul)};
}

// A page's scores are dot * score_scale + ev, with q negated where the scale of
// the scores is negative, so that the largest dot is the largest score; a scale
// of zero counts as 2^-120, because a masked dot is minus infinity, and one past
// fp32 as its largest number, because a dot may be zero.
__device__ __forceinline__ float score_scale(float sc, float k_scale) {
  return __builtin_amdgcn_fmed3f(fabsf(sc) * k_scale, 7.52316385e-37f, 3.40282347e38f);
}

__device__ __forceinline__ float quad_max(float v) {   // over the lanes l, l ^ 16, l ^ 32, l ^ 48
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

constexpr int kThreads = 256;

// ── parts ────────────────────────────────────────────────────────────────────

constexpr int kSc1 = 16;                   // cache-policy operand: agent-coherent access

__device__ __forceinline__ void st_agent(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// A part's sums, row by row of n_rows, are stored (agent-coherent, by every
// thread).  True in the workgroup that completes the set, which then joins it.
__device__ __forceinline__ bool arrive(const PartArgs& pa, const ItemHead& it, int n_kv, int g) {
  __shared__ int s_last;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // every store acknowledged
  __syncthreads();
  if (threadIdx.x == 0) {
    int32_t* c = pa.count + (int64_t)it.slot0 * n_kv + g;
    const int old = __hip_atomic_fetch_add(c, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = old + 1 == it.n_parts;
  }
  __syncthreads();
  return s_last;
}

// Joins the parts of a tile.  32 threads take a row's 128 dims; with fewer rows
// than such groups, several groups a row, each every pg-th part.  The
// tail of a call waits for this, and it waits for its loads, which go past the
// caches: sums, maxima and exponential sums of U parts of RB rows go out
// together, and are taken in with a running maximum.  smem: 16.1 bytes
// a thread.
template <bool BF16, int ROWS>
__device__ __forceinline__ void join_parts(const AttendArgs& a, const PartArgs& pa, const ItemHead& it, int g, int n_rows,
                                           float* smem) {
  constexpr int kGroups = kThreads / 32, RB = ROWS == kFewRows ? 1 : 4, U = ROWS == kFewRows ? 8 : 4;
  f32x4* s_y = reinterpret_cast<f32x4*>(smem);       // (kGroups, 32)
  float* s_M = smem + 4 * kThreads;
  float* s_L = s_M + kGroups;
  const int tid = threadIdx.x, grp = tid >> 5, lane = tid & 31, lg = a.group_log, n_parts = it.n_parts;
  const float ninf = -__builtin_inff();
  const int64_t base = ((int64_t)it.slot0 * a.n_kv + g) * ROWS;
  const int stride = a.n_kv * ROWS;                  // rows from a part to the next
  const uint32_t rows = (uint32_t)((n_parts - 1) * stride + ROWS);
  const rsrc_t ro = rsrc(pa.o + base * kHeadD, rows * (kHeadD * 4)), rml = rsrc(pa.ml + 2 * base, rows * 8);
  const int pg = n_rows < kGroups ? kGroups / n_rows : 1, per = n_rows < kGroups ? n_rows : kGroups;
  const int first = grp / per;
  for (int r0 = 0; r0 < n_rows; r0 += kGroups * RB) {
    f32x4 y[RB];
    float M[RB], L[RB];
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      M[i] = ninf;
      L[i] = 0.0f;
    }
    const int row0 = r0 + grp % per;                 // rows row0, row0 + kGroups, ..
    for (int k = first; k < n_parts && first < pg; k += U * pg) {
      u32x4 x[U][RB];
      u32x2v ml[U][RB];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < RB; ++i) {
          const int row = row0 + kGroups * i;
          const bool is = k + u * pg < n_parts && row < n_rows;
          const uint32_t at = (uint32_t)((k + u * pg) * stride + row);
          ml[u][i] = __builtin_amdgcn_raw_buffer_load_b64(rml, is ? 8 * at : kNoOff, 0, kSc1);
          x[u][i] = __builtin_amdgcn_raw_buffer_load_b128(ro, is ? at * (kHeadD * 4) + 16 * lane : kNoOff, 0, kSc1);
        }
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        float top = M[i], m[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          m[u] = k + u * pg < n_parts ? as_f32(ml[u][i].x) : ninf;
          top = fmaxf(top, m[u]);
        }
        const float f0 = M[i] == ninf ? 0.0f : __builtin_amdgcn_exp2f(M[i] - top);
        M[i] = top;
        L[i] *= f0;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[i][e] *= f0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          // 0 times a NaN sum, of a part whose every score is NaN, stays NaN
          const float f = m[u] == ninf ? 0.0f : __builtin_amdgcn_exp2f(m[u] - top);
          L[i] = fmaf(f, as_f32(ml[u][i].y), L[i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[i][e] = fmaf(f, as_f32(x[u][i][e]), y[i][e]);
        }
      }
    }
    if (pg > 1) {                                    // one row a group: a row's groups meet in its first one
      __syncthreads();
      s_y[tid] = y[0];
      if (lane == 0) {
        s_M[grp] = M[0];
        s_L[grp] = L[0];
      }
      __syncthreads();
      if (first == 0) {
        float top = M[0];
        for (int k = 1; k < pg; ++k) top = fmaxf(top, s_M[grp + k * per]);
        const float f0 = M[0] == ninf ? 0.0f : __builtin_amdgcn_exp2f(M[0] - top);
        L[0] *= f0;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[0][e] *= f0;
        for (int k = 1; k < pg; ++k) {
          const float m = s_M[grp + k * per], f = m == ninf ? 0.0f : __builtin_amdgcn_exp2f(m - top);
          L[0] = fmaf(f, s_L[grp + k * per], L[0]);
          const f32x4 x = s_y[tid + 32 * k * per];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[0][e] = fmaf(f, x[e], y[0][e]);
        }
      }
    }
    if (first > 0) continue;
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      const int row = row0 + kGroups * i;
      if (row >= n_rows) continue;
      const float inv = 1.0f / L[i];
      uint16_t z[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = narrow<BF16>(y[i][e] * inv);
      const int64_t to =
          ((int64_t)(it.token0 + (row >> lg)) * a.n_q + (g << lg) + (row & ((1 << lg) - 1))) * kHeadD + 4 * lane;
      *reinterpret_cast<u32x2v*>(a.out + to) = *reinterpret_cast<u32x2v*>(z);
    }
  }
}

// ── few rows ─────────────────────────────────────────────────────────────────

constexpr int kORow = kHeadD + 4;          // floats of an output row in LDS, padded
constexpr int kFewLds = (kFewWaves * kFewRows * (kORow + 2) + kHeadD) * 4;

// Lane (r = lane % 16, grp = lane / 16).  K's 16-row tile t of a page: row
// r = 4 a + i is position 16 a + 4 t + i; D's element i of lane (r, grp) is
// the score of query row r at position 16 grp + 4 t + i: in 4 tiles a lane has
// positions 16 grp .. 16 grp + 15 of its query row, which are the positions of
// the 16 bytes of V^T that it loads for each dim.
//
// A wave takes every fourth page, loads the next one (k and v, 16 KB) while it
// works on this one, and its page number by a scalar load two ahead; the four
// meet in LDS at the end.  Bound by the pages' loads: 56 tokens of 300 to 14000
// positions 71 us (378 MB, 5.3 TB/s), three of 40 to 110 thousand 46 (241 MB,
// 5.2); the same blocks, scattered over the pool and read alone, take 57 and 37
// (6.5 TB/s), so a fifth is the start, the last round, and the join.  One token
// of 700 positions 8.1, three rounds and the merge.  Tried without gain: 8 and
// 16 waves, pages dealt out in equal shares whatever row they belong to.
template <bool BF16>
__device__ __forceinline__ void attend_few(const AttendArgs& a, int b, uint8_t* smem) {
  const int item = b / a.n_kv, g = b - item * a.n_kv;
  const AttendItem& full = a.few.items[item];
  const ItemHead it = scalar_load(static_cast<const ItemHead*>(&full));
  if (item >= scalar_load(a.work + kNFew)) return;
  typedef float Rows[kFewRows];
  float (*s_o)[kFewRows][kORow] = reinterpret_cast<float (*)[kFewRows][kORow]>(smem);
  Rows* s_m = reinterpret_cast<Rows*>(smem + kFewWaves * kFewRows * kORow * 4);
  Rows* s_l = s_m + kFewWaves;
  int* s_nan = reinterpret_cast<int*>(s_l + kFewWaves);
  const int n_tok = min(it.n_tokens, a.n_tokens - it.token0);
  // a tile whose last part is not in the launch (fewer tokens than the plan's)
  // is left out whole: its arrivals would not be complete
  if (n_tok <= 0 || item - it.part + it.n_parts > a.few.groups / a.n_kv) return;
  const int tid = threadIdx.x, lane = lane_id(), r = lane & 15, grp = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lg = a.group_log, n_rows = n_tok << lg;
  if (tid < kHeadD) s_nan[tid] = kNoNan;
  __syncthreads();

  // the query row: B operand, MFMA (i, h) dims 16 (4 i + grp) + 8 h ..
  uint16_t qv[4][8];
  const int tok = r >> lg;
  {
    const uint16_t* pq = a.q + (int64_t)(it.token0 + min(tok, n_tok - 1)) * a.token_stride +
                         (int64_t)((g << lg) + (r & ((1 << lg) - 1))) * a.head_stride;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t* p = pq + 16 * (4 * (i >> 1) + grp) + 8 * (i & 1);
      if (a.wide) {
        *reinterpret_cast<u32x4*>(qv[i]) = *reinterpret_cast<const u32x4*>(p);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) qv[i][e] = p[e];
      }
    }
  }
  int qe = 0;
  if (BF16) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(bf16_bits_to_float(qv[i][e])));
    top = quad_max(top);
    qe = min(max((int)(as_u32(top) >> 23) - 127 - kTopExp, -126), 126);
  }
  h8 qf[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) qf[i] = q_frag<BF16>(qv[i], qe, a.scale < 0.0f);
  const float sc = BF16 ? ldexp2(a.scale, qe) : a.scale;
  const int lim = r < n_rows ? min(it.pos0 + tok + 1, it.kv_len) : 0;   // positions that this row sees
  const int all_see = min(it.pos0 + 1, it.kv_len);                      // ... and every row does

  const float ninf = -__builtin_inff();
  f32x4 o[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = ninf, l = 0.0f;

  // A page's k, then its v: each is loaded as soon as the products of the page
  // before have taken theirs, so a wave always has 8 KB in flight.  Past the
  // last page the descriptor's range is empty: nothing is read.
  const int32_t* table = a.table + (int64_t)it.row * a.width;
  auto block_of = [&](int page) {
    int id = scalar_load(table + min(page, it.page1 - 1));
    id = (unsigned)id < (unsigned)a.n_pages ? id : 0;
    return (int64_t)id * a.n_kv + g;
  };
  auto page_rsrc = [&](int64_t block, int page) { return rsrc(a.pages + block * kBlock, page < it.page1 ? kBlock : 0); };
  auto scale_of = [&](int64_t block) { return scalar_load(reinterpret_cast<const float2*>(a.scales) + block); };
  u32x4 kr[8], vr[8];
  auto load8 = [&](u32x4 (&x)[8], rsrc_t r, int at) {
#pragma unroll
    for (int n = 0; n < 8; ++n) x[n] = wld16(r, at + 1024 * n + 16 * lane);
  };
  const int first = it.page0 + w;
  int64_t next = 0;
  float2 scale = {1.0f, 1.0f};
  if (first < it.page1) {
    const int64_t block = (int64_t)scalar_load(full.ids + w) * a.n_kv + g;
    const rsrc_t r0 = page_rsrc(block, first);
    load8(kr, r0, 0);
    load8(vr, r0, kHalfBlock);
    scale = scale_of(block);
    next = block_of(first + kFewWaves);
  }
  for (int page = first; page < it.page1; page += kFewWaves) {
    const rsrc_t rn = page_rsrc(next, page + kFewWaves);
    const float ks = scale.x, vs = scale.y;
    scale = scale_of(next);
    next = block_of(page + 2 * kFewWaves);
    const float ev = (float)((int)((as_u32(vs) >> 23) & 0xFF) - 127);

    float s[16];
    const float ksc = score_scale(sc, ks);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc = mfma16(widen8(kr[2 * t + (i >> 1)][2 * (i & 1)], kr[2 * t + (i >> 1)][2 * (i & 1) + 1]), qf[i], acc);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * t + i] = acc[i];
    }
    __builtin_amdgcn_sched_barrier(0);
    load8(kr, rn, 0);
    __builtin_amdgcn_sched_barrier(0);
    const int p0 = page * kPage + 16 * grp;
    if (page * kPage + kPage > all_see) {
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j] = p0 + j < lim ? s[j] : ninf;
    }
    float cm = s[0];
#pragma unroll
    for (int j = 1; j < 16; ++j) cm = fmaxf(cm, s[j]);
    cm = fmaf(quad_max(cm), ksc, ev);
    const bool up = cm > m + kSlack;
    if (__any(up)) {
      const float mn = up ? cm : m;
      const float alpha = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      l *= alpha;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[d] *= alpha;
      m = mn;
    }
    const float rel = ev - ((m == ninf ? 0.0f : m) - kLift);
    float sum[2] = {0.0f, 0.0f};
    Probs p[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        e[j] = __builtin_amdgcn_exp2f(fmaf(s[8 * h + j], ksc, rel));
        sum[h] += e[j];
      }
      p[h] = to_probs(e);
    }
    l = fmaf(sum[0] + sum[1], ldexp2(1.0f, -(int)ev), l);
    // places behind the row's end hold whatever their page held before
    const int tail = it.kv_len - p0;
    if (page * kPage + kPage > it.kv_len) {
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k) vr[n][k] = first_bytes(vr[n][k], tail - 4 * k);
    }
    if (vs < 0.0f) {
#pragma unroll
      for (int n = 0; n < 8; ++n) take_nans(vr[n], p0, &s_nan[16 * n + r]);
    }
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const h8 vf = widen8(vr[d][2 * h], vr[d][2 * h + 1]);
        o[d] = mfma16(vf, p[h].hi, o[d]);
        o[d] = mfma16(vf, p[h].lo, o[d]);
      }
    __builtin_amdgcn_sched_barrier(0);
    load8(vr, rn, kHalfBlock);
    __builtin_amdgcn_sched_barrier(0);
  }

  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
#pragma unroll
  for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4*>(&s_o[w][r][16 * d + 4 * grp]) = o[d];
  if (grp == 0) {
    s_m[w][r] = m;
    s_l[w][r] = l;
  }
  __syncthreads();
  // thread: E dims from d0 of a query row
  constexpr int E = kFewRows * kHeadD / kThreads;
  const int row = tid * E / kHeadD, d0 = tid * E % kHeadD;
  float M = ninf, L = 0.0f, y[E];
#pragma unroll
  for (int k = 0; k < kFewWaves; ++k) M = fmaxf(M, s_m[k][row]);
#pragma unroll
  for (int e = 0; e < E; ++e) y[e] = 0.0f;
#pragma unroll
  for (int k = 0; k < kFewWaves; ++k) {
    const float mk = s_m[k][row], f = mk == ninf ? 0.0f : __builtin_amdgcn_exp2f(mk - M);
    L = fmaf(f, s_l[k][row], L);
    // 0 times a NaN sum, of a wave whose every score is NaN, stays NaN
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = fmaf(f, s_o[k][row][d0 + e], y[e]);
  }
  const int tk = row >> lg, head = (g << lg) + (row & ((1 << lg) - 1));
  const int sees = min(it.pos0 + tk + 1, it.kv_len);
#pragma unroll
  for (int e = 0; e < E; ++e) y[e] = s_nan[d0 + e] < sees ? __builtin_nanf("") : y[e];
  if (it.n_parts > 1) {
    const int64_t base = ((int64_t)(it.slot0 + it.part) * a.n_kv + g) * kFewRows;
    if (row < n_rows) {
      const rsrc_t ro = rsrc(a.few.o + base * kHeadD, kFewRows * kHeadD * 4);
#pragma unroll
      for (int e = 0; e < E; e += 2)
        __builtin_amdgcn_raw_buffer_store_b64(u32x2v{as_u32(y[e]), as_u32(y[e + 1])}, ro, (row * kHeadD + d0 + e) * 4, 0, kSc1);
      if (d0 == 0) {
        st_agent(a.few.ml + 2 * (base + row), M);
        st_agent(a.few.ml + 2 * (base + row) + 1, L);
      }
    }
    if (arrive(a.few, it, a.n_kv, g)) join_parts<BF16, kFewRows>(a, a.few, it, g, n_rows, reinterpret_cast<float*>(smem));
    return;
  }
  if (row >= n_rows) return;
  const float inv = it.kv_len > 0 ? 1.0f / L : 0.0f;     // a rejected row: zeros
  uint16_t z[E];
#pragma unroll
  for (int e = 0; e < E; ++e) z[e] = it.kv_len > 0 ? narrow<BF16>(y[e] * inv) : 0;
  uint16_t* to = a.out + ((int64_t)(it.token0 + tk) * a.n_q + head) * kHeadD + d0;
#pragma unroll
  for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(to + e) = z[e] | (uint32_t)z[e + 1] << 16;
}

// ── many rows ────────────────────────────────────────────────────────────────

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(h8 a, h8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// In LDS, fp16: two pages of k, rows of one position (256 bytes, 16 chunks of 8
// dims), and two of v, rows of one dim (128 bytes, 8 chunks of 8 positions).
// Chunks are swizzled within their rows so that staging stores (16 lanes in a
// row) and fragment reads touch all banks: k's by position p = 16 a + 4 t + i
// with i | (t ^ 3 (a % 2) ^ 2 (a / 2)) << 2, distinct for the rows of a store (one
// t) and for those that a 16-byte read takes in one cycle, which are lanes 0-3,
// 12-15 and 20-27, or 4-11, 16-19 and 28-31 (with a ^ t they met in pairs: 5000
// tokens 248 -> 233 us in bf16); v's by
// d / 2.  Every address is a lane's base with constant bits flipped and a
// constant added, which costs an instruction where a register each would spill.
constexpr int kHalfLds = kPage * 256, kVLds = 2 * kHalfLds;
static_assert(kHalfLds == kHeadD * 128, "a page of k and one of v");
__device__ __forceinline__ int k_swz(int p) { return (p & 3) | (((p >> 2 & 3) ^ (p >> 4 & 3) ^ (p >> 3 & 2)) << 2); }
__device__ __forceinline__ int k_lds(int p, int c) { return p * 256 + 16 * (c ^ k_swz(p)); }
__device__ __forceinline__ int v_lds(int d, int c) { return kVLds + d * 128 + 16 * (c ^ ((d >> 1) & 7)); }

// Four waves of 32 query rows.  A page is widened to fp16 once for all of them
// on its way into LDS (one barrier a page; its codes come a page ahead into
// registers).  Lane (r = lane % 32, h = lane / 32) has the scores of query row
// r: element j of tile T is position 32 T + 16 (j / 8) + 8 h + j % 8, because
// row 8 b + 4 h + i (+ 16 s) of the product is given position 8 h + 4 b + i
// (+ 16 s); eight consecutive ones are a fragment of P^T and a 16-byte chunk of
// a dim's row of V^T.
//
// The next page's staging stands between the products of the scores, and a
// fragment's exponentials between the products of the fragment before.  What
// bounds it: the products, a third of them for the probabilities' low parts;
// the matrix cores are busy 60 % of the time, and two waves a SIMD fill the rest
// by chance.  A call of 5000 tokens 288 to 306 us, boxes differ, in fp16 and 285 to
// 302 in bf16 (670 to 720 TFLOP/s of the formula's operations, a third more with
// the low parts'), 6 chunks beside 3 short rows 98 to 102.  With one fp16 part of a
// probability, of 249 us before k's conflicts went, the exponentials alone made
// 38, staging 35, the fragments' reads 55, the products 68, and there was tried
// without gain: fragments read three steps ahead; raised priority around
// the products; one wave a SIMD with 64 rows and the next page's scores between
// this one's exponentials, whose accumulators in AGPRs cost more copies than the
// shared fragments save (326 us in bf16); the same with 32 rows, which spilled
// (272); eight waves over 256 rows, four of them half a page behind, products
// beside the others' softmax: that hides the softmax, but leaves the 10 us of a
// workgroup's start and end bare, with one workgroup a CU (251).
constexpr int kManyLds = 4 * kHalfLds + kHeadD * 4;

template <bool BF16>
__device__ __forceinline__ void attend_many(const AttendArgs& a, int b, uint8_t* s_page) {
  int* s_nan = reinterpret_cast<int*>(s_page + 4 * kHalfLds);
  // the last tiles, which see most, first
  const int back = b / a.n_kv, g = b - back * a.n_kv;
  const int item = min(scalar_load(a.work + kNMany), a.many.groups / a.n_kv) - 1 - back;
  if (item < 0) return;
  const AttendItem& full = a.many.items[item];
  const ItemHead it = scalar_load(static_cast<const ItemHead*>(&full));
  const int n_tok = min(it.n_tokens, a.n_tokens - it.token0);
  if (n_tok <= 0 || item - it.part + it.n_parts > a.many.groups / a.n_kv) return;
  const int tid = threadIdx.x, lane = lane_id(), r = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lg = a.group_log, n_rows = n_tok << lg;
  if (tid < kHeadD) s_nan[tid] = kNoNan;
  __syncthreads();

  // this lane's query row: B operand, step st dims 16 st + 8 h ..
  const int row = 32 * w + r, tok = row >> lg;
  h8 qf[8];
  int qe = 0;
  {
    uint16_t qv[8][8];
    const uint16_t* pq = a.q + (int64_t)(it.token0 + min(tok, n_tok - 1)) * a.token_stride +
                         (int64_t)((g << lg) + (row & ((1 << lg) - 1))) * a.head_stride + 8 * h;
#pragma unroll
    for (int st = 0; st < 8; ++st) {
      if (a.wide) {
        *reinterpret_cast<u32x4*>(qv[st]) = *reinterpret_cast<const u32x4*>(pq + 16 * st);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) qv[st][e] = pq[16 * st + e];
      }
    }
    if (BF16) {
      float top = 0.0f;
#pragma unroll
      for (int st = 0; st < 8; ++st)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(bf16_bits_to_float(qv[st][e])));
      top = fmaxf(top, __shfl_xor(top, 32));
      qe = min(max((int)(as_u32(top) >> 23) - 127 - kTopExp, -126), 126);
    }
#pragma unroll
    for (int st = 0; st < 8; ++st) qf[st] = q_frag<BF16>(qv[st], qe, a.scale < 0.0f);
  }
  const float sc = BF16 ? ldexp2(a.scale, qe) : a.scale;
  const int lim = row < n_rows ? min(it.pos0 + tok + 1, it.kv_len) : 0;   // positions that this row sees
  // ... that every row of the wave sees
  const int all_see = min(it.pos0 + (32 * w >> lg) + 1, it.kv_len);

  const float ninf = -__builtin_inff();
  f32x16 o[4];
#pragma unroll
  for (int d = 0; d < 4; ++d) o[d] = f32x16{};
  float m = ninf, l = 0.0f;

  const int32_t* table = a.table + (int64_t)it.row * a.width;
  auto block_of = [&](int page) {
    int id = scalar_load(table + min(page, it.page1 - 1));
    id = (unsigned)id < (unsigned)a.n_pages ? id : 0;
    return (int64_t)id * a.n_kv + g;
  };
  u32x4 kr[2], vr[2];                  // codes on their way into LDS: vectors tid and tid + 256
  auto load = [&](u32x4 (&x)[2], int64_t block, int half) {
    const uint8_t* b = a.pages + block * kBlock + half;
#pragma unroll
    for (int n = 0; n < 2; ++n) x[n] = load16(b + 16 * tid + 4096 * n);
  };
  // lane bases of the stores and reads
  const int st_p = 16 * ((tid & 15) >> 2) + 4 * (tid >> 7) + (tid & 3), st_d = 16 * (tid >> 6) + (tid & 15);
  const int k_st = k_lds(st_p, 2 * ((tid >> 4) & 7)), v_st = v_lds(st_d, 2 * ((tid >> 4) & 3));
  const int k_rd = k_lds((r & 19) | ((r >> 3) & 1) << 2 | ((r >> 2) & 1) << 3, h), v_rd = v_lds(r, h);
  // part q of 4 of the staged vectors, widened into LDS
  auto put_k = [&](int ka, int q) {    // 8 positions (2 t) further: the swizzle's bit 3 flips
    const int n = q >> 1, e = q & 1;
    *reinterpret_cast<h8*>(s_page + (ka ^ (128 * n) ^ (16 * e)) + 2048 * n) = widen8(kr[n][2 * e], kr[n][2 * e + 1]);
  };
  auto put_v = [&](int va, int q) {    // 64 dims further
    const int n = q >> 1, e = q & 1;
    *reinterpret_cast<h8*>(s_page + (va ^ (16 * e)) + 8192 * n) = widen8(vr[n][2 * e], vr[n][2 * e + 1]);
  };
  auto fix_v = [&](int page, float v_scale) {
    const int tail = it.kv_len - page * kPage - 16 * ((tid >> 4) & 3);
    if (page * kPage + kPage > it.kv_len) {   // behind the row's end: whatever the page held before
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k) vr[n][k] = first_bytes(vr[n][k], tail - 4 * k);
    }
    if (v_scale < 0.0f) {
#pragma unroll
      for (int n = 0; n < 2; ++n) take_nans(vr[n], page * kPage + 16 * ((tid >> 4) & 3), &s_nan[st_d + 64 * n]);
    }
  };
  auto scale_of = [&](int64_t block) { return scalar_load(reinterpret_cast<const float2*>(a.scales) + block); };

  h8 kf[2][2], vf[4];
  auto read_k = [&](int ka, int st) {
#pragma unroll
    for (int T = 0; T < 2; ++T)        // a 2 further: the swizzle's bit 3
      kf[st & 1][T] = *reinterpret_cast<const h8*>(s_page + (ka ^ (32 * st) ^ (128 * T)) + 8192 * T);
  };
  auto read_v = [&](int va, int i) {   // fragment f = i / 4, dims 32 (i % 4) ..
    vf[i & 3] = *reinterpret_cast<const h8*>(s_page + (va ^ (32 * (i >> 2))) + 4096 * (i & 3));
  };
  // `page` is in buffers i % 2; the next one goes from kr and vr to the others,
  // the one after it is loaded.
  auto round = [&](int page, int i, float2 scale, float2 next_scale, int64_t after) {
    const int at = (i & 1) * kHalfLds, other = kHalfLds - at;
    fix_v(page + 1, next_scale.y);
    int k_to = other + k_st, v_to = other + v_st;
    int ka = at + k_rd, va = at + v_rd;
    asm volatile("" : "+v"(ka), "+v"(va), "+v"(k_to), "+v"(v_to));
    read_k(ka, 0);
    f32x16 s[2] = {};
#pragma unroll
    for (int st = 0; st < 8; ++st) {
      if (st < 7) read_k(ka, st + 1);
      if (st >= 5) read_v(va, st - 5);
#pragma unroll
      for (int T = 0; T < 2; ++T) s[T] = mfma32(kf[st & 1][T], qf[st], s[T]);
      if (st & 1) put_v(v_to, st >> 1);
      else put_k(k_to, st >> 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    load(kr, after, 0);
    load(vr, after, kHalfBlock);
    __builtin_amdgcn_sched_barrier(0);
    const float ev = (float)((int)((as_u32(scale.y) >> 23) & 0xFF) - 127), ksc = score_scale(sc, scale.x);
    if (page * kPage + kPage > all_see) {
      const int p0 = page * kPage + 8 * h;
#pragma unroll
      for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[T][j] = p0 + 32 * T + 16 * (j >> 3) + (j & 7) < lim ? s[T][j] : ninf;
    }
    float cm = ninf;
#pragma unroll
    for (int T = 0; T < 2; ++T)
#pragma unroll
      for (int j = 0; j < 16; ++j) cm = fmaxf(cm, s[T][j]);
    cm = fmaf(fmaxf(cm, __shfl_xor(cm, 32)), ksc, ev);
    const bool up = cm > m + kSlack;
    if (__any(up)) {
      const float mn = up ? cm : m;
      const float alpha = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      l *= alpha;
#pragma unroll
      for (int d = 0; d < 4; ++d) o[d] *= alpha;
      m = mn;
    }
    const float rel = ev - ((m == ninf ? 0.0f : m) - kLift);
    // fragment f of the probabilities: positions 16 f + 8 h ..
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f}, e[8];
    auto exps = [&](int f, int j0, int j1) {
#pragma unroll
      for (int j = j0; j < j1; ++j) {
        e[j] = __builtin_amdgcn_exp2f(fmaf(s[f >> 1][8 * (f & 1) + j], ksc, rel));
        sum[f] += e[j];
      }
    };
    Probs p;
    exps(0, 0, 8);
    p = to_probs(e);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int f = 0; f < 4; ++f) {
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        if (4 * f + d < 13) read_v(va, 4 * f + d + 3);
        o[d] = mfma32(vf[d], p.hi, o[d]);
        o[d] = mfma32(vf[d], p.lo, o[d]);
        if (f < 3) exps(f + 1, 2 * d, 2 * d + 2);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (f < 3) p = to_probs(e);
    }
    l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), ldexp2(1.0f, -(int)ev), l);
  };

  if (it.page0 < it.page1) {
    const int64_t b0 = (int64_t)scalar_load(full.ids) * a.n_kv + g;
    const int64_t b1 = (int64_t)scalar_load(full.ids + 1) * a.n_kv + g;
    int64_t b2 = block_of(it.page0 + 2);
    load(kr, b0, 0);
    load(vr, b0, kHalfBlock);
    float2 sc0 = scale_of(b0), sc1 = scale_of(b1);
    fix_v(it.page0, sc0.y);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      put_k(k_st, q);
      put_v(v_st, q);
    }
    load(kr, b1, 0);
    load(vr, b1, kHalfBlock);
    for (int page = it.page0; page < it.page1; ++page) {
      __syncthreads();                 // the page is in LDS, the last one is read
      const float2 sc2 = scale_of(b2);
      const int64_t b3 = block_of(page + 3);
      round(page, page - it.page0, sc0, sc1, b2);   // past the last page: that one again, not used
      b2 = b3;
      sc0 = sc1;
      sc1 = sc2;
    }
  }

  l += __shfl_xor(l, 32);
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j)
      o[d][j] = s_nan[32 * d + 8 * (j >> 2) + 4 * h + (j & 3)] < lim ? __builtin_nanf("") : o[d][j];
  if (it.n_parts > 1) {
    // through LDS (chunks of a row swizzled by it), so that rows leave whole
    static_assert(kManyRows * 512 <= 4 * kHalfLds, "a tile's sums");
    __syncthreads();
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(s_page + row * 512 + 16 * ((8 * d + 2 * q + h) ^ r)) =
            f32x4{o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
    const int64_t base = ((int64_t)(it.slot0 + it.part) * a.n_kv + g) * kManyRows;
    const rsrc_t ro = rsrc(a.many.o + base * kHeadD, kManyRows * kHeadD * 4);
    __syncthreads();
    for (int i = tid; i < n_rows * 32; i += kThreads)
      __builtin_amdgcn_raw_buffer_store_b128(*reinterpret_cast<const u32x4*>(s_page + (i >> 5) * 512 + 16 * ((i ^ (i >> 5)) & 31)),
                                             ro, 16 * i, 0, kSc1);
    if (h == 0 && row < n_rows) {
      st_agent(a.many.ml + 2 * (base + row), m);
      st_agent(a.many.ml + 2 * (base + row) + 1, l);
    }
    if (arrive(a.many, it, a.n_kv, g)) join_parts<BF16, kManyRows>(a, a.many, it, g, n_rows, reinterpret_cast<float*>(s_page));
    return;
  }
  if (row >= n_rows) return;
  const float inv = it.kv_len > 0 ? 1.0f / l : 0.0f;   // a rejected row: zeros
  uint16_t* po = a.out + ((int64_t)(it.token0 + tok) * a.n_q + (g << lg) + (row & ((1 << lg) - 1))) * kHeadD + 4 * h;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint16_t z[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = narrow<BF16>(o[d][4 * q + e] * inv);
      *reinterpret_cast<u32x2v*>(po + 32 * d + 8 * q) = *reinterpret_cast<u32x2v*>(z);
    }
}

// Zeros for the rows past the step's last token.
__device__ __forceinline__ void zero_rest(const AttendArgs& a, int b) {
  const int row = a.n_q * (kHeadD / 8);    // 16-byte vectors of a token
  u32x4* out = reinterpret_cast<u32x4*>(a.out);
  for (int t = max(scalar_load(a.total), 0) + b; t < a.n_tokens; t += a.zero_groups)
    for (int i = threadIdx.x; i < row; i += kThreads) out[(int64_t)t * row + i] = u32x4{0, 0, 0, 0};
}

// Steps whose rows all have few query rows, and steps with rows of either kind:
// the long tiles first, the others fill the chip behind and beside them.
template <bool BF16>
__global__ __launch_bounds__(kThreads, 2) void k_attend_few(AttendArgs a) {
  __shared__ __align__(16) uint8_t smem[kFewLds];
  const int b = blockIdx.x;
  if (b < a.few.groups) attend_few<BF16>(a, b, smem);
  else zero_rest(a, b - a.few.groups);
}

template <bool BF16>
__global__ __launch_bounds__(kThreads, 2) void k_attend(AttendArgs a) {
  static_assert(kManyLds >= kFewLds && kThreads == 64 * kFewWaves, "one workgroup for either");
  __shared__ __align__(1024) uint8_t smem[kManyLds];
  const int b = blockIdx.x;
  if (b < a.many.groups) attend_many<BF16>(a, b, smem);
  else if (b - a.many.groups < a.few.groups) attend_few<BF16>(a, b - a.many.groups, smem);
  else zero_rest(a, b - a.many.groups - a.few.groups);
}

// Arrivals of the parts: in the workspace, which is the call's own, and cleared
// by the call, so that calls of one plan (other layers, other queries) may run
// at the same time.
__global__ __launch_bounds__(1024) void k_clear(int32_t* count, int n) {
  const int i = blockIdx.x * 1024 + threadIdx.x;
  if (i < n) count[i] = 0;
}

// The workspace: the partial sums of either kernel's parts, out and then m, l;
// the parts' counters.
size_t few_floats(const PlanLayout& l, int n_kv) { return (size_t)l.cap_parts_few * n_kv * kFewRows * (kHeadD + 2); }
size_t many_floats(const PlanLayout& l, int n_kv) { return (size_t)l.cap_parts_many * n_kv * kManyRows * (kHeadD + 2); }
size_t counters(const PlanLayout& l, int n_kv) { return (size_t)(l.cap_parts_few + l.cap_parts_many) * n_kv; }
size_t attend_bytes(const PlanLayout& l, int n_kv) { return (few_floats(l, n_kv) + many_floats(l, n_kv) + counters(l, n_kv)) * 4; }

}  // namespace
}  // namespace oi2

using namespace oi2;

extern "C" {

size_t oi2_kv_attend_workspace_bytes(const oi2_paged* c, int32_t max_tokens, int32_t max_new) {
  if (!oi2_page_plan_bytes(c, max_tokens, max_new)) return 0;
  const PlanLayout l = plan_layout(*c, max_tokens, max_new);
  const size_t n = attend_bytes(l, c->n_kv);
  return n ? n : 16;
}

int oi2_kv_attend(const oi2_paged* c, const oi2_page_plan* p, int32_t layer, int32_t dtype, int32_t n_tokens,
                  const oi2_heads* q, float scale, void* out, void* workspace, size_t workspace_bytes,
                  void* stream) {
  clear_error();
  if (int rc = check_paged(c, layer, true)) return rc;
  if (int rc = check_plan(c, p)) return rc;
  const bool zero = dtype & OI2_ZERO_LEFT_OUT;
  dtype &= ~OI2_ZERO_LEFT_OUT;
  OI2_CHECK_ARG(dtype == OI2_DTYPE_F16 || dtype == OI2_DTYPE_BF16, "dtype %d: fp16 or bf16", dtype);
  OI2_CHECK_ARG(n_tokens >= 0 && n_tokens <= p->max_tokens, "%d tokens in a plan of %d", n_tokens, p->max_tokens);
  OI2_CHECK_ARG(q && q->heads == c->n_q, "q needs the cache's %d query heads", c->n_q);
  OI2_CHECK_ARG(scale == scale && scale - scale == 0.0f, "the scale of the scores is not finite");
  if (n_tokens == 0) return OI2_OK;
  OI2_CHECK_ARG(q->data && (uintptr_t)q->data % 2 == 0, "q must be non-null and 2-byte aligned");
  OI2_CHECK_ARG(out && (uintptr_t)out % 16 == 0, "out must be non-null and 16-byte aligned");
  const PlanLayout l = plan_layout(*c, p->max_tokens, p->max_new), now = plan_layout(*c, n_tokens, p->max_new);
  const size_t need = attend_bytes(l, c->n_kv);
  OI2_CHECK_ARG(!need || (workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need),
                "workspace of %zu bytes, %zu needed, 16-byte aligned", workspace_bytes, need);
  OI2_CHECK_ARG(!clashes(true, out, c->n_q, q, n_tokens, kHeadD), "out shares memory with q, and is not q");
  AttendArgs a{};
  a.work = p->work;
  a.table = c->block_table;
  a.pages = c->pages + (size_t)layer * c->n_pages * c->n_kv * kBlock;
  a.scales = c->scales + (size_t)layer * c->n_pages * c->n_kv * 2;
  a.n_q = c->n_q;
  a.n_kv = c->n_kv;
  a.group_log = 0;
  while (c->n_kv << a.group_log < c->n_q) ++a.group_log;
  a.width = (c->max_len + kPage - 1) / kPage;
  a.n_pages = c->n_pages;
  a.n_tokens = n_tokens;
  a.q = (const uint16_t*)q->data;
  a.token_stride = q->token_stride;
  a.head_stride = q->head_stride;
  a.wide = (uintptr_t)q->data % 16 == 0 && q->token_stride % 8 == 0 && q->head_stride % 8 == 0;
  a.scale = scale * kLog2e;
  a.out = (uint16_t*)out;
  hipStream_t st = (hipStream_t)stream;
  const bool bf = dtype == OI2_DTYPE_BF16;
  const int64_t few = (int64_t)now.cap_few * c->n_kv, many = (int64_t)now.cap_many * c->n_kv;
  OI2_CHECK_ARG(few + many < 1 << 23, "%d tokens are too many for one call", n_tokens);
  a.few.items = reinterpret_cast<const AttendItem*>(p->work + l.few);
  a.few.groups = (int)few;
  a.few.o = (float*)workspace;
  a.few.ml = a.few.o + (size_t)l.cap_parts_few * c->n_kv * kFewRows * kHeadD;
  a.many.items = reinterpret_cast<const AttendItem*>(p->work + l.many);
  a.many.groups = (int)many;
  a.many.o = a.few.o + few_floats(l, c->n_kv);
  a.many.ml = a.many.o + (size_t)l.cap_parts_many * c->n_kv * kManyRows * kHeadD;
  a.few.count = (int32_t*)(a.few.o + few_floats(l, c->n_kv) + many_floats(l, c->n_kv));
  a.many.count = a.few.count + (size_t)l.cap_parts_few * c->n_kv;
  if (need) {
    const int n = (int)counters(l, c->n_kv);
    hipLaunchKernelGGL(k_clear, dim3((n + 1023) / 1024), dim3(1024), 0, st, a.few.count, n);
    OI2_CHECK_LAUNCH();
  }
  a.total = p->cu + c->n_seqs;
  a.zero_groups = zero ? (n_tokens < 128 ? n_tokens : 128) : 0;
  const dim3 grid((uint32_t)(few + many + a.zero_groups)), block(kThreads);
  if (many && bf) hipLaunchKernelGGL(k_attend<true>, grid, block, 0, st, a);
  else if (many) hipLaunchKernelGGL(k_attend<false>, grid, block, 0, st, a);
  else if (bf) hipLaunchKernelGGL(k_attend_few<true>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(k_attend_few<false>, grid, block, 0, st, a);
  OI2_CHECK_LAUNCH();
  return OI2_OK;
}

}  // extern "C"
