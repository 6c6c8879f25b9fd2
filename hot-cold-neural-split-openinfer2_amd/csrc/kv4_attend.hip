// Attention of a step's query tokens over the paged 4-bit KV cache: the plan, the
// parts and the products of the 8-bit cache's, on pages whose groups of 32 dims
// have a scale at every position.
//
// Codes times scales, exact in fp16, are the products' operands, so that scales
// cost one packed multiplication for two values and nothing behind it:
//   p = exp2(score - m),  out = sum p v,  l = sum p
// The cache stores a page so that a lane's 16 bytes of k are 32 dims of one
// position, one group, and its 16 bytes of v 8 dims, of one group, of four
// positions: a scale serves all that a lane has of a position.
#include "attend.h"
#include "kv4.h"

namespace oi2 {
namespace {

// A dword of k, dims in order, times its scale.
__device__ __forceinline__ h8 k_values(uint32_t d, f16x2 s) {
  const uint32_t lo = low4(d), hi = high4(d);
  const f16x2 a = whole2(lo, false) * s, b = whole2(lo, true) * s, c = whole2(hi, false) * s, e = whole2(hi, true) * s;
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
}
__device__ __forceinline__ f16x2 twice(uint32_t d, bool hi) {
  return as_f16x2(__builtin_amdgcn_perm(d, d, hi ? 0x03020302u : 0x01000100u));
}

// Dims 2 q and 2 q + 1 of two positions' dwords x, y as e4m3 bytes: (x, y) of the
// first, (x, y) of the second.
__device__ __forceinline__ uint32_t v_bytes(uint32_t x, uint32_t y, int q) {
  return __builtin_amdgcn_perm(y, x, q & 1 ? 0x07030602u : 0x05010400u);
}

// Scales of v at positions pos, pos + 1 .. in pairs: behind the row's end 0,
// whatever the page held before; a NaN that some row may not see 0, and noted for
// the 8 dims from dim0 on.
template <int N>
__device__ __forceinline__ void fix_scales(uint32_t (&s)[N], int pos, int kv_len, int dim0, int* nan) {
#pragma unroll
  for (int k = 0; k < 2 * N; ++k) {
    const uint32_t shift = 16 * (k & 1);
    const bool out = pos + k >= kv_len, odd = (s[k / 2] >> shift & 0x7C00u) == 0x7C00u;
    if (out || odd) s[k / 2] &= ~(0xFFFFu << shift);
    if (odd && !out)
      for (int e = 0; e < 8; ++e) atomicMin(&nan[dim0 + e], pos + k);
  }
}

// ── few rows ─────────────────────────────────────────────────────────────────

// Lane (r = lane % 16, grp = lane / 16).  K's 16-row tile t of a page: row
// r = 4 a + i is position 16 a + 4 t + i, and the lane has dims 32 grp .. of it,
// eight a step; D's element i of lane (r, grp) is the score of query row r at
// position 16 grp + 4 t + i: in 4 tiles a lane has positions 16 grp .. 16 grp + 15
// of its query row.  V's row r of tile d is dim 8 r + d, at those positions.
//
// A wave takes every fourth page, loads the next one (9 KB) while it works on
// this one, and its page number by a scalar load two ahead; the four meet in
// LDS at the end.
//
// Bound by loads and instructions alike: 48 tokens over 500 to 20000 positions
// 57.7 us (258 MB, 4.5 TB/s); their loads alone 50, the products alone 52; two
// over 60 and 150 thousand 37.3 (34 and 34), 20 rows of 4 tokens 19.7 (18 and 18).
// Besides: 4 us to the first scores, parts of unequal length, 4 for arrivals and
// joins.  158 registers, three workgroups a CU: with two 48 tokens take 65, with
// four (128 registers) 92.  Measured slower: pages two ahead (66.5), equal shares of
// all pages (61.5, and 54 instead of 20 for the drafts), a second launch that joins
// (the two long ones 41.4), the query loaded behind the first page (59.2).  Shorter
// parts: every part halved 64 instead of 61 (an earlier form), the two long ones 46
// instead of 40, the drafts 27.5 instead of 21; cut three times as fine only where
// a step has 256 tiles or more 55.3 instead of 57.4, and nothing elsewhere.  That is
// not done: the plan, which is laid out for either cache, cuts the rows.
//
// SETS: of 16 query rows.  Two where all rows have 17 to 32: a page is decoded
// once for both, and 244 registers leave two workgroups a CU (126 scalars are kept
// in lanes of vector registers; none goes to memory).  24 drafts of 8 tokens over
// 300 to 14000 positions 44 us (110 MB, 2.5 TB/s) instead of 91 the way of many
// rows, 40 of 5 over 200 to 4000 34 instead of 68.  33 to 64 rows stay there: 56 of them took 72.8
// with four sets (414 registers) and 63.2 with two workgroups a tile, and there 65.
template <bool BF16, int SETS>
__device__ __forceinline__ bool attend_few(const AttendArgs& a, const Found& found, uint8_t* smem) {
  const FewLds<SETS> lds(smem);
  FewTile<SETS> t;
  few_open<BF16>(a, found, lds, t, [](int grp, int i) { return 32 * grp + 8 * i; });
  const ItemHead& it = t.it;
  const int g = t.g, w = t.w, lane = t.lane, r = t.r, grp = t.grp, all_see = t.all_see;

  const float ninf = -__builtin_inff();
  f32x4 o[SETS][8];
  float m[SETS], l[SETS], ksc[SETS];
#pragma unroll
  for (int z = 0; z < SETS; ++z) {
#pragma unroll
    for (int d = 0; d < 8; ++d) o[z][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[z] = ninf;
    l[z] = 0.0f;
    ksc[z] = score_scale(t.sc[z], 1.0f);
  }

  const int32_t* table = a.table + (int64_t)it.row * a.width;
  auto block_of = [&](int page) {
    int id = scalar_load(table + min(page, it.page1 - 1));
    id = (unsigned)id < (unsigned)a.n_pages ? id : 0;
    return (int64_t)id * a.n_kv + g;
  };
  // Past the last page the descriptor's range is empty: nothing is read.
  auto page_rsrc = [&](int64_t block, int page) { return rsrc(a.pages + block * k4Block, page < it.page1 ? k4Block : 0); };
  u32x4 kr[4], vr[4];
  u32x2v ks;
  uint32_t vs[8];
  // The scales first, and in one order everywhere: a wait is for a number of
  // loads, and where two orders meet for the larger one (at the loop's head that
  // was all of them: 48 tokens over long contexts 61.2 -> 57.6 us).
  auto load_k = [&](rsrc_t x) {
    ks = wld8(x, k4KScale + 8 * lane);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 4; ++n) kr[n] = wld16(x, 1024 * n + 16 * lane);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto load_v = [&](rsrc_t x) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const u32x4 s = wld16(x, k4VScale + 128 * (r >> 2) + 32 * grp + 16 * n);
#pragma unroll
      for (int k = 0; k < 4; ++k) vs[4 * n + k] = s[k];
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 4; ++n) vr[n] = wld16(x, k4V + 1024 * n + 16 * lane);
    __builtin_amdgcn_sched_barrier(0);
  };
  const int first = it.page0 + w;
  int64_t next = 0;
  if (first < it.page1) {
    const rsrc_t r0 = page_rsrc((int64_t)scalar_load(t.full->ids + w) * a.n_kv + g, first);
    load_k(r0);
    load_v(r0);
    next = block_of(first + kFewWaves);
  }
  for (int page = first; page < it.page1; page += kFewWaves) {
    const rsrc_t rn = page_rsrc(next, page + kFewWaves);
    next = block_of(page + 2 * kFewWaves);

    float s[SETS][16];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f32x4 acc[SETS] = {};
      const f16x2 sk = twice(k < 2 ? ks.x : ks.y, k & 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const h8 kv = k_values(kr[k][i], sk);
#pragma unroll
        for (int z = 0; z < SETS; ++z) acc[z] = mfma16(kv, t.q[z][i], acc[z]);
      }
#pragma unroll
      for (int z = 0; z < SETS; ++z)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[z][4 * k + i] = acc[z][i];
    }
    __builtin_amdgcn_sched_barrier(0);
    load_k(rn);
    const int p0 = page * kPage + 16 * grp;
    const bool whole = page * kPage + kPage <= all_see;
    if (!whole) {
#pragma unroll
      for (int z = 0; z < SETS; ++z)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[z][j] = p0 + j < t.lim[z] ? s[z][j] : ninf;
      fix_scales(vs, p0, it.kv_len, 8 * r, lds.nan);
    }
    Probs p[SETS][2];
#pragma unroll
    for (int z = 0; z < SETS; ++z) {
      float cm = s[z][0];
#pragma unroll
      for (int j = 1; j < 16; ++j) cm = fmaxf(cm, s[z][j]);
      cm = quad_max(cm) * ksc[z];
      const bool up = cm > m[z] + kSlack;
      if (__any(up)) {
        const float mn = up ? cm : m[z];
        const float alpha = m[z] == mn ? 1.0f : __builtin_amdgcn_exp2f(m[z] - mn);
        l[z] *= alpha;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[z][d] *= alpha;
        m[z] = mn;
      }
      const float rel = kLift - (m[z] == ninf ? 0.0f : m[z]);
      float sum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          e[j] = __builtin_amdgcn_exp2f(fmaf(s[z][8 * h + j], ksc[z], rel));
          sum[h] += e[j];
        }
        p[z][h] = to_probs(e);
      }
      l[z] += sum[0] + sum[1];
    }
    // positions 16 grp + 8 h + 2 k, + 1 are dwords 2 (k % 2), + 1 of vector 2 h + k / 2
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < 4; ++q) {        // dims 8 r + 2 q, + 1
        f16x2 v0[4], v1[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t x = vr[2 * h + k / 2][2 * (k % 2)], y = vr[2 * h + k / 2][2 * (k % 2) + 1];
          const uint32_t d = q < 2 ? v_bytes(low4(x), low4(y), q) : v_bytes(high4(x), high4(y), q);
          const f16x2 sv = as_f16x2(vs[4 * h + k]);
          v0[k] = whole2(d, false) * sv;
          v1[k] = whole2(d, true) * sv;
        }
        const h8 f0 = {v0[0][0], v0[0][1], v0[1][0], v0[1][1], v0[2][0], v0[2][1], v0[3][0], v0[3][1]};
        const h8 f1 = {v1[0][0], v1[0][1], v1[1][0], v1[1][1], v1[2][0], v1[2][1], v1[3][0], v1[3][1]};
#pragma unroll
        for (int z = 0; z < SETS; ++z) {
          o[z][2 * q] = mfma16(f0, p[z][h].hi, o[z][2 * q]);
          o[z][2 * q] = mfma16(f0, p[z][h].lo, o[z][2 * q]);
          o[z][2 * q + 1] = mfma16(f1, p[z][h].hi, o[z][2 * q + 1]);
          o[z][2 * q + 1] = mfma16(f1, p[z][h].lo, o[z][2 * q + 1]);
        }
      }
    __builtin_amdgcn_sched_barrier(0);
    load_v(rn);
  }

#pragma unroll
  for (int z = 0; z < SETS; ++z) {
    const int row = kFewRows * z + r;
    l[z] += __shfl_xor(l[z], 16);
    l[z] += __shfl_xor(l[z], 32);
#pragma unroll
    for (int i = 0; i < 4; ++i)            // dims 8 (4 grp + i) ..
#pragma unroll
      for (int d = 0; d < 8; d += 4)
        *reinterpret_cast<f32x4*>(&lds.o[w][row][8 * (4 * grp + i) + d]) =
            f32x4{o[z][d][i], o[z][d + 1][i], o[z][d + 2][i], o[z][d + 3][i]};
    if (grp == 0) {
      lds.m[w][row] = m[z];
      lds.l[w][row] = l[z];
    }
  }
  return few_close<BF16>(a, t, lds);
}

// Zeros for the tokens of a rejected row.
__device__ __forceinline__ void zero_tile(const AttendArgs& a, const Found& f) {
  const int lg = a.group_log;
  for (int i = threadIdx.x; i < f.n_tok << lg << 4; i += kThreads) {   // 16 vectors of 8 dims a row
    const int row = i >> 4, head = (f.g << lg) + (row & ((1 << lg) - 1));
    *reinterpret_cast<u32x4*>(a.out + ((int64_t)(f.it.token0 + (row >> lg)) * a.n_q + head) * kHeadD + 8 * (i & 15)) = u32x4{0, 0, 0, 0};
  }
}

// ── many rows ────────────────────────────────────────────────────────────────

// Thread (n = tid / 64, lane): the 16 bytes of k of one position and group, and
// those of v of positions 16 grp + 4 n .. + 3, dims 8 r ...  Row 16 e + r of V^T
// in LDS is dim 8 r + e, so that a wave's stores are to 16 rows side by side.
//
// A prompt of 4100 tokens 206 us (667 TFLOP/s of the formula's operations, half as
// much again with the low parts'), 10 chunks of 1 to 800 tokens over 400 to 9000
// positions 104 (472).  The CUs are busy 83 and 70 % of the time (the rest is
// start, unequal parts, joins), in it the matrix cores 56 and 45 %, vector
// instructions 62 %, LDS 33 %; two waves a SIMD overlap them by chance.  A page's
// staging is 97 of its 340 vector instructions; low parts to nearest, which are 16
// fewer, took 1 % off the prompt alone.
struct Pages4 {
  const AttendArgs& a;
  const ItemHead& it;
  int tid, *nan;
  int k_st, v_st;                      // lane bases of the staging stores
  int at_ks, at_vs;                    // of the scales in a block
  u32x4 kr, vr;
  uint32_t ks, vs[2];

  __device__ __forceinline__ Pages4(const AttendArgs& args, const ItemHead& item, int thread, int* s_nan)
      : a(args), it(item), tid(thread), nan(s_nan) {
    const int n = tid >> 6, hi = (tid >> 4) & 3, r = tid & 15;    // hi: k's group, v's grp
    k_st = k_lds(16 * (r >> 2) + 4 * n + (r & 3), 4 * hi);
    v_st = v_lds(r, 2 * hi + (n >> 1)) + 8 * (n & 1);
    at_ks = k4KScale + 8 * (tid & 63) + 2 * n;
    at_vs = k4VScale + 128 * (r >> 2) + 2 * (16 * hi + 4 * n);
  }
  __device__ __forceinline__ int first_pos() const { return 16 * ((tid >> 4) & 3) + 4 * (tid >> 6); }
  __device__ __forceinline__ void load(int64_t block) {
    const uint8_t* b = a.pages + block * k4Block;
    kr = load16(b + 16 * tid);
    vr = load16(b + k4V + 16 * tid);
    ks = *reinterpret_cast<const uint16_t*>(b + at_ks);
    const u32x2v s = *reinterpret_cast<const u32x2v*>(b + at_vs);
    vs[0] = s.x;
    vs[1] = s.y;
  }
  __device__ __forceinline__ float2 scale_of(int64_t) const { return float2{1.0f, 1.0f}; }
  __device__ __forceinline__ void fix(int page, float) {
    if (page * kPage + kPage > min(it.pos0 + 1, it.kv_len)) fix_scales(vs, page * kPage + first_pos(), it.kv_len, 8 * (tid & 15), nan);
  }
  __device__ __forceinline__ void put_k(uint8_t* s_page, int ka, int q) const {
    *reinterpret_cast<h8*>(s_page + (ka ^ (16 * q))) = k_values(kr[q], twice(ks, false));
  }
  __device__ __forceinline__ void put_v(uint8_t* s_page, int va, int q) const {   // dims 8 r + 2 q, + 1: rows 32 q + r, + 16
    f16x2 v[2][2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t x = vr[2 * k], y = vr[2 * k + 1];
      const uint32_t d = q < 2 ? v_bytes(low4(x), low4(y), q) : v_bytes(high4(x), high4(y), q);
      v[0][k] = whole2(d, false) * as_f16x2(vs[k]);
      v[1][k] = whole2(d, true) * as_f16x2(vs[k]);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<u32x2v*>(s_page + va + 128 * (32 * q + 16 * e)) =
          u32x2v{__builtin_bit_cast(uint32_t, v[e][0]), __builtin_bit_cast(uint32_t, v[e][1])};
  }
  // element j of o[d] in half h is row 32 d + 8 (j / 4) + j % 4, + 4 h, of V^T
  static __device__ __forceinline__ int dim(int row, int h) { return 8 * ((row & 15) + 4 * h) + (row >> 4); }
  template <class F>
  static __device__ __forceinline__ void each_four(const f32x16 (&o)[4], int h, F f) {   // of dims 4 chunk ..
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e)          // dims 8 (8 q + 4 h + e) ..: rows 16 apart
#pragma unroll
        for (int d = 0; d < 4; d += 2)
          f(2 * (8 * q + 4 * h + e) + d / 2,
            f32x4{o[d][4 * q + e], o[d][8 + 4 * q + e], o[d + 1][4 * q + e], o[d + 1][8 + 4 * q + e]});
  }
};

template <bool BF16>
__global__ __launch_bounds__(kThreads, 2) void k_kv4_attend_few(AttendArgs a) {
  __shared__ __align__(16) uint8_t smem[kFewLds<1>];
  const int b = blockIdx.x;
  Found f;
  if (b >= a.few.groups) zero_rest(a, b - a.few.groups);
  else if (few_find(a, b, f) && attend_few<BF16, 1>(a, f, smem)) join_parts<BF16, kFewRows>(a, a.few, f, smem);
}

// Steps whose rows all have kSetsRows query rows at most (max_new says so), and
// some more than one set.  A kernel of its own: beside attend_many and chosen by
// the tile it made every step with chunks 2 us longer, by its 20 KB of code and
// the registers that its arguments hold.
constexpr int kSets = 2, kSetsRows = kSets * kFewRows;

template <bool BF16>
__global__ __launch_bounds__(kThreads, 2) void k_kv4_attend_sets(AttendArgs a) {
  __shared__ __align__(16) uint8_t smem[kFewLds<kSets>];
  const int b = blockIdx.x;
  Found f;
  if (b < a.many.groups) {
    if (!many_find(a, b, f)) return;
    if (f.it.n_tokens << a.group_log > kSetsRows) zero_tile(a, f);     // only a rejected row has more
    else if (attend_few<BF16, kSets>(a, f, smem)) join_parts<BF16, kManyRows>(a, a.many, f, smem);
  } else if (b - a.many.groups >= a.few.groups) {
    zero_rest(a, b - a.many.groups - a.few.groups);
  } else if (few_find(a, b - a.many.groups, f) && attend_few<BF16, 1>(a, f, smem)) {
    join_parts<BF16, kFewRows>(a, a.few, f, smem);
  }
}

template <bool BF16>
__global__ __launch_bounds__(kThreads, 2) void k_kv4_attend(AttendArgs a) {
  static_assert(kManyLds >= kFewLds<1> && kThreads == 64 * kFewWaves, "one workgroup for either");
  __shared__ __align__(1024) uint8_t smem[kManyLds];
  const int b = blockIdx.x;
  Found f;
  if (b < a.many.groups) {
    if (many_find(a, b, f) && attend_many<BF16, Pages4>(a, f, smem)) join_parts<BF16, kManyRows>(a, a.many, f, smem);
  } else if (b - a.many.groups >= a.few.groups) {
    zero_rest(a, b - a.many.groups - a.few.groups);
  } else if (few_find(a, b - a.many.groups, f) && attend_few<BF16, 1>(a, f, smem)) {
    join_parts<BF16, kFewRows>(a, a.few, f, smem);
  }
}

}  // namespace

int kv4_counters(const oi2_paged* c, const oi2_page_plan* p, void* workspace, int32_t** at) {
  const PlanLayout l = plan_layout(*c, p->max_tokens, p->max_new);
  *at = counters_at(l, c->n_kv, workspace);
  return (int)counters(l, c->n_kv);
}

int kv4_attend(const oi2_paged* c, const oi2_page_plan* p, int32_t layer, int32_t dtype, int32_t n_tokens, const oi2_heads* q, float scale,
               void* out, void* workspace, size_t workspace_bytes, bool cleared, void* stream) {
  if (int rc = check_paged4(c, layer)) return rc;
  hipStream_t st = (hipStream_t)stream;
  AttendCall call;
  if (int rc = attend_call(call, c, p, dtype, n_tokens, q, scale, out, workspace, workspace_bytes, st, cleared)) return rc;
  if (!call.groups) return OI2_OK;
  AttendArgs& a = call.a;
  a.pages = c->pages + (size_t)layer * c->n_pages * c->n_kv * k4Block;
  const dim3 grid(call.groups), block(kThreads);
  const bool sets = a.many.groups && (int64_t)p->max_new << a.group_log <= kSetsRows;
  if (sets && call.bf16) hipLaunchKernelGGL(k_kv4_attend_sets<true>, grid, block, 0, st, a);
  else if (sets) hipLaunchKernelGGL(k_kv4_attend_sets<false>, grid, block, 0, st, a);
  else if (a.many.groups && call.bf16) hipLaunchKernelGGL(k_kv4_attend<true>, grid, block, 0, st, a);
  else if (a.many.groups) hipLaunchKernelGGL(k_kv4_attend<false>, grid, block, 0, st, a);
  else if (call.bf16) hipLaunchKernelGGL(k_kv4_attend_few<true>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(k_kv4_attend_few<false>, grid, block, 0, st, a);
  OI2_CHECK_LAUNCH();
  return OI2_OK;
}

}  // namespace oi2

extern "C" int oi2_kv4_attend(const oi2_paged* c, const oi2_page_plan* p, int32_t layer, int32_t dtype, int32_t n_tokens,
                              const oi2_heads* q, float scale, void* out, void* workspace, size_t workspace_bytes,
                              void* stream) {
  oi2::clear_error();
  return oi2::kv4_attend(c, p, layer, dtype, n_tokens, q, scale, out, workspace, workspace_bytes, false, stream);
}
