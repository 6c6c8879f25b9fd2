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
#include "attend.h"

namespace oi2 {
namespace {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ h8 widen8(uint32_t d0, uint32_t d1) {
  const h4 lo = __builtin_shufflevector(fp8x2_to_f16x2(d0, false), fp8x2_to_f16x2(d0, true), 0, 1, 2, 3);
  const h4 hi = __builtin_shufflevector(fp8x2_to_f16x2(d1, false), fp8x2_to_f16x2(d1, true), 0, 1, 2, 3);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Bytes [0, n) of a dword's four kept, the rest zero.
__device__ __forceinline__ uint32_t first_bytes(uint32_t d, int n) {
  return n >= 4 ? d : n <= 0 ? 0u : d & ((1u << (8 * n)) - 1);
}

// Pages that hold a NaN are marked; its code becomes 0 and its position is noted.
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

// ── few rows ─────────────────────────────────────────────────────────────────

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
__device__ __forceinline__ bool attend_few(const AttendArgs& a, const Found& found, uint8_t* smem) {
  const FewLds<1> lds(smem);
  FewTile<1> t;
  few_open<BF16>(a, found, lds, t, [](int grp, int i) { return 16 * (4 * (i >> 1) + grp) + 8 * (i & 1); });
  const ItemHead& it = t.it;
  const int g = t.g, w = t.w, lane = t.lane, r = t.r, grp = t.grp, lim = t.lim[0], all_see = t.all_see;
  const h8 (&qf)[4] = t.q[0];
  const float sc = t.sc[0];

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
    const int64_t block = (int64_t)scalar_load(t.full->ids + w) * a.n_kv + g;
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
    for (int k = 0; k < 4; ++k) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc = mfma16(widen8(kr[2 * k + (i >> 1)][2 * (i & 1)], kr[2 * k + (i >> 1)][2 * (i & 1) + 1]), qf[i], acc);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * k + i] = acc[i];
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
      for (int n = 0; n < 8; ++n) take_nans(vr[n], p0, &lds.nan[16 * n + r]);
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
  for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4*>(&lds.o[w][r][16 * d + 4 * grp]) = o[d];
  if (grp == 0) {
    lds.m[w][r] = m;
    lds.l[w][r] = l;
  }
  return few_close<BF16>(a, t, lds);
}

// ── many rows ────────────────────────────────────────────────────────────────

// What bounds many rows: the products, a third of them for the probabilities' low
// parts; the matrix cores are busy 60 % of the time, and two waves a SIMD fill the
// rest by chance.  A call of 5000 tokens 287 us in fp16 (714 TFLOP/s of the
// formula's operations, half as much again with the low parts'), 6 chunks beside 3
// short rows 97, where a low part by a subtraction and a conversion took 291 and
// 98 (boxes differ: 288 to 306, in bf16 285 to 302).  With one fp16 part of a
// probability, of 249 us before k's conflicts went, the exponentials alone made
// 38, staging 35, the fragments' reads 55, the products 68, and there was tried
// without gain: fragments read three steps ahead; raised priority around
// the products; one wave a SIMD with 64 rows and the next page's scores between
// this one's exponentials, whose accumulators in AGPRs cost more copies than the
// shared fragments save (326 us in bf16); the same with 32 rows, which spilled
// (272); eight waves over 256 rows, four of them half a page behind, products
// beside the others' softmax: that hides the softmax, but leaves the 10 us of a
// workgroup's start and end bare, with one workgroup a CU (251).
struct Pages8 {
  const AttendArgs& a;
  const ItemHead& it;
  int tid, st_d, *nan;
  int k_st, v_st;                      // lane bases of the staging stores
  u32x4 kr[2], vr[2];                  // codes on their way into LDS: vectors tid and tid + 256

  __device__ __forceinline__ Pages8(const AttendArgs& args, const ItemHead& item, int thread, int* s_nan)
      : a(args), it(item), tid(thread), nan(s_nan) {
    const int st_p = 16 * ((tid & 15) >> 2) + 4 * (tid >> 7) + (tid & 3);
    st_d = 16 * (tid >> 6) + (tid & 15);
    k_st = k_lds(st_p, 2 * ((tid >> 4) & 7));
    v_st = v_lds(st_d, 2 * ((tid >> 4) & 3));
  }
  __device__ __forceinline__ void load(int64_t block) {
    const uint8_t* b = a.pages + block * kBlock + 16 * tid;
#pragma unroll
    for (int n = 0; n < 2; ++n) kr[n] = load16(b + 4096 * n);
#pragma unroll
    for (int n = 0; n < 2; ++n) vr[n] = load16(b + kHalfBlock + 4096 * n);
  }
  __device__ __forceinline__ float2 scale_of(int64_t block) const {
    return scalar_load(reinterpret_cast<const float2*>(a.scales) + block);
  }
  __device__ __forceinline__ void fix(int page, float v_scale) {
    const int tail = it.kv_len - page * kPage - 16 * ((tid >> 4) & 3);
    if (page * kPage + kPage > it.kv_len) {   // behind the row's end: whatever the page held before
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k) vr[n][k] = first_bytes(vr[n][k], tail - 4 * k);
    }
    if (v_scale < 0.0f) {
#pragma unroll
      for (int n = 0; n < 2; ++n) take_nans(vr[n], page * kPage + 16 * ((tid >> 4) & 3), &nan[st_d + 64 * n]);
    }
  }
  __device__ __forceinline__ void put_k(uint8_t* s_page, int ka, int q) const {    // 8 positions (2 t) further: the swizzle's bit 3 flips
    const int n = q >> 1, e = q & 1;
    *reinterpret_cast<h8*>(s_page + (ka ^ (128 * n) ^ (16 * e)) + 2048 * n) = widen8(kr[n][2 * e], kr[n][2 * e + 1]);
  }
  __device__ __forceinline__ void put_v(uint8_t* s_page, int va, int q) const {    // 64 dims further
    const int n = q >> 1, e = q & 1;
    *reinterpret_cast<h8*>(s_page + (va ^ (16 * e)) + 8192 * n) = widen8(vr[n][2 * e], vr[n][2 * e + 1]);
  }
  // a row of V^T is that dim: element j of o[d] in half h is row 32 d + 8 (j / 4) + j % 4, + 4 h
  static __device__ __forceinline__ int dim(int row, int h) { return row + 4 * h; }
  template <class F>
  static __device__ __forceinline__ void each_four(const f32x16 (&o)[4], int h, F f) {   // of dims 4 chunk ..
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) f(8 * d + 2 * q + h, f32x4{o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]});
  }
};

// Steps whose rows all have few query rows, and steps with rows of either kind:
// the long tiles first, the others fill the chip behind and beside them.
template <bool BF16>
__global__ __launch_bounds__(kThreads, 2) void k_attend_few(AttendArgs a) {
  __shared__ __align__(16) uint8_t smem[kFewLds<1>];
  const int b = blockIdx.x;
  Found f;
  if (b >= a.few.groups) zero_rest(a, b - a.few.groups);
  else if (few_find(a, b, f) && attend_few<BF16>(a, f, smem)) join_parts<BF16, kFewRows>(a, a.few, f, smem);
}

template <bool BF16>
__global__ __launch_bounds__(kThreads, 2) void k_attend(AttendArgs a) {
  static_assert(kManyLds >= kFewLds<1> && kThreads == 64 * kFewWaves, "one workgroup for either");
  __shared__ __align__(1024) uint8_t smem[kManyLds];
  const int b = blockIdx.x;
  Found f;
  if (b < a.many.groups) {
    if (many_find(a, b, f) && attend_many<BF16, Pages8>(a, f, smem)) join_parts<BF16, kManyRows>(a, a.many, f, smem);
  } else if (b - a.many.groups >= a.few.groups) {
    zero_rest(a, b - a.many.groups - a.few.groups);
  } else if (few_find(a, b - a.many.groups, f) && attend_few<BF16>(a, f, smem)) {
    join_parts<BF16, kFewRows>(a, a.few, f, smem);
  }
}

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
  hipStream_t st = (hipStream_t)stream;
  AttendCall call;
  if (int rc = attend_call(call, c, p, dtype, n_tokens, q, scale, out, workspace, workspace_bytes, st)) return rc;
  if (!call.groups) return OI2_OK;
  AttendArgs& a = call.a;
  a.pages = c->pages + (size_t)layer * c->n_pages * c->n_kv * kBlock;
  a.scales = c->scales + (size_t)layer * c->n_pages * c->n_kv * 2;
  const dim3 grid(call.groups), block(kThreads);
  if (a.many.groups && call.bf16) hipLaunchKernelGGL(k_attend<true>, grid, block, 0, st, a);
  else if (a.many.groups) hipLaunchKernelGGL(k_attend<false>, grid, block, 0, st, a);
  else if (call.bf16) hipLaunchKernelGGL(k_attend_few<true>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(k_attend_few<false>, grid, block, 0, st, a);
  OI2_CHECK_LAUNCH();
  return OI2_OK;
}

}  // extern "C"
