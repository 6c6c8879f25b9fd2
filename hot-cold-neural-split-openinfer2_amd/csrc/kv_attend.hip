// Attention of a step's query tokens over the paged 8-bit KV cache.
//
//   k_attend_few   up to 16 query rows (tokens times query heads of a kv head)
//                  over a range of a row's pages
//   k_attend_many  up to 128 query rows over a range of a row's pages
//   k_attend_join  joins the ranges where a row's pages were cut into parts
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
// p comes out times 2^kLift: its low fp16 part stays out of the subnormals.
constexpr float kLift = 10.0f;
// The running maximum follows the row's once that is 2^kSlack above it.
constexpr float kSlack = 5.0f;

struct AttendArgs {
  const int32_t* work;        // the plan's
  int items_at, merge_at;     // its lists of this kernel, in ints
  const int32_t* table;
  const uint8_t* pages;       // of the layer
  const float* scales;
  int n_q, n_kv, group_log, width, n_pages, n_tokens;
  const uint16_t* q;
  int64_t token_stride, head_stride;
  int wide;                   // 16-byte loads of q
  float scale;                // of the scores, times log2 e
  uint16_t* out;
  float* part_o;              // (slot, kv head, rows, 128)
  float* part_ml;             // (slot, kv head, rows, 2)
};

__device__ __forceinline__ h8 widen8(uint32_t d0, uint32_t d1) {
  const h4 lo = __builtin_shufflevector(fp8x2_to_f16x2(d0, false), fp8x2_to_f16x2(d0, true), 0, 1, 2, 3);
  const h4 hi = __builtin_shufflevector(fp8x2_to_f16x2(d1, false), fp8x2_to_f16x2(d1, true), 0, 1, 2, 3);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ __forceinline__ f32x4 mfma16(h8 a, h8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
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
// A row of bf16 values over its largest one's power of two is exact in fp16 but
// for what lies 2^-24 below that one.
template <bool BF16>
__device__ __forceinline__ h8 q_frag(const uint16_t (&v)[8], int e) {
  h8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    r[i] = BF16 ? (_Float16)ldexp2(bf16_bits_to_float(v[i]), -e) : __builtin_bit_cast(_Float16, v[i]);
  return r;
}

__device__ __forceinline__ float quad_max(float v) {   // over the lanes l, l ^ 16, l ^ 32, l ^ 48
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

constexpr int kFewWaves = 4, kFewThreads = 64 * kFewWaves;
constexpr int kORow = kHeadD + 4;          // floats of an output row in LDS, padded

// Lane (r = lane % 16, grp = lane / 16).  K's 16-row tile t of a page: row
// r = 4 a + i is position 16 a + 4 t + i; D's element i of lane (r, grp) is
// the score of query row r at position 16 grp + 4 t + i: in 4 tiles a lane has
// positions 16 grp .. 16 grp + 15 of its query row, which are the positions of
// the 16 bytes of V^T that it loads for each dim.
template <bool BF16>
__global__ __launch_bounds__(kFewThreads) void k_attend_few(AttendArgs a) {
  __shared__ __align__(16) float s_o[kFewWaves][kFewRows][kORow];
  __shared__ float s_m[kFewWaves][kFewRows], s_l[kFewWaves][kFewRows];
  __shared__ int s_nan[kHeadD];
  const int item = blockIdx.x / a.n_kv, g = blockIdx.x - item * a.n_kv;
  if (item >= a.work[kNFew]) return;
  const AttendItem it = reinterpret_cast<const AttendItem*>(a.work + a.items_at)[item];
  const int n_tok = min(it.n_tokens, a.n_tokens - it.token0);
  if (n_tok <= 0) return;
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
    qe = min(max((int)(as_u32(top) >> 23) - 127, -126), 126);
  }
  h8 qf[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) qf[i] = q_frag<BF16>(qv[i], qe);
  const float sc = BF16 ? ldexp2(a.scale, qe) : a.scale;
  const int lim = r < n_rows ? min(it.pos0 + tok + 1, it.kv_len) : 0;   // positions that this row sees
  const int all_see = min(it.pos0 + 1, it.kv_len);                      // ... and every row does

  const float ninf = -__builtin_inff();
  f32x4 o[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = ninf, l = 0.0f;

  const int32_t* table = a.table + (int64_t)it.row * a.width;
  for (int page = it.page0 + w; page < it.page1; page += kFewWaves) {
    int id = table[page];
    id = (unsigned)id < (unsigned)a.n_pages ? id : 0;
    id = __builtin_amdgcn_readfirstlane(id);
    const int64_t block = (int64_t)id * a.n_kv + g;
    const uint8_t* kb = a.pages + block * kBlock;
    u32x4 kr[8], vr[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) kr[n] = load16_nt(kb + 1024 * n + 16 * lane);
#pragma unroll
    for (int n = 0; n < 8; ++n) vr[n] = load16_nt(kb + kHalfBlock + 1024 * n + 16 * lane);
    const float ks = a.scales[2 * block], vs = a.scales[2 * block + 1];
    const float ev = (float)((int)((as_u32(vs) >> 23) & 0xFF) - 127);

    float s[16];
    const float ksc = sc * ks;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc = mfma16(widen8(kr[2 * t + (i >> 1)][2 * (i & 1)], kr[2 * t + (i >> 1)][2 * (i & 1) + 1]), qf[i], acc);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * t + i] = fmaf(acc[i], ksc, ev);
    }
    const int p0 = page * kPage + 16 * grp;
    if (page * kPage + kPage > all_see) {
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j] = p0 + j < lim ? s[j] : ninf;
    }
    float cm = s[0];
#pragma unroll
    for (int j = 1; j < 16; ++j) cm = fmaxf(cm, s[j]);
    cm = quad_max(cm);
    const bool up = cm > m + kSlack;
    if (__any(up)) {
      const float mn = up ? cm : m;
      const float alpha = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      l *= alpha;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[d] *= alpha;
      m = mn;
    }
    const float ref = (m == ninf ? 0.0f : m) - kLift;
    float p[16], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      p[j] = __builtin_amdgcn_exp2f(s[j] - ref);
      sum += p[j];
    }
    l = fmaf(sum, ldexp2(1.0f, -(int)ev), l);
    h8 ph[2], pl[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 uh, ul;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float e0 = p[8 * h + 2 * k], e1 = p[8 * h + 2 * k + 1];
        const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(e0, e1));
        uh[k] = hi;
        ul[k] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(e0 - half_lo(hi), e1 - half_hi(hi)));
      }
      ph[h] = __builtin_bit_cast(h8, uh);
      pl[h] = __builtin_bit_cast(h8, ul);
    }
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
        o[d] = mfma16(vf, ph[h], o[d]);
        o[d] = mfma16(vf, pl[h], o[d]);
      }
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
  // thread: query row tid / 16, dims 8 (tid % 16) ..
  const int row = tid >> 4, d0 = 8 * (tid & 15);
  if (row >= n_rows) return;
  float M = ninf, L = 0.0f;
#pragma unroll
  for (int k = 0; k < kFewWaves; ++k) M = fmaxf(M, s_m[k][row]);
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = 0.0f;
#pragma unroll
  for (int k = 0; k < kFewWaves; ++k) {
    const float mk = s_m[k][row], f = mk == ninf ? 0.0f : __builtin_amdgcn_exp2f(mk - M);
    L = fmaf(f, s_l[k][row], L);
    // 0 times a NaN sum, of a wave whose every score is NaN, stays NaN
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = fmaf(f, s_o[k][row][d0 + e], y[e]);
  }
  const int tk = row >> lg, head = (g << lg) + (row & ((1 << lg) - 1));
  const int sees = min(it.pos0 + tk + 1, it.kv_len);
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = s_nan[d0 + e] < sees ? __builtin_nanf("") : y[e];
  if (it.part >= 0) {
    const int64_t at = ((int64_t)it.part * a.n_kv + g) * kFewRows + row;
    f32x4* po = reinterpret_cast<f32x4*>(a.part_o + at * kHeadD + d0);
    po[0] = f32x4{y[0], y[1], y[2], y[3]};
    po[1] = f32x4{y[4], y[5], y[6], y[7]};
    if (d0 == 0) {
      a.part_ml[2 * at] = M;
      a.part_ml[2 * at + 1] = L;
    }
    return;
  }
  const float inv = it.kv_len > 0 ? 1.0f / L : 0.0f;     // a rejected row: zeros
  uint16_t z[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) z[e] = it.kv_len > 0 ? narrow<BF16>(y[e] * inv) : 0;
  *reinterpret_cast<u32x4*>(a.out + ((int64_t)(it.token0 + tk) * a.n_q + head) * kHeadD + d0) = *reinterpret_cast<u32x4*>(z);
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(h8 a, h8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

constexpr int kManyThreads = 256;

// A page in LDS, fp16: k's rows of one position (256 bytes, 16 chunks of 8
// dims), then v's rows of one dim (128 bytes, 8 chunks of 8 positions).  Chunks
// are swizzled within their rows so that staging stores and fragment reads
// touch all banks: k's by position p = 16 a + 4 t + i with i | (a ^ t) << 2,
// distinct for the 16 rows of a store (one t) and of a read (one a); v's by
// d / 2.  Every address is a lane's base with constant bits flipped and a
// constant added, which costs an instruction where a register each would spill.
constexpr int kPageLds = kPage * 256 + kHeadD * 128, kVLds = kPage * 256;
__device__ __forceinline__ int k_swz(int p) { return (p & 3) | ((((p >> 4) ^ (p >> 2)) & 3) << 2); }
__device__ __forceinline__ int k_lds(int p, int c) { return p * 256 + 16 * (c ^ k_swz(p)); }
__device__ __forceinline__ int v_lds(int d, int c) { return kVLds + d * 128 + 16 * (c ^ ((d >> 1) & 7)); }

// Four waves of 32 query rows.  A page is widened to fp16 once for all of them
// on its way into LDS (two buffers, one barrier a page; its codes come two pages
// ahead into registers).  Lane (r = lane % 32, h = lane / 32) has the scores of
// query row r: element j of tile T is position 32 T + 16 (j / 8) + 8 h + j % 8,
// because row 8 b + 4 h + i (+ 16 s) of the product is given position
// 8 h + 4 b + i (+ 16 s); eight consecutive ones are a fragment of P^T and a
// 16-byte chunk of a dim's row of V^T.
template <bool BF16>
__global__ __launch_bounds__(kManyThreads, 2) void k_attend_many(AttendArgs a) {
  __shared__ __align__(1024) uint8_t s_page[2 * kPageLds];
  __shared__ int s_nan[kHeadD];
  const int item = blockIdx.x / a.n_kv, g = blockIdx.x - item * a.n_kv;
  if (item >= a.work[kNMany]) return;
  const AttendItem it = reinterpret_cast<const AttendItem*>(a.work + a.items_at)[item];
  const int n_tok = min(it.n_tokens, a.n_tokens - it.token0);
  if (n_tok <= 0) return;
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
      qe = min(max((int)(as_u32(top) >> 23) - 127, -126), 126);
    }
#pragma unroll
    for (int st = 0; st < 8; ++st) qf[st] = q_frag<BF16>(qv[st], qe);
  }
  const float sc = BF16 ? ldexp2(a.scale, qe) : a.scale;
  const int lim = row < n_rows ? min(it.pos0 + tok + 1, it.kv_len) : 0;   // positions that this row sees
  // ... that every row of the wave sees, and that some row of it does
  const int all_see = min(it.pos0 + (32 * w >> lg) + 1, it.kv_len);
  const int some_see = 32 * w < n_rows ? min(it.pos0 + (min(32 * w + 31, n_rows - 1) >> lg) + 1, it.kv_len) : 0;

  const float ninf = -__builtin_inff();
  f32x16 o[4];
#pragma unroll
  for (int d = 0; d < 4; ++d) o[d] = f32x16{};
  float m = ninf, l = 0.0f;

  const int32_t* table = a.table + (int64_t)it.row * a.width;
  auto block_of = [&](int page) {
    int id = table[min(page, it.page1 - 1)];
    id = (unsigned)id < (unsigned)a.n_pages ? id : 0;
    return (int64_t)__builtin_amdgcn_readfirstlane(id) * a.n_kv + g;
  };
  u32x4 kr[2], vr[2];
  auto load = [&](int64_t block) {
    const uint8_t* b = a.pages + block * kBlock;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      kr[n] = load16(b + 16 * tid + 4096 * n);
      vr[n] = load16(b + kHalfBlock + 16 * tid + 4096 * n);
    }
  };
  // lane bases: stores of vectors tid (and tid + 256), reads
  const int st_p = 16 * ((tid & 15) >> 2) + 4 * (tid >> 7) + (tid & 3), st_d = 16 * (tid >> 6) + (tid & 15);
  const int k_st = k_lds(st_p, 2 * ((tid >> 4) & 7)), v_st = v_lds(st_d, 2 * ((tid >> 4) & 3));
  const int k_rd = k_lds((r & 19) | ((r >> 3) & 1) << 2 | ((r >> 2) & 1) << 3, h), v_rd = v_lds(r, h);
  auto store = [&](int page, int at, float v_scale) {
    int ka = at + k_st, va = at + v_st;
    asm volatile("" : "+v"(ka), "+v"(va));
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      // 8 positions (2 t) further: the swizzle's bit 3 flips
      uint8_t* k0 = s_page + (ka ^ (128 * n)) + 2048 * n;
      uint8_t* k1 = s_page + (ka ^ (128 * n) ^ 16) + 2048 * n;
      *reinterpret_cast<h8*>(k0) = widen8(kr[n][0], kr[n][1]);
      *reinterpret_cast<h8*>(k1) = widen8(kr[n][2], kr[n][3]);
      u32x4 x = vr[n];
      if (page * kPage + kPage > it.kv_len) {   // behind the row's end: whatever the page held before
        const int tail = it.kv_len - page * kPage - 16 * ((tid >> 4) & 3);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = first_bytes(x[k], tail - 4 * k);
      }
      if (v_scale < 0.0f) take_nans(x, page * kPage + 16 * ((tid >> 4) & 3), &s_nan[st_d + 64 * n]);
      *reinterpret_cast<h8*>(s_page + va + 8192 * n) = widen8(x[0], x[1]);           // 64 dims further
      *reinterpret_cast<h8*>(s_page + (va ^ 16) + 8192 * n) = widen8(x[2], x[3]);
    }
  };
  auto scale_of = [&](int64_t block) { return *reinterpret_cast<const float2*>(a.scales + 2 * block); };

  auto compute = [&](int page, int at, float2 scale) {
    int ka = at + k_rd, va = at + v_rd;
    asm volatile("" : "+v"(ka), "+v"(va));
    const float ev = (float)((int)((as_u32(scale.y) >> 23) & 0xFF) - 127), ksc = sc * scale.x;
    f32x16 s[2] = {};
#pragma unroll
    for (int st = 0; st < 8; ++st)
#pragma unroll
      for (int T = 0; T < 2; ++T)
        s[T] = mfma32(*reinterpret_cast<const h8*>(s_page + (ka ^ (32 * st) ^ (128 * T)) + 8192 * T), qf[st], s[T]);   // a 2 further: bit 3
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int T = 0; T < 2; ++T)
#pragma unroll
      for (int j = 0; j < 16; ++j) s[T][j] = fmaf(s[T][j], ksc, ev);
    const int p0 = page * kPage + 8 * h;
    if (page * kPage + kPage > all_see) {
#pragma unroll
      for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[T][j] = p0 + 32 * T + 16 * (j >> 3) + (j & 7) < lim ? s[T][j] : ninf;
    }
    float cm = s[0][0];
#pragma unroll
    for (int T = 0; T < 2; ++T)
#pragma unroll
      for (int j = 0; j < 16; ++j) cm = fmaxf(cm, s[T][j]);
    cm = fmaxf(cm, __shfl_xor(cm, 32));
    const bool up = cm > m + kSlack;
    if (__any(up)) {
      const float mn = up ? cm : m;
      const float alpha = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      l *= alpha;
#pragma unroll
      for (int d = 0; d < 4; ++d) o[d] *= alpha;
      m = mn;
    }
    const float ref = (m == ninf ? 0.0f : m) - kLift;
    float sum = 0.0f;
    h8 ph, pl;
    // fragment f of the probabilities: positions 16 f + 8 h ..
    auto probabilities = [&](int f) {
      u32x4 uh, ul;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = 8 * (f & 1) + 2 * k;
        const float e0 = __builtin_amdgcn_exp2f(s[f >> 1][j] - ref), e1 = __builtin_amdgcn_exp2f(s[f >> 1][j + 1] - ref);
        sum += e0;
        sum += e1;
        const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(e0, e1));
        uh[k] = hi;
        ul[k] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(fmaf(half_lo(hi), -1.0f, e0), fmaf(half_hi(hi), -1.0f, e1)));
      }
      ph = __builtin_bit_cast(h8, uh);
      pl = __builtin_bit_cast(h8, ul);
    };
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      probabilities(f);
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const h8 vf = *reinterpret_cast<const h8*>(s_page + (va ^ (32 * f)) + 4096 * d);
        o[d] = mfma32(vf, ph, o[d]);
        o[d] = mfma32(vf, pl, o[d]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    l = fmaf(sum, ldexp2(1.0f, -(int)ev), l);
  };

  if (it.page0 < it.page1) {
    int64_t b0 = block_of(it.page0), b1 = block_of(it.page0 + 1);
    load(b0);
    float2 sc0 = scale_of(b0), sc1 = scale_of(b1);
    store(it.page0, 0, sc0.y);
    load(b1);
    for (int page = it.page0; page < it.page1; ++page) {
      const int cur = (page - it.page0) & 1;
      const int64_t b2 = block_of(page + 2);
      __syncthreads();                 // the page is in LDS; its other buffer is read
      if (page + 1 < it.page1) store(page + 1, (cur ^ 1) * kPageLds, sc1.y);
      load(b2);
      const float2 sc2 = scale_of(b2);
      if (page * kPage < some_see) compute(page, cur * kPageLds, sc0);
      sc0 = sc1;
      sc1 = sc2;
    }
  }

  l += __shfl_xor(l, 32);
  if (row >= n_rows) return;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j)
      o[d][j] = s_nan[32 * d + 8 * (j >> 2) + 4 * h + (j & 3)] < lim ? __builtin_nanf("") : o[d][j];
  if (it.part >= 0) {
    const int64_t at = ((int64_t)it.part * a.n_kv + g) * kManyRows + row;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(a.part_o + at * kHeadD + 32 * d + 8 * q + 4 * h) =
            f32x4{o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
    if (h == 0) {
      a.part_ml[2 * at] = m;
      a.part_ml[2 * at + 1] = l;
    }
    return;
  }
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

// Joins the parts of one tile of query tokens and kv head: a row of 128 dims by
// 32 threads.
template <bool BF16, int ROWS>
__global__ __launch_bounds__(256) void k_attend_join(AttendArgs a, int count) {
  const int item = blockIdx.x / a.n_kv, g = blockIdx.x - item * a.n_kv;
  if (item >= a.work[count]) return;
  const MergeItem it = reinterpret_cast<const MergeItem*>(a.work + a.merge_at)[item];
  const int n_tok = min(it.n_tokens, a.n_tokens - it.token0), lg = a.group_log;
  const int n_rows = max(n_tok, 0) << lg;
  const float ninf = -__builtin_inff();
  const int64_t stride = (int64_t)a.n_kv * ROWS;
  for (int row = threadIdx.x >> 5; row < n_rows; row += 8) {
    const int d0 = 4 * (threadIdx.x & 31);
    const int64_t at = ((int64_t)it.part0 * a.n_kv + g) * ROWS + row;
    float M = ninf;
    for (int k = 0; k < it.n_parts; ++k) M = fmaxf(M, a.part_ml[2 * (at + k * stride)]);
    float L = 0.0f;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < it.n_parts; ++k) {
      const float mk = a.part_ml[2 * (at + k * stride)], f = mk == ninf ? 0.0f : __builtin_amdgcn_exp2f(mk - M);
      L = fmaf(f, a.part_ml[2 * (at + k * stride) + 1], L);
      const f32x4 x = *reinterpret_cast<const f32x4*>(a.part_o + (at + k * stride) * kHeadD + d0);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = fmaf(f, x[e], y[e]);
    }
    const float inv = 1.0f / L;
    uint16_t z[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = narrow<BF16>(y[e] * inv);
    const int64_t to = ((int64_t)(it.token0 + (row >> lg)) * a.n_q + (g << lg) + (row & ((1 << lg) - 1))) * kHeadD + d0;
    *reinterpret_cast<u32x2v*>(a.out + to) = *reinterpret_cast<u32x2v*>(z);
  }
}

// The workspace: the partial sums of either kernel's parts, out and then m, l.
size_t few_floats(const PlanLayout& l, int n_kv) { return (size_t)l.cap_parts_few * n_kv * kFewRows * (kHeadD + 2); }
size_t many_floats(const PlanLayout& l, int n_kv) { return (size_t)l.cap_parts_many * n_kv * kManyRows * (kHeadD + 2); }

}  // namespace
}  // namespace oi2

using namespace oi2;

extern "C" {

size_t oi2_kv_attend_workspace_bytes(const oi2_paged* c, int32_t max_tokens, int32_t max_new) {
  if (!oi2_page_plan_bytes(c, max_tokens, max_new)) return 0;
  const PlanLayout l = plan_layout(*c, max_tokens, max_new);
  const size_t n = (few_floats(l, c->n_kv) + many_floats(l, c->n_kv)) * 4;
  return n ? n : 16;
}

int oi2_kv_attend(const oi2_paged* c, const oi2_page_plan* p, int32_t layer, int32_t dtype, int32_t n_tokens,
                  const oi2_heads* q, float scale, void* out, void* workspace, size_t workspace_bytes,
                  void* stream) {
  clear_error();
  if (int rc = check_paged(c, layer, true)) return rc;
  if (int rc = check_plan(c, p)) return rc;
  OI2_CHECK_ARG(dtype == OI2_DTYPE_F16 || dtype == OI2_DTYPE_BF16, "dtype %d: fp16 or bf16", dtype);
  OI2_CHECK_ARG(n_tokens >= 0 && n_tokens <= p->max_tokens, "%d tokens in a plan of %d", n_tokens, p->max_tokens);
  OI2_CHECK_ARG(q && q->heads == c->n_q, "q needs the cache's %d query heads", c->n_q);
  OI2_CHECK_ARG(scale == scale && scale - scale == 0.0f, "the scale of the scores is not finite");
  if (n_tokens == 0) return OI2_OK;
  OI2_CHECK_ARG(q->data && (uintptr_t)q->data % 2 == 0, "q must be non-null and 2-byte aligned");
  OI2_CHECK_ARG(out && (uintptr_t)out % 16 == 0, "out must be non-null and 16-byte aligned");
  const PlanLayout l = plan_layout(*c, p->max_tokens, p->max_new), now = plan_layout(*c, n_tokens, p->max_new);
  const size_t need = (few_floats(l, c->n_kv) + many_floats(l, c->n_kv)) * 4;
  OI2_CHECK_ARG(!need || (workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need),
                "workspace of %zu bytes, %zu needed, 16-byte aligned", workspace_bytes, need);
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
  OI2_CHECK_ARG(few < 1 << 23 && many < 1 << 23, "%d tokens are too many for one call", n_tokens);
  AttendArgs b = a;
  b.items_at = (int)l.many;
  b.merge_at = (int)l.merge_many;
  b.part_o = (float*)workspace + few_floats(l, c->n_kv);
  b.part_ml = b.part_o + (size_t)l.cap_parts_many * c->n_kv * kManyRows * kHeadD;
  a.items_at = (int)l.few;
  a.merge_at = (int)l.merge_few;
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o + (size_t)l.cap_parts_few * c->n_kv * kFewRows * kHeadD;
  if (many) {
    if (bf) hipLaunchKernelGGL(k_attend_many<true>, dim3((uint32_t)many), dim3(kManyThreads), 0, st, b);
    else hipLaunchKernelGGL(k_attend_many<false>, dim3((uint32_t)many), dim3(kManyThreads), 0, st, b);
    OI2_CHECK_LAUNCH();
  }
  if (bf) hipLaunchKernelGGL(k_attend_few<true>, dim3((uint32_t)few), dim3(kFewThreads), 0, st, a);
  else hipLaunchKernelGGL(k_attend_few<false>, dim3((uint32_t)few), dim3(kFewThreads), 0, st, a);
  OI2_CHECK_LAUNCH();
  if (const uint32_t n = (uint32_t)now.cap_merge_few * c->n_kv) {
    if (bf) hipLaunchKernelGGL((k_attend_join<true, kFewRows>), dim3(n), dim3(256), 0, st, a, kNMergeFew);
    else hipLaunchKernelGGL((k_attend_join<false, kFewRows>), dim3(n), dim3(256), 0, st, a, kNMergeFew);
    OI2_CHECK_LAUNCH();
  }
  if (const uint32_t n = (uint32_t)now.cap_merge_many * c->n_kv) {
    if (bf) hipLaunchKernelGGL((k_attend_join<true, kManyRows>), dim3(n), dim3(256), 0, st, b, kNMergeMany);
    else hipLaunchKernelGGL((k_attend_join<false, kManyRows>), dim3(n), dim3(256), 0, st, b, kNMergeMany);
    OI2_CHECK_LAUNCH();
  }
  return OI2_OK;
}

}  // extern "C"
