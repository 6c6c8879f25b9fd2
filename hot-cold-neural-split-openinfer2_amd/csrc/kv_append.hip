// k and v of a step into the pages of the 8-bit KV cache, q and k rotated on
// the way.
//
// A page's scale needs the largest of its new values before the first of them
// is coded.  Steps of up to eight tokens a row: a wave takes one (touched page,
// kv head), a pair of dims a lane, without a barrier; codes go out by bytes.
// Longer ones: a workgroup takes a touched page and one or several kv heads (the
// cosines and sines of its tokens stay in LDS for all of them); codes are
// put together in LDS in the cache's own order and leave 16 bytes at a time,
// v's, which run along positions there, byte by byte where the step fills a
// group of 16 positions in part.  Codes that the page already holds are touched
// only where its scale grows.  q has workgroups of its own behind them in the
// same launch.
//
// Bound by the bytes of k, v and q in prompts (7110 tokens of 32 + 8 + 8 heads,
// out of cache, 35.8 us, 4.4 TB/s; k and v alone 17, the chain of a page's
// heads); a step of single tokens by the chain of its loads, the reduction and
// the stores (16 rows 4.5 us, 40 rows of four tokens 8.7).  These are steps whose
// pages keep their scales.  Where every partly filled page's scales grow, 16
// rows take 11 us more, 40 rows of four tokens 12, prompts the same: most of a
// page's steps do not, as a scale that has seen some tokens is seldom passed.
#include "capi_util.h"
#include "kv_cache.h"
#include "rotary.h"

namespace oi2 {
namespace {

struct AppendArgs {
  const int32_t* work;        // the plan's
  int append_at;              // its list, in ints
  int n_kv, n_pages, n_tokens, page_groups;   // page_groups: workgroups of pages, before q's
  int heads_each;             // kv heads of a workgroup
  const uint16_t* src[2];     // k, v
  int64_t token_stride[2], head_stride[2];
  int rotate;
  uint8_t* pages;             // of the layer
  float* scales;
  RotaryArgs rope;            // q's tensors; its frequencies serve k too
};

__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = as_u32(v) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}

// The smallest e in [kExpMin, kExpMax] with amax <= 448 2^e = 1.75 2^(e + 8).
__device__ __forceinline__ int exponent_for(uint32_t amax_bits) {
  if (amax_bits == 0) return kExpMin;
  const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return min(max(e, kExpMin), kExpMax);
}

__device__ __forceinline__ float two_to(int e) { return as_f32((uint32_t)(e + 127) << 23); }

__device__ __forceinline__ int exponent_of(float scale) {
  return min(max((int)((as_u32(scale) >> 23) & 0xFF) - 127, kExpMin), kExpMax);
}

// The code of x (already over the scale), nearest, ties to even; NaN past 448.
__device__ __forceinline__ uint32_t code(float x) {
  if (!(fabsf(x) <= kCodeMax)) return 0x7Fu;
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false) & 0xFFu;
}

// The codes of a dword times f, a power of two below 1.
__device__ __forceinline__ uint32_t recode(uint32_t d, float f) {
  const f32x2 a = fp8x2_to_f32x2(d, false), b = fp8x2_to_f32x2(d, true);
  return code(a.x * f) | code(a.y * f) << 8 | code(b.x * f) << 16 | code(b.y * f) << 24;
}

// Byte offsets of 16-byte vectors in a half block: k's of token p, dims 16 c ..
__device__ __forceinline__ int k_vec(int p, int c) { return 2048 * (p / 4 % 4) + 256 * c + 16 * (4 * (p / 16) + p % 4); }
// ... and v's of dim d, positions 16 g ..
__device__ __forceinline__ int v_vec(int d, int g) { return 1024 * (d / 16) + 256 * g + 16 * (d % 16); }

// Dims of pair j of a head: what turns together, behind the rotated part dims
// 2 j and 2 j + 1.
struct PairDims {
  int a, b;
};
__device__ __forceinline__ PairDims pair_dims(int j, int rot, bool interleaved) {
  return 2 * j < rot && !interleaved ? PairDims{j, j + rot / 2} : PairDims{2 * j, 2 * j + 1};
}

__device__ __forceinline__ CosSin turn_of(const RotaryArgs& r, int j, int pos) {
  CosSin t = turn(r.freq[j], pos);
  t.c *= r.magnitude;
  t.s *= r.magnitude;
  return t;
}

// A page of one head: where it is, its scales, and which places are new.
struct PageHead {
  float2* scale;
  uint8_t* k;
  uint8_t* v;
  int held, upto;
};
__device__ __forceinline__ PageHead page_head(const AppendArgs& a, const AppendItem& it, int g) {
  const int64_t block = (int64_t)it.page * a.n_kv + g;
  uint8_t* k = a.pages + block * kBlock;
  return {reinterpret_cast<float2*>(a.scales) + block, k, k + kHalfBlock, it.held,
          min(it.upto, it.held + max(a.n_tokens - it.token0, 0))};
}

// Codes of the vectors [i0, i0 + n) of the page, of places that were held
// before, over a scale grown by 1 / f.
__device__ __forceinline__ void grow_k(uint8_t* kb, int i, int held, float f) {
  if (4 * (i >> 7) + 16 * ((i & 15) >> 2) + (i & 3) >= held) return;
  u32x4 x = *reinterpret_cast<const u32x4*>(kb + 16 * i);
#pragma unroll
  for (int q = 0; q < 4; ++q) x[q] = recode(x[q], f);
  *reinterpret_cast<u32x4*>(kb + 16 * i) = x;
}
__device__ __forceinline__ void grow_v(uint8_t* vb, int i, int held, float f) {
  const int lo = min(held - 16 * ((i >> 4) & 3), 16);
  if (lo <= 0) return;
  u32x4 x = *reinterpret_cast<const u32x4*>(vb + 16 * i);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int keep = min(max(lo - 4 * q, 0), 4);             // bytes of the dword that were held
    const uint32_t mask = keep == 4 ? 0xFFFFFFFFu : (1u << (8 * keep)) - 1;
    x[q] = (recode(x[q], f) & mask) | (x[q] & ~mask);
  }
  *reinterpret_cast<u32x4*>(vb + 16 * i) = x;
}

// ── few tokens ───────────────────────────────────────────────────────────────

constexpr int kWaveTokens = 8;

// One page and head by a wave: lane j the pair j of every new token.
template <bool BF16>
__device__ __forceinline__ void append_few(const AppendArgs& a, int task) {
  const int item = task / a.n_kv, g = task - item * a.n_kv, j = lane_id();
  const AppendItem it = reinterpret_cast<const AppendItem*>(a.work + a.append_at)[item];
  if (item >= a.work[kNAppend] || (unsigned)it.page >= (unsigned)a.n_pages) return;
  const PageHead ph = page_head(a, it, g);
  const int n = min(ph.upto - ph.held, kWaveTokens);
  if (n <= 0) return;
  const float2 before = *ph.scale;
  const RotaryArgs& r = a.rope;
  const PairDims dk = a.rotate ? pair_dims(j, r.rot, r.interleaved) : PairDims{2 * j, 2 * j + 1};
  const bool turns = a.rotate && 2 * j < r.rot;
  float k[kWaveTokens][2], v[kWaveTokens][2];
#pragma unroll
  for (int t = 0; t < kWaveTokens; ++t) {
    k[t][0] = k[t][1] = v[t][0] = v[t][1] = 0.0f;
    if (t < n) {
      const uint16_t* pk = a.src[0] + (int64_t)(it.token0 + t) * a.token_stride[0] + g * a.head_stride[0];
      const uint16_t* pv = a.src[1] + (int64_t)(it.token0 + t) * a.token_stride[1] + g * a.head_stride[1];
      k[t][0] = widen<BF16>(pk[dk.a]);
      k[t][1] = widen<BF16>(pk[dk.b]);
      v[t][0] = widen<BF16>(pv[2 * j]);
      v[t][1] = widen<BF16>(pv[2 * j + 1]);
    }
  }
  if (turns) {
#pragma unroll
    for (int t = 0; t < kWaveTokens; ++t)
      if (t < n) {
        const f32x2 o = turned(k[t][0], k[t][1], turn_of(r, j, r.positions[it.token0 + t]));
        k[t][0] = widen<BF16>(narrow<BF16>(o.x));
        k[t][1] = widen<BF16>(narrow<BF16>(o.y));
      }
  }
  uint32_t mk = 0, mv = 0;
#pragma unroll
  for (int t = 0; t < kWaveTokens; ++t) {
    mk = max(mk, max(finite_bits(k[t][0]), finite_bits(k[t][1])));
    mv = max(mv, max(finite_bits(v[t][0]), finite_bits(v[t][1])));
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    mk = max(mk, (uint32_t)__shfl_xor((int)mk, d));
    mv = max(mv, (uint32_t)__shfl_xor((int)mv, d));
  }
  int ek = exponent_for(mk), ev = exponent_for(mv);
  const int ek0 = exponent_of(before.x), ev0 = exponent_of(before.y);
  if (ph.held > 0) {
    ek = max(ek, ek0);
    ev = max(ev, ev0);
    if (ek > ek0)
      for (int i = j; i < 512; i += 64) grow_k(ph.k, i, ph.held, two_to(ek0 - ek));
    if (ev > ev0)
      for (int i = j; i < 512; i += 64) grow_v(ph.v, i, ph.held, two_to(ev0 - ev));
    // the byte stores below may share a vector with what another lane has just
    // written whole: behind it
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  const float ik = two_to(-ek), iv = two_to(-ev);
  bool nan = false;
#pragma unroll
  for (int t = 0; t < kWaveTokens; ++t)
    if (t < n) {
      const int p = ph.held + t;
      ph.k[k_vec(p, dk.a / 16) + dk.a % 16] = (uint8_t)code(k[t][0] * ik);
      ph.k[k_vec(p, dk.b / 16) + dk.b % 16] = (uint8_t)code(k[t][1] * ik);
      const uint32_t c0 = code(v[t][0] * iv), c1 = code(v[t][1] * iv);
      nan = nan || c0 == 0x7F || c1 == 0x7F;
      ph.v[v_vec(2 * j, p / 16) + p % 16] = (uint8_t)c0;
      ph.v[v_vec(2 * j + 1, p / 16) + p % 16] = (uint8_t)c1;
    }
  const bool flag = __any(nan) || (ph.held > 0 && as_u32(before.y) >> 31);
  if (j == 0) *ph.scale = float2{two_to(ek), flag ? -two_to(ev) : two_to(ev)};
}

template <bool BF16>
__device__ __forceinline__ float lower(uint32_t d) {
  return widen<BF16>((uint16_t)(d & 0xFFFFu));
}
template <bool BF16>
__device__ __forceinline__ float upper(uint32_t d) {
  return widen<BF16>((uint16_t)(d >> 16));
}

// Largest of two 16-bit values each; the magnitudes of fp16 and bf16 are in the
// order of their bits.
__device__ __forceinline__ uint32_t max_u16(uint32_t a, uint32_t b) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
template <bool BF16>
constexpr uint32_t kInfBits = BF16 ? 0x7F80u : 0x7C00u;

// The largest magnitude of 16 values in pairs, of the finite ones alone with FINITE.
template <bool BF16, bool FINITE>
__device__ __forceinline__ uint32_t top_of(const uint32_t (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    uint32_t d = x[e] & 0x7FFF7FFFu;
    if (FINITE) {
      if ((d & 0xFFFFu) >= kInfBits<BF16>) d &= 0xFFFF0000u;
      if (d >> 16 >= kInfBits<BF16>) d &= 0xFFFFu;
    }
    m = max_u16(m, d);
  }
  return max(m & 0xFFFFu, m >> 16);
}
__device__ __forceinline__ uint32_t wave_top(uint32_t top) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = max_u16(top, (uint32_t)__shfl_xor((int)top, d));
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)top);
}

// The codes of two pairs, whose values over the scale are 448 at most.
template <bool BF16>
__device__ __forceinline__ uint32_t codes4(uint32_t lo, uint32_t hi, float inv) {
  const int x = __builtin_amdgcn_cvt_pk_fp8_f32(lower<BF16>(lo) * inv, upper<BF16>(lo) * inv, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(lower<BF16>(hi) * inv, upper<BF16>(hi) * inv, x, true);
}

// ── many tokens ──────────────────────────────────────────────────────────────

// Vectors of the codes in LDS, in the cache's order but for a swizzle that
// spreads a wave's stores (8 tokens of 8 groups of dims) over the banks.
__device__ __forceinline__ int k_img(int off) { return off ^ ((off >> 8 & 3) << 6); }    // by dims 16 c: the token's a
__device__ __forceinline__ int v_img(int off) { return off ^ ((off >> 10 & 7) << 4); }   // by d / 16: d % 16

// A page of heads [g0, g1) by a workgroup.  Thread (u = tid % 8, p = tid / 8)
// takes the pairs 8 u .. of token p of the page; WIDE: rows of k and v at
// 16-byte addresses and whole groups of eight pairs to turn.
constexpr int kPageThreads = 512;
template <bool BF16, bool WIDE>
__device__ __forceinline__ void append_page(const AppendArgs& a, int item, int g0, int g1) {
  __shared__ __align__(16) uint8_t s_kc[kHalfBlock], s_vc[kHalfBlock];
  __shared__ uint32_t s_max[2][kPageThreads / 64], s_nan[2];
  const int tid = threadIdx.x, lane = lane_id(), wave = tid >> 6, u = tid & 7;
  const AppendItem it = reinterpret_cast<const AppendItem*>(a.work + a.append_at)[item];
  if (item >= a.work[kNAppend] || (unsigned)it.page >= (unsigned)a.n_pages) return;   // the whole workgroup
  const RotaryArgs& r = a.rope;
  const int held = it.held, upto = page_head(a, it, 0).upto;
  if (held >= upto) return;
  const int p = tid >> 3;
  const bool mine = p >= held && p < upto;
  const int64_t t = it.token0 + p - held;
  // cosines and sines of this thread's pairs, for every head; in LDS, but for
  // the last pair's (two workgroups share a CU's 160 KB), they leave the
  // registers to the next head's loads
  __shared__ __align__(16) CosSin s_cs[7][kPageThreads];
  CosSin last{};
  if (a.rotate && mine) {
    const int pos = r.positions[t];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (2 * (8 * u + e) < r.rot) (e < 7 ? s_cs[e][tid] : last) = turn_of(r, 8 * u + e, pos);
  }
  // WIDE: the first dims of this thread's pairs' two runs of eight
  const PairDims run = a.rotate && 16 * u < r.rot && !r.interleaved ? PairDims{8 * u, 8 * u + r.rot / 2} : PairDims{16 * u, 16 * u + 8};
  const bool halves = a.rotate && 16 * u < r.rot && !r.interleaved;   // else the runs are 16 neighbouring dims
  uint32_t raw[16];                        // k's and v's of the next head
  auto load = [&](int g) {
    const uint16_t* pk = a.src[0] + t * a.token_stride[0] + g * a.head_stride[0];
    const uint16_t* pv = a.src[1] + t * a.token_stride[1] + g * a.head_stride[1] + 16 * u;
    if constexpr (WIDE) {
      *reinterpret_cast<u32x4*>(raw) = *reinterpret_cast<const u32x4*>(pk + run.a);
      *reinterpret_cast<u32x4*>(raw + 4) = *reinterpret_cast<const u32x4*>(pk + run.b);
      *reinterpret_cast<u32x4*>(raw + 8) = *reinterpret_cast<const u32x4*>(pv);
      *reinterpret_cast<u32x4*>(raw + 12) = *reinterpret_cast<const u32x4*>(pv + 8);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const PairDims d = a.rotate ? pair_dims(8 * u + e, r.rot, r.interleaved) : PairDims{16 * u + 2 * e, 16 * u + 2 * e + 1};
        raw[e] = pk[d.a] | (uint32_t)pk[d.b] << 16;
        raw[8 + e] = pv[2 * e] | (uint32_t)pv[2 * e + 1] << 16;
      }
    }
  };
  if (mine) load(g0);
  for (int g = g0; g < g1; ++g) {
    const int par = (g - g0) & 1;          // the reduction's words: the last head's may still be read
    const PageHead ph = page_head(a, it, g);
    const float2 before = *ph.scale;
    uint32_t kx[8], vx[8];                 // k's pairs 8 u + e; v's dims 16 u + 2 e, + 1
#pragma unroll
    for (int e = 0; e < 8; ++e) kx[e] = vx[e] = 0;
    if (mine) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        vx[e] = raw[8 + e];
        if (WIDE && halves) kx[e] = __builtin_amdgcn_perm(raw[4 + e / 2], raw[e / 2], e % 2 ? 0x07060302u : 0x05040100u);
        else kx[e] = raw[e];
      }
      if (g + 1 < g1) load(g + 1);
      if (a.rotate)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (2 * (8 * u + e) < r.rot) {
            const f32x2 o = turned(lower<BF16>(kx[e]), upper<BF16>(kx[e]), e < 7 ? s_cs[e][tid] : last);
            kx[e] = narrow<BF16>(o.x) | (uint32_t)narrow<BF16>(o.y) << 16;
          }
    }

    // the largest finite values, k's in the low half
    uint32_t top = top_of<BF16, false>(kx) | top_of<BF16, false>(vx) << 16;
    top = wave_top(top);
    const bool odd = (top & 0xFFFFu) >= kInfBits<BF16> || top >> 16 >= kInfBits<BF16>;   // the wave's
    if (odd) top = wave_top(top_of<BF16, true>(kx) | top_of<BF16, true>(vx) << 16);
    if (lane == 0) s_max[par][wave] = top;
    if (tid == 0) s_nan[par] = 0;
    __syncthreads();                       // the last head's codes have left LDS too
#pragma unroll
    for (int w = 0; w < kPageThreads / 64; ++w) top = max_u16(top, s_max[par][w]);
    const uint32_t mk = as_u32(lower<BF16>(top)), mv = as_u32(upper<BF16>(top));
    int ek = exponent_for(mk), ev = exponent_for(mv);
    const int ek0 = exponent_of(before.x), ev0 = exponent_of(before.y);
    if (held > 0) {
      ek = max(ek, ek0);
      ev = max(ev, ev0);
    }

    // codes, in the cache's order
    const float ik = two_to(-ek), iv = two_to(-ev);
    const bool plain = !odd && ek < kExpMax && ev < kExpMax;   // nothing past the codes
    bool nan = false;
    if (mine) {
      uint32_t c[4], y[4];                 // codes of two pairs each
      if (plain) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          c[e] = codes4<BF16>(kx[2 * e], kx[2 * e + 1], ik);
          y[e] = codes4<BF16>(vx[2 * e], vx[2 * e + 1], iv);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          c[e] = y[e] = 0;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t kd = kx[2 * e + h], vd = vx[2 * e + h];
            const uint32_t v0 = code(lower<BF16>(vd) * iv), v1 = code(upper<BF16>(vd) * iv);
            c[e] |= (code(lower<BF16>(kd) * ik) | code(upper<BF16>(kd) * ik) << 8) << 16 * h;
            y[e] |= (v0 | v1 << 8) << 16 * h;
            nan = nan || v0 == 0x7F || v1 == 0x7F;
          }
        }
      }
      if constexpr (WIDE) {
        if (halves) {                      // every pair's first codes, then its second
          *reinterpret_cast<u32x2v*>(s_kc + k_img(k_vec(p, run.a / 16)) + run.a % 16) =
              u32x2v{__builtin_amdgcn_perm(c[1], c[0], 0x06040200u), __builtin_amdgcn_perm(c[3], c[2], 0x06040200u)};
          *reinterpret_cast<u32x2v*>(s_kc + k_img(k_vec(p, run.b / 16)) + run.b % 16) =
              u32x2v{__builtin_amdgcn_perm(c[1], c[0], 0x07050301u), __builtin_amdgcn_perm(c[3], c[2], 0x07050301u)};
        } else {
          *reinterpret_cast<u32x4*>(s_kc + k_img(k_vec(p, u))) = u32x4{c[0], c[1], c[2], c[3]};
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const PairDims d = a.rotate ? pair_dims(8 * u + e, r.rot, r.interleaved) : PairDims{16 * u + 2 * e, 16 * u + 2 * e + 1};
          s_kc[k_img(k_vec(p, d.a / 16)) + d.a % 16] = (uint8_t)(c[e / 2] >> 16 * (e % 2));
          s_kc[k_img(k_vec(p, d.b / 16)) + d.b % 16] = (uint8_t)(c[e / 2] >> 16 * (e % 2) + 8);
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e)
        s_vc[v_img(v_vec(16 * u + e, p / 16)) + p % 16] = (uint8_t)(y[e / 4] >> 8 * (e % 4));
    }
    if (nan) s_nan[par] = 1;
    __syncthreads();

    const bool more_k = held > 0 && ek > ek0, more_v = held > 0 && ev > ev0;
    {
      const int i = tid;                   // vector 16 i of the half block
      const int kp = 4 * (i >> 7) + 16 * ((i & 15) >> 2) + (i & 3);   // k: of token kp
      if (kp >= held && kp < upto) *reinterpret_cast<u32x4*>(ph.k + 16 * i) = *reinterpret_cast<const u32x4*>(s_kc + k_img(16 * i));
      else if (more_k) grow_k(ph.k, i, held, two_to(ek0 - ek));
      // v: positions 16 w .. 16 w + 15 of a dim
      const int w = (i >> 4) & 3, lo = max(held - 16 * w, 0), hi = min(upto - 16 * w, 16);
      const uint8_t* s = s_vc + v_img(16 * i);
      uint8_t* dst = ph.v + 16 * i;
      if (lo == 0 && hi == 16) {
        *reinterpret_cast<u32x4*>(dst) = *reinterpret_cast<const u32x4*>(s);
      } else {
        if (more_v) grow_v(ph.v, i, held, two_to(ev0 - ev));
        for (int b = lo; b < hi; ++b) dst[b] = s[b];
      }
    }
    if (tid == 0) {
      const bool flag = s_nan[par] || (held > 0 && as_u32(before.y) >> 31);
      *ph.scale = float2{two_to(ek), flag ? -two_to(ev) : two_to(ev)};
    }
  }
}

// WIDE and KWIDE: the forms for q's rows and for k's and v's.
template <bool BF16, bool WIDE>
__global__ __launch_bounds__(256) void k_kv_append_few(AppendArgs a) {
  const int b = blockIdx.x;
  if (b < a.page_groups) append_few<BF16>(a, 4 * b + (int)(threadIdx.x >> 6));
  else rotate_tokens<BF16, WIDE, 256>(a.rope, b - a.page_groups);
}

template <bool BF16, bool WIDE, bool KWIDE>
__global__ __launch_bounds__(kPageThreads, 4) void k_kv_append(AppendArgs a) {
  const int b = blockIdx.x;
  if (b < a.page_groups) {
    const int per = (a.n_kv + a.heads_each - 1) / a.heads_each, item = b / per, g = (b - item * per) * a.heads_each;
    append_page<BF16, KWIDE>(a, item, g, min(g + a.heads_each, a.n_kv));
  } else {
    rotate_tokens<BF16, WIDE, kPageThreads>(a.rope, b - a.page_groups);
  }
}

template <bool BF16, bool WIDE>
void launch_append(const AppendArgs& a, bool few, bool kwide, uint32_t groups, hipStream_t st) {
  const dim3 grid(groups), block(few ? 256 : kPageThreads);
  if (few) hipLaunchKernelGGL((k_kv_append_few<BF16, WIDE>), grid, block, 0, st, a);
  else if (kwide) hipLaunchKernelGGL((k_kv_append<BF16, WIDE, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((k_kv_append<BF16, WIDE, false>), grid, block, 0, st, a);
}

}  // namespace
}  // namespace oi2

using namespace oi2;

extern "C" int oi2_kv_append(const oi2_paged* c, const oi2_page_plan* p, int32_t layer, int32_t dtype, int32_t n_tokens,
                             const oi2_heads* k, const oi2_heads* v, const oi2_rotary* r, const oi2_heads* q,
                             void* q_out, void* stream) {
  clear_error();
  if (int rc = check_paged(c, layer, true)) return rc;
  if (int rc = check_plan(c, p)) return rc;
  const bool zero = dtype & OI2_ZERO_LEFT_OUT;
  dtype &= ~OI2_ZERO_LEFT_OUT;
  OI2_CHECK_ARG(dtype == OI2_DTYPE_F16 || dtype == OI2_DTYPE_BF16, "dtype %d: fp16 or bf16", dtype);
  OI2_CHECK_ARG(n_tokens >= 0 && n_tokens <= p->max_tokens, "%d tokens in a plan of %d", n_tokens, p->max_tokens);
  OI2_CHECK_ARG(k && v && k->heads == c->n_kv && v->heads == c->n_kv, "k and v need the cache's %d heads", c->n_kv);
  OI2_CHECK_ARG(!q || r, "q is rotated: it needs the rotary frequencies");
  if (r) {
    if (int rc = check_rotary(r)) return rc;
    OI2_CHECK_ARG(r->head_dim == kHeadD, "rotary head_dim %d: the cache's heads have %d", r->head_dim, kHeadD);
  }
  if (n_tokens == 0) return OI2_OK;
  OI2_CHECK_ARG(k->data && v->data && (uintptr_t)k->data % 2 == 0 && (uintptr_t)v->data % 2 == 0, "k and v must be non-null and 2-byte aligned");
  OI2_CHECK_ARG(!q || (q->heads >= 1 && q->heads <= 1 << 16 && q->data && q_out && (uintptr_t)q->data % 2 == 0 && (uintptr_t)q_out % 2 == 0),
                "q and its output must be non-null and 2-byte aligned, with heads");
  AppendArgs a{};
  const PlanLayout l = plan_layout(*c, p->max_tokens, p->max_new), now = plan_layout(*c, n_tokens, p->max_new);
  a.work = p->work;
  a.append_at = (int)l.append;
  a.n_kv = c->n_kv;
  a.n_pages = c->n_pages;
  a.n_tokens = n_tokens;
  bool kwide = !r || r->rotary_dim % 16 == 0;
  const oi2_heads* in[2] = {k, v};
  for (int w = 0; w < 2; ++w) {
    a.src[w] = (const uint16_t*)in[w]->data;
    a.token_stride[w] = in[w]->token_stride;
    a.head_stride[w] = in[w]->head_stride;
    if ((uintptr_t)in[w]->data % 16 || in[w]->token_stride % 8 || in[w]->head_stride % 8) kwide = false;
  }
  a.pages = c->pages + (size_t)layer * c->n_pages * c->n_kv * kBlock;
  a.scales = c->scales + (size_t)layer * c->n_pages * c->n_kv * 2;
  // A wave takes up to eight tokens of a page and head.  In longer steps a
  // workgroup takes up to four heads, and leaves 128 workgroups at least: 7061
  // tokens of 8 heads, inputs out of cache, with 1, 2, 4, 8 of them 42.2, 38.2,
  // 35.8 (4.4 TB/s), 36.3 us.
  const bool few = p->max_new <= kWaveTokens;
  const int64_t full = (int64_t)(n_tokens / kPage + 1) * c->n_kv;
  a.heads_each = full >= 512 ? 4 : full >= 256 ? 2 : 1;
  const int64_t pages = few ? ((int64_t)now.cap_append * c->n_kv + 3) / 4
                            : (int64_t)now.cap_append * ((c->n_kv + a.heads_each - 1) / a.heads_each);
  int64_t rows = 0;
  bool wide = true;
  a.rotate = r ? 1 : 0;
  if (r) {
    rotary_describe(a.rope, r, n_tokens, p->positions, zero);
    wide = rotary_fill(a.rope, q, q_out, nullptr, nullptr);
    rows = rotary_workgroups(a.rope);
  }
  OI2_CHECK_ARG(pages + rows < 1 << 23, "%d tokens are too many for one call", n_tokens);
  OI2_CHECK_ARG(!q || (!clashes(true, q_out, q->heads, q, n_tokens, kHeadD) && !clashes(false, q_out, q->heads, k, n_tokens, kHeadD) &&
                       !clashes(false, q_out, q->heads, v, n_tokens, kHeadD)),
                "q's output shares memory with q, and is not q, or with k or v");
  a.page_groups = (int)pages;
  hipStream_t st = (hipStream_t)stream;
  const uint32_t groups = (uint32_t)(pages + rows);
  const bool bf = dtype == OI2_DTYPE_BF16;
  if (bf && wide) launch_append<true, true>(a, few, kwide, groups, st);
  else if (bf) launch_append<true, false>(a, few, kwide, groups, st);
  else if (wide) launch_append<false, true>(a, few, kwide, groups, st);
  else launch_append<false, false>(a, few, kwide, groups, st);
  OI2_CHECK_LAUNCH();
  return OI2_OK;
}
