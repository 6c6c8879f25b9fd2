// k and v of a step into the pages of the 8-bit KV cache, q and k rotated on
// the way.
//
// A workgroup takes one (touched page, kv head): the page's scale needs the
// largest of its new values before the first of them is coded.  k goes through
// LDS (the pairs that turn together lie in different threads), its codes and
// v's are put together in LDS in the cache's own order and leave 16 bytes at a
// time; v's codes run along positions there, so a group of 16 positions that
// the step fills in part is written byte by byte.  Codes that the page already
// holds are touched only where its scale grows.  q has workgroups of its own
// behind them in the same launch.
//
// Bound by the bytes of k, v and q in prompts; a step of single tokens by the
// chain of its loads, the reduction and the stores.
#include "capi_util.h"
#include "kv_cache.h"
#include "rotary.h"

namespace oi2 {
namespace {

struct AppendArgs {
  const int32_t* work;        // the plan's
  int append_at;              // its list, in ints
  int n_kv, n_pages, n_tokens, page_groups;   // page_groups: workgroups of pages, before q's
  const uint16_t* src[2];     // k, v
  int64_t token_stride[2], head_stride[2];
  int wide;                   // 16-byte loads of k and v
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

constexpr int kRow = kHeadD + 8;           // fp16 row of k in LDS, padded

template <bool BF16>
__device__ void append_page(const AppendArgs& a, int item, int g) {
  __shared__ __align__(16) uint16_t s_k[kPage * kRow];
  __shared__ __align__(16) uint8_t s_kc[kHalfBlock], s_vc[kHalfBlock];
  __shared__ uint32_t s_max[2][4];
  __shared__ uint32_t s_nan;
  const int tid = threadIdx.x, lane = lane_id(), wave = tid >> 6;
  const AppendItem it = reinterpret_cast<const AppendItem*>(a.work + a.append_at)[item];
  const int held = it.held, upto = min(it.upto, it.held + max(a.n_tokens - it.token0, 0));
  if (held >= upto || (unsigned)it.page >= (unsigned)a.n_pages) return;   // the whole workgroup
  float2* scale = reinterpret_cast<float2*>(a.scales) + (int64_t)it.page * a.n_kv + g;
  uint8_t* kb = a.pages + ((int64_t)it.page * a.n_kv + g) * kBlock;
  uint8_t* vb = kb + kHalfBlock;
  const float2 before = *scale;

  // piece n of this thread: token 16 n + tid / 16, dims 8 (tid % 16) ..
  const int pt = tid >> 4, d0 = 8 * (tid & 15);
  uint16_t kx[4][8], vx[4][8];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int p = 16 * n + pt;
    *reinterpret_cast<u32x4*>(kx[n]) = u32x4{0, 0, 0, 0};
    *reinterpret_cast<u32x4*>(vx[n]) = u32x4{0, 0, 0, 0};
    if (p >= held && p < upto) {
      const int64_t t = it.token0 + p - held;
      const uint16_t* pk = a.src[0] + t * a.token_stride[0] + g * a.head_stride[0] + d0;
      const uint16_t* pv = a.src[1] + t * a.token_stride[1] + g * a.head_stride[1] + d0;
      if (a.wide) {
        *reinterpret_cast<u32x4*>(kx[n]) = *reinterpret_cast<const u32x4*>(pk);
        *reinterpret_cast<u32x4*>(vx[n]) = *reinterpret_cast<const u32x4*>(pv);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          kx[n][e] = pk[e];
          vx[n][e] = pv[e];
        }
      }
    }
  }
  if (a.rotate) {
#pragma unroll
    for (int n = 0; n < 4; ++n) *reinterpret_cast<u32x4*>(s_k + (16 * n + pt) * kRow + d0) = *reinterpret_cast<u32x4*>(kx[n]);
    __syncthreads();
    const RotaryArgs& r = a.rope;
    const int half = r.rot / 2;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int p = 16 * n + pt;
      if (p < held || p >= upto) continue;
      const int pos = r.positions[it.token0 + p - held];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = d0 + e;
        if (d >= r.rot) continue;
        // the pair's number and its other dim; `second`: this one is its second
        const int j = r.interleaved ? d >> 1 : (d < half ? d : d - half);
        const int o = r.interleaved ? d ^ 1 : (d < half ? d + half : d - half);
        const bool second = r.interleaved ? d & 1 : d >= half;
        CosSin cs = turn(r.freq[j], pos);
        cs.c *= r.magnitude;
        cs.s *= r.magnitude;
        const float mine = widen<BF16>(kx[n][e]), other = widen<BF16>(s_k[p * kRow + o]);
        const f32x2 t = second ? turned(other, mine, cs) : turned(mine, other, cs);
        kx[n][e] = narrow<BF16>(second ? t.y : t.x);
      }
    }
  }

  // the largest finite values
  uint32_t mk = 0, mv = 0;
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      mk = max(mk, finite_bits(widen<BF16>(kx[n][e])));
      mv = max(mv, finite_bits(widen<BF16>(vx[n][e])));
    }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    mk = max(mk, (uint32_t)__shfl_xor((int)mk, d));
    mv = max(mv, (uint32_t)__shfl_xor((int)mv, d));
  }
  if (lane == 0) {
    s_max[0][wave] = mk;
    s_max[1][wave] = mv;
  }
  if (tid == 0) s_nan = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    mk = max(mk, s_max[0][w]);
    mv = max(mv, s_max[1][w]);
  }
  int ek = exponent_for(mk), ev = exponent_for(mv);
  const int ek0 = exponent_of(before.x), ev0 = exponent_of(before.y);
  if (held > 0) {
    ek = max(ek, ek0);
    ev = max(ev, ev0);
  }

  // codes, in the cache's order
  const float ik = two_to(-ek), iv = two_to(-ev);
  bool nan = false;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int p = 16 * n + pt;
    if (p < held || p >= upto) continue;
    uint32_t c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = code(widen<BF16>(kx[n][e]) * ik);
    *reinterpret_cast<u32x2v*>(s_kc + k_vec(p, d0 / 16) + d0 % 16) =
        u32x2v{c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t x = code(widen<BF16>(vx[n][e]) * iv);
      nan = nan || x == 0x7F;
      s_vc[v_vec(d0 + e, p / 16) + p % 16] = (uint8_t)x;
    }
  }
  if (nan) s_nan = 1;
  __syncthreads();

  const bool grow_k = held > 0 && ek > ek0, grow_v = held > 0 && ev > ev0;
  const float fk = two_to(max(ek0 - ek, -126)), fv = two_to(max(ev0 - ev, -126));
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int i = tid + 256 * n;           // vector 16 i of the half block
    // k: dims 16 c .. of token p
    const int p = 4 * (i >> 7) + 16 * ((i & 15) >> 2) + (i & 3);
    if (p >= held && p < upto) {
      *reinterpret_cast<u32x4*>(kb + 16 * i) = *reinterpret_cast<const u32x4*>(s_kc + 16 * i);
    } else if (p < held && grow_k) {
      u32x4 x = *reinterpret_cast<const u32x4*>(kb + 16 * i);
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] = recode(x[q], fk);
      *reinterpret_cast<u32x4*>(kb + 16 * i) = x;
    }
    // v: positions 16 w .. 16 w + 15 of dim d
    const int w = (i >> 4) & 3, lo = max(held - 16 * w, 0), hi = min(upto - 16 * w, 16);
    const uint8_t* s = s_vc + 16 * i;
    uint8_t* dst = vb + 16 * i;
    if (lo == 0 && hi == 16) {
      *reinterpret_cast<u32x4*>(dst) = *reinterpret_cast<const u32x4*>(s);
    } else {
      if (grow_v && lo > 0) {
        u32x4 x = *reinterpret_cast<const u32x4*>(dst);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int keep = min(max(lo - 4 * q, 0), 4);       // bytes of the dword that were held
          const uint32_t mask = keep == 4 ? 0xFFFFFFFFu : (1u << (8 * keep)) - 1;
          x[q] = (recode(x[q], fv) & mask) | (x[q] & ~mask);
        }
        *reinterpret_cast<u32x4*>(dst) = x;
      }
      for (int b = lo; b < hi; ++b) dst[b] = s[b];
    }
  }
  if (tid == 0) {
    const bool flag = s_nan || (held > 0 && as_u32(before.y) >> 31);
    *scale = float2{two_to(ek), flag ? -two_to(ev) : two_to(ev)};
  }
}

template <bool BF16, bool WIDE>
__global__ __launch_bounds__(256) void k_kv_append(AppendArgs a) {
  const int b = blockIdx.x;
  if (b < a.page_groups) {
    const int item = b / a.n_kv;
    if (item < a.work[kNAppend]) append_page<BF16>(a, item, b - item * a.n_kv);
    return;
  }
  rotate_heads<BF16, WIDE>(a.rope, (uint32_t)(b - a.page_groups) * 256 + threadIdx.x);
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
  a.wide = 1;
  const oi2_heads* in[2] = {k, v};
  for (int w = 0; w < 2; ++w) {
    a.src[w] = (const uint16_t*)in[w]->data;
    a.token_stride[w] = in[w]->token_stride;
    a.head_stride[w] = in[w]->head_stride;
    if ((uintptr_t)in[w]->data % 16 || in[w]->token_stride % 8 || in[w]->head_stride % 8) a.wide = 0;
  }
  a.pages = c->pages + (size_t)layer * c->n_pages * c->n_kv * kBlock;
  a.scales = c->scales + (size_t)layer * c->n_pages * c->n_kv * 2;
  const int64_t pages = (int64_t)now.cap_append * c->n_kv;
  int64_t rows = 0;
  bool wide = true;
  a.rotate = r ? 1 : 0;
  if (r) {
    rotary_describe(a.rope, r, n_tokens, p->positions);
    wide = rotary_fill(a.rope, q, q_out, nullptr, nullptr);
    rows = (rotary_threads(a.rope) + 255) / 256;
  }
  OI2_CHECK_ARG(pages + rows < 1 << 23, "%d tokens are too many for one call", n_tokens);
  a.page_groups = (int)pages;
  const dim3 grid((uint32_t)(pages + rows)), block(256);
  hipStream_t st = (hipStream_t)stream;
  const bool bf = dtype == OI2_DTYPE_BF16;
  if (bf && wide) hipLaunchKernelGGL((k_kv_append<true, true>), grid, block, 0, st, a);
  else if (bf) hipLaunchKernelGGL((k_kv_append<true, false>), grid, block, 0, st, a);
  else if (wide) hipLaunchKernelGGL((k_kv_append<false, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((k_kv_append<false, false>), grid, block, 0, st, a);
  OI2_CHECK_LAUNCH();
  return OI2_OK;
}
