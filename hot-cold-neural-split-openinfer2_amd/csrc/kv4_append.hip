// k and v of a step into the pages of the 4-bit KV cache, q and k rotated on the
// way.
//
// A group of 32 values has a scale of its own, so every token is coded by
// itself: 16 lanes take a token of the packed order and kv head, 8 dims a lane;
// the largest magnitude goes over four lanes.  A workgroup takes 16 tokens, the
// next one other heads of them: those of 64 tokens and one head, which share lines
// of a page, are as far apart as a set of tokens has workgroups (`chunks`).  Where
// that is a multiple of 8 (8, 16 or 32 heads, one a workgroup) they are on one XCD;
// elsewhere (4 heads; long rotated steps, whose workgroups take several heads)
// lines are written in parts from several.  q has workgroups of its own behind
// them in the same launch.
//
// Bound by the chain of slot, loads, reduction and stores for a step (24 tokens 6
// us), by bytes for prompts: 5875 tokens of 8 heads 9.8 us (31 MB, behind 600 MB of
// writes).  Rotated, by the fp64 turns: the same with q's 32 heads 34 us, with
// turns made by every thread for its own dims instead of once a token 53.
//
// k, v and q are read by non-temporal loads, for calls whose inputs are no longer
// in the caches: with cached ones the 9.8 us are 14.0, the rotated step's 34 are
// 45.  In a captured layer, where the projection has just written them, cached
// ones are as fast or little faster: a token 23.0 us a layer instead of 23.4, a
// prompt of 512 75.6 instead of 76.0, of 2000 and of 5000 the same (236.5, 835).
#include "capi_util.h"
#include "kv4.h"
#include "rotary.h"

namespace oi2 {
namespace {

struct Append4Args {
  const int32_t* slots;       // the plan's
  int n_kv, n_pages, n_tokens, groups;    // groups: workgroups for k and v, before q's
  int heads_each, chunks;     // kv heads of a workgroup, and how many take a token's
  const uint16_t* src[2];     // k, v
  int64_t token_stride[2], head_stride[2];
  int q_wide;
  uint8_t* pages;             // of the layer
  int32_t* clear;             // n_clear ints for the attention behind it
  int n_clear;
  RotaryArgs rope;            // q's tensors; its frequencies serve k too
};

// How k's pairs lie.  kAligned: rotary_dim a multiple of 16, so that the eight
// partners of a lane's dims are another lane's.
enum Turns { kNone, kAligned, kHalves, kNeighbours };

__device__ __forceinline__ uint32_t quad_top(uint32_t v) {     // over the four lanes of a group
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
}

// Eight values of a group, in pairs: their dword, and the group's scale in fp16.
template <bool BF16>
__device__ __forceinline__ uint32_t code8(const uint32_t (&x)[4], uint16_t& scale) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) m = max_u16(m, x[e] & 0x7FFF7FFFu);
  const uint32_t top = quad_top(max(m & 0xFFFFu, m >> 16));
  const bool bad = top >= kInfBits<BF16>;
  const float most = widen<BF16>((uint16_t)top), s = scale4(most), unit = s * 512.0f;
  scale = bad ? 0x7E00u : float_to_half_bits(s);
  // x / unit, exact where it is a tie between two codes: the quotient of the
  // reciprocal, corrected by its own remainder
  const float inv = s > 0.0f ? __builtin_amdgcn_rcpf(unit) : 0.0f;
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float v = e & 1 ? upper<BF16>(x[e / 2]) : lower<BF16>(x[e / 2]);
    const float q0 = v * inv;
    q[e] = fmaf(fmaf(-q0, unit, v), inv, q0);
  }
  // more than 7: past fp16's range, or where 2^-24 is a large part of the scale
  if (__any(most > 7.25f * s)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = __builtin_amdgcn_fmed3f(q[e], -0.013671875f, 0.013671875f);
  }
  const uint32_t lo = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false), true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false), true);
  return bad ? 0u : lo | __builtin_rotateleft32(hi, 4);
}

template <bool BF16, bool WIDE>
__device__ __forceinline__ void load8(uint32_t (&x)[4], const uint16_t* p) {
  if constexpr (WIDE) {
    *reinterpret_cast<u32x4*>(x) = load16_nt(reinterpret_cast<const uint8_t*>(p));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = p[2 * e] | (uint32_t)p[2 * e + 1] << 16;
  }
}

// A workgroup has 16 tokens of one kv head or several, whose cosines and sines its
// threads share.
constexpr int kTokens = 16, kPairs = kHeadD / 2;

template <bool BF16, bool WIDE, Turns TURNS>
__device__ __forceinline__ void append4(const Append4Args& a, int b) {
  const int set = b / a.chunks, g0 = (b - set * a.chunks) * a.heads_each, g1 = min(g0 + a.heads_each, a.n_kv);
  const int tid = threadIdx.x, u = tid & 15, in = tid >> 4;
  const int64_t t = kTokens * (int64_t)set + in;
  const bool have = t < a.n_tokens;
  const RotaryArgs& r = a.rope;
  const int64_t row = have ? t : a.n_tokens - 1;
  const uint16_t* pk = a.src[0] + row * a.token_stride[0] + 8 * u;
  const uint16_t* pv = a.src[1] + row * a.token_stride[1] + 8 * u;
  uint32_t nk[4], nv[4];
  load8<BF16, WIDE>(nk, pk + g0 * a.head_stride[0]);
  load8<BF16, WIDE>(nv, pv + g0 * a.head_stride[1]);
  const int slot = have ? a.slots[t] : -1;

  // Cosines and sines of this lane's pairs, for every head; the first dim of a
  // pair is turned as c a - s b, the second as s a + c b.
  constexpr int N = TURNS == kNone ? 1 : TURNS == kNeighbours ? 4 : 8;
  CosSin cs[N];
  const int pairs = r.rot / 2;
  if constexpr (TURNS != kNone) {
    __shared__ __align__(16) CosSin s_turn[kTokens * kPairs];
    // thread: pairs u, u + 16 .. of its token
    const int pos = r.positions[row];
#pragma unroll
    for (int e = 0; e < kPairs / 16; ++e) {
      const int j = u + 16 * e;
      if (j >= pairs) continue;
      CosSin x = turn(r.freq[j], pos);
      x.c *= r.magnitude;
      x.s *= r.magnitude;
      s_turn[in * kPairs + j] = x;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int d = 8 * u + (TURNS == kNeighbours ? 2 * e : e);
      if (d >= r.rot) continue;
      const int j = TURNS == kNeighbours ? d / 2 : d < pairs ? d : d - pairs;
      cs[e] = s_turn[in * kPairs + j];
      if (TURNS != kNeighbours && d >= pairs) cs[e] = CosSin{cs[e].s, cs[e].c};
    }
  }
  if (slot < 0 || slot / kPage >= a.n_pages) return;     // a token's lanes together
  const int p = slot % kPage, lane = lane_id();
  const int other = TURNS != kAligned || 8 * u >= r.rot ? lane : 8 * u < pairs ? lane + pairs / 8 : lane - pairs / 8;

  for (int g = g0; g < g1; ++g) {
    uint32_t k[4], v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      k[e] = nk[e];
      v[e] = nv[e];
    }
    if (g + 1 < g1) {
      load8<BF16, WIDE>(nk, pk + (g + 1) * a.head_stride[0]);
      load8<BF16, WIDE>(nv, pv + (g + 1) * a.head_stride[1]);
    }
    if constexpr (TURNS == kNeighbours) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (8 * u + 2 * e < r.rot) {
          const f32x2 o = turned(lower<BF16>(k[e]), upper<BF16>(k[e]), cs[e]);
          k[e] = narrow<BF16>(o.x) | (uint32_t)narrow<BF16>(o.y) << 16;
        }
    } else if constexpr (TURNS != kNone) {
      uint32_t b[4];                       // the partners
      if constexpr (TURNS == kAligned) {
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = (uint32_t)__shfl((int)k[e], other);
      } else {
        const uint16_t* row = pk - 8 * u + g * a.head_stride[0];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t w[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int d = 8 * u + 2 * e + h;
            w[h] = d < r.rot ? row[d < pairs ? d + pairs : d - pairs] : 0;
          }
          b[e] = w[0] | w[1] << 16;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int d = 8 * u + 2 * e + h;
          const float x = h ? upper<BF16>(k[e]) : lower<BF16>(k[e]), y = h ? upper<BF16>(b[e]) : lower<BF16>(b[e]);
          const bool first = d < pairs;
          const CosSin z = cs[2 * e + h];
          // the products and their order are turned()'s
          float o = (float)fma((double)(first ? x : y), z.c, (double)(first ? -y : x) * z.s);
          asm("" : "+v"(o));
          w[h] = d < r.rot ? narrow<BF16>(o) : h ? k[e] >> 16 : k[e] & 0xFFFFu;
        }
        k[e] = w[0] | w[1] << 16;
      }
    }
    uint8_t* block = a.pages + ((int64_t)(slot / kPage) * a.n_kv + g) * k4Block;
    uint16_t ks, vs;
    const uint32_t kd = code8<BF16>(k, ks), vd = code8<BF16>(v, vs);
    *reinterpret_cast<uint32_t*>(block + k4_at(p, u)) = kd;
    *reinterpret_cast<uint32_t*>(block + v4_at(p, u)) = vd;
    if (u % 4 == 0) {
      *reinterpret_cast<uint16_t*>(block + k4_scale_at(p, u / 4)) = ks;
      *reinterpret_cast<uint16_t*>(block + v4_scale_at(p, u / 4)) = vs;
    }
  }
}

template <bool BF16, bool WIDE, Turns TURNS>
__global__ __launch_bounds__(256) void k_kv4_append(Append4Args a) {
  const int b = blockIdx.x;
  for (int i = 256 * b + threadIdx.x; i < a.n_clear; i += 256 * gridDim.x) a.clear[i] = 0;
  if (b < a.groups) append4<BF16, WIDE, TURNS>(a, b);
  else if constexpr (TURNS != kNone) {
    if (a.q_wide) rotate_tokens<BF16, true, 256, true>(a.rope, b - a.groups);
    else rotate_tokens<BF16, false, 256, true>(a.rope, b - a.groups);
  }
}

template <bool BF16, bool WIDE>
void launch_append4(const Append4Args& a, Turns turns, uint32_t groups, hipStream_t st) {
  const dim3 grid(groups), block(256);
  switch (turns) {
    case kNone: hipLaunchKernelGGL((k_kv4_append<BF16, WIDE, kNone>), grid, block, 0, st, a); break;
    case kAligned: hipLaunchKernelGGL((k_kv4_append<BF16, WIDE, kAligned>), grid, block, 0, st, a); break;
    case kHalves: hipLaunchKernelGGL((k_kv4_append<BF16, WIDE, kHalves>), grid, block, 0, st, a); break;
    case kNeighbours: hipLaunchKernelGGL((k_kv4_append<BF16, WIDE, kNeighbours>), grid, block, 0, st, a); break;
  }
}

}  // namespace

int check_paged4(const oi2_paged* c, int32_t layer) {
  if (int rc = check_paged(c, layer, false)) return rc;
  OI2_CHECK_ARG(layer >= 0 && layer < c->n_layers, "layer %d of a cache of %d", layer, c->n_layers);
  OI2_CHECK_ARG(c->pages && (uintptr_t)c->pages % 16 == 0, "pages must be non-null and 16-byte aligned");
  OI2_CHECK_ARG(!c->scales, "a cache of 4 bits has its scales in its pages");
  return OI2_OK;
}

int kv4_append(const oi2_paged* c, const oi2_page_plan* p, int32_t layer, int32_t dtype, int32_t n_tokens, const oi2_heads* k,
               const oi2_heads* v, const oi2_rotary* r, const oi2_heads* q, void* q_out, int32_t* clear, int n_clear, void* stream) {
  if (int rc = check_paged4(c, layer)) return rc;
  if (int rc = check_plan(c, p)) return rc;
  bool zero;
  if (int rc = check_append(c, p, dtype, zero, n_tokens, k, v, r, q, q_out)) return rc;
  if (n_tokens == 0) return OI2_OK;
  Append4Args a{};
  a.slots = p->slots;
  a.n_kv = c->n_kv;
  a.n_pages = c->n_pages;
  a.n_tokens = n_tokens;
  a.clear = clear;
  a.n_clear = n_clear;
  bool wide = true;
  const oi2_heads* in[2] = {k, v};
  for (int w = 0; w < 2; ++w) {
    a.src[w] = (const uint16_t*)in[w]->data;
    a.token_stride[w] = in[w]->token_stride;
    a.head_stride[w] = in[w]->head_stride;
    if ((uintptr_t)in[w]->data % 16 || in[w]->token_stride % 8 || in[w]->head_stride % 8) wide = false;
  }
  a.pages = c->pages + (size_t)layer * c->n_pages * c->n_kv * k4Block;
  // heads share their turns while 1024 workgroups are left: 5875 tokens with q's 32
  // heads 34 us (8 kv heads) and 55 (32); while 512 are 32 and 60
  const int64_t sets = ((int64_t)n_tokens + kTokens - 1) / kTokens;
  a.heads_each = 1;
  while (r && a.heads_each < c->n_kv && sets * c->n_kv / (2 * a.heads_each) >= 1024) a.heads_each *= 2;
  a.chunks = (c->n_kv + a.heads_each - 1) / a.heads_each;
  const int64_t pages = sets * a.chunks;
  int64_t rows = 0;
  Turns turns = kNone;
  if (r) {
    rotary_describe(a.rope, r, n_tokens, p->positions, zero);
    a.q_wide = rotary_fill(a.rope, q, q_out, nullptr, nullptr) ? 1 : 0;
    rows = rotary_workgroups(a.rope);
    turns = r->interleaved ? kNeighbours : r->rotary_dim % 16 == 0 ? kAligned : kHalves;
  }
  OI2_CHECK_ARG(pages + rows < 1 << 23, "%d tokens are too many for one call", n_tokens);
  a.groups = (int)pages;
  hipStream_t st = (hipStream_t)stream;
  const uint32_t groups = (uint32_t)(pages + rows);
  const bool bf = dtype == OI2_DTYPE_BF16;
  if (bf && wide) launch_append4<true, true>(a, turns, groups, st);
  else if (bf) launch_append4<true, false>(a, turns, groups, st);
  else if (wide) launch_append4<false, true>(a, turns, groups, st);
  else launch_append4<false, false>(a, turns, groups, st);
  OI2_CHECK_LAUNCH();
  return OI2_OK;
}

}  // namespace oi2

extern "C" int oi2_kv4_append(const oi2_paged* c, const oi2_page_plan* p, int32_t layer, int32_t dtype, int32_t n_tokens,
                              const oi2_heads* k, const oi2_heads* v, const oi2_rotary* r, const oi2_heads* q,
                              void* q_out, void* stream) {
  oi2::clear_error();
  return oi2::kv4_append(c, p, layer, dtype, n_tokens, k, v, r, q, q_out, nullptr, 0, stream);
}
