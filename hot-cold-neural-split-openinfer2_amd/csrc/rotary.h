// Rotary positions from 64-bit fixed-point turns, shared by the rotary operator
// and the cache's append.
//
// Cosines, sines and products are fp64; a result is rounded to fp32 and then to
// its type.  The append codes rotated keys to 4 bits, where an fp32 sum moves
// one value in 2^16 across the edge of a code, and the operator's forms agree
// bit for bit without being compiled alike.  It costs no time: the operator is
// bound by its bytes (12001 tokens of 32 + 8 heads, half of each head rotated:
// 54.4 us, with fp32 sums 58.2).
#pragma once
#include "decode_util.h"
#include "oi2.h"

namespace oi2 {

struct CosSin {
  double c, s;
};

// cos and sin of position * freq / 2^64 turns.  The product modulo 2^64 is the
// angle's fraction of a turn without any error, however far the position.
// Its top bits, rounded, name the quadrant; the rest is an angle in [-pi/4,
// pi/4] for Taylor polynomials of sin (to x^13, off by x^15 / 15! < 3e-14) and
// cos (to x^14, off by x^16 / 16! < 2e-15).
__device__ __forceinline__ CosSin turn(uint64_t freq, int position) {
  const uint64_t t = freq * (uint64_t)(uint32_t)position;
  const uint32_t top = (uint32_t)(t >> 32), low = (uint32_t)t;
  const uint32_t quad = (top + 0x20000000u) >> 30;
  const int32_t rest = (int32_t)(top - (quad << 30));   // from the quadrant's axis, in 2^-32 turns
  const double x = fma((double)rest, 4294967296.0, (double)low) * 3.4061215800304185e-19;   // 2 pi / 2^64
  const double x2 = x * x;
  double s = fma(x2, 1.0 / 6227020800.0, -1.0 / 39916800.0);
  s = fma(x2, s, 1.0 / 362880.0);
  s = fma(x2, s, -1.0 / 5040.0);
  s = fma(x2, s, 1.0 / 120.0);
  s = fma(x2, s, -1.0 / 6.0);
  s = fma(x2 * x, s, x);
  double c = fma(x2, -1.0 / 87178291200.0, 1.0 / 479001600.0);
  c = fma(x2, c, -1.0 / 3628800.0);
  c = fma(x2, c, 1.0 / 40320.0);
  c = fma(x2, c, -1.0 / 720.0);
  c = fma(x2, c, 1.0 / 24.0);
  c = fma(x2, c, -0.5);
  c = fma(x2, c, 1.0);
  const bool odd = quad & 1;
  CosSin r;
  r.c = odd ? s : c;
  r.s = odd ? c : s;
  r.c = ((quad + 1) & 2) ? -r.c : r.c;
  r.s = (quad & 2) ? -r.s : r.s;
  return r;
}

// The pair (a, b) turned, rounded to fp32; the caller rounds it to its type.
// The empty asm keeps the two roundings apart: without it some instantiations
// rounded to bf16 otherwise than others.
__device__ __forceinline__ f32x2 turned(float a, float b, CosSin t) {
  float x = (float)fma((double)a, t.c, -((double)b * t.s)), y = (float)fma((double)a, t.s, (double)b * t.c);
  asm("" : "+v"(x), "+v"(y));
  return f32x2{x, y};
}

// fp16 and bf16 values by type.
template <bool BF16>
__device__ __forceinline__ float widen(uint16_t v) {
  return BF16 ? bf16_bits_to_float(v) : half_bits_to_float(v);
}
template <bool BF16>
__device__ __forceinline__ uint16_t narrow(float v) {
  if (BF16) return __builtin_bit_cast(uint16_t, (__bf16)v);
  return float_to_half_bits(v);
}

struct RotaryArgs {
  const uint64_t* freq;
  const int32_t* positions;
  float magnitude;
  int n_tokens, head_dim, rot, interleaved;
  const uint16_t* src[2];     // q, k
  uint16_t* dst[2];           // dense
  int64_t token_stride[2], head_stride[2];
  int heads[2];
  uint32_t per_head;          // threads of a head
  uint32_t groups;            // threads' groups of heads of a token
  int heads_each;             // heads of a thread
};

// Thread i of the tokens' heads.  WIDE: eight pairs of a head, 16-byte loads
// and stores: pairs 8 u .. of the rotated part, or 16 dims of the part behind
// it.  Needs a rotary_dim and head_dim that 16 divides and rows at 16-byte
// addresses; otherwise one pair, or two dims behind the rotated part.
template <bool BF16, bool WIDE>
__device__ __forceinline__ void rotate_heads(const RotaryArgs& a, uint32_t i) {
  constexpr int P = WIDE ? 8 : 1;
  const uint32_t u = i % a.per_head, tg = i / a.per_head, t = tg / a.groups, g = tg % a.groups;
  if (t >= (uint32_t)a.n_tokens) return;
  const int pos = a.positions[t];
  if (pos < 0) return;
  const bool rotate = 2 * P * (int)u < a.rot;
  const bool halves = rotate && !a.interleaved;
  const int d0 = halves ? P * u : 2 * P * u, d1 = halves ? P * u + a.rot / 2 : 2 * P * u + P;
  CosSin cs[P];
#pragma unroll
  for (int e = 0; e < P; ++e) {
    cs[e] = rotate ? turn(a.freq[P * u + e], pos) : CosSin{1.0, 0.0};
    cs[e].c *= a.magnitude;
    cs[e].s *= a.magnitude;
  }
  const int all = a.heads[0] + a.heads[1], h1 = min((int)(g + 1) * a.heads_each, all);
  for (int hh = (int)g * a.heads_each; hh < h1; ++hh) {
    const int w = hh >= a.heads[0], h = w ? hh - a.heads[0] : hh;
    const uint16_t* src = (w ? a.src[1] : a.src[0]) + (int64_t)t * (w ? a.token_stride[1] : a.token_stride[0]) +
                          h * (w ? a.head_stride[1] : a.head_stride[0]);
    uint16_t* dst = (w ? a.dst[1] : a.dst[0]) + ((int64_t)t * (w ? a.heads[1] : a.heads[0]) + h) * a.head_dim;
    uint16_t v[2 * P];
    if constexpr (WIDE) {
      *reinterpret_cast<u32x4*>(v) = *reinterpret_cast<const u32x4*>(src + d0);
      *reinterpret_cast<u32x4*>(v + 8) = *reinterpret_cast<const u32x4*>(src + d1);
    } else {
      v[0] = src[d0];
      v[1] = src[d1];
    }
    if (rotate) {
      if (a.interleaved) {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const f32x2 o = turned(widen<BF16>(v[2 * e]), widen<BF16>(v[2 * e + 1]), cs[e]);
          v[2 * e] = narrow<BF16>(o.x);
          v[2 * e + 1] = narrow<BF16>(o.y);
        }
      } else {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const f32x2 o = turned(widen<BF16>(v[e]), widen<BF16>(v[e + P]), cs[e]);
          v[e] = narrow<BF16>(o.x);
          v[e + P] = narrow<BF16>(o.y);
        }
      }
    }
    if constexpr (WIDE) {
      *reinterpret_cast<u32x4*>(dst + d0) = *reinterpret_cast<const u32x4*>(v);
      *reinterpret_cast<u32x4*>(dst + d1) = *reinterpret_cast<const u32x4*>(v + 8);
    } else {
      dst[d0] = v[0];
      dst[d1] = v[1];
    }
  }
}

inline void rotary_describe(RotaryArgs& a, const oi2_rotary* r, int n_tokens, const int32_t* positions) {
  a.freq = r->freq;
  a.positions = positions;
  a.magnitude = r->magnitude;
  a.n_tokens = n_tokens;
  a.head_dim = r->head_dim;
  a.rot = r->rotary_dim;
  a.interleaved = r->interleaved ? 1 : 0;
}

// The tensors, how the work is cut, and whether the wide form serves them.
inline bool rotary_fill(RotaryArgs& a, const oi2_heads* q, void* q_out, const oi2_heads* k, void* k_out) {
  const oi2_heads* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  bool wide = a.rot % 16 == 0 && a.head_dim % 16 == 0;
  for (int w = 0; w < 2; ++w) {
    a.heads[w] = in[w] ? in[w]->heads : 0;
    if (!a.heads[w]) continue;
    a.src[w] = (const uint16_t*)in[w]->data;
    a.dst[w] = (uint16_t*)out[w];
    a.token_stride[w] = in[w]->token_stride;
    a.head_stride[w] = in[w]->head_stride;
    wide = wide && (uintptr_t)in[w]->data % 16 == 0 && (uintptr_t)out[w] % 16 == 0 && in[w]->token_stride % 8 == 0 &&
           in[w]->head_stride % 8 == 0;
  }
  a.per_head = a.head_dim / (wide ? 16 : 2);
  const int all = a.heads[0] + a.heads[1];
  // as many heads a thread as still leave 2^18 threads (4 waves a SIMD)
  a.heads_each = 1;
  auto groups = [&](int each) { return (all + each - 1) / each; };
  while (a.heads_each < 8 && (int64_t)a.n_tokens * a.per_head * groups(2 * a.heads_each) >= 1 << 18) a.heads_each *= 2;
  a.groups = groups(a.heads_each);
  return wide;
}

inline int64_t rotary_threads(const RotaryArgs& a) { return (int64_t)a.n_tokens * a.per_head * a.groups; }

int check_rotary(const oi2_rotary* r);

}  // namespace oi2
