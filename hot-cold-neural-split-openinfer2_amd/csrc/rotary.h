// Rotary positions from 64-bit fixed-point turns, shared by the rotary operator
// and the cache's append.
//
// Cosines, sines and products are fp64; a result is rounded to fp32 and then to
// its type.  The append codes rotated keys to 4 bits, where an fp32 sum moves
// one value in 2^16 across the edge of a code, and the operator's forms agree
// bit for bit without being compiled alike.
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
  int per_head;               // threads of a head
  int tokens_each;            // tokens of a workgroup
  int zero;                   // tokens at negative positions get zeros
};

// Cosines and sines of a workgroup's tokens: kTurns at most.
constexpr int kTurns = 256;

// The heads of tokens_each tokens by a workgroup of NT threads.  Their cosines
// and sines are made once, in LDS, while the first heads are on their way; a
// thread takes eight pairs of a head in WIDE (16-byte loads and stores: pairs
// 8 u .. of the rotated part, or 16 dims behind it; needs a rotary_dim and
// head_dim that 16 divides and rows at 16-byte addresses), otherwise one pair,
// and then the same of the head NT / per_head further on, whose loads are under
// way while this one is turned.  12001 tokens of 32 + 8 heads out of cache 47 us
// (5.2 TB/s); with the turns made by each thread for up to 8 heads of its own
// 51.5, for 2 of them 56.
template <bool BF16, bool WIDE, int NT>
__device__ __forceinline__ void rotate_tokens(const RotaryArgs& a, int b) {
  constexpr int P = WIDE ? 8 : 1;
  static_assert(NT >= kTurns);
  __shared__ __align__(16) CosSin s_turn[kTurns];
  __shared__ int s_pos[kTurns];
  const int tid = threadIdx.x, t0 = b * a.tokens_each, nt = min(a.tokens_each, a.n_tokens - t0);
  const int pairs = a.rot / 2, lanes = pairs / P, all = a.heads[0] + a.heads[1];
  const int slot = tid / a.per_head, slots = NT / a.per_head, u = tid - slot * a.per_head;
  const bool rotate = u < lanes, halves = rotate && !a.interleaved;
  const int d0 = halves ? P * u : 2 * P * u, d1 = halves ? P * u + pairs : 2 * P * u + P;
  uint16_t v[2 * P], ahead[2 * P];
  auto load = [&](uint16_t* x, int t, int h) {
    const int w = h >= a.heads[0];
    const uint16_t* p = (w ? a.src[1] : a.src[0]) + (int64_t)(t0 + t) * (w ? a.token_stride[1] : a.token_stride[0]) +
                        (w ? h - a.heads[0] : h) * (w ? a.head_stride[1] : a.head_stride[0]);
    if constexpr (WIDE) {
      *reinterpret_cast<u32x4*>(x) = *reinterpret_cast<const u32x4*>(p + d0);
      *reinterpret_cast<u32x4*>(x + 8) = *reinterpret_cast<const u32x4*>(p + d1);
    } else {
      x[0] = p[d0];
      x[1] = p[d1];
    }
  };
  int t = slot / all, h = slot - t * all;
  if (slot >= slots) t = nt;                     // threads past the last whole head
  if (t < nt) load(v, t, h);
  if (tid < nt) s_pos[tid] = a.positions[t0 + tid];
  if (tid < nt * pairs) {
    const int tok = tid / pairs, i = tid - tok * pairs;      // pair 8 u + e at e * lanes + u: no bank conflicts
    CosSin x = turn(a.freq[WIDE ? i % lanes * P + i / lanes : i], a.positions[t0 + tok]);
    x.c *= a.magnitude;
    x.s *= a.magnitude;
    s_turn[tid] = x;
  }
  __syncthreads();
  while (t < nt) {
    int next = t, nh = h + slots;
    while (nh >= all) {
      nh -= all;
      ++next;
    }
    if (next < nt) load(ahead, next, nh);
    if (rotate) {
      const CosSin* cs = s_turn + t * pairs + u;
      if (a.interleaved) {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const f32x2 o = turned(widen<BF16>(v[2 * e]), widen<BF16>(v[2 * e + 1]), cs[e * lanes]);
          v[2 * e] = narrow<BF16>(o.x);
          v[2 * e + 1] = narrow<BF16>(o.y);
        }
      } else {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const f32x2 o = turned(widen<BF16>(v[e]), widen<BF16>(v[e + P]), cs[e * lanes]);
          v[e] = narrow<BF16>(o.x);
          v[e + P] = narrow<BF16>(o.y);
        }
      }
    }
    const bool left_out = s_pos[t] < 0;
    if (left_out) {
#pragma unroll
      for (int e = 0; e < 2 * P; ++e) v[e] = 0;
    }
    if (!left_out || a.zero) {
      const int w = h >= a.heads[0];
      uint16_t* p = (w ? a.dst[1] : a.dst[0]) + ((int64_t)(t0 + t) * (w ? a.heads[1] : a.heads[0]) + (w ? h - a.heads[0] : h)) * a.head_dim;
      if constexpr (WIDE) {
        *reinterpret_cast<u32x4*>(p + d0) = *reinterpret_cast<const u32x4*>(v);
        *reinterpret_cast<u32x4*>(p + d1) = *reinterpret_cast<const u32x4*>(v + 8);
      } else {
        p[d0] = v[0];
        p[d1] = v[1];
      }
    }
    t = next;
    h = nh;
#pragma unroll
    for (int e = 0; e < 2 * P; ++e) v[e] = ahead[e];
  }
}

inline void rotary_describe(RotaryArgs& a, const oi2_rotary* r, int n_tokens, const int32_t* positions, bool zero) {
  a.freq = r->freq;
  a.positions = positions;
  a.magnitude = r->magnitude;
  a.n_tokens = n_tokens;
  a.head_dim = r->head_dim;
  a.rot = r->rotary_dim;
  a.interleaved = r->interleaved ? 1 : 0;
  a.zero = zero ? 1 : 0;
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
  // as many tokens a workgroup as there is room for their turns, and as leave
  // 512 workgroups
  a.tokens_each = kTurns / (a.rot / 2);
  while (a.tokens_each > 1 && a.n_tokens / a.tokens_each < 512) a.tokens_each /= 2;
  return wide;
}

inline int64_t rotary_workgroups(const RotaryArgs& a) {
  return a.heads[0] + a.heads[1] ? ((int64_t)a.n_tokens + a.tokens_each - 1) / a.tokens_each : 0;
}

int check_rotary(const oi2_rotary* r);

// Whether the dense (n_tokens, out_heads, dim) values at out share memory with
// in's: a workgroup would read what another has written.  own: in is what out
// is computed from, and may be it where it is as dense: every value of it is
// read by the thread that writes it, or before.
inline bool clashes(bool own, const void* out, int out_heads, const oi2_heads* in, int n_tokens, int dim) {
  if (!in || !in->heads || !out_heads || n_tokens < 1) return false;
  if (own && out == in->data && out_heads == in->heads && (in->heads == 1 || in->head_stride == dim) &&
      (n_tokens == 1 || in->token_stride == (int64_t)in->heads * dim))
    return false;
  int64_t lo = 0, hi = dim;                // of in, in elements
  const int64_t far[2] = {(n_tokens - 1) * in->token_stride, (in->heads - 1) * in->head_stride};
  for (int64_t f : far) (f < 0 ? lo : hi) += f;
  const intptr_t o0 = (intptr_t)out, o1 = o0 + 2 * (int64_t)n_tokens * out_heads * dim, i = (intptr_t)in->data;
  return o0 < i + 2 * hi && i + 2 * lo < o1;
}

}  // namespace oi2
