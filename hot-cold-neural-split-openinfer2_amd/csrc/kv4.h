// The paged 4-bit KV cache: where a page's codes and scales are, how a group of
// values is coded and what it stands for.
//
// A head's 128 values are four groups of 32 dims, a group n s with whole n in
// [-7, 7] and one scale s, its largest magnitude over 7 rounded to 8 significant
// bits (a multiple of 2^-24, 2^-24 to 9344, 0 for zeros).  So n s has 3 + 8 bits
// and is exact in fp16, and codes times scales are the matrix products' operands.
// A group with a NaN or an infinity has a NaN for its scale.
//
// Sign and magnitude, because e4m3's bytes s0000mmm are (-1)^s m 2^-9: the fp8
// conversions code and decode, two values each, after one and (values 0-3 of a
// dword, a byte each: sign at its bit 7, magnitude at bits 0-2) or one rotation
// by 4 and one and (values 4-7).  Two's complement nibbles cost two instructions
// more for each eight.
#pragma once
#include "kv_cache.h"
#include "oi2_device.h"

namespace oi2 {

// Blocks of a page and kv head: k's codes, v's, k's scales (fp16), v's.
constexpr int k4Codes = kPage * kHeadD / 2, k4Scales = kPage * 4 * 2;
constexpr int k4V = k4Codes, k4KScale = 2 * k4Codes, k4VScale = k4KScale + k4Scales;
constexpr int k4Block = k4VScale + k4Scales;
static_assert(k4Block == OI2_KV4_BLOCK, "the header's");

constexpr float k4TopScale = 9344.0f;      // the largest with 7 s in fp16
constexpr float k4Least = 5.9604644775390625e-8f;   // 2^-24

// Byte offsets in a block: the dword of position p, dims 8 u ..; the scale of its
// group c = u / 4.  The attention's loads, 16 bytes a lane, are consecutive.
__device__ __forceinline__ int k4_at(int p, int u) {
  return 1024 * (p >> 2 & 3) + 256 * (u >> 2) + 16 * (4 * (p >> 4) + (p & 3)) + 4 * (u & 3);
}
__device__ __forceinline__ int v4_at(int p, int u) { return k4V + 1024 * (p >> 2 & 3) + 256 * (p >> 4) + 16 * u + 4 * (p & 3); }
__device__ __forceinline__ int k4_scale_at(int p, int c) {
  return k4KScale + 8 * (16 * c + 4 * (p >> 4) + (p & 3)) + 2 * (p >> 2 & 3);
}
__device__ __forceinline__ int v4_scale_at(int p, int c) { return k4VScale + 128 * c + 2 * p; }

// A dword's values 0-3 and 4-7 as bytes of e4m3, in 2^-9.
constexpr uint32_t k4Mask = 0x87878787u;
__device__ __forceinline__ uint32_t low4(uint32_t d) { return d & k4Mask; }
__device__ __forceinline__ uint32_t high4(uint32_t d) { return __builtin_rotateright32(d, 4) & k4Mask; }

// Bytes 0, 1 or 2, 3 of those as whole numbers in fp16.
__device__ __forceinline__ f16x2 whole2(uint32_t bytes, bool hi) {
  return hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, 512.0f, true)
            : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, 512.0f, false);
}

// The scale of a group whose largest magnitude is top >= 0, as fp32 with at
// most 8 significant bits.  Exact: top has at most 11 bits, so top / 7 is either
// a tie, and then exact in fp32, or 2^-12 of itself away from one.
__device__ __forceinline__ float scale4(float top) {
  const float y = top / 7.0f;
  const uint32_t b = as_u32(y);
  const float wide = as_f32((b + 0x7FFFu + (b >> 16 & 1)) & 0xFFFF0000u);
  const float s = y < 1.52587890625e-5f ? fmaxf(rintf(y * 16777216.0f) * k4Least, k4Least) : fminf(wide, k4TopScale);
  return top > 0.0f ? s : 0.0f;
}

}  // namespace oi2
