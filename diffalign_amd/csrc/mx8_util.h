// MXINT8 (OCP microscaling): 32 consecutive channels of a row share a power-of-two scale X = 2^(b - 127), one byte b; an element is an
// int8 q and stands for q / 64 * X.  b is the smallest exponent at which the group's largest magnitude rounds to 127 or less, so
// every value is within half a step, X / 128, of its element (an amax over 127.5 / 64 * 2^127 has no such b and saturates at 127; KEEP lifts
// an element below half a step to a whole one).
// b as written is in [MX8_B_MIN, 254]: X >= 2^-100 keeps every element a normal bf16 / fp32 (smaller values round to zero at that step); any
// byte is read.
// A group with an infinity or NaN gets b = 255 and stands for NaN throughout.  An element has 7 significant bits: exact in bf16.
#pragma once
#include "common.h"

#define MX8_GROUP 32
#define MX8_B_MIN 27

// largest |x| bits of the group -> b
__device__ __forceinline__ unsigned mx8_scale(unsigned amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  const unsigned b = (amax_bits + (0x800000u - 0x7f0000u)) >> 23;      // mantissa >= 127.5 / 128 of the next power: one exponent up
  return b < MX8_B_MIN ? MX8_B_MIN : (b > 254u ? 254u : b);
}
// 64 / X: what a value is multiplied by; 0 for the NaN group (its codes are 0)
__device__ __forceinline__ float mx8_inv(unsigned b) { return __builtin_bit_cast(float, b == 255u ? 0u : (260u - b) << 23); }
// X / 64 = 2^(b - 133): what a code stands for.  A caller's own scale bytes may lie below MX8_B_MIN: up to 6 the step is a subnormal, of which
// fp32 holds every multiple by a code exactly
__device__ __forceinline__ float mx8_step(unsigned b) {
  return __builtin_bit_cast(float, b == 255u ? 0x7fc00000u : b < 7u ? 0x10000u << b : (b - 6u) << 23);
}
// round to nearest even of x * inv in the low byte of a word: 1.5 * 2^23 has a unit of 1 and x * inv is exact (a power of two) unless it is
// far below one half, so the fused sum rounds once.  The clamp acts only where the scale is saturated (or x is not finite: inv = 0, and
// that group's codes are 0).
__device__ __forceinline__ unsigned mx8_round(float x, float inv) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_fmed3f(__builtin_fmaf(x, inv, 12582912.f), 12582912.f - 127.f, 12582912.f + 127.f));
}
// KEEP: an element other than zero never gets code 0 (+-1 instead), so the codes still tell what a ReLU let through.
template <bool KEEP>
__device__ __forceinline__ unsigned mx8_code(float x, float inv) {
  unsigned w = inv == 0.f ? 0u : mx8_round(x, inv) & 0xffu;
  if (KEEP && w == 0u && x != 0.f) w = x > 0.f ? 1u : 0xffu;
  return w;
}
// four codes (element order) in one word
template <bool KEEP>
__device__ __forceinline__ unsigned mx8_pack4(float a, float b, float c, float d, float inv) {
  if constexpr (KEEP) return mx8_code<true>(a, inv) | mx8_code<true>(b, inv) << 8 | mx8_code<true>(c, inv) << 16 | mx8_code<true>(d, inv) << 24;
  const unsigned ab = __builtin_amdgcn_perm(mx8_round(b, inv), mx8_round(a, inv), 0x0c0c0400u);
  const unsigned cd = __builtin_amdgcn_perm(mx8_round(d, inv), mx8_round(c, inv), 0x0c0c0400u);
  return inv == 0.f ? 0u : __builtin_amdgcn_perm(cd, ab, 0x05040100u);
}
// signed byte k of a word as a float
template <int K>
__device__ __forceinline__ float mx8_elem(unsigned w) { return (float)(((int)(w << (24 - 8 * K))) >> 24); }

// maximum over the 4 / 8 lanes of an aligned group (DPP: no LDS)
__device__ __forceinline__ unsigned dpp_max_u32(unsigned v, unsigned o) { return v > o ? v : o; }
#define MX8_DPP(v, ctrl) ((unsigned)__builtin_amdgcn_mov_dpp((int)(v), ctrl, 0xf, 0xf, true))
__device__ __forceinline__ unsigned quad_max(unsigned v) {
  v = dpp_max_u32(v, MX8_DPP(v, 0xB1));                                // lanes 1,0,3,2
  return dpp_max_u32(v, MX8_DPP(v, 0x4E));                             // lanes 2,3,0,1
}
__device__ __forceinline__ unsigned oct_max(unsigned v) {
  v = quad_max(v);
  return dpp_max_u32(v, MX8_DPP(v, 0x141));                            // row_half_mirror: the other quad of the eight
}
__device__ __forceinline__ unsigned abs_bits(float x) { return __builtin_bit_cast(unsigned, x) & 0x7fffffffu; }
