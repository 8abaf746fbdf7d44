// The 8-bit paged KV cache: e4m3 codes [blocks + 1][page][hkv][128] and, for
// every 16 consecutive slots (a "scale block") and kv head, one power of two
// for K and one for V, scales[slot / 16][hkv][2]; a value is code * scale.
//
// A floating code keeps its precision whatever the power of two is, so a
// block's scale only has to hold its largest value, it can grow later by an
// exact rescale of the codes (but for those that become subnormal), and the
// hardware's scaled converter turns codes into 16-bit values with the scale
// applied at no cost.
#pragma once
#include "device_util.hpp"

namespace feattn {

constexpr int kScaleTokens = 16;                // slots of one scale block
constexpr uint32_t kMinScale = 9u << 23;        // 2^-118: the smallest value of such a block is 2^-127
constexpr uint32_t kInfBits = 0x7f800000u;

// The largest magnitude of the 16-bit type that four significand bits hold:
// what is stored, so that a cached value is always finite in that type.
template <bool BF16>
__device__ __forceinline__ constexpr float kv8_cap() { return BF16 ? 0x1.ep127f : 61440.f; }

// Bits of the smallest power of two s (2^-118 at least) with amax <= 448 s;
// 448 = 1.75 * 2^8.  amax finite, as bits.
__device__ __forceinline__ uint32_t kv8_need(uint32_t amax) {
  const uint32_t e = (amax + 0x1fffffu) >> 23;  // the exponent, one more above 1.75 of it
  return max(e << 23, kMinScale + (8u << 23)) - (8u << 23);
}

// 1 / s for a power of two s in [2^-118, 2^120], as bits.
__device__ __forceinline__ float kv8_inverse(uint32_t s) { return __uint_as_float((254u << 23) - s); }

// Four fp32 values to four codes, round to nearest even; what overflows or is
// no number becomes the NaN code.
__device__ __forceinline__ uint32_t kv8_encode4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Codes 2 HI, 2 HI + 1 of a word as a packed pair of 16-bit values, scaled by
// the power of two `s` (the converter takes its exponent only).
template <bool BF16, bool HI>
__device__ __forceinline__ uint32_t kv8_pair(uint32_t w, float s) {
  if constexpr (BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, HI));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, HI));
}

// Eight codes as eight 16-bit values: the first four scaled by s0, the others by s1.
template <bool BF16>
__device__ __forceinline__ u32x4 kv8_decode8(uint32_t w0, uint32_t w1, float s0, float s1) {
  return u32x4{kv8_pair<BF16, false>(w0, s0), kv8_pair<BF16, true>(w0, s0), kv8_pair<BF16, false>(w1, s1),
               kv8_pair<BF16, true>(w1, s1)};
}

// Split-KV partial rows of these kernels: fp16 under a power of two of the
// row's own, three bits more than a bf16 row at the same size.  For fp16 results
// of tiles, whose probabilities are rounded as well, that would be a third
// rounding (1.7 times the error of the output's alone, 1.4 without it): there the
// remainder of each value, at most 2^-11 of the scale, goes along as an e4m3 code
// in units of 2^-19.  (Calls
// without tiles have none: their probabilities have two parts, and 24 sequences
// of 5 rows took 52.3 us with remainders and one part, 46.4 so.  32 draft blocks
// take 143 us with them, 139 without.)
// mx: the row's largest magnitude; returns the scale s with mx in [s, 2 s), and
// its inverse.
constexpr float kPartLo = 0x1p19f;
__device__ __forceinline__ float part_scale_of(float mx, float& inverse) {
  const uint32_t s = min(max(__float_as_uint(mx) & kInfBits, 1u << 23), 253u << 23);
  inverse = __uint_as_float((254u << 23) - s);
  return __uint_as_float(s);
}

}  // namespace feattn
