// Paged KV cache held in 8 bits: e4m3 codes in 16-token pages, one scale per (page, kv head) for the keys and one for the values.
//
//   k codes [pages][Hkv][4][16][D/4]  four runs of D/4 dims, within a run the page's tokens: a lane of an MFMA A operand (16 tokens x 4
//                                     k-groups) finds its D/4 dims in one piece, a page and run is contiguous (512 B at D = 128)
//   v codes [pages][Hkv][D][16]       a dim's 16 tokens in one 16-byte load (the A operand of O^T = V^T P^T)
//   scales  [pages][Hkv][2]           fp32: keys', values'
//
// A scale is the least power of two s with amax <= 448 s (448: e4m3's largest number), at least 2^-100.  A power of two costs no
// precision - e4m3 is a floating type, a scale between two powers only moves its binade - and it makes three things exact: code * s
// has e4m3's 4 significant bits, so it is a bf16 number (v_cvt_scalef32_pk_bf16_fp8 yields two of them in one instruction, with the
// scale in it); x / s only moves the exponent; and a page whose scale grows when a later token is larger has its codes rounded anew
// without error, but for those that become subnormal.
#pragma once
#include "common.h"

namespace k8sllm {

constexpr int kPage = 16;
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// 448 = 1.75 * 2^8: the mantissa's carry past 1.75 takes the next power of two
__device__ __forceinline__ float kv8_scale(float amax) {
  const int e = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 8;
  return __uint_as_float((uint32_t)max(e, 27) << 23);  // 27: 2^-100
}
// 1 / s of a power of two between 2^-100 and 2^120
__device__ __forceinline__ float kv8_inverse(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

__device__ __forceinline__ float kv8_finite(float x) {  // |x|, 0 for infinities and NaN
  const float a = __builtin_fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// Four numbers over s as codes, the first in the low byte (to nearest, halves to even).  Non-finite ones become NaN codes.
__device__ __forceinline__ uint32_t kv8_codes(float a, float b, float c, float d, float inv) {
  const float nan = __uint_as_float(0x7fc00000u);
  a = __builtin_fabsf(a) < INFINITY ? a * inv : nan;
  b = __builtin_fabsf(b) < INFINITY ? b * inv : nan;
  c = __builtin_fabsf(c) < INFINITY ? c * inv : nan;
  d = __builtin_fabsf(d) < INFINITY ? d * inv : nan;
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}

// Two packed pairs of bf16 numbers over s, as above: the conversion takes bf16 as it lies and s with it.  Infinities and NaN are NaN codes.
typedef short s16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t kv8_codes_bf16(uint32_t a, uint32_t b, float s) {
  s16x2 r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(s16x2{0, 0}, __builtin_bit_cast(bf16x2, a), s, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, b), s, true);
  return __builtin_bit_cast(uint32_t, r);
}

// Larger magnitudes of packed bf16 pairs, as 16-bit patterns; 0x7f80 and more: not finite
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t kv8_max_bits(uint32_t m, uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
}
__device__ __forceinline__ uint32_t kv8_finite_bits(uint32_t w) {  // numbers that are not finite as zeros
  const uint32_t lo = (w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu, hi = (w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u;
  return lo | hi;
}

// Codes under a scale that grew: ratio = old / new
__device__ __forceinline__ uint32_t kv8_again(uint32_t w, float ratio) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  return __builtin_amdgcn_cvt_pk_fp8_f32(b[0] * ratio, b[1] * ratio, __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * ratio, a[1] * ratio, 0, false),
                                         true);
}

// eight codes times their scale as bf16 (exact)
__device__ __forceinline__ bf16x8 kv8_values(uint32_t lo, uint32_t hi, float s) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// the bytes of word w (tokens 4 w .. 4 w + 3 of a page) that are below n
__device__ __forceinline__ uint32_t kv8_below(int n, int w) {
  const int k = n - 4 * w;
  return k >= 4 ? 0xffffffffu : k <= 0 ? 0u : (1u << (8 * k)) - 1u;
}

}  // namespace k8sllm
