// 8-bit floating point with block scales: the power of two of a block, and conversions to e4m3 (4 exponent bits, 3 of fraction, largest 448).
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

namespace bspec {

// the bits of max |x| -> the e8m0 code of the block, and 1 / s
__device__ __forceinline__ int scale_code(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255;
  if (amax_bits == 0u) return 127;
  const int code = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);   // above 1.75 x 2^e: 448 = 1.75 x 2^8
  return code < 0 ? 0 : code;
}
__device__ __forceinline__ float inverse_scale(int code) {
  return code == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)(254 - code) << 23);
}
// two float32 numbers -> two e4m3 numbers, the first in the low byte
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t to_e4m3x4(const float* v, float inv) {
  return to_e4m3x2(v[0] * inv, v[1] * inv) | (to_e4m3x2(v[2] * inv, v[3] * inv) << 16);
}
// the value of an e8m0 code
__device__ __forceinline__ float scale_value(uint32_t code) {
  return __uint_as_float(code == 0u ? 0x00400000u : (code == 255u ? 0x7fc00000u : code << 23));
}
// Whether the product f of two scales leaves float32's normal range although neither is 0 or infinite: such a product keeps few bits or none
// (a sum of 128 products of e4m3 numbers, up to 2^25, brings 2^-140 back into the range), or turns a sum of 0 into NaN.
__device__ __forceinline__ bool leaves_range(float x, float w, float f) {
  return (fabsf(f) < 1.17549435e-38f && x != 0.f && w != 0.f) || (isinf(f) && !isinf(x) && !isinf(w));
}
// whether f is a normal number: what leaves_range holds for is not
__device__ __forceinline__ bool is_ordinary(float f) { return ((__float_as_uint(f) & 0x7fffffffu) - 0x00800000u) < 0x7f000000u; }
// Such a product as two factors with half of its exponent each: a sum that meets one after the other stays in the range if the result does.
__device__ __forceinline__ void split_scales(float x, float w, float& first, float& second) {
  int ex, ew;
  const float mx = frexpf(x, &ex), mw = frexpf(w, &ew);
  const int half = (ex + ew) >> 1;
  first = ldexpf(mx, half);
  second = ldexpf(mw, ex + ew - half);
}
// Two e4m3 numbers for one: v * inv = a + b / 16, a the nearest e4m3 number, b what is left, times 16 (|b| <= |a| where a is not among
// the smallest numbers; exact for a v of 8 bits).  Two values, and four, packed with the first in the low byte.
__device__ __forceinline__ void two_e4m3x2(float v0, float v1, float inv, uint32_t& a, uint32_t& b) {
  v0 *= inv;
  v1 *= inv;
  a = to_e4m3x2(v0, v1);
  uint32_t halves;                               // two e4m3 numbers as float16 numbers
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(halves) : "h"((uint16_t)a));
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&halves));
  b = to_e4m3x2((v0 - f.x) * 16.f, (v1 - f.y) * 16.f);
}
__device__ __forceinline__ void two_e4m3x4(const float* v, float inv, uint32_t& a, uint32_t& b) {
  uint32_t a0, a1, b0, b1;
  two_e4m3x2(v[0], v[1], inv, a0, b0);
  two_e4m3x2(v[2], v[3], inv, a1, b1);
  a = a0 | (a1 << 16);
  b = b0 | (b1 << 16);
}

}  // namespace bspec
