// The 8-bit paged cache: e4m3 values with a scale for each block of tokens and kv head.  A cache is
// [pages, page_size, kv_heads, dim] bytes, its scales fp32 [pages, page_size / block, kv_heads]; an element is its
// byte's value times its block's scale.  Blocks are 16, 32 or 64 tokens, pages whole numbers of blocks.
//
// Scales are powers of two: dividing by one is exact, so an element is rounded once, and a block that takes
// another scale (a larger element is appended, a token comes from another block) keeps its elements' bits, but for
// those that fall below e4m3's normal numbers, 2^-14 of the block's largest.  With any other scale each change would
// round all elements again.  A power of two leaves up to one bit of the exponent's range unused, which costs
// subnormals only.
#pragma once

#include "fnx_common.cuh"
#include "fnx_kernels.h"

namespace fnx {

constexpr int kLowestScale = -40;  // exponent of the smallest scale: blocks of zeros have it

// Scales that no append writes (not positive, infinite, NaN or below the smallest) count as the smallest.
__device__ __forceinline__ float scale_or_least(float s) {
  return s >= 0x1p-40f && s <= 0x1p120f ? s : 0x1p-40f;
}
// The smallest power of two, 2^kLowestScale at least, by which `amax` (finite) divided is at most 448 = 7/4 2^8.
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x007FFFFFu) > 0x00600000u ? 1 : 0);
  return __uint_as_float((uint32_t)((e < kLowestScale ? kLowestScale : e) + 127) << 23);
}
// The smallest power of two that is at least s (finite, not below the smallest scale).
__device__ __forceinline__ float power_above(float s) {
  const uint32_t bits = __float_as_uint(s);
  return __uint_as_float((bits + 0x007FFFFFu) & 0xFF800000u);
}

// Two 16-bit elements as floats, and two floats rounded to 16 bits.
template <typename T> __device__ __forceinline__ float2 two_floats(uint32_t w);
template <> __device__ __forceinline__ float2 two_floats<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <> __device__ __forceinline__ float2 two_floats<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
template <typename T> __device__ __forceinline__ uint32_t round_pair(float lo, float hi);
template <> __device__ __forceinline__ uint32_t round_pair<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
template <> __device__ __forceinline__ uint32_t round_pair<__half>(float lo, float hi) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// Two values rounded to e4m3 (to the nearest, ties to even; NaN stays NaN), the first in the low byte.
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_four(const float* x) {
  return e4m3_pair(x[0], x[1]) | (e4m3_pair(x[2], x[3]) << 16);
}
// Four bytes' values times `ratio`, rounded again.
__device__ __forceinline__ uint32_t e4m3_scaled(uint32_t w, float ratio) {
  uint32_t lo, hi;
  deq_fp8_word(w, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo)), b = __half22float2(*reinterpret_cast<__half2*>(&hi));
  return e4m3_pair(a.x * ratio, a.y * ratio) | (e4m3_pair(b.x * ratio, b.y * ratio) << 16);
}

}  // namespace fnx
