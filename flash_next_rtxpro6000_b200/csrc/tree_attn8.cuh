// What both forms of tree attention over an 8-bit cache share: places with their scales, and how scales and query
// rows enter the softmax.
//
// A key is s_k(block) k8, a value s_v(block) v8, with k8 and v8 bytes that fp16 holds exactly, so both products run
// on fp16 operands.  In base-2 units the score is t = c (q k8) s_k, and a row's result
//
//   sum_j 2^t_j s_v v8_j / sum_j 2^t_j  =  sum_j w_j v8_j / sum_j w_j / s_v(j),     w_j = 2^(t_j + log2 s_v(j) - ref):
//
// the value's scale goes into the exponent, where it costs an addend that is there anyway, and the sum divides it out
// again, once a group of 16 keys (blocks are whole groups).  The running reference is of w, so fp16 weights keep
// their bits whatever the scales of the values are (tree_attn.cuh says why and by what margin).
//
// A query row takes a power of two that brings its largest element to [2^14, 2^15), exact for bf16 elements down to
// 2^-28 of the row's largest, and gives it back in c.
#pragma once

#include "cache8.cuh"
#include "tree_attn.cuh"

namespace fnx {

constexpr int kGroup = 16;  // keys with one scale

// Byte offsets of key position pos of request b (its head included) in the caches, and of its block's scales; -1
// where there is none.
struct Place8 {
  int64_t k, v, ks, vs;
};
__device__ __forceinline__ Place8 attn8_place(const Attn8Args& a, int b, int pos, int len, int head) {
  Place8 r{-1, -1, -1, -1};
  if (pos >= len) return r;
  const int p = pos / a.page_size, in = pos - p * a.page_size;
  const int page = a.page_table[(int64_t)b * a.table_ld + p];
  if (page < 0 || page >= a.num_pages) {
    record_error(a.err, ERR_PAGE);
    return r;
  }
  const int blk = in / a.block;
  r.k = (int64_t)page * a.kc_st[0] + (int64_t)in * a.kc_st[1] + (int64_t)head * a.kc_st[2];
  r.v = (int64_t)page * a.vc_st[0] + (int64_t)in * a.vc_st[1] + (int64_t)head * a.vc_st[2];
  r.ks = (int64_t)page * a.ks_st[0] + (int64_t)blk * a.ks_st[1] + (int64_t)head * a.ks_st[2];
  r.vs = (int64_t)page * a.vs_st[0] + (int64_t)blk * a.vs_st[1] + (int64_t)head * a.vs_st[2];
  return r;
}

// A group's (s_k, log2 s_v, 1 / s_v); ones where there are no keys.
__device__ __forceinline__ float4 group_scales(const Attn8Args& a, const Place8& p) {
  if (p.ks < 0) return make_float4(1.f, 0.f, 1.f, 0.f);
  float ks = a.k_scale[p.ks], vs = a.v_scale[p.vs];
  const float k = scale_or_least(ks), v = scale_or_least(vs);
  if (!(k == ks) || !(v == vs)) record_error(a.err, ERR_SCALE);
  return make_float4(k, log2f(v), 1.f / v, 0.f);
}

// Whether one of the four bytes is a NaN.
__device__ __forceinline__ bool has_nan(uint32_t w) { return (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0u; }

__device__ __forceinline__ float e4m3_value(uint8_t v) {
  uint32_t lo, hi;
  deq_fp8_word(v, lo, hi);
  return __half2float(*reinterpret_cast<const __half*>(&lo));
}

// Two query elements as floats.
template <typename T> __device__ __forceinline__ float2 query_two(uint32_t w);
template <> __device__ __forceinline__ float2 query_two<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <> __device__ __forceinline__ float2 query_two<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }

template <typename T> __device__ __forceinline__ uint32_t round_pair(float lo, float hi);
template <> __device__ __forceinline__ uint32_t round_pair<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
template <> __device__ __forceinline__ uint32_t round_pair<__half>(float lo, float hi) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// Exponent of the power of two that a row with this largest magnitude takes; 0 where it is not finite.
__device__ __forceinline__ int row_exponent(float amax) {
  if (!(amax > 0.f) || !(amax < INFINITY)) return 0;
  const int e = 14 + 127 - (int)(__float_as_uint(amax) >> 23);
  return e > 100 ? 100 : e;
}

}  // namespace fnx
