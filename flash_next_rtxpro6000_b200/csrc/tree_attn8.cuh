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
// In two steps, since the first waits for nothing: a warp that asks for a page number and tests it at once stands still
// for an L2 access.
struct Look8 {
  int page, in, head;  // in -1: no such key
};
__device__ __forceinline__ Look8 attn8_look(const Attn8Args& a, int b, int pos, int len, int head) {
  Look8 l{0, -1, head};
  if (pos < len) {
    const int p = pos / a.page_size;
    l.in = pos - p * a.page_size;
    l.page = __ldg(a.page_table + (int64_t)b * a.table_ld + p);
  }
  return l;
}
__device__ __forceinline__ Place8 attn8_place(const Attn8Args& a, const Look8& l) {
  Place8 r{-1, -1, -1, -1};
  if (l.in < 0) return r;
  if (l.page < 0 || l.page >= a.num_pages) {
    record_error(a.err, ERR_PAGE);
    return r;
  }
  const int blk = l.in / a.block;
  r.k = (int64_t)l.page * a.kc_st[0] + (int64_t)l.in * a.kc_st[1] + (int64_t)l.head * a.kc_st[2];
  r.v = (int64_t)l.page * a.vc_st[0] + (int64_t)l.in * a.vc_st[1] + (int64_t)l.head * a.vc_st[2];
  r.ks = (int64_t)l.page * a.ks_st[0] + (int64_t)blk * a.ks_st[1] + (int64_t)l.head * a.ks_st[2];
  r.vs = (int64_t)l.page * a.vs_st[0] + (int64_t)blk * a.vs_st[1] + (int64_t)l.head * a.vs_st[2];
  return r;
}
__device__ __forceinline__ Place8 attn8_place(const Attn8Args& a, int b, int pos, int len, int head) {
  return attn8_place(a, attn8_look(a, b, pos, len, head));
}

// What the softmax needs of a group's scales (s_k, s_v): s_k, log2 s_v, 1 / s_v.
__device__ __forceinline__ float4 group_factors(const Attn8Args& a, float2 s) {
  const float k = scale_or_least(s.x), v = scale_or_least(s.y);
  if (!(k == s.x) || !(v == s.y)) record_error(a.err, ERR_SCALE);
  return make_float4(k, __log2f(v), __fdividef(1.f, v), 0.f);
}
// Those of the key at p; ones where there is none.
__device__ __forceinline__ float4 group_scales(const Attn8Args& a, const Place8& p) {
  return group_factors(a, p.ks < 0 ? make_float2(1.f, 1.f) : make_float2(a.k_scale[p.ks], a.v_scale[p.vs]));
}

// 16 bytes into shared memory, zeros where they are not there.
__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// Whether one of the four bytes is a NaN.
__device__ __forceinline__ bool has_nan(uint32_t w) { return (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0u; }

__device__ __forceinline__ float e4m3_value(uint8_t v) {
  uint32_t lo, hi;
  deq_fp8_word(v, lo, hi);
  return __half2float(*reinterpret_cast<const __half*>(&lo));
}

// Exponent of the power of two that a row with this largest magnitude takes; 0 where it is not finite.
__device__ __forceinline__ int row_exponent(float amax) {
  if (!(amax > 0.f) || !(amax < INFINITY)) return 0;
  const int e = 14 + 127 - (int)(__float_as_uint(amax) >> 23);
  return e > 100 ? 100 : e;
}

}  // namespace fnx
