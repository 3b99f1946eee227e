// Sampling with temperature, top-k, top-p and min-p from given random numbers.
//
// With m the row's maximum, token i has the weight  w_i = trunc(2^40 exp((x_i - m) / T)), a whole
// number, and all sums are sums of whole numbers in 64 bits: exact, so neither the split of a row nor
// the order of atomics changes a result.  In the order of falling logits (lower token first on ties):
//   top-k   keeps the first k;                                     S_k = their sum
//   top-p   keeps tokens until their sum reaches p S_k;
//   min-p   keeps tokens with exp((x_i - m) / T) >= min_p;
// each is a prefix of that order, so what is kept is the shortest of them, with the smallest of their
// sums S.  The token drawn is the one at which the running sum passes u S.  Every question is of one
// kind: at which token does the running count, or sum, reach a value.
//
// Bound: one read of the logits (memory); below about a megabyte, the chain of steps.
// A row belongs to a cluster of CTAs that read their slices from global memory once.  Steps:
// (1) maximum and minimum.
// (2) Where top-k leaves up to kFew tokens: each thread has the maximum of its own logits, and the
//     r-th largest of a CTA's 512 is a value that at least r of its logits reach; the smallest of
//     these over C CTAs is one that r C >= k tokens of the row reach, in practice not many more.  They
//     go to the first CTA, which sorts them and has all answers in their running sums.
// (3) Elsewhere, or where those tokens do not fit into the list: a histogram of sums (and counts, if
//     there is a top-k) over kBins intervals of m - x of equal width, which is a partition in the
//     right order because m - x falls as x grows.
// (4) The first CTA finds the intervals in which the values are reached, the cluster sends it their
//     tokens, and it sorts them and reads the token off their running sums.  The last value, the
//     random share of what top-p keeps, is known within the weight of top-p's interval beforehand, so
//     both values' intervals are sent at once.  An interval with more tokens than the list holds
//     (many ties, or one token far from the others) is split again by order key and token index
//     until it fits.
// Measured (B200): one row of 151,936 bf16 logits 10 us with a top-k of 50, 21 to 25 without filters or with top-p or
// min-p, 36 where top-p's interval holds more tokens than the list, 37 with a top-k of 5,000 (of some 57,000 cycles the
// histogram's pass takes 15,000 to 19,000, its exponentials and shared-memory adds in equal parts, the gathering 9,000, the
// exchanges about 1,500 each); 16 such rows in fp32 19, 41 to 44 and 62 us; 128 rows of 248,320 51 and 144 to 151 us (175 to
// 234 with a division and a 64-bit shift a logit in place of quotient() and add_share()).  Two other ways were measured: a list of the likely tokens, made while all weights are added up, in
// place of the histogram (31 and 92 us where it decides, 65 and 240 where it does not and the histogram follows), and a
// histogram of counts, then exact sums around the interval that it points at (44 to 52, 128 to 240 us).  The form for
// many rows has 64 registers a thread and spills some 500 bytes of them.
#pragma once

#include <cooperative_groups.h>

#include <type_traits>

#include "fnx_common.cuh"
#include "fnx_kernels.h"

namespace fnx {

namespace {

// Lambdas are inlined by force.  Where the compiler left one out (the third kernel of a unit, say), all that it captures went
// to local memory: 16 rows of 151,936 logits without top-k took 77 us instead of 56.
#define FNX_INLINE __attribute__((always_inline))
// The steps' lambdas, unless the unit leaves them to the compiler (sample.cu).
#ifndef FNX_INLINE_STEP
#define FNX_INLINE_STEP FNX_INLINE
#endif

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kST = 512;          // threads
constexpr int kBins = 2048;       // intervals of m - x
constexpr int kSub = kST;         // intervals of a stretch, or a split
constexpr int kCap = 2048;        // tokens of the list
constexpr int kShort = 256;       // tokens of a list that is ranked token by token
constexpr int kFew = 1024;        // largest top-k served by the list alone
constexpr u64 kOne = 1ull << 40;  // the weight of the most likely token
// exp(-28) < 2^-40: tokens further below the maximum have no weight and are not looked at
constexpr float kReach = 28.0f;
constexpr uint32_t kLowest = 0x00800000u;  // order bits of the lowest finite fp32 value

enum Want : int { WANT_COUNT = 0, WANT_SHARE = 1, WANT_SUM = 2 };
enum Op : int { OP_DONE = 0, OP_GATHER = 1, OP_SPLIT = 2 };
constexpr int kCluster = 8;  // CTAs of a row, at most

struct Control {  // written by the first CTA, read by the cluster
  int op;
  int bin_lo, bin_hi, bin2_lo, bin2_hi;  // the tokens of two ranges of intervals ...
  u64 key_lo, key_hi;                    // ... with keys in this range
};

struct Local {  // written by each CTA, read by the others
  u64 best;       // largest key of the slice
  uint32_t floor;  // order bits that as many logits of the slice reach as are its part of the list
  float low;      // smallest finite logit
  u64 min_sum;    // sum of the weights that min-p keeps
  u64 key_lo, key_hi;  // smallest and largest key of a split
};

struct Bins {
  uint32_t count[kBins], w0[kBins], w1[kBins], w2[kBins];
};

struct Found {  // a token: the running sum up to and with it, its weight
  u64 sum, weight;
  int token;
};

struct SampleSmem {
  alignas(16) Bins h;
  u64 list[kCap];  // first CTA: the tokens sent to it
  u64 mine_found[kCap];  // this CTA's finds, before they are sent
  // first CTA: exclusive running counts and sums of the row's intervals, and of a split's
  u64 sum[kBins + 1];
  uint32_t count[kBins + 1];
  union {
    struct { u64 sub_sum[kSub + 1]; uint32_t sub_count[kSub + 1]; };
    uint32_t pick[2][kST];
  };
  u64 likely;
  int at_bin[8];
  Found found_token;
  // two buffers of kCap keys for the first CTA, where its histogram was
  __device__ __forceinline__ u64* scratch() { return reinterpret_cast<u64*>(&h); }
  Control ctl;
  Local mine;
  uint32_t listed;  // first CTA: tokens sent to the list
  uint32_t finds;   // tokens found by this CTA
  uint32_t place;   // and their place in the list
  uint32_t picked;  // tokens of an interval that is looked at closely
  int found;
  u64 red[kST / 32];
  uint32_t red_c[kST / 32];
  float red_f[kST / 32];
};

__device__ __forceinline__ uint32_t order_bits(float f) {
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
}
// Larger for larger logits, then for lower tokens; -0 counts as 0 so that the two tie.
__device__ __forceinline__ u64 make_key(float x, uint32_t token) {
  return ((u64)order_bits(x + 0.0f) << 32) | (0xFFFFFFFFu - token);
}
__device__ __forceinline__ float key_value(u64 k) { return order_value((uint32_t)(k >> 32)); }
__device__ __forceinline__ int key_token(u64 k) { return (int)(0xFFFFFFFFu - (uint32_t)k); }

__device__ __forceinline__ float logit(const float v) { return v; }
__device__ __forceinline__ float logit(const __nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float logit(const __half v) { return __half2float(v); }

// The nearest whole number to x in [0, 2^22]: the low bits of x + 2^23.
__device__ __forceinline__ int nearest(float x) { return (int)(__float_as_uint(x + 8388608.0f) & 0x007FFFFFu); }

// The row's scale: everything a thread needs to place a logit.
struct Scale {
  float m, T, range, inv, min_p;
  // exp((x - m) / T); the maximum's is 1 also where it is infinite
  __device__ __forceinline__ float share(float x) const {
    if (x == m) return 1.0f;
    return expf(T == 1.0f ? x - m : (x - m) / T);
  }
  // trunc(2^40 e) for e in [0, 1]: the significand, shifted (the conversion instruction shares its
  // slow unit with the exponential)
  static __device__ __forceinline__ u64 weight(float e) {
    const uint32_t bits = __float_as_uint(e);
    const int up = (int)(bits >> 23) - (127 + 23 - 40);
    const u64 m = (bits & 0x007FFFFFu) | 0x00800000u;
    return up >= 0 ? m << up : m >> min(-up, 63);
  }
  // (x - m) / T for tokens with weight, something without for others; `by` is T's reciprocal in two parts.  a by.x + a by.y
  // is the quotient but for one unit in its last place at most and its remainder is exact, so one more step gives the
  // correctly rounded quotient (Markstein's theorem; by.x is the correctly rounded reciprocal).  Where `plain`: finite m
  // and T in [2^-60, 2^60]; quotients so small that the remainder is not exact have an exponential of 1 all the same.
  __device__ __forceinline__ bool plain() const { return m < INFINITY && T >= 0x1p-60f && T <= 0x1p60f; }
  __device__ __forceinline__ float2 reciprocal() const {
    const float y = __frcp_rn(T);
    return make_float2(y, fmaf(-y, T, 1.0f) * y);
  }
  __device__ __forceinline__ float quotient(float x, float2 by) const {
    const float a = fmaxf(x - m, -kReach * T);  // of NaN, too
    const float q = fmaf(a, by.x, a * by.y);
    return fmaf(fmaf(-q, T, a), by.x, q);
  }
  // the interval of x, or -1 for a token without weight (NaN and -inf among them)
  __device__ __forceinline__ int bin(float x) const {
    const float d = x == m ? 0.0f : m - x;
    return d <= range ? nearest(fminf(d * inv, (float)(kBins - 1))) : -1;
  }
};

__device__ __forceinline__ u64 warp_max(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  return v;
}
__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Exclusive running count and sum over the block of one pair per thread; the totals come back too.
__device__ __forceinline__ void block_scan(SampleSmem& s, uint32_t c, u64 v, uint32_t& c_before, u64& v_before,
                                           uint32_t& c_all, u64& v_all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t ci = c;
  u64 vi = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t cu = __shfl_up_sync(0xffffffffu, ci, o);
    const u64 vu = __shfl_up_sync(0xffffffffu, vi, o);
    if (lane >= o) ci += cu, vi += vu;
  }
  __syncthreads();  // the scratch may still be read from the call before
  if (lane == 31) s.red_c[warp] = ci, s.red[warp] = vi;
  __syncthreads();
  c_before = ci - c, v_before = vi - v, c_all = 0, v_all = 0;
#pragma unroll
  for (int w = 0; w < kST / 32; ++w) {
    const uint32_t cw = s.red_c[w];
    const u64 vw = s.red[w];
    if (w < warp) c_before += cw, v_before += vw;
    c_all += cw, v_all += vw;
  }
}

// Adds to a word of this CTA's shared memory, without a branch where there is nothing to add.
__device__ __forceinline__ void add_shared(uint32_t addr, uint32_t v) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "@p red.relaxed.cta.shared::cta.add.u32 [%0], %1;\n\t}" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t next_shared(uint32_t addr) {
  uint32_t old;
  asm volatile("atom.relaxed.cta.shared::cta.add.u32 %0, [%1], 1;" : "=r"(old) : "r"(addr) : "memory");
  return old;
}

// Adds a weight (41 bits) to an interval's sum, kept as three 32-bit sums of 14 bits each (shared
// memory has no 64-bit add): 2^18 weights fit, and a CTA has no more logits.  Nothing is waited for,
// and most tokens' weights are too small for the upper ones.
__device__ __forceinline__ void add_sum(uint32_t w0_of_bin, u64 w) {
  const uint32_t w0 = (uint32_t)w & 0x3FFFu, w1 = (uint32_t)(w >> 14) & 0x3FFFu, w2 = (uint32_t)(w >> 28);
  add_shared(w0_of_bin, w0);
  add_shared(w0_of_bin + kBins * 4, w1);
  add_shared(w0_of_bin + kBins * 8, w2);
}
// The same of trunc(2^40 e): adding 2^(23 - k), rounded towards 0, leaves the whole number of 2^-k in a float's lowest bits.
__device__ __forceinline__ void add_share(uint32_t w0_of_bin, float e) {
  const float h = __fadd_rz(e, 0x1p11f), a = e - (h - 0x1p11f);     // 2^-12
  const float i = __fadd_rz(a, 0x1p-3f), b = a - (i - 0x1p-3f);     // 2^-26
  const float l = __fadd_rz(b, 0x1p-17f);                          // 2^-40
  add_shared(w0_of_bin, __float_as_uint(l) - 0x37000000u);
  add_shared(w0_of_bin + kBins * 4, __float_as_uint(i) - 0x3E000000u);
  add_shared(w0_of_bin + kBins * 8, __float_as_uint(h) - 0x45000000u);
}
__device__ __forceinline__ u64 sum_of(const Bins& h, int b) {
  return h.w0[b] + ((u64)h.w1[b] << 14) + ((u64)h.w2[b] << 28);
}

// Sorts n keys in falling order: a bitonic network with E keys a thread, exchanged within the thread,
// then by shuffles, and through shared memory only from 32 E keys apart on.  `a` holds the keys and
// the answer; it takes turns with `b`, one barrier a step.
template <int E>
__device__ __forceinline__ void sort_keys(u64* a, u64* b, int n, int p) {
  const int tid = threadIdx.x;
  u64 v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = tid * E + e < n ? a[tid * E + e] : 0ull;
  __syncthreads();
  bool odd = false;
  for (int size = 2; size <= p; size <<= 1) {
    for (int d = size >> 1; d > 0; d >>= 1) {
      u64 w[E];
      if (d >= 32 * E) {
        u64* buf = odd ? b : a;
        odd = !odd;
#pragma unroll
        for (int e = 0; e < E; ++e) buf[tid * E + e] = v[e];
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) w[e] = buf[(tid * E + e) ^ d];
      } else if (d >= E) {
#pragma unroll
        for (int e = 0; e < E; ++e) w[e] = __shfl_xor_sync(0xffffffffu, v[e], d / E);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) w[e] = d == 1 ? v[E > 1 ? e ^ 1 : e] : v[E == 4 ? e ^ 2 : e];
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = tid * E + e;
        const bool larger = ((i & d) == 0) == ((i & size) == 0);
        v[e] = (v[e] > w[e]) == larger ? v[e] : w[e];
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) a[tid * E + e] = v[e];
  __syncthreads();
}

// The r-th largest (from 1) of one 32-bit value per thread.
__device__ __forceinline__ uint32_t rth_largest(SampleSmem& s, uint32_t v, int r) {
  const int tid = threadIdx.x;
  bool odd = false;
  for (int size = 2; size <= kST; size <<= 1) {
    for (int d = size >> 1; d > 0; d >>= 1) {
      uint32_t w;
      if (d >= 32) {
        uint32_t* buf = s.pick[odd];
        odd = !odd;
        buf[tid] = v;
        __syncthreads();
        w = buf[tid ^ d];
      } else {
        w = __shfl_xor_sync(0xffffffffu, v, d);
      }
      const bool larger = ((tid & d) == 0) == ((tid & size) == 0);
      v = larger ? max(v, w) : min(v, w);
    }
  }
  if (tid == r - 1) s.found = (int)v;
  __syncthreads();
  return (uint32_t)s.found;
}

// Whether a running count / sum has reached the wanted value.
__device__ __forceinline__ bool reached(int want, u64 count, u64 sum, u64 value, double share) {
  return want == WANT_COUNT ? count >= value : want == WANT_SHARE ? (double)sum >= share : sum >= value;
}

// The first of nb intervals (exclusive running counts / sums, nb + 1 entries) in which it is reached.
__device__ __forceinline__ int find_bin(SampleSmem& s, const uint32_t* count, const u64* sum, int nb, u64 base_count,
                                        u64 base_sum, int want, u64 value, double share) {
  __syncthreads();
  if (threadIdx.x == 0) s.found = nb - 1;
  __syncthreads();
  for (int b = threadIdx.x; b < nb; b += kST) {
    if (reached(want, base_count + count[b + 1], base_sum + sum[b + 1], value, share) &&
        !reached(want, base_count + count[b], base_sum + sum[b], value, share))
      s.found = b;
  }
  __syncthreads();
  return s.found;
}

// A short list: thread i has the i-th token and what lies ahead of it.
struct Ranked {
  u64 key, weight, sum;
  uint32_t count;
};
__device__ __forceinline__ Ranked rank_list(SampleSmem& s, const Scale& sc, int held, u64& likely) {
  const int tid = threadIdx.x;
  Ranked r{0ull, 0ull, 0ull, 0u};
  __syncthreads();
  if (tid == 0) s.likely = 0ull;
  u64* weight = s.scratch();
  if (tid < held) {
    r.key = s.list[tid];
    const float e = sc.share(key_value(r.key));
    r.weight = Scale::weight(e);
    weight[tid] = r.weight;
  }
  __syncthreads();
  if (tid < held) {
#pragma unroll 4
    for (int j = 0; j < held; ++j) {
      const bool ahead = s.list[j] > r.key;
      r.sum += ahead ? weight[j] : 0ull;
      r.count += ahead ? 1u : 0u;
    }
    if (sc.min_p > 0.0f && sc.share(key_value(r.key)) >= sc.min_p) atomicAdd(&s.likely, r.weight);
  }
  __syncthreads();
  likely = s.likely;
  return r;
}
__device__ __forceinline__ Found answer(SampleSmem& s, const Ranked& r, int held, u64 base_count, u64 base_sum, int want,
                                        u64 value, double share) {
  if ((int)threadIdx.x < held && reached(want, base_count + r.count + 1, base_sum + r.sum + r.weight, value, share) &&
      !reached(want, base_count + r.count, base_sum + r.sum, value, share))
    s.found_token = Found{base_sum + r.sum + r.weight, r.weight, key_token(r.key)};
  __syncthreads();
  const Found f = s.found_token;
  __syncthreads();
  return f;
}

// The running sum at which the token for u is reached: u of what is kept, and 1.
__device__ __forceinline__ u64 target_of(double u, u64 kept) {
  const u64 t = __double2ull_rz(u * (double)kept);
  return (t < kept - 1 ? t : kept - 1) + 1;
}

// The answer, of `kept` weight in all.
__device__ __forceinline__ void draw(const SampleArgs& a, int row, const Found& f, u64 kept) {
  if (threadIdx.x != 0) return;
  a.tokens[row] = f.token;
  a.probs[row] = (float)((double)f.weight / (double)kept);
}

// A stretch of the order, all of whose tokens are in the list: those with bin >= 0 (bin < 0: all of the
// list), cut into kSub intervals by  (m - x) scale - offset  in [0, 1].
struct Stretch {
  int bin;
  float scale, offset;
  // the interval of x, -1 for a token outside the stretch
  __device__ __forceinline__ int sub(const Scale& sc, float x) const {
    if (bin >= 0 && sc.bin(x) != bin) return -1;
    const float d = x == sc.m ? 0.0f : sc.m - x;
    return nearest(fminf(fmaxf((d * scale - offset) * (float)kSub, 0.0f), (float)(kSub - 1)));
  }
};

// Running counts and sums of a stretch's intervals; returns what min-p keeps of it.
__device__ __forceinline__ u64 measure(SampleSmem& s, const Scale& sc, const Stretch& st, int held) {
  const int tid = threadIdx.x;
  const uint32_t count0 = smem_u32(s.h.count), sum0 = smem_u32(s.h.w0);
  __syncthreads();
  for (int b = tid; b < kSub; b += kST) s.h.count[b] = s.h.w0[b] = s.h.w1[b] = s.h.w2[b] = 0u;
  if (tid == 0) s.likely = 0ull;
  __syncthreads();
  u64 likely = 0ull;
  for (int i = tid; i < held; i += kST) {
    const float x = key_value(s.list[i]);
    const int b = st.sub(sc, x);
    if (b < 0) continue;
    const float e = sc.share(x);
    const u64 w = Scale::weight(e);
    add_shared(count0 + b * 4, 1u);
    add_sum(sum0 + b * 4, w);
    if (e >= sc.min_p) likely += w;
  }
  if (sc.min_p > 0.0f) {
    likely = warp_sum(likely);
    if ((tid & 31) == 0 && likely) atomicAdd(&s.likely, likely);
  }
  __syncthreads();
  static_assert(kSub == kST, "one interval a thread");
  uint32_t cb, c_all;
  u64 vb, v_all;
  block_scan(s, s.h.count[tid], sum_of(s.h, tid), cb, vb, c_all, v_all);
  s.sub_count[tid] = cb, s.sub_sum[tid] = vb;
  if (tid == 0) s.sub_count[kSub] = c_all, s.sub_sum[kSub] = v_all;
  __syncthreads();
  return s.likely;
}

// The token of a measured stretch at which the value is reached (base_count tokens of base_sum weight
// lie ahead of the stretch).
__device__ __forceinline__ Found answer(SampleSmem& s, const Scale& sc, const Stretch& st, int held, u64 base_count,
                                        u64 base_sum, int want, u64 value, double share) {
  const int tid = threadIdx.x, lane = tid & 31;
  const int b = find_bin(s, s.sub_count, s.sub_sum, kSub, base_count, base_sum, want, value, share);
  base_count += s.sub_count[b];
  base_sum += s.sub_sum[b];
  u64* few = s.scratch();  // the interval's tokens
  if (tid == 0) s.picked = 0u;
  __syncthreads();
  for (int i = tid; i < held; i += kST) {
    const u64 key = s.list[i];
    if (st.sub(sc, key_value(key)) == b) few[next_shared(smem_u32(&s.picked))] = key;
  }
  __syncthreads();
  const int n = (int)s.picked;
  if (n <= 32) {  // one warp: each lane's token gets what is ahead of it, in whatever order they lie
    if (tid < 32) {
      const u64 key = lane < n ? few[lane] : 0ull;
      const u64 w = lane < n ? Scale::weight(sc.share(key_value(key))) : 0ull;
      u64 sum = base_sum + w;
      int count = 1;
      for (int i = 0; i < n; ++i) {
        const u64 k = __shfl_sync(0xffffffffu, key, i), v = __shfl_sync(0xffffffffu, w, i);
        if (k > key) sum += v, ++count;
      }
      const bool here = reached(want, base_count + count, sum, value, share) &&
                        !reached(want, base_count + count - 1, sum - w, value, share);
      const bool last = count == n;  // taken where rounding lets no token reach the value
      const unsigned any = __ballot_sync(0xffffffffu, lane < n && here);
      if (lane < n && (any ? here : last)) s.found_token = Found{sum, w, key_token(key)};
    }
  } else {  // many ties
    int p = 64;
    while (p < n) p <<= 1;
    u64* spare = few + kCap;
    if (p <= kST) sort_keys<1>(few, spare, n, p);
    else if (p <= 2 * kST) sort_keys<2>(few, spare, n, p);
    else sort_keys<4>(few, spare, n, p);
    constexpr int kPer = kCap / kST;
    u64 w[kPer], mine = 0;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int i = tid * kPer + q;
      w[q] = i < n ? Scale::weight(sc.share(key_value(few[i]))) : 0ull;
      mine += w[q];
    }
    uint32_t c0, ca;
    u64 sum, all;
    block_scan(s, 0u, mine, c0, sum, ca, all);
    sum += base_sum;
    if (tid == 0) s.found = 0;
    __syncthreads();
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {  // second: the last token, if none reached the value
      u64 run = sum;
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        const int i = tid * kPer + q;
        if (i < n) {
          const bool here = reached(want, base_count + i + 1, run + w[q], value, share) &&
                            !reached(want, base_count + i, run, value, share);
          if (pass == 0 ? here : (s.found == 0 && i == n - 1)) {
            s.found_token = Found{run + w[q], w[q], key_token(few[i])};
            if (pass == 0) s.found = 1;
          }
        }
        run += w[q];
      }
      __syncthreads();
    }
  }
  __syncthreads();
  const Found f = s.found_token;
  __syncthreads();
  return f;
}

}  // namespace

// kMany: two CTAs on an SM, slices read from global memory (the L2 cache after the first time).
// kAll: not a token but what keeps a row's tokens apart from the others is wanted (token_probs).  The last token that is
// kept is the one that a random number of 1 draws.
template <typename T, bool kMany, bool kAll>
__global__ void __launch_bounds__(kST, kMany ? 2 : 1) sample_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  SampleSmem& s = *reinterpret_cast<SampleSmem*>(smem);
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), C = (int)cl.num_blocks();
  const int row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  SampleSmem& first = *cl.map_shared_rank(&s, 0);
  const uint32_t count0 = smem_u32(s.h.count), sum0 = smem_u32(s.h.w0), finds0 = smem_u32(&s.finds);
  const int v0 = rank * a.per;
  const int n = v0 >= a.V ? 0 : (a.V - v0 < a.per ? a.V - v0 : a.per);
  constexpr int kVec = 16 / sizeof(T);
  pdl_wait();
  const float uniform = kAll ? 1.0f : a.uniforms[row];
  const float Tm = a.temperature ? a.temperature[row] : 1.0f, top_p = a.top_p ? a.top_p[row] : 1.0f,
              min_p = a.min_p ? a.min_p[row] : 0.0f;
  const int top_k = a.top_k ? a.top_k[row] : 0;

  // --- (1) the slice into shared memory, with its maximum and minimum
  const T* g = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.ldl + v0;
  T* slice = reinterpret_cast<T*>(smem + ((sizeof(SampleSmem) + 15) & ~(size_t)15));
  const int off = (int)((reinterpret_cast<uintptr_t>(g) & 15) / sizeof(T));  // same place modulo 16 bytes
  const T* xs = kMany || !a.in_smem ? g : slice + off;
  const int head = min(n, off ? kVec - off : 0), vecs = (n - head) / kVec;

  // Calls f(number of logits, their values, place of the first) for the thread's logits of the
  // slice, a 16-byte vector at a time where the alignment allows; places rise within a thread.
  auto sweep = [&](auto&& f) FNX_INLINE {
    if (tid < head) {
      const float x[1] = {logit(xs[tid])};
      f(std::integral_constant<int, 1>{}, x, tid);
    }
    const uint4* xv = reinterpret_cast<const uint4*>(xs + head);
    uint4 ahead[2];  // slices that stay in global memory are read two vectors ahead
    int j = tid;
    if (j < vecs) ahead[0] = xv[j];
    if (j + kST < vecs) ahead[1] = xv[j + kST];
    while (j < vecs) {
#pragma unroll
      for (int z = 0; z < 2; ++z, j += kST) {
        if (j >= vecs) break;
        const uint4 v = ahead[z];
        if (j + 2 * kST < vecs) ahead[z] = xv[j + 2 * kST];
        const T* e = reinterpret_cast<const T*>(&v);
        float x[kVec];
#pragma unroll
        for (int q = 0; q < kVec; ++q) x[q] = logit(e[q]);
        f(std::integral_constant<int, kVec>{}, x, head + j * kVec);
      }
    }
    const int i = head + vecs * kVec + tid;
    if (i < n) {
      const float x[1] = {logit(xs[i])};
      f(std::integral_constant<int, 1>{}, x, i);
    }
  };

  float top = -INFINITY, low = INFINITY;
  int top_at = -1;
  auto look = [&](float x, int i) FNX_INLINE {
    if (x > top) top = x, top_at = i;  // strictly: the first of equal logits stays
    low = fminf(low, x > -INFINITY ? x : low);
  };
  {
    T* to = slice + off;
    if (tid < head) {
      const T v = g[tid];
      if (!kMany && a.in_smem) to[tid] = v;
      look(logit(v), tid);
    }
    const uint4* gv = reinterpret_cast<const uint4*>(g + head);
    uint4* tv = reinterpret_cast<uint4*>(to + head);
#pragma unroll 8
    for (int j = tid; j < vecs; j += kST) {
      const uint4 v = ldg_cg_u4(gv + j);
      if (!kMany && a.in_smem) tv[j] = v;
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int q = 0; q < kVec; ++q) look(logit(e[q]), head + j * kVec + q);
    }
    const int i = head + vecs * kVec + tid;
    if (i < n) {
      const T v = g[i];
      if (!kMany && a.in_smem) to[i] = v;
      look(logit(v), i);
    }
  }
  u64 best = top_at < 0 ? 0ull : make_key(top, (uint32_t)(v0 + top_at));
  const bool quick = top_k > 0 && top_k <= kFew;
  uint32_t floor = 0u;
  if (quick) floor = rth_largest(s, (uint32_t)(best >> 32), (top_k + C - 1) / C);  // at most kST: C >= 2
  best = warp_max(best);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  if (lane == 0) s.red[warp] = best, s.red_f[warp] = low;
  if (tid == 0) s.listed = s.finds = 0u;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kST / 32; ++w) {
      best = s.red[w] > best ? s.red[w] : best;
      low = fminf(low, s.red_f[w]);
    }
    s.mine.best = best;
    s.mine.low = low;
    s.mine.floor = floor;
  }
  cl.sync();
  best = 0ull;
  low = INFINITY;
#pragma unroll
  for (int c = 0; c < kCluster; ++c) {
    if (c >= C) break;
    const Local& o = cl.map_shared_rank(&s, c)->mine;
    best = o.best > best ? o.best : best;
    low = fminf(low, o.low);
    floor = min(floor, o.floor);
  }
  // Thread 0 of the first CTA leaves the row's kept tokens for the launch that writes the probabilities.
  auto leave = [&](int what, const Scale& sc, int last, u64 kept) FNX_INLINE {
    if (rank != 0 || tid != 0) return;
    KeptTokens k;
    k.what = what;
    k.m = sc.m;
    k.T = sc.T;
    k.last = last;
    k.low = what != KEPT_PREFIX ? 0.0f : last < 0 ? -INFINITY : logit(reinterpret_cast<const T*>(a.logits)[(int64_t)row * a.ldl + last]);
    k.kept = kept;
    a.rows[row] = k;
  };
  if (best == 0ull || !(Tm > 0.0f)) {  // nothing to draw from, or the most likely token
    if (kAll) {
      leave(KEPT_ONE, Scale{}, best ? key_token(best) : -1, 1ull);
    } else if (rank == 0 && tid == 0) {
      a.tokens[row] = best ? key_token(best) : -1;
      a.probs[row] = best ? 1.0f : 0.0f;
    }
    cl.sync();  // no CTA leaves while another reads its shared memory
    pdl_trigger();
    return;
  }
  Scale sc;
  sc.m = key_value(best);
  sc.T = fminf(Tm, 3.0e38f);
  sc.range = fminf(kReach * sc.T, sc.m - low);
  sc.inv = sc.range > 0.0f ? (float)(kBins - 1) / sc.range : 0.0f;
  const bool use_p = top_p < 1.0f;
  sc.min_p = min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f;

  const double u = uniform > 0.0f ? (double)uniform : 0.0;  // NaN and negative numbers draw the most likely token

  // A found token goes to the CTA's own finds, and these to the first CTA's list in one piece.
  auto find = [&](u64 key) FNX_INLINE_STEP {
    const uint32_t at = next_shared(finds0);
    if (at < (uint32_t)kCap) s.mine_found[at] = key;
  };
  auto send = [&]() FNX_INLINE_STEP {
    __syncthreads();
    const uint32_t m = s.finds;
    if (tid == 0) s.place = atomicAdd(&first.listed, m);
    __syncthreads();
    const uint32_t at = s.place;
    for (uint32_t i = tid; i < m && at + i < (uint32_t)kCap; i += kST) first.list[at + i] = s.mine_found[i];
    __syncthreads();
    if (tid == 0) s.finds = 0u;
  };

  // --- (2) the tokens that reach the floor
  if (quick) {
    const float least = order_value(floor > kLowest ? floor : kLowest);
    sweep([&](auto count, const float* x, int i0) FNX_INLINE {
      float most = x[0];
#pragma unroll
      for (int q = 1; q < count; ++q) most = fmaxf(most, x[q]);
      if (most >= least) {
#pragma unroll
        for (int q = 0; q < count; ++q)
          if (x[q] >= least) find(make_key(x[q], (uint32_t)(v0 + i0 + q)));
      }
    });
    send();
    cl.sync();
    const int held = (int)first.listed;
    if (held <= kCap) {
      if (rank == 0) {
        const float depth = sc.m - least;
        const Stretch st{-1, depth > 0.0f && depth < INFINITY ? 1.0f / depth : 0.0f, 0.0f};
        const bool few = held <= kShort;
        u64 by_share, kept;
        Ranked r;
        if (few) r = rank_list(s, sc, held, by_share);
        else by_share = measure(s, sc, st, held);
        auto ask = [&](int what, u64 value, double share) FNX_INLINE_STEP {
          return few ? answer(s, r, held, 0, 0, what, value, share) : answer(s, sc, st, held, 0, 0, what, value, share);
        };
        // the list holds at least top_k tokens, or all there are
        kept = ask(WANT_COUNT, (u64)min(top_k, held), 0.0).sum;
        if (use_p) {
          const double want = (double)top_p * (double)kept;
          kept = want > 0.0 ? ask(WANT_SHARE, 0ull, want).sum : kOne;
        }
        if (sc.min_p > 0.0f) kept = by_share < kept ? by_share : kept;
        const Found f = ask(WANT_SUM, target_of(u, kept), 0.0);
        if (kAll) leave(KEPT_PREFIX, sc, f.token, kept);
        else draw(a, row, f, kept);
      }
      cl.sync();  // the first CTA's count has been read by all before it leaves
      pdl_trigger();
      return;
    }
  }

  // --- all tokens are kept: their sum is the answer, no histogram is needed (16 rows 48 -> 22 us, 128 rows 230 -> 120,
  // with the probabilities' launch)
  if (kAll && top_k <= 0 && !use_p && !(sc.min_p > 0.0f) && sc.plain()) {
    const float2 by = sc.reciprocal();
    // whole numbers of 2^-17, and the rest (as in add_share); a thread has fewer than 2^15 tokens
    uint32_t high = 0u;
    u64 all = 0ull;
    sweep([&](auto count, const float* x, int) FNX_INLINE {
      uint32_t rest = 0u;
#pragma unroll
      for (int q = 0; q < count; ++q) {
        const float e = expf(sc.quotient(x[q], by));
        const float h = __fadd_rz(e, 64.0f), l = __fadd_rz(e - (h - 64.0f), 0x1p-17f);
        high += __float_as_uint(h) - 0x42800000u;
        rest += __float_as_uint(l) - 0x37000000u;
      }
      all += rest;
    });
    all = warp_sum(all + ((u64)high << 23));
    if (lane == 0) s.red[warp] = all;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kST / 32; ++w) all += s.red[w];
      s.mine.min_sum = all;
    }
    cl.sync();
    if (rank == 0) {
      all = 0ull;
      for (int r = 0; r < C; ++r) all += cl.map_shared_rank(&s, r)->mine.min_sum;
      leave(KEPT_PREFIX, sc, -1, all);
    }
    cl.sync();  // no CTA leaves while another reads its shared memory
    pdl_trigger();
    return;
  }

  // --- (3) histogram, with counts where there is a top-k
  const bool counts = top_k > 0;
  {
    for (int b = tid; b < kBins; b += kST) s.h.count[b] = s.h.w0[b] = s.h.w1[b] = s.h.w2[b] = 0u;
    __syncthreads();
    u64 min_sum = 0ull;
    // Weights of a whole vector first, so that their chains overlap.
    const float2 by = sc.reciprocal();
    auto fill = [&](auto plain) FNX_INLINE {
      sweep([&](auto count, const float* x, int) FNX_INLINE {
        float e[count];
#pragma unroll
        for (int q = 0; q < count; ++q) {
          if (plain) {
            e[q] = expf(sc.quotient(x[q], by));
            continue;
          }
          float d = x[q] - sc.m;
          const bool none = !(-d <= sc.range);  // NaN and -inf among them
          if (none || x[q] == sc.m) d = 0.0f;  // the division is slow where it meets an infinity
          e[q] = expf(d / sc.T);
          if (none && x[q] != sc.m) e[q] = 0.0f;
        }
#pragma unroll
        for (int q = 0; q < count; ++q) {
          const int b = sc.bin(x[q]);  // -1: the weight is 0
          if (counts) add_shared(count0 + b * 4, b >= 0 ? 1u : 0u);
          add_share(sum0 + b * 4, e[q]);
          if (sc.min_p > 0.0f && e[q] >= sc.min_p) min_sum += Scale::weight(e[q]);
        }
      });
    };
    if (sc.plain()) fill(std::true_type{});
    else fill(std::false_type{});
    min_sum = warp_sum(min_sum);
    if (lane == 0) s.red[warp] = min_sum;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kST / 32; ++w) min_sum += s.red[w];
      s.mine.min_sum = min_sum;
    }
    cl.sync();
    // each CTA adds up its share of the intervals over the cluster, for all of them
    const int share = (kBins + C - 1) / C;
    for (int b = rank * share + tid; b < min(kBins, (rank + 1) * share); b += kST) {
      uint32_t cnt = 0u;
      u64 sum = 0ull;
#pragma unroll
      for (int c = 0; c < kCluster; ++c) {
        if (c >= C) break;
        const SampleSmem& o = *cl.map_shared_rank(&s, c);
        if (counts) cnt += o.h.count[b];
        sum += sum_of(o.h, b);
      }
#pragma unroll
      for (int c = 0; c < kCluster; ++c) {
        if (c >= C) break;
        SampleSmem& o = *cl.map_shared_rank(&s, c);
        if (counts) o.count[b] = cnt;
        o.sum[b] = sum;
      }
    }
    cl.sync();
  }
  // running counts and sums of the row's intervals, in every CTA; a thread has kPer of them
  constexpr int kPer = kBins / kST;
  uint32_t own_count[kPer + 1];
  u64 own_sum[kPer + 1];
  {
    uint32_t cs = 0u, c_all;
    u64 vs = 0ull, v_all;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      own_count[q + 1] = counts ? s.count[tid * kPer + q] : 0u;
      own_sum[q + 1] = s.sum[tid * kPer + q];
      cs += own_count[q + 1];
      vs += own_sum[q + 1];
    }
    block_scan(s, cs, vs, own_count[0], own_sum[0], c_all, v_all);
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      own_count[q + 1] += own_count[q];
      own_sum[q + 1] += own_sum[q];
      s.count[tid * kPer + q] = own_count[q];
      s.sum[tid * kPer + q] = own_sum[q];
    }
    if (tid == 0) s.count[kBins] = c_all, s.sum[kBins] = v_all;
    if (tid < 8) s.at_bin[tid] = kBins - 1;
    __syncthreads();
  }
  // The interval in which the value is reached; each question has a place of its own for the answer.
  auto bin_of = [&](int place, int want, u64 value, double share) FNX_INLINE_STEP {
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      if (reached(want, own_count[q + 1], own_sum[q + 1], value, share) &&
          !reached(want, own_count[q], own_sum[q], value, share))
        s.at_bin[place] = tid * kPer + q;
    }
    __syncthreads();
    return s.at_bin[place];
  };
  u64 by_share = ~0ull;  // what min-p keeps
  if (sc.min_p > 0.0f) {
    by_share = 0ull;
    for (int r = 0; r < C; ++r) by_share += cl.map_shared_rank(&s, r)->mine.min_sum;
  }

  // Calls f(key, logit) for the slice's tokens that the first CTA asks for.
  auto asked = [&](const Control& c, auto&& f) FNX_INLINE {
    sweep([&](auto count, const float* x, int i0) FNX_INLINE {
#pragma unroll
      for (int q = 0; q < count; ++q) {
        const int b = sc.bin(x[q]);
        if ((b < c.bin_lo || b > c.bin_hi) && (b < c.bin2_lo || b > c.bin2_hi)) continue;
        const u64 key = make_key(x[q], (uint32_t)(v0 + i0 + q));
        if (key >= c.key_lo && key <= c.key_hi) f(key, x[q]);
      }
    });
  };

  // Sends them to its list.
  auto gather = [&](const Control& c) FNX_INLINE_STEP {
    asked(c, [&](u64 key, float) FNX_INLINE { find(key); });
    send();
    cl.sync();
  };

  // Splits their range of keys into intervals of 2^shift and adds up the counts and sums of these in the
  // first CTA.
  u64 klo = 0ull, khi = 0ull;
  int shift = 0;
  auto split = [&](const Control& c) FNX_INLINE_STEP {
    klo = ~0ull, khi = 0ull;
    asked(c, [&](u64 key, float) FNX_INLINE {
      klo = key < klo ? key : klo;
      khi = key > khi ? key : khi;
    });
    khi = warp_max(khi);
    klo = ~warp_max(~klo);
    if (tid == 0) s.mine.key_lo = ~0ull, s.mine.key_hi = 0ull;
    __syncthreads();
    if (lane == 0) atomicMax(&s.mine.key_hi, khi), atomicMin(&s.mine.key_lo, klo);
    for (int b = tid; b < kSub; b += kST) s.h.count[b] = s.h.w0[b] = s.h.w1[b] = s.h.w2[b] = 0u;
    cl.sync();
    for (int r = 0; r < C; ++r) {
      const Local& o = cl.map_shared_rank(&s, r)->mine;
      klo = o.key_lo < klo ? o.key_lo : klo;
      khi = o.key_hi > khi ? o.key_hi : khi;
    }
    shift = 0;
    while (((khi - klo) >> shift) >= (u64)kSub) ++shift;
    asked(c, [&](u64 key, float x) FNX_INLINE {
      const int at = (int)((khi - key) >> shift);
      add_shared(count0 + at * 4, 1u);
      add_sum(sum0 + at * 4, Scale::weight(sc.share(x)));
    });
    cl.sync();
    if (rank == 0 && tid < kSub) {
      uint32_t cnt = 0u;
      u64 sum = 0ull;
      for (int r = 0; r < C; ++r) {
        const SampleSmem& o = *cl.map_shared_rank(&s, r);
        cnt += o.h.count[tid];
        sum += sum_of(o.h, tid);
      }
      s.sub_count[tid] = cnt;
      s.sub_sum[tid] = sum;
    }
    cl.sync();
  };

  // Without top-k every CTA knows what to send: the tokens of top-p's interval, and of the intervals in
  // which the random share of what it keeps can lie.
  Control c{OP_GATHER, 0, -1, 0, -1, 0ull, ~0ull};
  u64 kept = s.sum[kBins];
  double want = (double)top_p * (double)kept;
  if (!counts) {
    if (use_p && want > 0.0) {
      const int bp = bin_of(0, WANT_SHARE, 0ull, want);
      const u64 least = s.sum[bp] + 1, most = s.sum[bp + 1];
      c.bin_lo = bin_of(1, WANT_SUM, target_of(u, least < by_share ? least : by_share), 0.0);
      c.bin_hi = bin_of(2, WANT_SUM, target_of(u, most < by_share ? most : by_share), 0.0);
      c.bin2_lo = c.bin2_hi = bp;
    } else {
      if (use_p) kept = kOne;
      c.bin_lo = c.bin_hi = bin_of(3, WANT_SUM, target_of(u, kept < by_share ? kept : by_share), 0.0);
    }
    gather(c);
  }

  if (rank != 0) {  // the other CTAs do as they are told
    cl.sync();
    for (;;) {
      c = first.ctl;
      if (c.op == OP_DONE) break;
      if (c.op == OP_GATHER) gather(c);
      else split(c);
      cl.sync();
    }
  } else {
    auto tell = [&](const Control& c) FNX_INLINE_STEP {
      __syncthreads();
      if (tid == 0) {
        s.ctl = c;
        s.listed = 0u;
      }
      cl.sync();
    };
    // The token of interval b at which the value is reached; the list is loaded.
    auto query = [&](int b, int want, u64 value, double share) FNX_INLINE_STEP -> Found {
      c = Control{OP_GATHER, b, b, 0, -1, 0ull, ~0ull};
      u64 base_count = s.count[b], base_sum = s.sum[b];
      for (;;) {
        c.op = OP_GATHER;
        tell(c);
        gather(c);
        const int held = (int)s.listed;
        if (held <= kCap) {
          const Stretch st{b, sc.inv, (float)b - 0.5f};
          measure(s, sc, st, held);
          return answer(s, sc, st, held, base_count, base_sum, want, value, share);
        }
        c.op = OP_SPLIT;
        tell(c);
        split(c);
        uint32_t cb, c_all;
        u64 vb, v_all;
        block_scan(s, s.sub_count[tid], s.sub_sum[tid], cb, vb, c_all, v_all);
        s.sub_count[tid] = cb, s.sub_sum[tid] = vb;
        if (tid == 0) s.sub_count[kSub] = c_all, s.sub_sum[kSub] = v_all;
        const int q = find_bin(s, s.sub_count, s.sub_sum, kSub, base_count, base_sum, want, value, share);
        base_count += s.sub_count[q];
        base_sum += s.sub_sum[q];
        const u64 width = (1ull << shift) - 1ull;
        c.key_hi = khi - ((u64)q << shift);
        c.key_lo = c.key_hi - klo > width ? c.key_hi - width : klo;
      }
    };
    if (counts) {
      if ((uint32_t)top_k < s.count[kBins]) {
        kept = query(bin_of(4, WANT_COUNT, (u64)top_k, 0.0), WANT_COUNT, (u64)top_k, 0.0).sum;
        want = (double)top_p * (double)kept;
      }
      if (use_p && want > 0.0) kept = query(bin_of(0, WANT_SHARE, 0ull, want), WANT_SHARE, 0ull, want).sum;
      else if (use_p) kept = kOne;
    }
    // a list that holds the intervals asked for above
    const int held = counts || s.listed > (uint32_t)kCap ? -1 : (int)s.listed;
    const bool few = held >= 0 && held <= kShort;
    Ranked r;
    u64 unused;
    if (few) r = rank_list(s, sc, held, unused);
    int measured = -1;
    auto from_list = [&](int b, int what, u64 value, double share) FNX_INLINE_STEP {
      if (few) {  // weight ahead of the list's tokens: that of an interval after the others is not in it
        u64 base = s.sum[c.bin_lo];
        if (b > c.bin_hi) base += s.sum[b] - s.sum[c.bin_hi + 1];
        return answer(s, r, held, 0, base, what, value, share);
      }
      const Stretch st{b, sc.inv, (float)b - 0.5f};
      if (measured != b) measure(s, sc, st, held);
      measured = b;
      return answer(s, sc, st, held, 0, s.sum[b], what, value, share);
    };
    if (!counts && use_p && want > 0.0) {
      const int bp = s.at_bin[0];
      kept = (held >= 0 ? from_list(bp, WANT_SHARE, 0ull, want) : query(bp, WANT_SHARE, 0ull, want)).sum;
    }
    kept = by_share < kept ? by_share : kept;
    const u64 target = target_of(u, kept);
    const int bt = bin_of(5, WANT_SUM, target, 0.0);
    const Found f = held >= 0 ? from_list(bt, WANT_SUM, target, 0.0) : query(bt, WANT_SUM, target, 0.0);
    if (kAll) leave(KEPT_PREFIX, sc, f.token, kept);
    else draw(a, row, f, kept);
    tell(Control{OP_DONE, 0, -1, 0, -1, 0ull, 0ull});
  }
  cl.sync();  // no CTA leaves while another reads its shared memory
  pdl_trigger();
}

namespace {

template <bool kMany, bool kAll>
const void* sample_fn(int type) {
  if (type == LOGITS_F32) return (const void*)sample_kernel<float, kMany, kAll>;
  if (type == LOGITS_F16) return (const void*)sample_kernel<__half, kMany, kAll>;
  return (const void*)sample_kernel<__nv_bfloat16, kMany, kAll>;
}

}  // namespace

// Each form is a unit of compilation: one takes the compiler a minute and a half.
const void* sample_fn_one(int type);
const void* sample_fn_many(int type);
const void* probs_fn_one(int type);
const void* probs_fn_many(int type);

namespace {

template <bool kAll>
int launch_rows(SampleArgs a, cudaStream_t stream) {
  const int size = a.type == LOGITS_F32 ? 4 : 2;
  // Rows for which clusters of 8 would not all run at once share the SMs two CTAs each, in clusters of 4.  Measured, in
  // clusters of 8 and of 4: sampling 14 fp32 rows of 151,936 without filters 24 and 36 us, 19 rows 44 and 36, 128 rows of
  // 248,320 with all kinds of filters 205 and 100; token_probs with top-p, 14 rows 29 and 41, 19 rows 52 and 41, the 128 rows
  // 248 and 150.  From 15 to 18 rows some clusters of 8 wait for others: rows of one kind would be faster in clusters
  // of 4 (16 rows 41 and 34), rows of several kinds, whose short ones end early, are not (24 and 35; token_probs 32 and 44).
  // (A CTA of a cluster of 4 may hold too many logits for its histogram's sums above 2^20.)
  const bool many = (int64_t)a.M * 8 > num_sms() && a.V <= 1 << 20;
  const int C = many ? 4 : 8;
  const void* k = kAll ? (many ? probs_fn_many(a.type) : probs_fn_one(a.type)) : many ? sample_fn_many(a.type) : sample_fn_one(a.type);
  if (!prepare_kernel(k)) return 2;
  a.per = ((a.V + C - 1) / C + 15) / 16 * 16;
  const size_t fixed = (sizeof(SampleSmem) + 15) & ~(size_t)15;
  const size_t whole = fixed + (size_t)a.per * size + 32;
  a.in_smem = !many && whole <= 227 * 1024 ? 1 : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.M * C);
  cfg.blockDim = dim3(kST);
  cfg.dynamicSmemBytes = a.in_smem ? whole : fixed;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.pdl ? 2 : 1;
  void* params[1] = {&a};
  return cudaLaunchKernelExC(&cfg, k, params) == cudaSuccess ? 0 : 2;
}

}  // namespace

}  // namespace fnx
