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
// A row belongs to a cluster of CTAs that hold their slices in shared memory, so global memory is
// read once.  Steps: (1) maximum and minimum; (2) a histogram of counts and sums over kBins intervals
// of m - x of equal width, which is a partition in the right order because m - x falls as x grows;
// (3) the first CTA finds the interval in which a value is reached, the cluster sends it the
// interval's tokens, and it sorts them and reads the token off their running sums.  Where top-k keeps
// few, the tokens of all intervals up to the k-th's are sent at once and answer every question.  An
// interval with more tokens than the list holds (many ties, or one token far from the others) is
// split again by order key and token index until it fits.
#include <cooperative_groups.h>

#include "fnx_common.cuh"
#include "fnx_kernels.h"

namespace fnx {

namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kST = 512;          // threads
constexpr int kBins = 2048;       // intervals of m - x
constexpr int kSub = 256;         // intervals of a split
constexpr int kCap = 2048;        // tokens of the sorted list
constexpr u64 kOne = 1ull << 40;  // the weight of the most likely token
// exp(-28) < 2^-40: tokens further below the maximum have no weight and are not looked at
constexpr float kReach = 28.0f;

enum Want : int { WANT_COUNT = 0, WANT_SHARE = 1, WANT_SUM = 2 };
enum Op : int { OP_DONE = 0, OP_GATHER = 1, OP_SPLIT = 2 };

struct Control {  // written by the first CTA, read by the cluster
  int op, bin_lo, bin_hi, shift;
  u64 key_lo, key_hi;
};

struct Local {  // written by each CTA, read by the others
  u64 best;       // largest key of the slice
  float low;      // smallest finite logit
  u64 min_sum;    // sum of the weights that min-p keeps
  u64 key_lo, key_hi;  // smallest and largest key sent to the list
};

struct SampleSmem {
  // histogram, then (it is dead by then) the list and its running sums
  union {
    struct { uint32_t count[kBins], lo[kBins], hi[kBins]; } h;
    struct { u64 key[kCap], sum[kCap]; } list;
  };
  // first CTA: exclusive running counts and sums of the row's intervals, and of a split's
  u64 sum[kBins + 1];
  uint32_t count[kBins + 1];
  uint32_t sub_count[kSub + 1];
  u64 sub_sum[kSub + 1];
  Control ctl;
  Local mine;
  uint32_t listed;
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

// The row's scale: everything a thread needs to place a logit.
struct Scale {
  float m, T, range, inv, min_p;
  // exp((x - m) / T); the maximum's is 1 also where it is infinite
  __device__ __forceinline__ float share(float x) const { return x == m ? 1.0f : expf((x - m) / T); }
  static __device__ __forceinline__ u64 weight(float e) { return __float2ull_rz(e * (float)kOne); }
  // the interval of x, or -1 for a token without weight (NaN and -inf among them)
  __device__ __forceinline__ int bin(float x) const {
    if (x == m) return 0;
    const float d = m - x;
    if (!(d <= range)) return -1;
    return (int)fminf(d * inv, (float)(kBins - 1));
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

// Adds a weight to the two 32-bit halves of an interval's sum (shared memory has no 64-bit add).
__device__ __forceinline__ void add_sum(uint32_t* lo, uint32_t* hi, u64 w) {
  const uint32_t l = (uint32_t)w;
  uint32_t h = (uint32_t)(w >> 32);
  if (l) {
    const uint32_t old = atomicAdd(lo, l);
    h += old + l < old ? 1u : 0u;
  }
  if (h) atomicAdd(hi, h);
}

// Sorts n keys (padded with zeros to a power of two) in falling order.
__device__ __forceinline__ void sort_list(SampleSmem& s, int n) {
  int p = 64;
  while (p < n) p <<= 1;
  for (int i = n + threadIdx.x; i < p; i += kST) s.list.key[i] = 0ull;
  __syncthreads();
  for (int size = 2; size <= p; size <<= 1) {
    for (int d = size >> 1; d > 0; d >>= 1) {
      for (int t = threadIdx.x; t < p / 2; t += kST) {
        const int i = 2 * t - (t & (d - 1)), j = i + d;
        const u64 a = s.list.key[i], b = s.list.key[j];
        if ((a < b) == ((i & size) == 0)) s.list.key[i] = b, s.list.key[j] = a;
      }
      __syncthreads();
    }
  }
}

// Running sums (inclusive) of the sorted list's weights.
__device__ __forceinline__ void sum_list(SampleSmem& s, const Scale& sc, int n) {
  constexpr int kPer = kCap / kST;
  u64 w[kPer], mine = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int i = threadIdx.x * kPer + q;
    w[q] = i < n ? Scale::weight(sc.share(key_value(s.list.key[i]))) : 0ull;
    mine += w[q];
  }
  uint32_t c0, ca;
  u64 before, all;
  block_scan(s, 0u, mine, c0, before, ca, all);
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    before += w[q];
    s.list.sum[threadIdx.x * kPer + q] = before;
  }
  __syncthreads();
}

// Whether a running count / sum has reached the wanted value.
__device__ __forceinline__ bool reached(int want, u64 count, u64 sum, u64 value, double share) {
  return want == WANT_COUNT ? count >= value : want == WANT_SHARE ? (double)sum >= share : sum >= value;
}

// The first entry of the sorted list at which the value is reached (the last one if none is).
__device__ __forceinline__ int find_in_list(SampleSmem& s, int n, u64 base_count, u64 base_sum, int want, u64 value,
                                            double share) {
  __syncthreads();
  if (threadIdx.x == 0) s.found = n - 1;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kST) {
    if (reached(want, base_count + i + 1, base_sum + s.list.sum[i], value, share) &&
        !(i > 0 && reached(want, base_count + i, base_sum + s.list.sum[i - 1], value, share)))
      s.found = i;
  }
  __syncthreads();
  return s.found;
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

}  // namespace

template <typename T>
__global__ void __launch_bounds__(kST) sample_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  SampleSmem& s = *reinterpret_cast<SampleSmem*>(smem);
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), C = (int)cl.num_blocks();
  const int row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  SampleSmem& first = *cl.map_shared_rank(&s, 0);
  const int v0 = rank * a.per;
  const int n = v0 >= a.V ? 0 : (a.V - v0 < a.per ? a.V - v0 : a.per);
  constexpr int kVec = 16 / sizeof(T);
  pdl_wait();

  // --- (1) the slice into shared memory, with its maximum and minimum
  const T* g = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.ldl + v0;
  T* slice = reinterpret_cast<T*>(smem + ((sizeof(SampleSmem) + 15) & ~(size_t)15));
  const int off = (int)((reinterpret_cast<uintptr_t>(g) & 15) / sizeof(T));  // same place modulo 16 bytes
  const T* xs = a.in_smem ? slice + off : g;
  u64 best = 0ull;
  float low = INFINITY;
  auto look = [&](float x, int i) {
    if (x > -INFINITY) {
      const u64 k = make_key(x, (uint32_t)(v0 + i));
      best = k > best ? k : best;
      low = fminf(low, x);
    }
  };
  {
    int head = off ? kVec - off : 0;
    head = head < n ? head : n;
    const int nv = (n - head) / kVec;
    T* to = slice + off;
    for (int i = tid; i < head; i += kST) {
      const T v = g[i];
      if (a.in_smem) to[i] = v;
      look(logit(v), i);
    }
    const uint4* gv = reinterpret_cast<const uint4*>(g + head);
    uint4* tv = reinterpret_cast<uint4*>(to + head);
#pragma unroll 4
    for (int j = tid; j < nv; j += kST) {
      const uint4 v = ldg_cg_u4(gv + j);
      if (a.in_smem) tv[j] = v;
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int q = 0; q < kVec; ++q) look(logit(e[q]), head + j * kVec + q);
    }
    for (int i = head + nv * kVec + tid; i < n; i += kST) {
      const T v = g[i];
      if (a.in_smem) to[i] = v;
      look(logit(v), i);
    }
  }
  best = warp_max(best);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  if (lane == 0) s.red[warp] = best, s.red_f[warp] = low;
  for (int b = tid; b < kBins; b += kST) s.h.count[b] = s.h.lo[b] = s.h.hi[b] = 0u;
  if (tid == 0) s.listed = 0u;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kST / 32; ++w) {
      best = s.red[w] > best ? s.red[w] : best;
      low = fminf(low, s.red_f[w]);
    }
    s.mine.best = best;
    s.mine.low = low;
  }
  cl.sync();
  best = 0ull;
  low = INFINITY;
  for (int c = 0; c < C; ++c) {
    const Local& o = cl.map_shared_rank(&s, c)->mine;
    best = o.best > best ? o.best : best;
    low = fminf(low, o.low);
  }
  float Tm = a.temperature ? a.temperature[row] : 1.0f;
  if (best == 0ull || !(Tm > 0.0f)) {  // nothing to draw from, or the most likely token
    if (rank == 0 && tid == 0) {
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
  sc.inv = sc.range > 0.0f ? (float)kBins / sc.range : 0.0f;
  const int top_k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.0f;
  const bool use_p = top_p < 1.0f;
  float min_p = a.min_p ? a.min_p[row] : 0.0f;
  sc.min_p = min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f;

  // --- (2) histogram; its sums are not needed where top-k leaves a list's worth of tokens
  bool sums = !(top_k > 0 && top_k <= kCap / 2);
  for (;;) {
    u64 min_sum = 0ull;
    for (int i = tid; i < n; i += kST) {
      const float x = logit(xs[i]);
      const int b = sc.bin(x);
      if (b < 0) continue;
      atomicAdd(&s.h.count[b], 1u);
      if (sums) {
        const float e = sc.share(x);
        const u64 w = Scale::weight(e);
        add_sum(&s.h.lo[b], &s.h.hi[b], w);
        if (e >= sc.min_p) min_sum += w;
      }
    }
    min_sum = warp_sum(min_sum);
    if (lane == 0) s.red[warp] = min_sum;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kST / 32; ++w) min_sum += s.red[w];
      s.mine.min_sum = min_sum;
    }
    cl.sync();
    // each CTA adds up its share of the intervals over the cluster and leaves them with the first
    const int share = (kBins + C - 1) / C;
    for (int b = rank * share + tid; b < min(kBins, (rank + 1) * share); b += kST) {
      uint32_t cnt = 0u;
      u64 sum = 0ull;
      for (int c = 0; c < C; ++c) {
        const SampleSmem& o = *cl.map_shared_rank(&s, c);
        cnt += o.h.count[b];
        sum += ((u64)o.h.hi[b] << 32) + o.h.lo[b];
      }
      first.count[b] = cnt;
      first.sum[b] = sum;
    }
    cl.sync();
    if (rank == 0) {
      constexpr int kPer = kBins / kST;
      uint32_t c[kPer], cs = 0u, c_all;
      u64 v[kPer], vs = 0ull, v_all;
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        c[q] = s.count[tid * kPer + q];
        v[q] = s.sum[tid * kPer + q];
        cs += c[q];
        vs += v[q];
      }
      uint32_t cb;
      u64 vb;
      block_scan(s, cs, vs, cb, vb, c_all, v_all);
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        s.count[tid * kPer + q] = cb;
        s.sum[tid * kPer + q] = vb;
        cb += c[q];
        vb += v[q];
      }
      if (tid == 0) s.count[kBins] = c_all, s.sum[kBins] = v_all;
      __syncthreads();
      if (!sums) {  // the k-th token's interval may hold too many for the list
        const u64 k = min((u64)top_k, (u64)c_all);
        const int b = find_bin(s, s.count, s.sum, kBins, 0, 0, WANT_COUNT, k, 0.0);
        if (tid == 0) s.ctl.op = s.count[b + 1] <= (uint32_t)kCap ? OP_GATHER : OP_SPLIT, s.ctl.bin_hi = b;
      }
    }
    if (sums) break;
    cl.sync();
    const bool fits = first.ctl.op == OP_GATHER;
    cl.sync();  // read by all before it is written again
    if (fits) break;
    sums = true;
    for (int b = tid; b < kBins; b += kST) s.h.count[b] = 0u;
    __syncthreads();
  }

  // Sends the tokens of intervals bin_lo .. bin_hi with keys in [key_lo, key_hi] to the first CTA.
  auto gather = [&](const Control& c) {
    u64 klo = ~0ull, khi = 0ull;
    const int rounds = (n + kST - 1) / kST;
    for (int r = 0; r < rounds; ++r) {
      const int i = r * kST + tid;
      bool hit = false;
      u64 key = 0ull;
      if (i < n) {
        const float x = logit(xs[i]);
        const int b = sc.bin(x);
        if (b >= c.bin_lo && b <= c.bin_hi) {
          key = make_key(x, (uint32_t)(v0 + i));
          hit = key >= c.key_lo && key <= c.key_hi;
        }
      }
      const unsigned who = __ballot_sync(0xffffffffu, hit);
      if (!who) continue;
      uint32_t at = 0u;
      if (lane == 0) at = atomicAdd(&first.listed, (uint32_t)__popc(who));
      at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1u));
      if (hit) {
        if (at < (uint32_t)kCap) first.list.key[at] = key;
        klo = key < klo ? key : klo;
        khi = key > khi ? key : khi;
      }
    }
    khi = warp_max(khi);
    klo = ~warp_max(~klo);
    __syncthreads();
    if (lane == 0) s.red[warp] = khi;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kST / 32; ++w) khi = s.red[w] > khi ? s.red[w] : khi;
      s.mine.key_hi = khi;
    }
    __syncthreads();
    if (lane == 0) s.red[warp] = klo;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kST / 32; ++w) klo = s.red[w] < klo ? s.red[w] : klo;
      s.mine.key_lo = klo;
    }
    cl.sync();
  };

  // Histogram of counts and sums over the intervals of a split, added up in the first CTA.
  auto split = [&](const Control& c) {
    for (int b = tid; b < kSub; b += kST) s.h.count[b] = s.h.lo[b] = s.h.hi[b] = 0u;
    __syncthreads();
    for (int i = tid; i < n; i += kST) {
      const float x = logit(xs[i]);
      const int b = sc.bin(x);
      if (b < c.bin_lo || b > c.bin_hi) continue;
      const u64 key = make_key(x, (uint32_t)(v0 + i));
      if (key < c.key_lo || key > c.key_hi) continue;
      const int q = (int)((c.key_hi - key) >> c.shift);
      atomicAdd(&s.h.count[q], 1u);
      add_sum(&s.h.lo[q], &s.h.hi[q], Scale::weight(sc.share(x)));
    }
    cl.sync();
    if (rank == 0 && tid < kSub) {
      uint32_t cnt = 0u;
      u64 sum = 0ull;
      for (int r = 0; r < C; ++r) {
        const SampleSmem& o = *cl.map_shared_rank(&s, r);
        cnt += o.h.count[tid];
        sum += ((u64)o.h.hi[tid] << 32) + o.h.lo[tid];
      }
      s.sub_count[tid] = cnt;
      s.sub_sum[tid] = sum;
    }
    cl.sync();
  };

  if (rank != 0) {  // the other CTAs do as they are told
    cl.sync();
    for (;;) {
      const Control c = first.ctl;
      if (c.op == OP_DONE) break;
      if (c.op == OP_GATHER) gather(c);
      else split(c);
      cl.sync();
    }
  } else {
    auto tell = [&](int op, int lo, int hi, int shift, u64 key_lo, u64 key_hi) {
      __syncthreads();
      if (tid == 0) {
        s.ctl = Control{op, lo, hi, shift, key_lo, key_hi};
        s.listed = 0u;
      }
      cl.sync();
    };
    const u64 tokens_in = s.count[kBins];
    const bool use_k = top_k > 0 && (u64)top_k < tokens_in;
    // The list's place in the row: tokens and weight ahead of it, and how many it holds; held_lo ..
    // held_hi are the intervals whose tokens are all in it.
    u64 base_count = 0ull, base_sum = 0ull;
    int held = 0, held_lo = 0, held_hi = -1;

    // The token at which the value is reached: its place in the list, which is loaded as needed.
    auto query = [&](int want, u64 value, double share) -> int {
      int b = 0;
      if (sums) b = find_bin(s, s.count, s.sum, kBins, 0, 0, want, value, share);
      if (sums && !(b >= held_lo && b <= held_hi)) {
        Control c{OP_GATHER, b, b, 0, 0ull, ~0ull};
        base_count = s.count[b];
        base_sum = s.sum[b];
        bool whole = true;
        for (;;) {
          tell(OP_GATHER, c.bin_lo, c.bin_hi, 0, c.key_lo, c.key_hi);
          gather(c);
          held = (int)s.listed;
          held_lo = b;
          held_hi = whole ? b : -1;
          if (held <= kCap) break;
          whole = false;  // the list will hold a part of the interval only
          u64 klo = ~0ull, khi = 0ull;
          for (int r = 0; r < C; ++r) {
            const Local& o = cl.map_shared_rank(&s, r)->mine;
            klo = o.key_lo < klo ? o.key_lo : klo;
            khi = o.key_hi > khi ? o.key_hi : khi;
          }
          c.key_lo = klo;
          c.key_hi = khi;
          c.shift = 0;
          while (((khi - klo) >> c.shift) >= (u64)kSub) ++c.shift;
          tell(OP_SPLIT, b, b, c.shift, klo, khi);
          split(c);
          uint32_t cnt = tid < kSub ? s.sub_count[tid] : 0u, cb, c_all;
          u64 sum = tid < kSub ? s.sub_sum[tid] : 0ull, vb, v_all;
          block_scan(s, cnt, sum, cb, vb, c_all, v_all);
          if (tid < kSub) s.sub_count[tid] = cb, s.sub_sum[tid] = vb;
          if (tid == 0) s.sub_count[kSub] = c_all, s.sub_sum[kSub] = v_all;
          const int q = find_bin(s, s.sub_count, s.sub_sum, kSub, base_count, base_sum, want, value, share);
          base_count += s.sub_count[q];
          base_sum += s.sub_sum[q];
          const u64 width = (1ull << c.shift) - 1ull;
          c.key_hi = khi - ((u64)q << c.shift);
          c.key_lo = c.key_hi - klo > width ? c.key_hi - width : klo;
        }
        sort_list(s, held);
        sum_list(s, sc, held);
      }
      return find_in_list(s, held, base_count, base_sum, want, value, share);
    };

    u64 min_sum = 0ull;
    if (!sums) {  // everything up to the k-th token's interval in one list
      const int b = s.ctl.bin_hi;
      Control c{OP_GATHER, 0, b, 0, 0ull, ~0ull};
      tell(OP_GATHER, 0, b, 0, 0ull, ~0ull);
      gather(c);
      held = (int)s.listed;
      sort_list(s, held);
      sum_list(s, sc, held);
      if (sc.min_p > 0.0f) {
        __syncthreads();
        if (tid == 0) s.found = 0;
        __syncthreads();
        for (int i = tid; i < held; i += kST)
          if (sc.share(key_value(s.list.key[i])) >= sc.min_p &&
              !(i + 1 < held && sc.share(key_value(s.list.key[i + 1])) >= sc.min_p))
            s.found = i;
        __syncthreads();
        min_sum = s.list.sum[s.found];
      }
    } else if (sc.min_p > 0.0f) {
      for (int r = 0; r < C; ++r) min_sum += cl.map_shared_rank(&s, r)->mine.min_sum;
    }
    u64 kept;
    if (use_k) {
      const int i = query(WANT_COUNT, (u64)top_k, 0.0);
      kept = base_sum + s.list.sum[i];
    } else {
      kept = sums ? s.sum[kBins] : s.list.sum[held - 1];
    }
    if (use_p) {
      const double want = (double)top_p * (double)kept;
      if (want > 0.0) {
        const int i = query(WANT_SHARE, 0ull, want);
        kept = base_sum + s.list.sum[i];
      } else {
        kept = kOne;
      }
    }
    if (sc.min_p > 0.0f) kept = min_sum < kept ? min_sum : kept;
    double u = (double)a.uniforms[row];
    u = u > 0.0 ? u : 0.0;  // NaN and negative numbers draw the most likely token
    u64 target = __double2ull_rz(u * (double)kept);
    target = target < kept - 1 ? target : kept - 1;
    const int i = query(WANT_SUM, target + 1, 0.0);
    if (tid == 0) {
      const u64 w = s.list.sum[i] - (i > 0 ? s.list.sum[i - 1] : 0ull);
      a.tokens[row] = key_token(s.list.key[i]);
      a.probs[row] = (float)((double)w / (double)kept);
    }
    tell(OP_DONE, 0, -1, 0, 0ull, 0ull);
  }
  cl.sync();  // no CTA leaves while another reads its shared memory
  pdl_trigger();
}

namespace {

const void* sample_fn(int type) {
  if (type == LOGITS_F32) return (const void*)sample_kernel<float>;
  if (type == LOGITS_F16) return (const void*)sample_kernel<__half>;
  return (const void*)sample_kernel<__nv_bfloat16>;
}

}  // namespace

int launch_sample(SampleArgs a, cudaStream_t stream) {
  const void* k = sample_fn(a.type);
  if (!prepare_kernel(k)) return 2;
  const int size = a.type == LOGITS_F32 ? 4 : 2;
  const int C = 8;
  a.per = ((a.V + C - 1) / C + 15) / 16 * 16;
  const size_t fixed = (sizeof(SampleSmem) + 15) & ~(size_t)15;
  const size_t whole = fixed + (size_t)a.per * size + 32;
  a.in_smem = whole <= 227 * 1024 ? 1 : 0;
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

}  // namespace fnx
