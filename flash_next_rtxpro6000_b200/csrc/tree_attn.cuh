// Shared parts of the tree attention kernels: the split of the work over the CTAs, the reading of
// lengths, pages and masks with their checks, and the form of partial results.
//
// Work.  For request b with context L, T nodes and G query heads per kv head, the G * T rows of one
// kv head are cut into row tiles of `rows`, and the L + T keys into key tiles of kKeyTile.  An item is
// (request, kv head, row tile); its units are its key tiles.  All units of the launch, item by item,
// are divided into contiguous ranges of equal size, one per CTA, so long and short requests load the
// GPU evenly whatever their lengths.  The range sizes follow from the lengths on the device: the host
// does not read them.  A CTA holds at most two items in part (its first and its last), whose partial
// sums go to two slots of its own; the combine kernel adds an item's slots up in a fixed order.
#pragma once

#include "fnx_common.cuh"
#include "fnx_kernels.h"

namespace fnx {

constexpr int kKeyTile = 64;
constexpr int kAttnMaxBatch = 128;  // requests of one launch
constexpr int kAttnMaxGrid = 256;   // CTAs of one launch (one per SM)

struct AttnReq {
  int ctx, nodes, n0;  // context length, drafted nodes, first row in q
  bool refused;
};

// Request b's lengths; anything inconsistent is recorded and leaves the request without nodes.
__device__ __forceinline__ AttnReq attn_request(const AttnArgs& a, int b, bool report) {
  AttnReq r;
  r.ctx = a.context_lens[b];
  r.n0 = a.node_offsets[b];
  r.nodes = a.node_offsets[b + 1] - r.n0;
  const int64_t room = (int64_t)a.table_width * a.page_size;
  r.refused = r.ctx < 0 || r.ctx > a.max_context || r.n0 < 0 || r.nodes < 0 || r.nodes > a.max_nodes ||
              r.n0 > a.N - r.nodes || (int64_t)r.ctx + r.nodes > room;
  if (r.refused) {
    if (report) record_error(a.err, ERR_LENGTHS);
    r.ctx = r.nodes = r.n0 = 0;
  }
  return r;
}

struct AttnShape {
  int row_tiles, key_tiles;
  long long units;  // of all kv heads
};

__device__ __forceinline__ AttnShape attn_shape(const AttnArgs& a, const AttnReq& r, int rows) {
  AttnShape s;
  s.row_tiles = (r.nodes * a.group + rows - 1) / rows;
  s.key_tiles = (r.ctx + r.nodes + kKeyTile - 1) / kKeyTile;
  s.units = (long long)a.Hk * s.row_tiles * s.key_tiles;
  return s;
}

// Fills before[b] = units of the requests ahead of b, before[B] = all units; returns whether a request was
// refused.  All threads of the block take part; `scratch` holds one value per warp.
__device__ __forceinline__ bool attn_prefix(const AttnArgs& a, int rows, long long* before, long long* scratch,
                                            bool report) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  long long base = 0;
  bool refused = false;
  for (int b0 = 0; b0 < a.B; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    long long u = 0;
    if (b < a.B) {
      const AttnReq r = attn_request(a, b, report);
      refused |= r.refused;
      u = attn_shape(a, r, rows).units;
    }
    long long v = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long w = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += w;
    }
    if (lane == 31) scratch[warp] = v;
    __syncthreads();
    long long ahead = base;
    for (int w = 0; w < nw; ++w) {
      if (w < warp) ahead += scratch[w];
      base += scratch[w];
    }
    if (b < a.B) before[b] = ahead + v - u;
    __syncthreads();
  }
  if (threadIdx.x == 0) before[a.B] = base;
  return __syncthreads_or(refused);
}

// Rows of q that no request has get 0 and -inf, as rows that see nothing do: those of refused requests, and
// those ahead of the first and behind the last (a captured call's, when it is replayed with fewer nodes).
__device__ __forceinline__ void attn_unowned(const AttnArgs& a, bool refused) {
  const int* off = a.node_offsets;
  if (!refused && !(a.head && off[0] > 0) && !(a.tail && off[a.B] < a.N)) return;
  for (int b = a.head ? -1 : 0; b < a.B + (a.tail ? 1 : 0); ++b) {
    if (b >= 0 && b < a.B && !attn_request(a, b, false).refused) continue;
    const int n0 = b < 0 ? 0 : max(off[b], 0), n1 = b == a.B ? a.N : min(off[b + 1], a.N);
    const int units = a.D / 8;
    const int64_t all = ((int64_t)n1 - n0) * a.Hq * units, step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t u = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; u < all; u += step) {
      const int64_t row = u / units, n = n0 + row / a.Hq;
      const int h = (int)(row % a.Hq), c = (int)(u % units);
      *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + n * a.o_sn + (int64_t)h * a.o_sh + c * 8) =
          make_uint4(0u, 0u, 0u, 0u);
      if (a.lse && c == 0) a.lse[n * a.Hq + h] = -INFINITY;
    }
  }
}

// The request that holds unit w: the last one with before[b] <= w (those without units are passed).
__device__ __forceinline__ int attn_find(const long long* before, int B, long long w) {
  int lo = 0, hi = B;  // before[lo] <= w < before[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (before[mid] <= w) lo = mid;
    else hi = mid;
  }
  return lo;
}

// First unit of CTA c of G, and the CTA that holds unit w.
__device__ __forceinline__ long long attn_first(long long c, long long total, long long G) { return c * total / G; }
__device__ __forceinline__ int attn_cta_of(long long w, long long total, long long G) {
  return (int)(((w + 1) * G - 1) / total);
}

// Partial result of a row: D sums, then (maximum, sum of weights), in base-2 units of the score.
__host__ __device__ constexpr int64_t attn_slot_floats(int rows, int D) { return (int64_t)rows * (D + 2); }

// Nodes that row r of the item's row tile belongs to, its head, and the tree bits it sees.
__device__ __forceinline__ unsigned long long attn_mask(const AttnArgs& a, const AttnReq& r, int node) {
  if (a.tree_mask) return a.tree_mask[r.n0 + node];
  return node >= 63 ? ~0ull : (2ull << node) - 1ull;  // a chain: the node and all before it
}

// Element offsets of key position pos of request b (its head included); -1 where there is none.
__device__ __forceinline__ void attn_place(const AttnArgs& a, int b, int pos, int len, int head, int64_t& k, int64_t& v) {
  k = v = -1;
  if (pos >= len) return;
  const int p = pos / a.page_size, in = pos - p * a.page_size;
  const int page = a.page_table[(int64_t)b * a.table_ld + p];
  if (page < 0 || page >= a.num_pages) {
    record_error(a.err, ERR_PAGE);
    return;
  }
  k = (int64_t)page * a.kc_st[0] + (int64_t)in * a.kc_st[1] + (int64_t)head * a.kc_st[2];
  v = (int64_t)page * a.vc_st[0] + (int64_t)in * a.vc_st[1] + (int64_t)head * a.vc_st[2];
}

// Weights are exp2(score - reference) of a row's own reference, which the row's sums and partial results
// carry along.  They are rounded to the cache's type for the second product.  bf16 has the exponents of
// fp32: the reference is the running maximum, and nothing is lost.  fp16 ends at 2^-24, and weights below
// that would count in the sum but not in the result, all of which may be theirs where the large weights'
// values are small (the first token's often are).  So with fp16 the reference lies some bits (the form's
// "head") below the running maximum, which uses fp16's range above 1, and where a key tile's largest score
// is more than kFall bits below the reference's, the reference follows it down, to kSpan bits below the
// running maximum at most (sums then stay below 2^102).  A tile's largest weight is 2^-7 at least.
template <typename T> constexpr bool kNarrow = false;  // few exponents
template <> constexpr bool kNarrow<__half> = true;
constexpr float kSpan = 40.0f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace fnx
