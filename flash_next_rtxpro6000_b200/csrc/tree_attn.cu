// Attention of drafted token trees over a paged cache.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i k_j - max_j),
//
// over the keys j < L of the request's context and the drafted tokens L + n whose bit n is set in node
// i's mask; lse_i = log sum_j exp(scale q_i k_j).  A row that sees nothing gives 0 and -inf.  One pass
// over the keys with a running maximum and sum; scores, weights' sums and outputs are held in fp32,
// the weights are rounded to the cache's type for the second product (as wide as its other operand, and
// relative to a reference that keeps fp16 weights in its range: tree_attn.cuh).
//
// Bound: the cache's bytes, each read once for all G query heads and all nodes that share a kv head:
// the G * T rows of a kv head are one matrix operand.  mma.sync.m16n8k16 with keys and values in
// shared memory (cp.async into a ring, 16-byte units swizzled by row so that ldmatrix is free of
// conflicts).  MT tiles of 16 rows; WK warps share a row tile and take WK-ths of each key tile, which
// keeps four or eight warps busy when there are few rows; they join their sums at the item's end.
#include "tree_attn.cuh"

namespace fnx {

namespace {

template <typename T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
    mma_bf16(d, x[0], x[1], x[2], x[3], b0, b1);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
  static __device__ __forceinline__ float one(__nv_bfloat16 v) { return __bfloat162float(v); }
  static constexpr uint32_t kExp = 0x7F807F80u;  // exponent bits of a pair
};
template <> struct Mma<__half> {
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
    mma_f16(d, x[0], x[1], x[2], x[3], b0, b1);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
  static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
  static constexpr uint32_t kExp = 0x7C007C00u;
};

// Whether one of the pair's two values is infinite or NaN.
template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  const uint32_t e = w & Mma<T>::kExp;
  return (e & 0xFFFFu) == (Mma<T>::kExp & 0xFFFFu) || (e >> 16) == (Mma<T>::kExp >> 16);
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int D, int MT, int WK>
struct AttnCfg {
  static constexpr int kThreads = 32 * MT * WK;
  static constexpr int kRows = 16 * MT;
  static constexpr int kRowBytes = D * 2;
  static constexpr int kTileBytes = kKeyTile * kRowBytes;  // keys or values of one tile
  static constexpr int kStages = D == 256 ? 2 : D == 128 ? 4 : 6;
  static constexpr int kKeys = kKeyTile / WK;  // keys of a tile per warp
  // joins the WK warps of a row tile after the item's last tile, in the ring's memory
  static constexpr int kJoinRow = D + 4;  // floats; pads the rows apart
  static_assert((WK - 1) * MT * 16 * (kJoinRow + 2) * 4 <= kStages * 2 * kTileBytes, "join area");
  struct Smem {
    alignas(128) uint8_t ring[kStages][2][kTileBytes];
    alignas(128) uint8_t q[kRows * kRowBytes];
    int64_t place[2][2][kKeyTile];  // element offsets of a tile's keys and values
    unsigned long long mask[kRows];
    long long before[kAttnMaxBatch + 1];
    long long scratch[32];
    uint32_t odd[2];  // drafted tokens of a tile whose values are not all finite
  };
};

}  // namespace

template <typename T, int D, int MT, int WK>
__global__ void __launch_bounds__(32 * MT * WK, 1) tree_attn_kernel(const __grid_constant__ AttnArgs a) {
  using Cfg = AttnCfg<D, MT, WK>;
  constexpr int kRows = Cfg::kRows, kStages = Cfg::kStages, kKeys = Cfg::kKeys, kThreads = Cfg::kThreads;
  constexpr int kUnits = D / 8;  // 16-byte units of a row
  extern __shared__ __align__(128) uint8_t raw[];
  typename Cfg::Smem& s = *reinterpret_cast<typename Cfg::Smem*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wr = warp / WK, wk = warp % WK;
  const T* kc = reinterpret_cast<const T*>(a.k_cache);
  const T* vc = reinterpret_cast<const T*>(a.v_cache);
  const float c2 = a.scale * 1.4426950408889634f;  // scores in base-2 units
  pdl_wait();
  attn_unowned(a, attn_prefix(a, kRows, s.before, s.scratch, blockIdx.x == 0));
  const long long total = s.before[a.B];
  const long long G = total < (long long)gridDim.x ? total : (long long)gridDim.x;
  pdl_trigger();  // the launch that joins the partials may get ready
  if (blockIdx.x >= G) return;
  long long w = attn_first(blockIdx.x, total, G);
  const long long end = attn_first(blockIdx.x + 1, total, G);
  int b = attn_find(s.before, a.B, w);

  while (w < end) {
    while (s.before[b + 1] <= w) ++b;
    const AttnReq rq = attn_request(a, b, false);
    const AttnShape sh = attn_shape(a, rq, kRows);
    const int item = (int)((w - s.before[b]) / sh.key_tiles);
    const int head = item / sh.row_tiles, row0 = (item % sh.row_tiles) * kRows;
    const int live = min(kRows, rq.nodes * a.group - row0);
    const long long item0 = s.before[b] + (long long)item * sh.key_tiles, item1 = item0 + sh.key_tiles;
    const long long w1 = end < item1 ? end : item1;
    const int t0 = (int)(w - item0), t1 = (int)(w1 - item0);
    const int len = rq.ctx + rq.nodes;

    // places of tile t's keys, one thread each, into buffer t & 1
    auto place = [&](int t) {
      if (tid < kKeyTile && t < t1) {
        int64_t k, v;
        attn_place(a, b, t * kKeyTile + tid, len, head, k, v);
        s.place[t & 1][0][tid] = k;
        s.place[t & 1][1][tid] = v;
      }
    };
    auto load = [&](int t) {
      if (t < t1) {
        const int st = (t - t0) % kStages;
#pragma unroll 4
        for (int u = tid; u < kKeyTile * kUnits; u += kThreads) {
          const int r = u / kUnits, c = u % kUnits;
          const uint32_t to = (uint32_t)(r * Cfg::kRowBytes + ((c ^ (r & 7)) << 4));
          const int64_t k = s.place[t & 1][0][r], v = s.place[t & 1][1][r];
          cp16_or_zero(smem_u32(s.ring[st][0]) + to, kc + (k < 0 ? 0 : k + c * 8), k >= 0);
          cp16_or_zero(smem_u32(s.ring[st][1]) + to, vc + (v < 0 ? 0 : v + c * 8), v >= 0);
        }
      }
      cp_commit();
    };

    __syncthreads();  // the item before is done with shared memory
    for (int u = tid; u < kRows * kUnits; u += kThreads) {
      const int r = u / kUnits, c = u % kUnits;
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (r < live) {
        const int node = (row0 + r) / a.group, h = head * a.group + (row0 + r) % a.group;
        x = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (int64_t)(rq.n0 + node) * a.q_sn +
                                            (int64_t)h * a.q_sh + c * 8);
      }
      *reinterpret_cast<uint4*>(s.q + r * Cfg::kRowBytes + ((c ^ (r & 7)) << 4)) = x;
    }
    for (int r = tid; r < kRows; r += kThreads) s.mask[r] = r < live ? attn_mask(a, rq, (row0 + r) / a.group) : 0ull;
    place(t0);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      load(t0 + i);
      place(t0 + i + 1);
      __syncthreads();
    }

    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    constexpr float kHead = kNarrow<T> ? 15.f : 0.f, kFall = 22.f;
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};  // reference, sum of weights
    float peak[2] = {-INFINITY, -INFINITY};                      // the highest reference so far
    const int g = lane >> 2, q2 = (lane & 3) * 2;

    for (int t = t0; t < t1; ++t) {
      cp_wait<kStages - 2>();
      __syncthreads();
      load(t + kStages - 1);
      const int st = (t - t0) % kStages;
      uint8_t* kt = s.ring[st][0];
      uint8_t* vt = s.ring[st][1];
      const int pos0 = t * kKeyTile;
      const bool tail = pos0 + kKeyTile > rq.ctx;  // drafted tokens, or places past the end
      unsigned long long odd = 0ull;
      if (tail) {
        // A drafted token hidden from a row has weight 0 there, but 0 times an infinite or NaN value
        // is NaN: such tokens' values are taken out of the product and added row by row below.
        if (tid < 2) s.odd[tid] = 0u;
        __syncthreads();
        for (int u = tid; u < kKeyTile * kUnits; u += kThreads) {
          const int r = u / kUnits;
          if (pos0 + r < rq.ctx) continue;
          const uint4 x = lds128(vt + u * 16);
          if (not_finite<T>(x.x) || not_finite<T>(x.y) || not_finite<T>(x.z) || not_finite<T>(x.w))
            atomicOr(&s.odd[r >> 5], 1u << (r & 31));
        }
        __syncthreads();
        odd = ((unsigned long long)s.odd[1] << 32) | s.odd[0];
        if (odd) {
          for (int u = tid; u < kKeyTile * kUnits; u += kThreads)
            if (odd >> (u / kUnits) & 1) *reinterpret_cast<uint4*>(vt + u * 16) = make_uint4(0u, 0u, 0u, 0u);
          __syncthreads();
        }
      }

      // scores of 16 rows x kKeys keys
      float sc[kKeys / 8][4];
#pragma unroll
      for (int i = 0; i < kKeys / 8; ++i) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.f;
#pragma unroll 4
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t qa[4];
        const int qr = wr * 16 + (lane & 15), qc = kk * 2 + (lane >> 4);
        ldsm4(qa, smem_u32(s.q) + qr * Cfg::kRowBytes + ((qc ^ (qr & 7)) << 4));
#pragma unroll
        for (int i = 0; i < kKeys / 16; ++i) {
          uint32_t kb[4];
          const int r = wk * kKeys + i * 16 + (lane & 7) + ((lane >> 4) << 3), c = kk * 2 + ((lane >> 3) & 1);
          ldsm4(kb, smem_u32(kt) + r * Cfg::kRowBytes + ((c ^ (r & 7)) << 4));
          Mma<T>::mma(sc[2 * i], qa, kb[0], kb[1]);
          Mma<T>::mma(sc[2 * i + 1], qa, kb[2], kb[3]);
        }
      }
#pragma unroll
      for (int i = 0; i < kKeys / 8; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[i][e] *= c2;
          if (tail) {
            const int pos = pos0 + wk * kKeys + i * 8 + q2 + (e & 1), d = pos - rq.ctx;
            const unsigned long long m = s.mask[wr * 16 + g + (e >> 1) * 8];
            if (d >= 0 && (d >= rq.nodes || !(m >> d & 1))) sc[i][e] = -INFINITY;
          }
        }
      }
      float rescale[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = kNarrow<T> ? -INFINITY : top[h];
#pragma unroll
        for (int i = 0; i < kKeys / 8; ++i) mx = fmaxf(mx, fmaxf(sc[i][2 * h], sc[i][2 * h + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        if (kNarrow<T>) {
          const float at = mx - kHead;
          peak[h] = fmaxf(peak[h], at);
          mx = at < top[h] - kFall && at > -INFINITY ? fmaxf(at, peak[h] - kSpan) : fmaxf(at, top[h]);
        }
        const float ref = mx == -INFINITY ? 0.f : mx;
        rescale[h] = exp2_fast(top[h] - ref);
        top[h] = mx;
        float add = 0.f;
#pragma unroll
        for (int i = 0; i < kKeys / 8; ++i) {
          sc[i][2 * h] = exp2_fast(sc[i][2 * h] - ref);
          sc[i][2 * h + 1] = exp2_fast(sc[i][2 * h + 1] - ref);
          add += sc[i][2 * h] + sc[i][2 * h + 1];
        }
        sum[h] = sum[h] * rescale[h] + add;
      }
      if (__any_sync(0xffffffffu, rescale[0] != 1.f || rescale[1] != 1.f)) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          o[i][0] *= rescale[0];
          o[i][1] *= rescale[0];
          o[i][2] *= rescale[1];
          o[i][3] *= rescale[1];
        }
      }
#pragma unroll
      for (int i = 0; i < kKeys / 16; ++i) {
        const uint32_t pa[4] = {Mma<T>::pack(sc[2 * i][0], sc[2 * i][1]), Mma<T>::pack(sc[2 * i][2], sc[2 * i][3]),
                                Mma<T>::pack(sc[2 * i + 1][0], sc[2 * i + 1][1]),
                                Mma<T>::pack(sc[2 * i + 1][2], sc[2 * i + 1][3])};
        const int r = wk * kKeys + i * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          uint32_t vb[4];
          const int c = j * 2 + (lane >> 4);
          ldsm4_t(vb, smem_u32(vt) + r * Cfg::kRowBytes + ((c ^ (r & 7)) << 4));
          Mma<T>::mma(o[2 * j], pa, vb[0], vb[1]);
          Mma<T>::mma(o[2 * j + 1], pa, vb[2], vb[3]);
        }
      }
      while (odd) {  // rare: values that are not finite, for the rows that see them
        const int j = __ffsll((long long)odd) - 1;
        odd &= odd - 1;
        const int jl = j - wk * kKeys, d = pos0 + j - rq.ctx;
        if (jl < 0 || jl >= kKeys || d >= rq.nodes) continue;
        float p[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kKeys / 8; ++i) {
          if (i != jl >> 3) continue;
          p[0] = (jl & 1) ? sc[i][1] : sc[i][0];
          p[1] = (jl & 1) ? sc[i][3] : sc[i][2];
        }
        const int src = (lane & 28) | ((jl & 7) >> 1);
        p[0] = __shfl_sync(0xffffffffu, p[0], src);
        p[1] = __shfl_sync(0xffffffffu, p[1], src);
        int64_t ko, vo;
        attn_place(a, b, pos0 + j, len, head, ko, vo);
        if (vo < 0) continue;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!(s.mask[wr * 16 + g + 8 * h] >> d & 1)) continue;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            o[i][2 * h] += p[h] * Mma<T>::one(vc[vo + i * 8 + q2]);
            o[i][2 * h + 1] += p[h] * Mma<T>::one(vc[vo + i * 8 + q2 + 1]);
          }
        }
      }
      place(t + kStages);
    }
    cp_wait<0>();
    __syncthreads();

    // join the row tile's warps
    float* join = reinterpret_cast<float*>(s.ring);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
    }
    if (WK > 1) {
      constexpr int kJ = Cfg::kJoinRow;
      float* stat = join + (WK - 1) * MT * 16 * kJ;
      if (wk > 0) {
        const int slot = (wk - 1) * MT + wr;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = g + 8 * h;
          float* to = join + (slot * 16 + r) * kJ;
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
            *reinterpret_cast<float2*>(to + i * 8 + q2) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
          if ((lane & 3) == 0) {
            stat[(slot * 16 + r) * 2] = top[h];
            stat[(slot * 16 + r) * 2 + 1] = sum[h];
          }
        }
      }
      __syncthreads();
      if (wk == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = g + 8 * h;
          float mx = top[h];
#pragma unroll
          for (int x = 0; x < WK - 1; ++x) mx = fmaxf(mx, stat[((x * MT + wr) * 16 + r) * 2]);
          const float ref = mx == -INFINITY ? 0.f : mx;
          float f = exp2_fast(top[h] - ref);
          sum[h] *= f;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) o[i][2 * h] *= f, o[i][2 * h + 1] *= f;
#pragma unroll
          for (int x = 0; x < WK - 1; ++x) {
            const int slot = x * MT + wr;
            f = exp2_fast(stat[(slot * 16 + r) * 2] - ref);
            sum[h] += f * stat[(slot * 16 + r) * 2 + 1];
            const float* from = join + (slot * 16 + r) * kJ;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
              const float2 y = *reinterpret_cast<const float2*>(from + i * 8 + q2);
              o[i][2 * h] += f * y.x;
              o[i][2 * h + 1] += f * y.y;
            }
          }
          top[h] = mx;
        }
      }
    }
    if (wk == 0) {
      const bool all = w == item0 && w1 == item1;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = wr * 16 + g + 8 * h;
        if (r >= live) continue;
        if (all) {
          const int node = rq.n0 + (row0 + r) / a.group, hq = head * a.group + (row0 + r) % a.group;
          const float inv = sum[h] > 0.f || sum[h] != sum[h] ? 1.f / sum[h] : 0.f;
          T* to = reinterpret_cast<T*>(a.out) + (int64_t)node * a.o_sn + (int64_t)hq * a.o_sh;
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
            *reinterpret_cast<uint32_t*>(to + i * 8 + q2) = Mma<T>::pack(o[i][2 * h] * inv, o[i][2 * h + 1] * inv);
          if (a.lse && (lane & 3) == 0)
            a.lse[(int64_t)node * a.Hq + hq] =
                sum[h] == 0.f ? -INFINITY : (top[h] + log2f(sum[h])) * 0.6931471805599453f;
        } else {
          float* slot = a.partials + (2ll * blockIdx.x + (w == item0 ? 1 : 0)) * attn_slot_floats(kRows, D);
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
            *reinterpret_cast<float2*>(slot + (int64_t)r * D + i * 8 + q2) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
          if ((lane & 3) == 0)
            *reinterpret_cast<float2*>(slot + (int64_t)kRows * D + 2 * r) = make_float2(top[h], sum[h]);
        }
      }
    }
    w = w1;
  }
}

// Where the partial results of (node n, head hq) are: the CTAs c0 .. c1 that held its item, and its row in
// their slots; c0 == c1 where one CTA held the item and wrote the result itself, or there is none.
struct Parts {
  int c0, c1, row;
};
__device__ __forceinline__ Parts find_parts(const AttnArgs& a, const AttnReq& rq, long long ahead, long long total,
                                            long long G, int rows, int n, int hq) {
  if (total == 0 || n < rq.n0 || n >= rq.n0 + rq.nodes) return Parts{0, 0, 0};
  const AttnShape sh = attn_shape(a, rq, rows);
  const int row = (n - rq.n0) * a.group + hq % a.group;
  const int item = hq / a.group * sh.row_tiles + row / rows;
  const long long item0 = ahead + (long long)item * sh.key_tiles, item1 = item0 + sh.key_tiles;
  return Parts{attn_cta_of(item0, total, G), attn_cta_of(item1 - 1, total, G), row % rows};
}

// The request that holds node n.
__device__ __forceinline__ int request_of(const AttnArgs& a, int n) {
  int lo = 0, hi = a.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.node_offsets[mid] <= n) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Adds up the partial results of the items that several CTAs held.  First the slots' maxima and sums, which
// give each slot its factor; then the sums, with several loads in flight.  WPR warps share a row (a node's
// query head): 8 where rows are few and their slots many, 1 where there are rows for every warp (measured
// at 24 ragged requests: 14 us less than a block a row; at 256 rows of 74 slots a block a row is faster).
template <typename T, int D, int WPR>
__global__ void __launch_bounds__(256) tree_attn_combine_kernel(const __grid_constant__ AttnArgs a, int rows, int grid) {
  constexpr int kPer = D / 32;  // columns of a lane: pairs or fours, 32 lanes apart
  constexpr int kVec = kPer < 4 ? kPer : 4, kN = kPer / kVec;
  __shared__ long long before[kAttnMaxBatch + 1];
  __shared__ long long scratch[8];
  __shared__ float factor[8 / WPR][kAttnMaxGrid];
  __shared__ float part[WPR == 8 ? 8 : 1][WPR == 8 ? D : 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // the lengths were there before the launch whose partials these are: only those are waited for
  attn_prefix(a, rows, before, scratch, false);
  const long long total = before[a.B];
  const long long G = total < (long long)grid ? total : (long long)grid;
  const int n = blockIdx.x, hq = WPR == 8 ? blockIdx.y : blockIdx.y * 8 + warp;
  const int b = request_of(a, n);
  const Parts p = hq < a.Hq ? find_parts(a, attn_request(a, b, false), before[b], total, G, rows, n, hq) : Parts{0, 0, 0};
  pdl_wait();
  if (p.c0 == p.c1) return;
  const int64_t size = attn_slot_floats(rows, D);
  // slot of contributor i: the item's first CTA holds its beginning, the others from their start
  auto slot = [&](int i) { return a.partials + (2ll * (p.c0 + i) + (i == 0 ? 1 : 0)) * size; };
  const int count = p.c1 - p.c0 + 1;  // at most the grid
  float2 st[kAttnMaxGrid / 32];
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int z = 0; z < kAttnMaxGrid / 32; ++z) {
    const int i = z * 32 + lane;
    st[z] = i < count ? __ldcg(reinterpret_cast<const float2*>(slot(i) + (int64_t)rows * D + 2 * p.row))
                      : make_float2(-INFINITY, 0.f);
    top = fmaxf(top, st[z].x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float ref = top == -INFINITY ? 0.f : top;
  float* mine = factor[WPR == 8 ? 0 : warp];  // WPR = 8: every warp writes the same
#pragma unroll
  for (int z = 0; z < kAttnMaxGrid / 32; ++z) {
    const float f = exp2_fast(st[z].x - ref);
    sum += st[z].y * f;
    if (z * 32 + lane < count) mine[z * 32 + lane] = f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncwarp();
  float acc[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
#pragma unroll 8
  for (int i = WPR == 8 ? warp : 0; i < count; i += WPR) {
    const float* from = slot(i) + (int64_t)p.row * D + lane * kVec;
    const float g = mine[i];
#pragma unroll
    for (int z = 0; z < kN; ++z) {
      if (kVec == 4) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(from + z * 128));
        acc[z * 4] += v.x * g, acc[z * 4 + 1] += v.y * g, acc[z * 4 + 2] += v.z * g, acc[z * 4 + 3] += v.w * g;
      } else {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(from));
        acc[0] += v.x * g, acc[1] += v.y * g;
      }
    }
  }
  if (WPR == 8) {
#pragma unroll
    for (int z = 0; z < kN; ++z)
#pragma unroll
      for (int e = 0; e < kVec; ++e) part[warp][z * 128 + lane * kVec + e] = acc[z * kVec + e];
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int z = 0; z < kN; ++z)
#pragma unroll
      for (int e = 0; e < kVec; ++e)
#pragma unroll
        for (int w = 1; w < WPR; ++w) acc[z * kVec + e] += part[w][z * 128 + lane * kVec + e];
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  T* to = reinterpret_cast<T*>(a.out) + (int64_t)n * a.o_sn + (int64_t)hq * a.o_sh + lane * kVec;
#pragma unroll
  for (int z = 0; z < kN; ++z)
#pragma unroll
    for (int e = 0; e < kVec; e += 2)
      *reinterpret_cast<uint32_t*>(to + z * 128 + e) =
          Mma<T>::pack(acc[z * kVec + e] * inv, acc[z * kVec + e + 1] * inv);
  if (a.lse && lane == 0)
    a.lse[(int64_t)n * a.Hq + hq] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

namespace {

template <typename T, int D, int MT, int WK>
int launch_form(const AttnArgs& a, cudaStream_t stream, int& grid, int& rows) {
  using Cfg = AttnCfg<D, MT, WK>;
  const void* k = (const void*)tree_attn_kernel<T, D, MT, WK>;
  if (!prepare_kernel(k)) return 2;
  const size_t smem = sizeof(typename Cfg::Smem);
  grid = num_sms();
  rows = Cfg::kRows;
  return launch_with_pdl(k, a, grid, Cfg::kThreads, smem, a.pdl, stream);
}

template <typename T, int D>
int launch_d(const AttnArgs& a, cudaStream_t stream) {
  int grid = 0, rows = 0, rc;
  const int most = a.max_nodes * a.group;
  // The tensor-memory form needs some tiles a CTA to pay for its start-up and its row tiles of 128.  In
  // key tiles an SM, times row tiles of 32: one token over 1,000 keys (0.2) 12.1 us here and 15.2 there,
  // 4 requests of 16 nodes over 1,000 (7.4) 23.7 and 29.1, one token over 32k (7) 29.4 and 32.3, 8 nodes
  // over 32k (14) 43.8 and 36.7, 16 nodes over 32k (28) 63.8 and 38.9, 16 requests of one token over 8k
  // (111) 117 and 88.
  const int64_t tiles = (int64_t)a.B * a.Hk * ((a.max_context + a.max_nodes + kKeyTile - 1) / kKeyTile);
  if (tiles * ((most + 31) / 32) > 8 * num_sms()) rc = launch_tree_attn_tc(a, stream, grid, rows);
  else if (most <= 16) rc = launch_form<T, D, 1, 4>(a, stream, grid, rows);
  else if (most <= 32) rc = launch_form<T, D, 2, 4>(a, stream, grid, rows);
  else rc = launch_form<T, D, 4, 2>(a, stream, grid, rows);
  if (rc) return rc;
  if (a.max_context + a.max_nodes <= kKeyTile) return 0;  // one key tile: no item is split
  cudaLaunchConfig_t cfg = {};
  const bool many = (int64_t)a.N * a.Hq >= 8 * num_sms();  // a row for each of eight warps an SM
  cfg.gridDim = dim3(a.N, many ? (a.Hq + 7) / 8 : a.Hq);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  AttnArgs args = a;
  void* params[3] = {&args, &rows, &grid};
  const void* k = many ? (const void*)tree_attn_combine_kernel<T, D, 1> : (const void*)tree_attn_combine_kernel<T, D, 8>;
  return cudaLaunchKernelExC(&cfg, k, params) == cudaSuccess ? 0 : 2;
}

template <typename T>
int launch_t(const AttnArgs& a, cudaStream_t stream) {
  if (a.D == 64) return launch_d<T, 64>(a, stream);
  if (a.D == 128) return launch_d<T, 128>(a, stream);
  return launch_d<T, 256>(a, stream);
}

}  // namespace

int64_t attn_workspace_floats() {
  // the widest slots: 256 rows of 128, 128 rows of 256
  return 2ll * num_sms() * attn_slot_floats(256, 128);
}

int launch_tree_attn(const AttnArgs& a, cudaStream_t stream) {
  return a.f16 ? launch_t<__half>(a, stream) : launch_t<__nv_bfloat16>(a, stream);
}

// What the other kernels need of a tree: one thread per node walks to the root.
__global__ void __launch_bounds__(128) tree_layout_kernel(const __grid_constant__ TreeArgs a) {
  pdl_wait();
  const int n = blockIdx.x * blockDim.x + threadIdx.x;
  if (n < a.N) {
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.node_offsets[mid] <= n) lo = mid;
      else hi = mid;
    }
    const int n0 = a.node_offsets[lo], n1 = a.node_offsets[lo + 1];
    // Nodes of no request, ahead of the first and behind the last, see nothing.  Then the attention's test of a
    // request: its nodes are rows of the arrays, 64 at most.
    const bool none = n < n0 || n >= n1;
    if (none || n0 < 0 || n1 > a.N || n1 - n0 > 64) {
      if (!none) record_error(a.err, ERR_LENGTHS);
      if (a.mask) a.mask[n] = 0ull;
      if (a.positions) a.positions[n] = 0;
      if (a.slots) a.slots[n] = -1;
    } else {
      const int i = n - n0;
      unsigned long long seen = 1ull << i;
      int depth = 0;
      for (int at = i;;) {
        const int p = a.parents[n0 + at];
        if (p == -1) break;
        if (p < 0 || p >= at) {
          record_error(a.err, ERR_TREE);
          break;
        }
        seen |= 1ull << p;
        ++depth;
        at = p;
      }
      const int64_t ctx = a.context_lens ? a.context_lens[lo] : 0;
      if (a.mask) a.mask[n] = seen;
      if (a.positions) a.positions[n] = ctx + depth;
      if (a.slots) {
        const int64_t at = ctx + i;
        int64_t slot = -1;
        if (ctx < 0 || at >= (int64_t)a.table_width * a.page_size) {
          record_error(a.err, ERR_LENGTHS);
        } else {
          const int64_t page = a.page_table[(int64_t)lo * a.table_ld + at / a.page_size];
          if (page < 0 || page >= a.num_pages) record_error(a.err, ERR_PAGE);
          else slot = page * a.page_size + at % a.page_size;
        }
        a.slots[n] = slot;
      }
    }
  }
  pdl_trigger();
}

int launch_tree_layout(const TreeArgs& a, cudaStream_t stream) {
  return launch_with_pdl((const void*)tree_layout_kernel, a, (a.N + 127) / 128, 128, 0, a.pdl, stream);
}

}  // namespace fnx
