// Attention of drafted token trees over an 8-bit paged cache: tree_attn.cu's operator (its formula, masks, split of
// the work and joining launch) on a cache of e4m3 values with a scale for each block of tokens and head
// (tree_attn8.cuh says how the scales enter).
//
// Bound: the cache's bytes, half of a 16-bit cache's.  Keys and values stay 8 bits wide in shared memory (cp.async
// into a ring) and become fp16 in the registers that feed mma.sync.m16n8k16:
//   scores  A lane reads 16 consecutive bytes of a key, which are its operands of four steps: the order of the head's
//           elements within 64 is permuted, for the queries alike, which a sum does not see.
//   output  ldmatrix with transposition moves pairs of bytes, so a lane gets two neighbouring elements d, d + 1 of
//           two keys; a byte permutation makes of them the two keys' d and the two keys' d + 1, operands of two
//           column tiles that have every other d each.  A lane's sums are then four neighbouring elements.
#include "tree_attn8.cuh"

namespace fnx {

namespace {

__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// MT row tiles of 16; WK warps share a row tile and a key tile; TG sets of these take key tiles in turn.
template <int D, int MT, int WK, int TG>
struct Attn8Cfg {
  static constexpr int kThreads = 32 * MT * WK * TG;
  static constexpr int kRows = 16 * MT;
  static constexpr int kUnits = D / 16;             // 16-byte units of a key
  static constexpr int kTileBytes = kKeyTile * D;   // keys or values of one tile
  static constexpr int kStages = (D == 256 ? 4 : D == 128 ? 8 : 12) / TG;  // of TG tiles
  static constexpr int kParts = WK * TG;            // warps that share a row tile
  static constexpr int kPass = kThreads / kUnits;   // rows that the block copies at a time
  static_assert(kPass % kGroup == 0 || kPass == 8, "a thread's rows have one place in their groups, or two");
  static constexpr int kKeys = kKeyTile / WK;       // keys of a tile per warp
  static constexpr int kJoinRow = D + 4;            // floats; pads the rows apart
  static_assert((kParts - 1) * MT * 16 * (kJoinRow + 2) * 4 <= kStages * TG * 2 * kTileBytes, "join area");
  static_assert(kKeys % kGroup == 0, "a warp has whole groups");
  struct Smem {
    alignas(128) uint8_t ring[kStages][2][TG * kTileBytes];
    alignas(128) uint8_t q[kRows * D * 2];
    float2 scales[kStages][TG * kKeyTile / kGroup];  // of the ring's groups: keys', values'
    Place8 place[2][TG * kKeyTile / kGroup];         // of a stage's groups, which one page and one block hold each
    unsigned long long mask[kRows];
    long long before[kAttnMaxBatch + 1];
    long long scratch[32];
    float factor[kRows];  // of a row's scores
    uint32_t odd[TG][2];  // drafted tokens of a tile with NaN values
  };
  // Places of 16-byte units in their rows, so that the eight lanes of one access meet eight different ones modulo
  // 128 bytes: two keys times four units of 16 for the scores, eight keys for the values.
  static __device__ __forceinline__ int key_unit(int r, int c) { return D == 64 ? c : c ^ ((r & 1) << 2); }
  static __device__ __forceinline__ int value_unit(int r, int c) { return D == 64 ? c ^ ((r >> 1) & 3) : c ^ (r & 7); }
};

}  // namespace

template <typename T, int D, int MT, int WK, int TG>
__global__ void __launch_bounds__(32 * MT * WK * TG, 1) tree_attn8_kernel(const __grid_constant__ Attn8Args a) {
  using Cfg = Attn8Cfg<D, MT, WK, TG>;
  constexpr int kRows = Cfg::kRows, kStages = Cfg::kStages, kKeys = Cfg::kKeys, kThreads = Cfg::kThreads;
  constexpr int kUnits = Cfg::kUnits, kGroups = kKeys / kGroup;
  constexpr bool kHold = D <= 128;  // the queries' operands stay in registers
  extern __shared__ __align__(128) uint8_t raw[];
  typename Cfg::Smem& s = *reinterpret_cast<typename Cfg::Smem*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tg = warp / (MT * WK), wr = warp / WK % MT, wk = warp % WK;
  const uint8_t* kc = reinterpret_cast<const uint8_t*>(a.k_cache);
  const uint8_t* vc = reinterpret_cast<const uint8_t*>(a.v_cache);
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

    // A stage is TG tiles from t on.  Its groups' places, one thread each, go to buffer `which`.
    constexpr int kStageGroups = TG * kKeyTile / kGroup;
    auto find = [&](int t) {
      return tid < kStageGroups && t < t1 ? attn8_look(a, b, t * kKeyTile + tid * kGroup, len, head) : Look8{0, -1, 0};
    };
    auto put = [&](int which, const Look8& l) {
      if (tid < kStageGroups) s.place[which][tid] = attn8_place(a, l);
    };
    const int row = tid / kUnits, unit = tid % kUnits;
    auto load = [&](int t, int stage) {
      if (t < t1) {
        const Place8* place = s.place[stage & 1];
        const int st = stage % kStages, end_row = min(t1, t + TG) * kKeyTile;
#pragma unroll
        for (int j = 0; j < TG * kKeyTile / Cfg::kPass; ++j) {
          const int r = j * Cfg::kPass + row;
          const Place8& p = place[r / kGroup];
          const int64_t k = p.k + (r % kGroup) * a.kc_st[1] + unit * 16, v = p.v + (r % kGroup) * a.vc_st[1] + unit * 16;
          const bool there = p.k >= 0 && t * kKeyTile + r < min(len, end_row);
          cp16_or_zero(smem_u32(s.ring[st][0]) + r * D + (Cfg::key_unit(r, unit) << 4), kc + (there ? k : 0), there);
          cp16_or_zero(smem_u32(s.ring[st][1]) + r * D + (Cfg::value_unit(r, unit) << 4), vc + (there ? v : 0), there);
        }
        if (tid < 2 * kStageGroups) {
          const int g = tid >> 1;
          const int64_t at = tid & 1 ? place[g].vs : place[g].ks;
          float* to = tid & 1 ? &s.scales[st][g].y : &s.scales[st][g].x;
          if (at >= 0) cp_async4(to, (tid & 1 ? a.v_scale : a.k_scale) + at);
          else *to = 1.f;
        }
      }
      cp_commit();
    };

    __syncthreads();  // the item before is done with shared memory
    put(0, find(t0));
    for (int r = warp; r < kRows; r += kThreads / 32) {  // a warp a row: two elements a lane and step
      constexpr int kSteps = D / 64;
      float2 x[kSteps];
      float amax = 0.f;
      const int node = (row0 + r) / a.group, h = head * a.group + (row0 + r) % a.group;
      const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)(rq.n0 + node) * a.q_sn + (int64_t)h * a.q_sh;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        x[i] = r < live ? two_floats<T>(*reinterpret_cast<const uint32_t*>(q + i * 64 + lane * 2)) : make_float2(0.f, 0.f);
        const float m = fmaxf(fabsf(x[i].x), fabsf(x[i].y));
        amax = fmaxf(amax, m);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const int e = row_exponent(amax);
      const float f = pow2f(e);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int c = i * 8 + (lane >> 2);
        *reinterpret_cast<uint32_t*>(s.q + r * (D * 2) + ((c ^ (r & 1)) << 4) + (lane & 3) * 4) =
            round_pair<__half>(x[i].x * f, x[i].y * f);
      }
      if (lane == 0) {
        s.factor[r] = c2 * pow2f(-e);
        s.mask[r] = r < live ? attn_mask(a, rq, node) : 0ull;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      load(t0 + i * TG, i);
      put((i + 1) & 1, find(t0 + (i + 1) * TG));
      __syncthreads();
    }

    const int g = lane >> 2, q4 = lane & 3, q2 = q4 * 2;
    // a row's 16 elements of 64: operands of four steps, rows g and g + 8
    auto query = [&](int kb, uint32_t (&x)[2][8]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = wr * 16 + g + 8 * h;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const uint4 v = lds128(s.q + r * (D * 2) + (((kb * 8 + q4 * 2 + z) ^ (r & 1)) << 4));
          x[h][4 * z] = v.x, x[h][4 * z + 1] = v.y, x[h][4 * z + 2] = v.z, x[h][4 * z + 3] = v.w;
        }
      }
    };
    uint32_t held[kHold ? D / 64 : 1][2][8];
    if (kHold) {
#pragma unroll
      for (int kb = 0; kb < D / 64; ++kb) query(kb, held[kHold ? kb : 0]);
    }
    const float factor[2] = {s.factor[wr * 16 + g], s.factor[wr * 16 + g + 8]};
    float o[kUnits][2][4];  // elements 16 c + 4 q4 + (0, 2), (1, 3) of rows g and g + 8
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) o[i][e][0] = o[i][e][1] = o[i][e][2] = o[i][e][3] = 0.f;
    constexpr float kHead = 15.f, kFall = 22.f;
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};  // reference, sum of weights
    float peak[2] = {-INFINITY, -INFINITY};                      // the highest reference so far

    Look8 ahead = find(t0 + kStages * TG);
    for (int ts = t0, stage = 0; ts < t1; ts += TG, ++stage) {
      cp_wait<kStages - 2>();
      __syncthreads();
      load(ts + (kStages - 1) * TG, stage + kStages - 1);
      put((stage + kStages) & 1, ahead);
      ahead = find(ts + (kStages + 1) * TG);  // a page number has an iteration to arrive
      const int st = stage % kStages, t = ts + tg;
      uint8_t* kt = s.ring[st][0] + tg * Cfg::kTileBytes;
      uint8_t* vt = s.ring[st][1] + tg * Cfg::kTileBytes;
      const int pos0 = t * kKeyTile;
      const bool tail = (ts + TG) * kKeyTile > rq.ctx;  // drafted tokens, or places past the end, in one of the tiles
      unsigned long long odd = 0ull;
      if (tail) {
        // A drafted token hidden from a row has weight 0 there, but 0 times NaN is NaN: such tokens' values are
        // taken out of the product and added row by row below.
        if (tid < 2 * TG) s.odd[tid >> 1][tid & 1] = 0u;
        __syncthreads();
        uint8_t* all = s.ring[st][1];
        const int rows = min(t1 - ts, TG) * kKeyTile;
        for (int u = tid; u < rows * kUnits; u += kThreads) {
          const int r = u / kUnits;
          if (ts * kKeyTile + r < rq.ctx) continue;
          const uint4 x = lds128(all + u * 16);
          if (has_nan(x.x) || has_nan(x.y) || has_nan(x.z) || has_nan(x.w))
            atomicOr(&s.odd[r / kKeyTile][(r >> 5) & 1], 1u << (r & 31));
        }
        __syncthreads();
        odd = ((unsigned long long)s.odd[tg][1] << 32) | s.odd[tg][0];
        bool any = false;
        for (int i = 0; i < TG; ++i) any |= (s.odd[i][0] | s.odd[i][1]) != 0u;
        if (any) {
          for (int u = tid; u < rows * kUnits; u += kThreads) {
            const int r = u / kUnits;
            if (s.odd[r / kKeyTile][(r >> 5) & 1] >> (r & 31) & 1) *reinterpret_cast<uint4*>(all + u * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          __syncthreads();
        }
      }
      if (TG > 1 && t >= t1) continue;  // the segment ends within the stage

      // scores of 16 rows x kKeys keys
      float sc[kKeys / 8][4];
#pragma unroll
      for (int i = 0; i < kKeys / 8; ++i) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.f;
#pragma unroll
      for (int kb = 0; kb < D / 64; ++kb) {
        uint32_t now[2][8];
        if (!kHold) query(kb, now);
        const uint32_t(&x)[2][8] = kHold ? held[kHold ? kb : 0] : now;
#pragma unroll
        for (int i = 0; i < kKeys / 8; ++i) {
          const int r = wk * kKeys + i * 8 + g;
          const uint4 v = lds128(kt + r * D + (Cfg::key_unit(r, kb * 4 + q4) << 4));
          const uint32_t y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            uint32_t b0, b1;
            deq_fp8_word(y[z], b0, b1);
            mma_f16(sc[i], x[0][2 * z], x[1][2 * z], x[0][2 * z + 1], x[1][2 * z + 1], b0, b1);
          }
        }
      }
      float4 gs[kGroups];
#pragma unroll
      for (int z = 0; z < kGroups; ++z) gs[z] = group_factors(a, s.scales[st][tg * (kKeyTile / kGroup) + wk * kGroups + z]);
#pragma unroll
      for (int i = 0; i < kKeys / 8; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // the factor stays above zero: a hidden key's -inf has to
          sc[i][e] = fmaf(sc[i][e], fmaxf(factor[e >> 1] * gs[i / 2].x, 1e-30f), gs[i / 2].y);
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
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < kKeys / 8; ++i) mx = fmaxf(mx, fmaxf(sc[i][2 * h], sc[i][2 * h + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float at = mx - kHead;
        peak[h] = fmaxf(peak[h], at);
        mx = at < top[h] - kFall && at > -INFINITY ? fmaxf(at, peak[h] - kSpan) : fmaxf(at, top[h]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        rescale[h] = exp2_fast(top[h] - ref);
        top[h] = mx;
        float add = 0.f;
#pragma unroll
        for (int z = 0; z < kGroups; ++z) {
          float part = 0.f;
#pragma unroll
          for (int i = 2 * z; i < 2 * z + 2; ++i) {
            sc[i][2 * h] = exp2_fast(sc[i][2 * h] - ref);
            sc[i][2 * h + 1] = exp2_fast(sc[i][2 * h + 1] - ref);
            part += sc[i][2 * h] + sc[i][2 * h + 1];
          }
          add = fmaf(part, gs[z].z, add);
        }
        sum[h] = sum[h] * rescale[h] + add;
      }
      if (__any_sync(0xffffffffu, rescale[0] != 1.f || rescale[1] != 1.f)) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            o[i][e][0] *= rescale[0];
            o[i][e][1] *= rescale[0];
            o[i][e][2] *= rescale[1];
            o[i][e][3] *= rescale[1];
          }
      }
#pragma unroll
      for (int z = 0; z < kGroups; ++z) {
        const uint32_t p0 = round_pair<__half>(sc[2 * z][0], sc[2 * z][1]), p1 = round_pair<__half>(sc[2 * z][2], sc[2 * z][3]),
                       p2 = round_pair<__half>(sc[2 * z + 1][0], sc[2 * z + 1][1]),
                       p3 = round_pair<__half>(sc[2 * z + 1][2], sc[2 * z + 1][3]);
        const int r = wk * kKeys + z * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < kUnits / 2; ++j) {
          uint32_t vb[4];  // keys 0 .. 7 and 8 .. 15 of unit 2 j, then of 2 j + 1
          ldsm4_t(vb, smem_u32(vt) + r * D + (Cfg::value_unit(r, 2 * j + (lane >> 4)) << 4));
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t even0, odd0, even1, odd1;  // a key pair's elements d, and d + 1
            deq_fp8_word(__byte_perm(vb[2 * y], 0, 0x3120), even0, odd0);
            deq_fp8_word(__byte_perm(vb[2 * y + 1], 0, 0x3120), even1, odd1);
            mma_f16(o[2 * j + y][0], p0, p1, p2, p3, even0, even1);
            mma_f16(o[2 * j + y][1], p0, p1, p2, p3, odd0, odd1);
          }
        }
      }
      while (odd) {  // rare: NaN values, for the rows that see them
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
        const int64_t vo = attn8_place(a, b, pos0 + j, len, head).v;
        if (vo < 0) continue;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!(s.mask[wr * 16 + g + 8 * h] >> d & 1)) continue;
#pragma unroll
          for (int i = 0; i < kUnits; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e & 1][2 * h + (e >> 1)] += p[h] * e4m3_value(vc[vo + i * 16 + q4 * 4 + e]);
        }
      }
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
    const int part = tg * WK + wk;
    {
      constexpr int kJ = Cfg::kJoinRow;
      float* stat = join + (Cfg::kParts - 1) * MT * 16 * kJ;
      if (part > 0) {
        const int slot = (part - 1) * MT + wr;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = g + 8 * h;
          float* to = join + (slot * 16 + r) * kJ + q4 * 4;
#pragma unroll
          for (int i = 0; i < kUnits; ++i)
            *reinterpret_cast<float4*>(to + i * 16) =
                make_float4(o[i][0][2 * h], o[i][1][2 * h], o[i][0][2 * h + 1], o[i][1][2 * h + 1]);
          if (q4 == 0) {
            stat[(slot * 16 + r) * 2] = top[h];
            stat[(slot * 16 + r) * 2 + 1] = sum[h];
          }
        }
      }
      __syncthreads();
      if (part == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = g + 8 * h;
          float mx = top[h];
#pragma unroll
          for (int x = 0; x < Cfg::kParts - 1; ++x) mx = fmaxf(mx, stat[((x * MT + wr) * 16 + r) * 2]);
          const float ref = mx == -INFINITY ? 0.f : mx;
          float f = exp2_fast(top[h] - ref);
          sum[h] *= f;
#pragma unroll
          for (int i = 0; i < kUnits; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) o[i][e][2 * h] *= f, o[i][e][2 * h + 1] *= f;
#pragma unroll
          for (int x = 0; x < Cfg::kParts - 1; ++x) {
            const int slot = x * MT + wr;
            f = exp2_fast(stat[(slot * 16 + r) * 2] - ref);
            sum[h] += f * stat[(slot * 16 + r) * 2 + 1];
            const float* from = join + (slot * 16 + r) * kJ + q4 * 4;
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
              const float4 y = *reinterpret_cast<const float4*>(from + i * 16);
              o[i][0][2 * h] += f * y.x, o[i][1][2 * h] += f * y.y;
              o[i][0][2 * h + 1] += f * y.z, o[i][1][2 * h + 1] += f * y.w;
            }
          }
          top[h] = mx;
        }
      }
    }
    if (part == 0) {
      const bool all = w == item0 && w1 == item1;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = wr * 16 + g + 8 * h;
        if (r >= live) continue;
        if (all) {
          const int node = rq.n0 + (row0 + r) / a.group, hq = head * a.group + (row0 + r) % a.group;
          const float inv = sum[h] > 0.f || sum[h] != sum[h] ? 1.f / sum[h] : 0.f;
          T* to = reinterpret_cast<T*>(a.out) + (int64_t)node * a.o_sn + (int64_t)hq * a.o_sh + q4 * 4;
#pragma unroll
          for (int i = 0; i < kUnits; ++i)
            *reinterpret_cast<uint2*>(to + i * 16) =
                make_uint2(round_pair<T>(o[i][0][2 * h] * inv, o[i][1][2 * h] * inv),
                           round_pair<T>(o[i][0][2 * h + 1] * inv, o[i][1][2 * h + 1] * inv));
          if (a.lse && q4 == 0)
            a.lse[(int64_t)node * a.Hq + hq] =
                sum[h] == 0.f ? -INFINITY : (top[h] + log2f(sum[h])) * 0.6931471805599453f;
        } else {
          float* slot = a.partials + (2ll * blockIdx.x + (w == item0 ? 1 : 0)) * attn_slot_floats(kRows, D);
#pragma unroll
          for (int i = 0; i < kUnits; ++i)
            *reinterpret_cast<float4*>(slot + (int64_t)r * D + i * 16 + q4 * 4) =
                make_float4(o[i][0][2 * h], o[i][1][2 * h], o[i][0][2 * h + 1], o[i][1][2 * h + 1]);
          if (q4 == 0)
            *reinterpret_cast<float2*>(slot + (int64_t)kRows * D + 2 * r) = make_float2(top[h], sum[h]);
        }
      }
    }
    w = w1;
  }
}

namespace {

template <typename T, int D, int MT, int WK, int TG>
int launch_form8(const Attn8Args& a, cudaStream_t stream, int& grid, int& rows) {
  using Cfg = Attn8Cfg<D, MT, WK, TG>;
  const void* k = (const void*)tree_attn8_kernel<T, D, MT, WK, TG>;
  if (!prepare_kernel(k)) return 2;
  grid = num_sms();
  rows = Cfg::kRows;
  return launch_with_pdl(k, a, grid, Cfg::kThreads, sizeof(typename Cfg::Smem), a.pdl, stream);
}

template <typename T, int D>
int launch_d8(const Attn8Args& a, cudaStream_t stream) {
  int grid = 0, rows = 0, rc;
  const int most = a.max_nodes * a.group;
  // Key tiles of the launch.  Up to 16 rows a kv head (decoding, narrow trees) stay here, where a tile costs the fewest
  // instructions, with more warps for the tiles where a CTA has several: one token over 1,000 keys 12.5 us with one set
  // of warps and 13.7 with two, 16 requests of a token over up to 8,192 keys (66 tiles a CTA) 132 and 88 (three or four
  // sets: 83 and 86; with heads of 64, 43, 37 and 36).  Only with tiles in plenty does the tensor-memory form draw level: 85
  // and 101 us against 88 and 104 at 112 tiles an SM.  More rows go there from three tiles an SM times row tiles of 32
  // on: at 1.8 17.7 us here and 19.5 there, at 3.5 30.3 and 25.7, at 7 30.6 and 27.8, at 28 66 and 39.
  const int64_t tiles = (int64_t)a.B * a.Hk * ((a.max_context + a.max_nodes + kKeyTile - 1) / kKeyTile), sms = num_sms();
  if (most <= 16 ? tiles > 100 * sms : tiles * ((most + 31) / 32) > 3 * sms) rc = launch_tree_attn8_tc(a, stream, grid, rows);
  else if (most <= 16 && tiles <= sms) rc = launch_form8<T, D, 1, 4, 1>(a, stream, grid, rows);
  else if (most <= 16) rc = launch_form8<T, D, 1, 4, D == 64 ? 3 : 2>(a, stream, grid, rows);
  else if (most <= 32) rc = launch_form8<T, D, 2, 4, 1>(a, stream, grid, rows);
  else rc = launch_form8<T, D, 4, 2, 1>(a, stream, grid, rows);
  return rc ? rc : launch_attn_join(a, stream, grid, rows);
}

template <typename T>
int launch_t8(const Attn8Args& a, cudaStream_t stream) {
  if (a.D == 64) return launch_d8<T, 64>(a, stream);
  if (a.D == 128) return launch_d8<T, 128>(a, stream);
  return launch_d8<T, 256>(a, stream);
}

}  // namespace

int launch_tree_attn8(const Attn8Args& a, cudaStream_t stream) {
  return a.f16 ? launch_t8<__half>(a, stream) : launch_t8<__nv_bfloat16>(a, stream);
}

}  // namespace fnx
