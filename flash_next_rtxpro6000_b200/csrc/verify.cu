// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// A request's nodes form a tree: node 0 is its last token, row i of `target` the target's distribution p of the token
// after node i, row i of `draft` the drafter's, q, that node i's children were drawn from.  The path starts at node 0.
// At its end the children are asked in order, with r = p and S = 1 at first:
//
//   child with token x, random number u:   accepted  iff  u q(x) < r(x) / S    (it joins the path, and is its end)
//   refused:                               r <- max(r / S - q, 0),  S <- sum r
//
// and without drafter probabilities (children chosen, not drawn: q is 1 at their token)
//
//   accepted  iff  u S < r(x);   refused:  S <- S - r(x),  r(x) <- 0.
//
// A refusal that would leave nothing leaves r and S as they are.  With drafter probabilities the refusal's own sum tells.
// Without, a row is not summed before the draw, so it is found there, when the refused tokens turn out to be all that the
// row has: the walk goes back to the refusal that took the last one and goes on from there with that token alone.
//
// Then the next token is drawn from r by the request's own random number: the path's tokens and this one have the
// target's distribution.  r, S and the tests are in 64-bit floating point, r / S - q in one rounding but for that of 1 / S:
// what cancels in one refusal keeps the bits that the next ones need.  (In 32 bits choices within some 2^-23 of their
// borders fell either way.)  Sums are of whole numbers (trunc(2^52 r), 64 bits), exact in any order: the split of a row
// changes nothing.  64 bits hold 4,096 in that unit, and a row that is no distribution could sum to more, so sums are
// capped on their way (by 128 a thread, warp and CTA) and one of 64 or more is an error.
//
// Bound: one read of the row at the path's end (of p, and of q where a child was refused there), since probabilities
// of drafted tokens alone decide all else; for few requests, the chain of steps.  A cluster of CTAs has a request,
// each a slice of the rows.  Every CTA walks the tree by itself, so the cluster only exchanges sums: one pass over
// the slice for each refusal by q, whose sums also serve the final draw.  The token is found from the sums of CTAs,
// then of warps, then by one more read of the 1/(16 x 8) of the row that holds it.
// Measured (B200): a chain of 6 nodes, vocabulary of 151,936, 8.4 us; 32 trees of 16 nodes 19.9 us, which is up to four
// passes over the 1.2 MB of one request's two rows, on 16 of the 148 SMs (in clusters of 8 25 us, with 512 threads 26,
// both with r in 32 bits, which took 8.5 and 19.5).
#include <cooperative_groups.h>

#include "fnx_common.cuh"
#include "fnx_kernels.h"

namespace fnx {

namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kVT = 256;             // threads
constexpr int kVW = kVT / 32;        // warps
constexpr int kNodes = 64;           // nodes of a request
constexpr int kVCluster = 16;        // CTAs of a request
constexpr int kTileV = 128;          // tokens of a warp's step: four a lane
constexpr int kFlight = 5;           // steps whose loads are in flight together
constexpr double kUnit = 4503599627370496.0;  // 2^52
constexpr u64 kHeavy = 1ull << 58;  // ... and a capped one stays above this when refused tokens (63 at most) are taken out

enum Step : int { STEP_PASS = 0, STEP_DRAW = 1 };

struct VerifySmem {
  int parent[kNodes];
  int64_t token[kNodes];
  float uniform[kNodes], p[kNodes], q[kNodes];  // of the node's token, in its parent's rows
  double inv[kNodes];      // 1 / S of the refusals at the path's end
  int refused[kNodes];     // their tokens (without drafter probabilities) ...
  int refused_node[kNodes];  // ... and nodes, and S before
  double left_before[kNodes];
  int path[kNodes];
  u64 warp_sum[kVW];       // of the last pass
  u64 total[2];            // this CTA's, of the last passes
  u64 tile_sum[kTileV];    // of the warp's part that holds the token
  // the walk
  int i, current, length, rounds, step;
  int sole;                // the only token left, or -1: its refusals change nothing (without drafter probabilities)
  bool summed;             // the last pass was over what is left now
  bool heavy;              // a row that is no distribution
  double left;             // S
};

__device__ __forceinline__ float probability(float v) { return __saturatef(v); }  // NaN counts as 0
// A float in [0, 1] as a double by its bits, since conversions have a quarter of the arithmetic's rate: half of a pair's are
// made this way.  Those below 2^-126, 0 among them, become some 2^-127: enough for a q, which is taken away, and for sums.
__device__ __forceinline__ double widen_bits(float v) {
  const uint32_t b = __float_as_uint(v);
  return __hiloint2double((int)((b >> 3) + 0x38000000u), (int)(b << 29));
}
// trunc(2^52 r) for r in [0, 1]: the lowest bits of 1 + r, rounded towards 0.
__device__ __forceinline__ u64 whole(double r) { return (u64)(__double_as_longlong(__dadd_rz(r, 1.0)) - 0x3FF0000000000000ll); }
__device__ __forceinline__ u64 part(float v) { return whole(widen_bits(probability(v))); }
// What `rounds` refusals leave of n tokens' r; negative numbers become 0 by their sign bit.
template <int N>
__device__ __forceinline__ void residual(const double* inv, int rounds, double (&r)[N], const double (&q)[N]) {
#pragma unroll 1
  for (int k = 0; k < rounds; ++k) {
    const double by = inv[k];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const double x = __fma_rn(r[e], by, -q[e]);
      const int hi = __double2hiint(x), keep = ~(hi >> 31);
      r[e] = __hiloint2double(hi & keep, __double2loint(x) & keep);
    }
  }
}

// At most 2^59 - 1, by the upper half.
__device__ __forceinline__ u64 capped(u64 v) {
  const uint32_t hi = min((uint32_t)(v >> 32), 0x07FFFFFFu);
  return ((u64)hi << 32) | (uint32_t)v;
}
__device__ __forceinline__ u64 warp_total(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Four tokens' probabilities, zeros past `end`.
template <bool kVec>
__device__ __forceinline__ float4 four(const float* row, int v, int end) {
  if (kVec) return v < end ? __ldg(reinterpret_cast<const float4*>(row + v)) : make_float4(0.f, 0.f, 0.f, 0.f);
  float4 x;
  x.x = v < end ? __ldg(row + v) : 0.f;
  x.y = v + 1 < end ? __ldg(row + v + 1) : 0.f;
  x.z = v + 2 < end ? __ldg(row + v + 2) : 0.f;
  x.w = v + 3 < end ? __ldg(row + v + 3) : 0.f;
  return x;
}

}  // namespace

// Four blocks an SM, at 64 registers and some 70 bytes of spills: 32 clusters of 16 run at once then (without drafter
// probabilities 16.0 us against 17.5 with three, with them 37.8 against 37.4 where most children are refused).
template <bool kVec>
__global__ void __launch_bounds__(kVT, 4) verify_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ VerifySmem s;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank();
  const int b = blockIdx.x / kVCluster, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  const int n0 = a.node_offsets[b], n = a.node_offsets[b + 1] - n0;
  const bool bad = n0 < 0 || n < 0 || n > a.width || n > a.N - n0;
  if (bad || n == 0) {  // the cluster's CTAs all leave here
    if (rank == 0) {
      if (tid < a.width) a.path[(int64_t)b * a.width + tid] = -1;
      if (tid == 0) {
        a.accepted[b] = 0;
        a.next[b] = -1;
        if (bad) record_error(a.err, ERR_LENGTHS);
      }
    }
    pdl_trigger();
    return;
  }
  if (tid < n) {
    const int parent = tid ? a.parents[n0 + tid] : -1;
    const int64_t x = a.tokens[n0 + tid];
    const bool known = parent >= 0 && parent < tid, word = x >= 0 && x < a.V;
    float p = 0.f, q = 0.f;
    if (known && word) {
      p = probability(a.target[(int64_t)(n0 + parent) * a.ldt + x]);
      q = a.draft ? probability(a.draft[(int64_t)(n0 + parent) * a.ldd + x]) : 1.f;
    }
    if (rank == 0 && tid > 0) {
      if (!known && parent != -1) record_error(a.err, ERR_TREE);
      if (known && !word) record_error(a.err, ERR_TOKEN);
    }
    s.parent[tid] = known ? parent : -1;
    s.token[tid] = word ? x : -1;
    s.uniform[tid] = fmaxf(a.node_uniforms[n0 + tid], 0.f);  // NaN and negative numbers count as 0
    s.p[tid] = p;
    s.q[tid] = q;
  }
  if (tid == 0) {
    s.i = 1;
    s.current = 0;
    s.length = 1;
    s.rounds = 0;
    s.left = 1.0;
    s.sole = -1;
    s.summed = s.heavy = false;
    s.path[0] = 0;
  }
  __syncthreads();

  const int v0 = rank * a.per + warp * (a.per / kVW);          // the warp's part of the row
  const int v1 = min(a.V, v0 + a.per / kVW);
  int phase = 0;
  // Sums of what `rounds` refusals leave of the current row: the warps', the CTA's and the cluster's.
  auto pass = [&](int rounds) {
    const float* prow = a.target + (int64_t)(n0 + s.current) * a.ldt;
    const float* qrow = a.draft ? a.draft + (int64_t)(n0 + s.current) * a.ldd : nullptr;
    u64 sum = 0;
    if (a.draft && rounds > 0) {
      for (int v = v0 + lane * 4; v < v1; v += kFlight * kTileV) {
        float p[4 * kFlight], q[4 * kFlight];
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
          const float4 x = four<kVec>(prow, v + f * kTileV, v1), y = four<kVec>(qrow, v + f * kTileV, v1);
          p[4 * f] = x.x, p[4 * f + 1] = x.y, p[4 * f + 2] = x.z, p[4 * f + 3] = x.w;
          q[4 * f] = y.x, q[4 * f + 1] = y.y, q[4 * f + 2] = y.z, q[4 * f + 3] = y.w;
        }
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
          double r[4], y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] = (double)probability(p[4 * f + e]), y[e] = widen_bits(probability(q[4 * f + e]));
          residual(s.inv, rounds, r, y);
#pragma unroll
          for (int e = 0; e < 4; ++e) sum += whole(r[e]);
        }
      }
      sum = capped(sum);
    } else {
      for (int v = v0 + lane * 4; v < v1; v += kFlight * kTileV) {
        float4 p[kFlight];
#pragma unroll
        for (int f = 0; f < kFlight; ++f) p[f] = four<kVec>(prow, v + f * kTileV, v1);
#pragma unroll
        for (int f = 0; f < kFlight; ++f)
          sum += part(p[f].x) + part(p[f].y) + part(p[f].z) + part(p[f].w);
      }
      sum = capped(sum);
      if (!a.draft && lane < rounds) {  // refused tokens' shares are taken out again
        for (int k = lane; k < rounds; k += 32)
          if (s.refused[k] >= v0 && s.refused[k] < v1) sum -= part(prow[s.refused[k]]);
      }
    }
    sum = warp_total(sum);
    __syncthreads();
    if (lane == 0) s.warp_sum[warp] = capped(sum);
    __syncthreads();
    if (tid == 0) {
      u64 all = 0;
      for (int w = 0; w < kVW; ++w) all += s.warp_sum[w];
      s.total[phase] = capped(all);
    }
    cl.sync();
    u64 all = 0;
#pragma unroll
    for (int c = 0; c < kVCluster; ++c) all += cl.map_shared_rank(&s, c)->total[phase];
    phase ^= 1;
    return all;
  };

  for (;;) {
    if (tid == 0) {  // the state in registers: a node costs no more than its loads
      int step = STEP_DRAW, i = s.i, current = s.current, length = s.length, rounds = s.rounds, sole = s.sole;
      double left = s.left;
      bool summed = s.summed;
      for (; i < n; ++i) {
        if (s.parent[i] != current) continue;
        const int x = (int)s.token[i];
        bool accept;
        if (a.draft) {
          double r[1] = {(double)s.p[i]};
          const double q[1] = {(double)s.q[i]};
          residual(s.inv, rounds, r, q);
          accept = (double)s.uniform[i] * q[0] * left < r[0];
          if (!accept) {
            s.inv[rounds] = 1.0 / left;
            step = STEP_PASS;
          }
        } else {
          double r = (double)s.p[i];
          for (int k = 0; k < rounds; ++k)
            if (s.refused[k] == x) r = 0.0;
          accept = (double)s.uniform[i] * left < r;
          if (!accept && r > 0.0 && x != sole) {
            s.left_before[rounds] = left;
            s.refused_node[rounds] = i;
            s.refused[rounds++] = x;
            left = fmax(left - r, 0.0);
          }
        }
        if (accept) {
          s.path[length++] = i;
          current = i;
          rounds = 0;
          left = 1.0;
          sole = -1;
          summed = false;
        }
        if (step == STEP_PASS) break;
      }
      s.step = step, s.i = i, s.current = current, s.length = length, s.rounds = rounds, s.sole = sole;
      s.left = left;
      s.summed = summed;
    }
    __syncthreads();
    if (s.step == STEP_DRAW) {
      if (s.summed || pass(s.rounds) > 0 || a.draft) break;
      // the last refusal that took something; those behind it took tokens below 2^-52
      int k = s.rounds - 1;
      while (k >= 0 && part(s.p[s.refused_node[k]]) == 0) --k;
      if (k < 0) break;  // the row is zeros
      __syncthreads();   // all have read what the next lines change
      if (tid == 0) {
        s.sole = s.refused[k];
        s.left = s.left_before[k];
        s.i = s.refused_node[k] + 1;
        s.rounds = k;
      }
      continue;
    }
    const u64 all = pass(s.rounds + 1);
    if (tid == 0) {
      ++s.i;
      s.summed = all > 0;
      if (all >= kHeavy) s.heavy = true;  // looked at in the end: a branch here took 38 -> 41 us (32 trees, most refused)
      if (all > 0) {
        ++s.rounds;
        s.left = (double)all * (1.0 / kUnit);
      }
    }
    __syncthreads();
  }
  // --- the draw
  u64 before = 0, all = 0;
  const u64 mine = s.total[phase ^ 1];
  for (int c = 0; c < kVCluster; ++c) {
    const u64 t = cl.map_shared_rank(&s, c)->total[phase ^ 1];
    if (c < rank) before += t;
    all += t;
  }
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");  // the others' sums have been read
  const bool heavy = s.heavy || all >= kHeavy;  // no distribution: as without nodes
  if (rank == 0) {
    const int length = heavy ? 0 : s.length;
    if (tid < a.width) a.path[(int64_t)b * a.width + tid] = tid < length ? s.path[tid] : -1;
    if (tid == 0) {
      a.accepted[b] = length;
      if (heavy) record_error(a.err, ERR_PROBS);
      if (heavy || all == 0) a.next[b] = -1;
    }
  }
  if (all > 0 && !heavy) {
    const float given = a.draw_uniforms[b];
    const double u = given > 0.f ? (double)given : 0.0;  // NaN and negative numbers draw the first token
    const u64 reach = __double2ull_rz(__dmul_rn(u, __ull2double_rn(all)));
    const u64 aim = reach < all - 1 ? reach : all - 1;
    if (aim >= before && aim < before + mine) {  // the CTA has the token
      int w = 0;
      while (w < kVW - 1 && aim >= before + s.warp_sum[w]) before += s.warp_sum[w++];
      const int p0 = rank * a.per + w * (a.per / kVW), p1 = min(a.V, p0 + a.per / kVW);
      const float* prow = a.target + (int64_t)(n0 + s.current) * a.ldt;
      const float* qrow = a.draft ? a.draft + (int64_t)(n0 + s.current) * a.ldd : nullptr;
      const bool pairs = a.draft && s.rounds > 0;
      auto weights = [&](int v, u64 (&x)[4]) {
        const float4 p = four<kVec>(prow, v, p1);
        const float4 q = pairs ? four<kVec>(qrow, v, p1) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float ps[4] = {p.x, p.y, p.z, p.w}, qs[4] = {q.x, q.y, q.z, q.w};
        double r[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = (double)probability(ps[e]), y[e] = widen_bits(probability(qs[e]));
        if (pairs) residual(s.inv, s.rounds, r, y);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = whole(r[e]);
          if (!a.draft)
            for (int k = 0; k < s.rounds; ++k)
              if (s.refused[k] == v + e) x[e] = 0;
        }
      };
      const int tiles = (p1 - p0 + kTileV - 1) / kTileV;  // at most kTileV: 2^21 tokens over 8 x 16 x 128
      for (int t = warp; t < tiles; t += kVW) {
        u64 x[4];
        weights(p0 + t * kTileV + lane * 4, x);
        const u64 sum = warp_total(x[0] + x[1] + x[2] + x[3]);
        if (lane == 0) s.tile_sum[t] = sum;
      }
      __syncthreads();  // of the CTA alone: the condition is the same for all of its threads
      if (warp == 0) {
        int t = 0;
        while (t < tiles - 1 && aim >= before + s.tile_sum[t]) before += s.tile_sum[t++];
        const int v = p0 + t * kTileV + lane * 4;
        u64 x[4];
        weights(v, x);
        const u64 own = x[0] + x[1] + x[2] + x[3];
        u64 sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 y = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += y;
        }
        u64 run = before + sum - own;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (aim >= run && aim < run + x[e]) a.next[b] = v + e;
          run += x[e];
        }
      }
    }
  }
  // no CTA leaves while another reads its sums
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  pdl_trigger();
}

int launch_verify(VerifyArgs a, cudaStream_t stream) {
  a.per = (a.V + kVCluster * kVW * kTileV - 1) / (kVCluster * kVW * kTileV) * (kVW * kTileV);
  const void* k = a.vectors ? (const void*)verify_kernel<true> : (const void*)verify_kernel<false>;
  if (!prepare_wide_cluster(k)) return 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.B * kVCluster);
  cfg.blockDim = dim3(kVT);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kVCluster;
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
