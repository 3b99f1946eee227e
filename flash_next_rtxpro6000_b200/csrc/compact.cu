// The accepted nodes of drafted trees moved behind their contexts, in the keys and values of all layers:
//
//   place context + d  <-  place context + path[d],   d < accepted,   path rising
//
// as if everything were read before anything is written.  In an 8-bit cache (cache8.cuh) a token may come to a block
// with another scale: the block's scale becomes the largest of those of the tokens that come to it and, if tokens of
// the context stay in it, its own; bytes whose scale changes are scaled and rounded again.
//
// Bound: latency.  A tree's path is some kilobytes a layer, so the launch and its chain of loads (path and length,
// page numbers, rows) are nearly all there is.  A warp has one request, one of a layer's two caches and 512 bytes of a
// token's heads, a lane 16 bytes of each token: nothing but its own lanes is waited for, and a batch over all layers fits
// on the GPU at once (24 requests, 48 layers, 8 bits: 44 us with a block of 256 threads for the same bytes, 10.4 this way).
// Tokens move in batches, each read before it is written: the path rises, so no token's place is written before
// that token has been read.  No other warp touches these bytes.
#include "cache8.cuh"

namespace fnx {

namespace {

constexpr int kCT = 128;                 // threads
constexpr int kMost = 64;                // nodes of a path
constexpr int kBatch = 4;                // tokens in registers
constexpr int kChunk = 512;              // bytes of a token
constexpr int kHeads = kChunk / 64;      // heads of a warp, at most (8 bits)
constexpr int kBlocks = kMost / 16 + 1;  // blocks that a path's tokens come to, at most

struct CompactWarp {
  int64_t from[kMost], to[kMost];  // byte offsets of the tokens in the cache
};
struct CompactScales {
  int64_t at[kMost], to[kBlocks];  // offsets of the tokens' scales, and of the blocks' that they come to
  float whose[kMost][kHeads], now[kBlocks][kHeads], own[kHeads];
};

}  // namespace

template <bool k8>
__global__ void __launch_bounds__(kCT, 8) compact_kernel(const __grid_constant__ CompactArgs a) {
  __shared__ CompactWarp rows_of[kCT / 32];
  __shared__ CompactScales scales_of[k8 ? kCT / 32 : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  CompactWarp& w = rows_of[warp];
  CompactScales& z = scales_of[k8 ? warp : 0];
  const int chunks = (a.Hk * a.row_bytes + kChunk - 1) / kChunk;
  int64_t at = (int64_t)blockIdx.x * (kCT / 32) + warp;
  const int chunk = (int)(at % chunks);
  at /= chunks;
  const bool key = at & 1;
  at >>= 1;
  const int layer = (int)(at % a.layers), b = (int)(at / a.layers);
  pdl_wait();
  if (b >= a.B) return;  // the last block's spare warps
  const bool speaks = chunk == 0 && layer == 0 && key;
  const int ctx = a.context_lens[b], n = a.accepted[b];
  const int64_t room = (int64_t)a.table_width * a.page_size;
  int code = ctx >= 0 && n >= 0 && n <= a.width && ctx <= room ? 0 : ERR_LENGTHS;
  const int64_t* st = key ? a.kc_st : a.vc_st;
  const int64_t* ss = key ? a.ks_st : a.vs_st;
  const int shift = k8 ? 31 - __clz(a.block) : 0;                // blocks are 16, 32 or 64 tokens
  const int first = k8 ? ctx & (a.block - 1) : 0;  // tokens of the context in the first block
  bool moves = false;
  if (code == 0) {
    const int* path = a.path + (int64_t)b * a.path_ld;
    const int* table = a.page_table + (int64_t)b * a.pt_ld;
#pragma unroll
    for (int i = 0; i < kMost / 32; ++i) {
      const int d = i * 32 + lane;
      if (d >= n) continue;
      const int p = path[d], before = d ? path[d - 1] : -1;
      if (p <= before || p < d) {  // rising from 0 on: a token never moves up, nor over one that is still to move
        code = ERR_TREE;
      } else if ((int64_t)ctx + p >= room) {
        code = ERR_LENGTHS;
      } else {
        const int64_t src = (int64_t)ctx + p, dst = (int64_t)ctx + d;
        const int64_t sp = src / a.page_size, dp = dst / a.page_size;
        const int si = (int)(src - sp * a.page_size), di = (int)(dst - dp * a.page_size);
        const int from = table[sp], to = table[dp];
        if (from < 0 || from >= a.num_pages || to < 0 || to >= a.num_pages) code = ERR_PAGE;
        w.from[d] = (int64_t)from * st[0] + (int64_t)si * st[1];
        w.to[d] = (int64_t)to * st[0] + (int64_t)di * st[1];
        if (k8) {
          z.at[d] = (int64_t)from * ss[0] + (int64_t)(si >> shift) * ss[1];
          if (d == 0 || ((first + d) & (a.block - 1)) == 0)
            z.to[(first + d) >> shift] = (int64_t)to * ss[0] + (int64_t)(di >> shift) * ss[1];
        }
        moves |= p != d;
      }
    }
  }
  if (code && speaks) record_error(a.err, code);
  const bool good = __all_sync(0xffffffffu, code == 0);
  moves = __any_sync(0xffffffffu, moves);
  if (speaks && lane == 0 && a.new_lens) a.new_lens[b] = good ? ctx + n : ctx;
  if (!good || !moves) {
    pdl_trigger();
    return;
  }
  __syncwarp();
  const int byte = chunk * kChunk + lane * 16, h = byte / a.row_bytes;
  const bool live = h < a.Hk;
  uint8_t* cache = reinterpret_cast<uint8_t*>(key ? a.k_cache : a.v_cache) + layer * (key ? a.k_layer : a.v_layer) +
                   (live ? (int64_t)h * st[2] + byte % a.row_bytes : 0);
  uint4 x[kBatch];
  auto load = [&](int d0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (live && d0 + i < n) x[i] = *reinterpret_cast<const uint4*>(cache + w.from[d0 + i]);
  };
  load(0);
  const int hs = k8 ? __clz(a.row_bytes) - __clz(kChunk) : 0, heads = 1 << hs, h0 = chunk << hs;  // of the warp, at most
  const int blocks = k8 ? ((first + n - 1) >> shift) + 1 : 0, hh = live && k8 ? h - h0 : 0;
  float* scales = nullptr;
  if (k8) {
    scales = (key ? a.k_scale : a.v_scale) + layer * (key ? a.ks_layer : a.vs_layer) + (int64_t)h0 * ss[2];
#pragma unroll 4
    for (int u = lane; u < n * heads; u += 32) {
      const int d = u >> hs, g = u & (heads - 1);
      z.whose[d][g] = h0 + g < a.Hk ? scale_or_least(scales[z.at[d] + g * ss[2]]) : 1.f;
    }
    // the first token's block is the only one that the context reaches into
    if (lane < heads && h0 + lane < a.Hk) z.own[lane] = scale_or_least(scales[z.to[0] + lane * ss[2]]);
    __syncwarp();
    for (int u = lane; u < blocks * heads; u += 32) {
      const int j = u >> hs, g = u & (heads - 1);
      float s = j == 0 && first > 0 && h0 + g < a.Hk ? z.own[g] : 0.f;
      const int d1 = min(n, (j + 1) * a.block - first);
      for (int d = max(0, j * a.block - first); d < d1; ++d) s = fmaxf(s, z.whose[d][g]);
      z.now[j][g] = s;
    }
    __syncwarp();
  }
  auto scaled = [](uint4 v, float ratio) {
    return make_uint4(e4m3_scaled(v.x, ratio), e4m3_scaled(v.y, ratio), e4m3_scaled(v.z, ratio), e4m3_scaled(v.w, ratio));
  };
  for (int d0 = 0; d0 < n; d0 += kBatch) {
    if (d0) load(d0);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int d = d0 + i;
      if (!live || d >= n) continue;
      const float ratio = k8 ? z.whose[d][hh] / z.now[(first + d) >> shift][hh] : 1.f;
      if (k8 && ratio != 1.f) x[i] = scaled(x[i], ratio);
      if (w.to[d] != w.from[d] || ratio != 1.f) *reinterpret_cast<uint4*>(cache + w.to[d]) = x[i];
    }
  }
  if (k8) {
    const float ratio = first > 0 && live ? z.own[hh] / z.now[0][hh] : 1.f;
    if (ratio != 1.f) {  // the context's tokens in the first block, which lie in front of the first accepted one
      for (int r = 1; r <= first; ++r) {
        uint4* y = reinterpret_cast<uint4*>(cache + w.to[0] - r * st[1]);
        *y = scaled(*y, ratio);
      }
    }
    for (int u = lane; u < blocks * heads; u += 32) {
      const int j = u >> hs, g = u & (heads - 1);
      if (h0 + g < a.Hk) scales[z.to[j] + g * ss[2]] = z.now[j][g];
    }
  }
  pdl_trigger();
}

int launch_compact(const CompactArgs& a, cudaStream_t stream) {
  const int chunks = (a.Hk * a.row_bytes + kChunk - 1) / kChunk;
  const int64_t warps = (int64_t)a.B * a.layers * 2 * chunks;
  const void* k = a.k_scale ? (const void*)compact_kernel<true> : (const void*)compact_kernel<false>;
  return launch_with_pdl(k, a, (int)((warps + kCT / 32 - 1) / (kCT / 32)), kCT, 0, a.pdl, stream);
}

}  // namespace fnx
