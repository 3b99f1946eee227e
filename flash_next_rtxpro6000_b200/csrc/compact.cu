// The accepted nodes of drafted trees moved behind their contexts, in the keys and values of all layers:
//
//   place context + d  <-  place context + path[d],   d < accepted,   path rising
//
// as if everything were read before anything is written.  In an 8-bit cache (cache8.cuh) a token may come to a block
// with another scale: the block's scale becomes the largest of those of the tokens that come to it and, if tokens of
// the context stay in it, its own; bytes whose scale changes are scaled and rounded again.
//
// Bound: latency.  A tree's path is some kilobytes a layer, so the launch and its chain of loads (path and length,
// page numbers, rows) are all there is.  A CTA has one request, one of a layer's two caches and 512 bytes of a
// token's heads: a warp a token, a lane 16 bytes.  All of its rows are in registers before the first is written, and
// no other CTA touches these bytes.
#include "cache8.cuh"

namespace fnx {

namespace {

constexpr int kCT = 256;                // threads
constexpr int kWarps = kCT / 32;
constexpr int kMost = 64;               // nodes of a path
constexpr int kEach = kMost / kWarps;   // tokens of a warp
constexpr int kChunk = 512;             // bytes of a token
constexpr int kHeads = kChunk / 64;     // heads of a CTA, at most (8 bits)
constexpr int kBlocks = kMost / 16 + 1;  // blocks that a path's tokens come to, at most

}  // namespace

template <bool k8>
__global__ void __launch_bounds__(kCT) compact_kernel(const __grid_constant__ CompactArgs a) {
  __shared__ int from_page[kMost], from_in[kMost], to_page[kMost], to_in[kMost];
  __shared__ float whose[k8 ? kMost : 1][kHeads], now[k8 ? kBlocks : 1][kHeads], own[kHeads];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int chunks = (a.Hk * a.row_bytes + kChunk - 1) / kChunk;
  int at = blockIdx.x;
  const int chunk = at % chunks;
  at /= chunks;
  const bool key = at & 1;
  const int layer = (at >> 1) % a.layers, b = (at >> 1) / a.layers;
  const bool speaks = tid == 0 && chunk == 0 && layer == 0 && key;
  pdl_wait();
  const int ctx = a.context_lens[b], n = a.accepted[b];
  const int64_t room = (int64_t)a.table_width * a.page_size;
  bool good = ctx >= 0 && n >= 0 && n <= a.width && ctx <= room;
  int code = good ? 0 : ERR_LENGTHS;
  bool moves = false;
  if (good && tid < n) {
    const int* path = a.path + (int64_t)b * a.path_ld;
    const int p = path[tid], before = tid ? path[tid - 1] : -1;
    if (p <= before || p < tid) {  // rising from 0 on: a token never moves up, nor over one that is still to move
      code = ERR_TREE;
    } else if ((int64_t)ctx + p >= room) {
      code = ERR_LENGTHS;
    } else {
      const int64_t src = (int64_t)ctx + p, dst = (int64_t)ctx + tid;
      const int* table = a.page_table + (int64_t)b * a.pt_ld;
      const int sp = table[src / a.page_size], dp = table[dst / a.page_size];
      if (sp < 0 || sp >= a.num_pages || dp < 0 || dp >= a.num_pages) code = ERR_PAGE;
      from_page[tid] = sp, from_in[tid] = (int)(src % a.page_size);
      to_page[tid] = dp, to_in[tid] = (int)(dst % a.page_size);
      moves = p != tid;
    }
  }
  if (code && chunk == 0 && layer == 0 && key) record_error(a.err, code);
  good = __syncthreads_and(code == 0);
  moves = __syncthreads_or(moves);
  if (speaks && a.new_lens) a.new_lens[b] = good ? ctx + n : ctx;
  if (!good || !moves) {
    pdl_trigger();
    return;
  }
  uint8_t* cache = reinterpret_cast<uint8_t*>(key ? a.k_cache : a.v_cache) + layer * (key ? a.k_layer : a.v_layer);
  const int64_t* st = key ? a.kc_st : a.vc_st;
  const int byte = chunk * kChunk + lane * 16, h = byte / a.row_bytes;
  const bool live = h < a.Hk;
  const int64_t head_at = (int64_t)h * st[2] + byte % a.row_bytes;
  uint4 x[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int d = warp + i * kWarps;
    if (live && d < n)
      x[i] = *reinterpret_cast<const uint4*>(cache + (int64_t)from_page[d] * st[0] + (int64_t)from_in[d] * st[1] + head_at);
  }
  const int heads = k8 ? kChunk / a.row_bytes : 1, h0 = chunk * heads;  // of the CTA, at most
  const int first = ctx % a.block;  // tokens of the context in the first block (k8)
  float* scales = nullptr;
  const int64_t* ss = key ? a.ks_st : a.vs_st;
  auto scale_of = [&](int page, int in, int hh) {
    return scales + (int64_t)page * ss[0] + (int64_t)(in / a.block) * ss[1] + (int64_t)(h0 + hh) * ss[2];
  };
  const int blocks = k8 ? (first + n - 1) / a.block + 1 : 0;
  if (k8) {
    scales = (key ? a.k_scale : a.v_scale) + layer * (key ? a.ks_layer : a.vs_layer);
    for (int u = tid; u < n * heads; u += kCT) {
      const int d = u / heads, hh = u % heads;
      if (h0 + hh < a.Hk) whose[d][hh] = scale_or_least(*scale_of(from_page[d], from_in[d], hh));
    }
    // the first token's block is the only one that the context reaches into
    if (tid < heads && h0 + tid < a.Hk) own[tid] = scale_or_least(*scale_of(to_page[0], to_in[0], tid));
    __syncthreads();
    for (int u = tid; u < blocks * heads; u += kCT) {
      const int j = u / heads, hh = u % heads;
      float s = j == 0 && first > 0 ? own[hh] : 0.f;
      const int d1 = min(n, (j + 1) * a.block - first);
      for (int d = max(0, j * a.block - first); d < d1; ++d) s = fmaxf(s, whose[d][hh]);
      now[j][hh] = s;
    }
  }
  __syncthreads();  // everything has been read
  const int hh = live && k8 ? h - h0 : 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int d = warp + i * kWarps;
    if (!live || d >= n) continue;
    if (k8) {
      const float ratio = whose[d][hh] / now[(first + d) / a.block][hh];
      if (ratio != 1.f) {
        x[i].x = e4m3_scaled(x[i].x, ratio), x[i].y = e4m3_scaled(x[i].y, ratio);
        x[i].z = e4m3_scaled(x[i].z, ratio), x[i].w = e4m3_scaled(x[i].w, ratio);
      }
    }
    *reinterpret_cast<uint4*>(cache + (int64_t)to_page[d] * st[0] + (int64_t)to_in[d] * st[1] + head_at) = x[i];
  }
  if (k8) {
    const float ratio = first > 0 && live ? own[hh] / now[0][hh] : 1.f;
    if (ratio != 1.f) {  // the context's tokens in the first block, which lie in front of the first accepted one
      uint8_t* rows = cache + (int64_t)to_page[0] * st[0] + (int64_t)(to_in[0] - first) * st[1] + head_at;
      for (int r = warp; r < first; r += kWarps) {
        uint4* y = reinterpret_cast<uint4*>(rows + (int64_t)r * st[1]);
        uint4 v = *y;
        v.x = e4m3_scaled(v.x, ratio), v.y = e4m3_scaled(v.y, ratio);
        v.z = e4m3_scaled(v.z, ratio), v.w = e4m3_scaled(v.w, ratio);
        *y = v;
      }
    }
    for (int u = tid; u < blocks * heads; u += kCT) {
      const int j = u / heads, g = u % heads, d = max(0, j * a.block - first);
      if (h0 + g < a.Hk) *scale_of(to_page[d], to_in[d], g) = now[j][g];
    }
  }
  pdl_trigger();
}

int launch_compact(const CompactArgs& a, cudaStream_t stream) {
  const int chunks = (a.Hk * a.row_bytes + kChunk - 1) / kChunk;
  const void* k = a.k_scale ? (const void*)compact_kernel<true> : (const void*)compact_kernel<false>;
  return launch_with_pdl(k, a, a.B * a.layers * 2 * chunks, kCT, 0, a.pdl, stream);
}

}  // namespace fnx
