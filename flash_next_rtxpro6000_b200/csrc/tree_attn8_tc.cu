// Tree attention over an 8-bit paged cache on the 5th-generation tensor cores, for launches with several key tiles
// an SM: tree_attn_tc.cu's products, roles and partial results, with the scales of tree_attn8.cuh.
//
// tcgen05 takes both operands of a product in one type, and queries and weights want 16 bits, so keys and values
// become fp16 on their way into shared memory: the loading warps copy 16 bytes a lane into a small ring (cp.async, a
// few tiles ahead), and each lane converts what it copied itself (exactly) and stores it in the swizzled layout that
// the products read, so that no barrier stands between copying and converting.  (Holding the tiles ahead in registers
// instead was slow: 216 us against 148 for 24 ragged requests, as a warp cannot wait for its oldest loads alone.)  The
// lanes that load keys also leave their group's scales for the softmax warps.  With heads of 256 the queries are in
// tensor memory (A of the first product), which leaves room for the rings.
//
// What bounds it is the instructions of the roles' loops, more than the tensor cores or memory: together they do not
// fit into the SM's instruction cache (18 % of its requests missed), and a warp waits for them.  So loops stay loops,
// and keys and values share the loading warps' code: 24 ragged requests, D = 128 fp16, 180 MB: 139 -> 105 us; up to 64
// keys a row in registers -> half of a tile, read twice from tensor memory: 541 -> 519 us for 4 requests of 64 nodes over 131,072
// keys, and 476 with the registers that this leaves.  Measured without gain: weights in columns of their own so that
// scores are computed earlier (670 against 552 us), the weights computed by the reference of the tile before while the
// maximum is found (772), a tile's rows shared by two warps (828), one loop for maximum and weights (119 against 105 us).
#include <type_traits>

#include "tree_attn8.cuh"
#include "tree_attn_tc.cuh"

namespace fnx {

namespace {

// RT sets of four softmax warps: of two row tiles (kAlt false, RT = 2), or of one row tile whose key tiles they take
// in turn, each with a reference and a result of its own that are joined at the segment's end (kAlt).
template <int D, int RT, bool kAlt>
struct Tc8 {
  static constexpr int kBlocks = D / 64;
  static constexpr int kChunk = kBlocks * kBlockBytes;  // keys or values of a tile, fp16
  static constexpr int kQTile = kBlocks * 128 * 128;    // a row tile of queries
  static constexpr int kK = D == 256 ? 2 : D == 128 ? (RT == 2 && !kAlt ? 2 : 3) : 5;  // chunks of the rings
  static constexpr int kV = D == 256 ? 2 : D == 128 ? (RT == 2 && !kAlt ? 3 : 4) : 5;
  static constexpr int kRows = kAlt ? 128 : 128 * RT;
  // Scales of tiles: those of tile i are written when the scores of tile i - kK have been computed, which is when its keys
  // get their chunk.  Scores wait for the output product of the same set's tile two before, and these products go tile by
  // tile, so while a set reads the scales of tile a, scores get no further than a + 1 where there is one set, and a + 3
  // where two take turns.  With two row tiles it is a + 2: where a is the second row tile's last and the next segment has
  // one row tile only, its scores wait for the first one's products alone, and a's has been issued.
  static constexpr int kScales = kK + (kAlt ? 4 : RT == 2 ? 3 : 2);
  static constexpr int kAhead = D == 256 ? 2 : D == 128 ? 4 : 6;  // 8-bit tiles in flight
  static constexpr bool kQInTmem = D == 256;
  static constexpr int kLoad = 4 * RT, kIssue = kLoad + 8;  // first loading, first issuing warp
  static constexpr int kThreads = (kIssue + 4) * 32;  // the issuing warps are the last two of four
  static constexpr int kQCol = RT * (D + 2 * kTile);  // tensor memory: results, scores (then weights), queries
  static constexpr int kUsed = kQCol + (kQInTmem ? D / 2 : 0), kCols = kUsed <= 256 ? 256 : 512;
  static_assert(kUsed <= 512, "tensor memory");
  struct Smem {
    uint8_t q[kRows / 128][kQInTmem ? 128 * 128 : kQTile];  // and room to turn the results of 128 rows
    uint8_t k[kK][kChunk];
    uint8_t v[kV][kChunk];
    uint4 raw[2][kAhead][kTile * D / 16];  // keys and values as they lie in the cache, by lane
    float2 raw_scales[kAhead][4];
    float4 scales[kScales][kTile / kGroup];
    float2 stat[kAlt ? 128 : 1];  // the second set's references and sums
    float factor[kQInTmem ? 128 : 1];  // of the rows' scores
    long long before[kAttnMaxBatch + 1];
    unsigned long long kfull[kK], kempty[kK], vfull[kV], vempty[kV];
    unsigned long long sfull[RT][2], pfull[RT][2], odone[RT][2], qfull[RT];
    unsigned long long joined[2];  // softmax warps of the first row tile, of both (kAlt: of each set)
    unsigned long long merged;
    unsigned long long drain;
    // drafted tokens with NaN values, of this segment, the one before and the next
    unsigned long long odd[3];
    uint32_t tmem;
  };
};

// The softmax warps take registers that the others do not need: with one row tile 128 * 144 + 384 * 120 are no more
// than the launch's 512 * 128, with two 256 * 104 + 384 * 88 no more than 640 * 96.
template <int RT> __device__ __forceinline__ void give_registers8() {
  if (RT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
}
template <int RT> __device__ __forceinline__ void take_registers8() {
  if (RT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
  else asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
}

// Two fp32 operations an instruction, and the largest of three.
__device__ __forceinline__ unsigned long long two(float lo, float hi) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void apart(unsigned long long v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ unsigned long long fma_two(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long add_two(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max_three(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ void st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// A place in a ring of N, and how often it has been used (its parity).
struct Turn {
  int N, at = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ explicit Turn(int n) : N(n) {}
  __device__ __forceinline__ void next() {
    if (++at == N) at = 0, parity ^= 1u;
  }
};

// Loads keys or values (kValues) of all tiles of the CTA, converts and stores them.
template <int D, int RT, bool kAlt>
__device__ __forceinline__ void load8(const Attn8Args& a, typename Tc8<D, RT, kAlt>::Smem& s, long long total, long long G, bool kValues, int pw) {
  using Cfg = Tc8<D, RT, kAlt>;
  constexpr int P = Cfg::kAhead;
  const int N = kValues ? Cfg::kV : Cfg::kK;
  constexpr int kLanesRow = D / 16;         // lanes of a row: 16 elements each
  constexpr int kRowsPer = 32 / kLanesRow;  // rows of one instruction
  constexpr int J = 16 / kRowsPer;          // instructions of a warp's 16 keys of a tile
  const int lane = threadIdx.x & 31, col = lane % kLanesRow;
  const uint8_t* from = reinterpret_cast<const uint8_t*>(kValues ? a.v_cache : a.k_cache) + col * 16;
  uint8_t* ring = kValues ? s.v[0] : s.k[0];
  unsigned long long* full = kValues ? s.vfull : s.kfull;
  unsigned long long* empty = kValues ? s.vempty : s.kempty;
  // The walk over the CTA's tiles.  A warp executes it alone, so each of its instructions counts: places advance by
  // a tile without a division, and a page number is used a tile after it has been asked for.
  Segments sg(a, s.before, Cfg::kRows, total, G);
  const int page_step = kTile / a.page_size, in_step = kTile % a.page_size;
  const int block_shift = 31 - __clz(a.block);
  int t = 0, t1 = 0, left = 0, queued = 0;  // tile of the segment, its end, keys from the warp's first on; tiles found
  int at_page = 0, at_in = 0;
  const int* table = nullptr;
  struct Spot {  // the warp's keys of a tile, a group: one page and one block hold them
    int page, in, head, live;
  };
  auto find = [&]() {
    Spot p{0, 0, 0, 0};
    if (t == t1) {
      if (!sg.next()) return p;
      t = sg.t0;
      t1 = sg.t1;
      table = a.page_table + (int64_t)sg.b * a.table_ld;
      const int pos = t * kTile + pw * kGroup;
      left = sg.rq.ctx + sg.rq.nodes - pos;
      at_page = pos / a.page_size;
      at_in = pos - at_page * a.page_size;
    }
    p.head = sg.head;
    p.live = left;
    if (left > 0) p.page = __ldg(table + at_page);
    p.in = at_in;
    at_page += page_step;
    at_in += in_step;
    if (at_in >= a.page_size) at_in -= a.page_size, ++at_page;
    left -= kTile;
    ++t;
    ++queued;
    return p;
  };
  const int row = lane / kLanesRow;
  const int64_t* st = kValues ? a.vc_st : a.kc_st;
  const int64_t step = st[1] * kRowsPer;
  from += st[1] * row;
  uint4* raw = s.raw[kValues][0] + pw * J * 32 + lane;  // the lane's own J places
  constexpr int kTileRaw = kTile * D / 16;
  auto issue = [&](int slot, const Spot& p) {
    int live = p.live;
    if (live > 0 && (p.page < 0 || p.page >= a.num_pages)) {
      if (lane == 0) record_error(a.err, ERR_PAGE);
      live = 0;
    }
    const uint8_t* at = from + (int64_t)p.page * st[0] + (int64_t)p.in * st[1] + (int64_t)p.head * st[2];
#pragma unroll
    for (int j = 0; j < J; ++j, at += step) {
      const bool there = j * kRowsPer + row < live;
      cp16_or_zero(smem_u32(raw + slot * kTileRaw + j * 32), there ? at : from, there);
    }
    if (!kValues && lane == 0) {
      float2* to = &s.raw_scales[slot][pw];
      if (p.live > 0 && p.page >= 0 && p.page < a.num_pages) {
        const int blk = p.in >> block_shift;
        cp_async4(&to->x, a.k_scale + (int64_t)p.page * a.ks_st[0] + (int64_t)blk * a.ks_st[1] + (int64_t)p.head * a.ks_st[2]);
        cp_async4(&to->y, a.v_scale + (int64_t)p.page * a.vs_st[0] + (int64_t)blk * a.vs_st[1] + (int64_t)p.head * a.vs_st[2]);
      } else {
        *to = make_float2(1.f, 1.f);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  Spot ahead;
  {
    Spot first[P];
#pragma unroll
    for (int p = 0; p < P; ++p) first[p] = find();
    ahead = find();
#pragma unroll
    for (int p = 0; p < P; ++p) issue(p, first[p]);
  }
  Turn ring_at(N), stage_at(P), scale_at(Cfg::kScales);
  for (int i = 0; i < queued; ++i) {  // `ahead` has been counted by the time it is the tile in turn
    const int slot = ring_at.at, stage = stage_at.at;
    asm volatile("cp.async.wait_group %0;" ::"n"(P - 1) : "memory");
    if (!all_wait(empty[slot], ring_at.parity ^ 1u)) {
      if (lane == 0) record_error(a.err, ERR_WAIT_EMPTY);
      break;
    }
    uint8_t* to = ring + slot * Cfg::kChunk + (col >> 2) * kBlockBytes;
    uint4 x[J];
#pragma unroll
    for (int j = 0; j < J; ++j) x[j] = raw[stage * kTileRaw + j * 32];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int r = pw * kGroup + j * kRowsPer + row;
      uint4 y[2];
      deq_fp8_word(x[j].x, y[0].x, y[0].y);
      deq_fp8_word(x[j].y, y[0].z, y[0].w);
      deq_fp8_word(x[j].z, y[1].x, y[1].y);
      deq_fp8_word(x[j].w, y[1].z, y[1].w);
      // lanes of neighbouring 64-element blocks take the two halves in turn: eight lanes, eight places
      const int odd = (col >> 2) & 1, u = (col & 3) * 2;
      *reinterpret_cast<uint4*>(to + r * 128 + (((u + odd) ^ (r & 7)) << 4)) = odd ? y[1] : y[0];
      *reinterpret_cast<uint4*>(to + r * 128 + (((u + 1 - odd) ^ (r & 7)) << 4)) = odd ? y[0] : y[1];
    }
    if (!kValues && lane == 0)  // which copied them
      s.scales[scale_at.at][pw] = group_factors(a, s.raw_scales[stage][pw]);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(full[slot]));
    issue(stage, ahead);
    ahead = find();
    ring_at.next();
    stage_at.next();
    if (!kValues) scale_at.next();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

}  // namespace

template <typename T, int D, int RT, bool kAlt>
__global__ void __launch_bounds__((4 * RT + 12) * 32, 1) tree_attn8_tc_kernel(const __grid_constant__ Attn8Args a) {
  using Cfg = Tc8<D, RT, kAlt>;
  using H = __half;  // operands of both products
  constexpr int NK = Cfg::kK, NV = Cfg::kV, kBlocks = Cfg::kBlocks, kRows = Cfg::kRows;
  extern __shared__ uint8_t raw[];
  uint8_t* base = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  typename Cfg::Smem& s = *reinterpret_cast<typename Cfg::Smem*>(base);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  attn_unowned(a, attn_prefix(a, kRows, s.before, reinterpret_cast<long long*>(s.q), blockIdx.x == 0));
  const long long total = s.before[a.B];
  const long long G = total < (long long)gridDim.x ? total : (long long)gridDim.x;
  pdl_trigger();  // the launch that joins the partials may get ready
  if (blockIdx.x >= G) return;
  if (tid == 0) {
    for (int i = 0; i < NK; ++i) mbar_init(bar(s.kfull[i]), 4), mbar_init(bar(s.kempty[i]), 1);
    for (int i = 0; i < NV; ++i) mbar_init(bar(s.vfull[i]), 4), mbar_init(bar(s.vempty[i]), 1);
    for (int r = 0; r < RT; ++r) {
      for (int i = 0; i < 2; ++i)
        mbar_init(bar(s.sfull[r][i]), 1), mbar_init(bar(s.pfull[r][i]), 4), mbar_init(bar(s.odone[r][i]), 1);
      mbar_init(bar(s.qfull[r]), 4);
    }
    mbar_init(bar(s.joined[0]), 4);
    mbar_init(bar(s.joined[1]), kAlt ? 4 : 8);
    mbar_init(bar(s.merged), 4);
    mbar_init(bar(s.drain), 2);
    s.odd[0] = s.odd[1] = s.odd[2] = 0ull;
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (warp == Cfg::kIssue) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem)),
                 "r"(Cfg::kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tm = s.tmem;
  if (warp >= Cfg::kLoad && warp < Cfg::kIssue) {
    // ------------------------------------------------------------------ loading and converting warps
    give_registers8<RT>();
    load8<D, RT, kAlt>(a, s, total, G, warp >= Cfg::kLoad + 4, warp & 3);
  } else if (warp == Cfg::kIssue + 2) {
    // ------------------------------------------------------------------ S = Q K^T
    give_registers8<RT>();
    Segments sg(a, s.before, kRows, total, G);
    constexpr uint32_t kId = attn_idesc(TcType<H>::kCode, 0, kTile);
    Turn ring(NK);
    int n[RT], segs[RT];       // tiles and segments of each row tile
#pragma unroll
    for (int r = 0; r < RT; ++r) n[r] = segs[r] = 0;
    int code = 0;
    auto scores = [&](int w, int chunk) {
      // the weights of the buffer's tile before have been used
      const int turn = n[w] & 1;
      if (!all_wait(s.odone[w][turn], ((n[w] >> 1) & 1) ^ 1)) { code = ERR_WAIT_RFREE; return; }
      fence_after();
      const uint32_t q = Cfg::kQInTmem ? tm + Cfg::kQCol : smem_u32(s.q[kAlt ? 0 : w]), k = smem_u32(s.k[chunk]);
      const uint32_t d = tm + RT * D + (w * 2 + turn) * kTile;
#pragma unroll 1
      for (int x = 0; x < D / 16; ++x) {
        const uint64_t kd = desc_sw128(k + (x >> 2) * kBlockBytes + (x & 3) * 32, 16, 1024);
        if (Cfg::kQInTmem) mma_ts(d, q + 8 * x, kd, kId, x > 0);
        else mma_ss(d, desc_sw128(q + (x >> 2) * (128 * 128) + (x & 3) * 32, 16, 1024), kd, kId, x > 0);
      }
      commit_to(s.sfull[w][turn]);
      ++n[w];
    };
    while (code == 0 && sg.next()) {
      const int rts = RT == 1 || kAlt ? 1 : (sg.live + 127) / 128;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if (r >= rts) break;
        if (!all_wait(s.qfull[r], segs[r] & 1)) code = ERR_WAIT_X;
        ++segs[r];
      }
      fence_after();
      for (int t = sg.t0; code == 0 && t < sg.t1; ++t, ring.next()) {
        const int c = ring.at;
        if (!all_wait(s.kfull[c], ring.parity)) { code = ERR_WAIT_FULL; break; }
        fence_after();
        const int set = (t - sg.t0) & 1;
#pragma unroll
        for (int r = 0; r < RT; ++r)
          if ((kAlt ? r == set : r < rts) && code == 0) scores(r, c);
        commit_to(s.kempty[c]);
      }
    }
    if (code && lane == 0) record_error(a.err, code);
    commit_to(s.drain);  // nothing runs any more when the tensor memory is freed
    if (!all_wait(s.drain, 0) && lane == 0) record_error(a.err, ERR_DRAIN);
  } else if (warp == Cfg::kIssue + 3) {
    // ------------------------------------------------------------------ O += P V
    give_registers8<RT>();
    Segments sg(a, s.before, kRows, total, G);
    constexpr uint32_t kId = attn_idesc(TcType<H>::kCode, 1, D);
    Turn ring(NV);
    int n[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) n[r] = 0;
    int code = 0;
    auto values = [&](int w, int chunk, bool add) {
      if (!all_wait(s.pfull[w][n[w] & 1], (n[w] >> 1) & 1)) { code = ERR_WAIT_RED; return; }
      fence_after();
      const uint32_t v = smem_u32(s.v[chunk]), p = tm + RT * D + (w * 2 + (n[w] & 1)) * kTile;
#pragma unroll 1
      for (int x = 0; x < kTile / 16; ++x)
        mma_ts(tm + w * D, p + 8 * x, desc_sw128(v + x * 2048, kBlockBytes, 1024), kId, add || x > 0);
      commit_to(s.odone[w][n[w] & 1]);
      ++n[w];
    };
    while (code == 0 && sg.next()) {
      const int rts = RT == 1 || kAlt ? 1 : (sg.live + 127) / 128;
      for (int t = sg.t0; code == 0 && t < sg.t1; ++t, ring.next()) {
        const int c = ring.at;
        if (!all_wait(s.vfull[c], ring.parity)) { code = ERR_WAIT_FULL; break; }
        const int set = (t - sg.t0) & 1;
#pragma unroll
        for (int r = 0; r < RT; ++r)
          if ((kAlt ? r == set : r < rts) && code == 0) values(r, c, t > sg.t0 + (kAlt ? r : 0));
        commit_to(s.vempty[c]);
      }
    }
    if (code && lane == 0) record_error(a.err, code);
    commit_to(s.drain);
    if (!all_wait(s.drain, 0) && lane == 0) record_error(a.err, ERR_DRAIN);
  } else if (warp < Cfg::kLoad) {
    // ------------------------------------------------------------------ softmax
    take_registers8<RT>();
    Segments sg(a, s.before, kRows, total, G);
    const int rt = warp >> 2, quad = warp & 3;
    const int row = quad * 32 + lane;  // of the row tile, and its lane in tensor memory
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    int n = 0, tiles = 0, seg = 0;  // tiles of the row tile and of the CTA, segments
    bool ok = true;
    int joins[2] = {0, 0};
    auto join = [&](int who) {  // a barrier of the live row tiles' warps, with a bounded wait
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(s.joined[who]));
      return all_wait(s.joined[who], joins[who]++ & 1);
    };
    auto o_is_done = [&]() { return all_wait(s.odone[rt][(n - 1) & 1], ((n - 1) >> 1) & 1); };
    while (ok && sg.next()) {
      const int first_tile = tiles;
      tiles += sg.t1 - sg.t0;
      unsigned long long* odds = &s.odd[seg % 3];
      ++seg;
      const int r0 = kAlt ? 0 : rt * 128;
      if (r0 >= sg.live) continue;
      const int who = kAlt ? rt : RT == 2 && sg.live > 128 ? 1 : 0, threads = who && !kAlt ? 256 : 128;
      const int r = r0 + row;
      const bool mine = r < sg.live;
      const bool busy = r0 + quad * 32 < sg.live;  // the warp has a live row
      const int node = mine ? (sg.row0 + r) / a.group : 0;
      const int hq = sg.head * a.group + sg.row0 + r - node * a.group;  // where the row is live
      const int64_t qn = sg.rq.n0 + node;
      const unsigned long long mask = mine ? attn_mask(a, sg.rq, node) : 0ull;
      float factor = a.scale * 1.4426950408889634f;  // of the row's scores, in base-2 units
      if (Cfg::kQInTmem) {
        // Into tensor memory, a row a lane, by way of the warp's part of s.q: 64 elements at a time, eight lanes a row,
        // so that loads are whole lines (one 16-node tree over 32,768 keys 39 -> 36 us).  First each row's largest
        // element, then its elements times its power of two.
        const int64_t my = mine ? qn * a.q_sn + (int64_t)hq * a.q_sh : -1;
        const T* q = reinterpret_cast<const T*>(a.q) + (lane & 7) * 8;
        const T* from[8];
        float top[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int64_t at = __shfl_sync(0xffffffffu, my, 4 * k + (lane >> 3));
          from[k] = at < 0 ? nullptr : q + at;
          top[k] = 0.f;
        }
        auto eight = [&](int k, int c) {
          return from[k] ? *reinterpret_cast<const uint4*>(from[k] + c * 64) : make_uint4(0u, 0u, 0u, 0u);
        };
        constexpr int kHold = 2;  // times 64 elements of a row at a time
        static_assert(!Cfg::kQInTmem || D / 64 % kHold == 0, "whole steps");
        uint4 held[kHold][8];
#pragma unroll 1
        for (int c0 = 0; c0 < D / 64; c0 += kHold) {
#pragma unroll
          for (int c = 0; c < kHold; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) held[c][k] = eight(k, c0 + c);
#pragma unroll
          for (int c = 0; c < kHold; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t w[4] = {held[c][k].x, held[c][k].y, held[c][k].z, held[c][k].w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 y = two_floats<T>(w[e]);
                top[k] = max_three(top[k], fabsf(y.x), fabsf(y.y));
              }
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], o));
          const int e2 = row_exponent(top[k]);
          if ((lane & 7) == 0) s.factor[quad * 32 + 4 * k + (lane >> 3)] = factor * pow2f(-e2);
          top[k] = pow2f(e2);
        }
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          uint8_t* to = s.q[0] + quad * 32 * 128;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint4 x = eight(k, c);
            const int y = 4 * k + (lane >> 3);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            uint32_t z[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 v = two_floats<T>(w[e]);
              z[e] = pack2<H>(v.x * top[k], v.y * top[k]);
            }
            *reinterpret_cast<uint4*>(to + y * 128 + (((lane & 7) ^ (y & 7)) << 4)) = make_uint4(z[0], z[1], z[2], z[3]);
          }
          __syncwarp();
          uint32_t z[32];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint4 x = lds128(to + lane * 128 + ((e ^ (lane & 7)) << 4));
            z[4 * e] = x.x, z[4 * e + 1] = x.y, z[4 * e + 2] = x.z, z[4 * e + 3] = x.w;
          }
          st32(tm + lanes + Cfg::kQCol + 32 * c, z);
          __syncwarp();
        }
        wait_st();
        fence_before();
        __syncwarp();
        factor = s.factor[row];
      } else {
        const T* q = reinterpret_cast<const T*>(a.q) + qn * a.q_sn + (int64_t)hq * a.q_sh;
        uint8_t* to = s.q[kAlt ? 0 : rt] + row * 128;
        float amax = 0.f;
        if (mine) {
#pragma unroll 8
          for (int c = 0; c < D / 8; ++c) {
            const uint4 x = *reinterpret_cast<const uint4*>(q + c * 8);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 y = two_floats<T>(w[e]);
              amax = fmaxf(amax, fmaxf(fabsf(y.x), fabsf(y.y)));
            }
          }
        }
        const int e2 = row_exponent(amax);
        const float up = pow2f(e2);
        factor *= pow2f(-e2);
        auto eight = [&](int c, uint32_t* y) {
          const uint4 x = mine ? *reinterpret_cast<const uint4*>(q + c * 8) : make_uint4(0u, 0u, 0u, 0u);
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 z = two_floats<T>(w[e]);
            y[e] = pack2<H>(z.x * up, z.y * up);
          }
        };
        if (!(kAlt && rt == 1)) {  // the other set stores them
#pragma unroll 8
          for (int c = 0; c < D / 8; ++c) {
            uint32_t y[4];
            eight(c, y);
            *reinterpret_cast<uint4*>(to + (c >> 3) * (128 * 128) + (((c & 7) ^ (row & 7)) << 4)) =
                make_uint4(y[0], y[1], y[2], y[3]);
          }
        }
      }
      {
        if (tid == 0) s.odd[seg % 3] = 0ull;  // the next segment's
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && !(kAlt && rt == 1)) mbar_arrive(bar(s.qfull[rt]));
      }
      // the second set may have no tile of a segment, and must not tell of the next one before this one's are joined
      if (kAlt && rt == 1 && !all_wait(s.qfull[0], (seg - 1) & 1)) {
        if (lane == 0) record_error(a.err, ERR_WAIT_X);
        break;
      }
      float ref = -INFINITY, sum = 0.f, peak = -INFINITY;  // reference, weights' sum, highest reference so far
      // held by each thread: the other row tile's warps may be segments ahead of these, or behind
      unsigned long long odd = 0ull;
      const int len = sg.rq.ctx + sg.rq.nodes;
      constexpr int kStep = kAlt ? 2 : 1;
      const int begin = sg.t0 + (kAlt ? rt : 0);
      int scales_at = (first_tile + begin - sg.t0) % Cfg::kScales;
      for (int t = begin; t < sg.t1; t += kStep, ++n, scales_at += kStep, scales_at -= scales_at >= Cfg::kScales ? Cfg::kScales : 0) {
        const int pos0 = t * kTile;
        const bool tail = pos0 + kTile > sg.rq.ctx;
        if (!all_wait(s.sfull[rt][n & 1], (n >> 1) & 1)) {
          if (lane == 0) record_error(a.err, ERR_WAIT_RED);
          ok = false;
          break;
        }
        fence_after();
        const uint32_t sp = tm + lanes + RT * D + (rt * 2 + (n & 1)) * kTile;
        if (tail) {
          // A drafted token hidden from a row has weight 0 there, but 0 times NaN is NaN: such tokens' values
          // are cleared here and added at the end for the rows that see them.
          const int chunk = first_tile + t - sg.t0;
          ok = all_wait(s.vfull[chunk % NV], (chunk / NV) & 1) && join(who);
          uint8_t* v = s.v[chunk % NV];
          for (int u = r; u < kTile * kBlocks * 8; u += threads) {
            const int j = (u >> 3) % kTile;  // unit u: block, row, place
            if (pos0 + j < sg.rq.ctx || pos0 + j >= len) continue;
            const uint4 x = lds128(v + u * 16);
            if (odd_pair<H>(x.x) || odd_pair<H>(x.y) || odd_pair<H>(x.z) || odd_pair<H>(x.w))
              atomicOr(odds, 1ull << (pos0 + j - sg.rq.ctx));
          }
          ok = ok && join(who);
          const unsigned long long seen = *reinterpret_cast<volatile unsigned long long*>(odds);
          if (kAlt) {  // this tile's
            const int d0 = pos0 - sg.rq.ctx;
            odd |= seen & (d0 >= 64 ? 0ull : d0 >= 0 ? ~0ull << d0 : d0 > -64 ? ~0ull >> -d0 : 0ull);
          } else {  // and those before
            odd = seen;
          }
          if (odd) {
            for (int u = r; u < kTile * kBlocks * 8; u += threads) {
              const int d = pos0 + (u >> 3) % kTile - sg.rq.ctx;
              if (d >= 0 && d < sg.rq.nodes && (odd >> d & 1)) *reinterpret_cast<uint4*>(v + u * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();
          }
          ok = ok && join(who);
          if (!ok) {
            if (lane == 0) record_error(a.err, ERR_WAIT_RED);
            break;
          }
        }
        if (busy) {
          const float4* group = s.scales[scales_at];
          // Half a tile's scores at a time, in loops that stay loops: the roles' code has to fit into the instruction caches.
          auto half_scores = [&](int h, float (&x)[32]) {
            ld32(sp + 32 * h, reinterpret_cast<uint32_t*>(x));
            wait_ld();
            if (tail) {
              const int d0 = pos0 + 32 * h - sg.rq.ctx;
              const unsigned long long m = d0 >= 64 ? 0ull : d0 >= 0 ? mask >> d0 : mask << -max(d0, -63);
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const int d = d0 + j;
                if (d >= 0 && (d >= sg.rq.nodes || !(m >> j & 1))) x[j] = -INFINITY;
              }
            }
          };
          float mx = -INFINITY;
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            float x[32];
            half_scores(h, x);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const float4 y = group[2 * h + g];
            const float* z = x + g * kGroup;
            float m = max_three(max_three(z[0], z[1], z[2]), max_three(z[3], z[4], z[5]), max_three(z[6], z[7], z[8]));
            m = max_three(m, max_three(z[9], z[10], z[11]), max_three(z[12], z[13], fmaxf(z[14], z[15])));
            // the factor stays above zero: a hidden key's -inf has to
            mx = fmaxf(mx, fmaf(m, fmaxf(factor * y.x, 1e-30f), y.y));
          }
          }
          mx -= kHead<H>;
          bool move = mx > ref + kRise || (ref == -INFINITY && mx > ref);
          float next = mx;
          peak = fmaxf(peak, mx);
          if (mx < ref - kFall && mx > -INFINITY) {
            next = fmaxf(mx, peak - kSpan);
            move = next < ref;
          }
          if (t == begin) {
            ref = mx;
          } else if (__any_sync(0xffffffffu, move)) {
            if (!o_is_done()) {
              if (lane == 0) record_error(a.err, ERR_WAIT_RED);
              ok = false;
              break;
            }
            fence_after();
            const float to = move ? next : ref;
            const float f = to == ref ? 1.f : exp2_fast(ref - to);
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              float o[32];
              ld32(tm + lanes + rt * D + c, reinterpret_cast<uint32_t*>(o));
              wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] *= f;
              st32(tm + lanes + rt * D + c, reinterpret_cast<const uint32_t*>(o));
            }
            sum *= f;
            ref = to;
          }
          const float zero = ref == -INFINITY ? 0.f : -ref;
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            uint32_t p[kTile / 4];  // half a tile's, stored while the other half is computed
            float x[32];
            half_scores(half, x);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const float4 y = group[2 * half + g];
              const float ks = fmaxf(factor * y.x, 1e-30f), lv = y.y + zero;
              const unsigned long long ks2 = two(ks, ks), lv2 = two(lv, lv);
              unsigned long long part[2] = {0ull, 0ull};
#pragma unroll
              for (int j = 0; j < kGroup; j += 2) {
                float e0, e1;
                apart(fma_two(two(x[g * kGroup + j], x[g * kGroup + j + 1]), ks2, lv2), e0, e1);
                e0 = exp2_fast(e0);
                e1 = exp2_fast(e1);
                part[j / 2 & 1] = add_two(part[j / 2 & 1], two(e0, e1));
                p[((g & 1) * kGroup + j) / 2] = pack2<H>(e0, e1);
              }
              float e0, e1;
              apart(add_two(part[0], part[1]), e0, e1);
              sum = fmaf(e0 + e1, y.z, sum);
            }
            st16(sp + half * (kTile / 4), p);
          }
          wait_st();
          fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(s.pfull[rt][n & 1]));
      }
      if (!ok) break;
      if (begin < sg.t1 && !o_is_done()) {
        if (lane == 0) record_error(a.err, ERR_WAIT_RED);
        break;
      }
      fence_after();
      if (busy) {
        const uint32_t oa = tm + lanes + rt * D;
        while (odd) {  // rare: NaN values, for the rows that see them
          const int d = __ffsll((long long)odd) - 1;
          odd &= odd - 1;
          const Place8 at = attn8_place(a, sg.b, sg.rq.ctx + d, len, sg.head);
          const bool add = mine && (mask >> d & 1) && at.v >= 0;
          float wgt = 0.f;
          if (add) {
            const T* q = reinterpret_cast<const T*>(a.q) + qn * a.q_sn + (int64_t)hq * a.q_sh;
            const uint8_t* k = reinterpret_cast<const uint8_t*>(a.k_cache) + at.k;
            const float4 y = group_scales(a, at);
            float dot = 0.f;
            for (int e = 0; e < D; ++e) dot += to_f32(q[e]) * e4m3_value(k[e]);
            wgt = exp2_fast(fmaf(dot, a.scale * 1.4426950408889634f * y.x, y.y) - (ref == -INFINITY ? 0.f : ref));
          }
          const uint8_t* v = reinterpret_cast<const uint8_t*>(a.v_cache) + (at.v >= 0 ? at.v : 0);
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            float o[32];
            __syncwarp();
            ld32(oa + c, reinterpret_cast<uint32_t*>(o));
            wait_ld();
            if (add) {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] += wgt * e4m3_value(v[c + e]);
            }
            __syncwarp();
            st32(oa + c, reinterpret_cast<const uint32_t*>(o));
          }
          wait_st();
        }
      }
      float mine_by = 1.f, its_by = 0.f;  // factors of the two sets' results
      if (kAlt) {
        if (rt == 1) {
          if (busy) s.stat[row] = make_float2(ref, sum);
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(s.merged));
          continue;
        }
        if (!all_wait(s.merged, (seg - 1) & 1)) {
          if (lane == 0) record_error(a.err, ERR_WAIT_RED);
          break;
        }
        fence_after();
        if (busy && sg.t1 - sg.t0 > 1) {
          const float2 other = s.stat[row];
          const float top = fmaxf(ref, other.x), zero = top == -INFINITY ? 0.f : top;
          mine_by = exp2_fast(ref - zero);
          its_by = exp2_fast(other.x - zero);
          sum = sum * mine_by + other.y * its_by;
          ref = top;
        }
      }
      if (busy) {
        const uint32_t oa = tm + lanes + r0 / 128 * D;
        const bool all = sg.first && sg.last;
        const float inv = all ? (sum > 0.f || sum != sum ? 1.f / sum : 0.f) : 1.f;
        T* out = reinterpret_cast<T*>(a.out) + qn * a.o_sn + (int64_t)hq * a.o_sh;
        float* slot = a.partials + (2ll * blockIdx.x + (sg.first ? 1 : 0)) * attn_slot_floats(kRows, D);
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float o[32];
          __syncwarp();
          ld32(oa + c, reinterpret_cast<uint32_t*>(o));
          if (kAlt && sg.t1 - sg.t0 > 1) {
            float other[32];
            ld32(oa + D + c, reinterpret_cast<uint32_t*>(other));
            wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = (o[e] * mine_by + other[e] * its_by) * inv;
          } else {
            wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= inv;
          }
          if (mine && all) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint4 y;
              y.x = pack2<T>(o[e], o[e + 1]);
              y.y = pack2<T>(o[e + 2], o[e + 3]);
              y.z = pack2<T>(o[e + 4], o[e + 5]);
              y.w = pack2<T>(o[e + 6], o[e + 7]);
              *reinterpret_cast<uint4*>(out + c + e) = y;
            }
          }
          if (!all) {
            // A row a thread would touch 32 lines a store: the warp's 32 rows x 32 columns go through the
            // queries' place of its rows (they have been used), and out four whole lines a store.
            uint8_t* turn = s.q[kAlt ? 0 : rt] + quad * 32 * 128;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<float4*>(turn + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                  make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int y = e * 4 + (lane >> 3), k = lane & 7, ry = r0 + quad * 32 + y;
              const float4 v = *reinterpret_cast<const float4*>(turn + y * 128 + ((k ^ (y & 7)) << 4));
              if (ry < sg.live) *reinterpret_cast<float4*>(slot + (int64_t)ry * D + c + 4 * k) = v;
            }
          }
        }
        if (mine && all && a.lse)
          a.lse[qn * a.Hq + hq] = sum == 0.f ? -INFINITY : (ref + log2f(sum)) * 0.6931471805599453f;
        if (mine && !all)
          *reinterpret_cast<float2*>(slot + (int64_t)kRows * D + 2 * r) = make_float2(ref, sum);
      }
      __syncwarp();
      fence_before();
    }
  } else {
    give_registers8<RT>();
  }
  fence_before();
  __syncthreads();
  if (warp == Cfg::kIssue) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(Cfg::kCols) : "memory");
  }
}

namespace {

template <typename T, int D, int RT, bool kAlt>
int launch_tc8(const Attn8Args& a, cudaStream_t stream, int& grid, int& rows) {
  using Cfg = Tc8<D, RT, kAlt>;
  static_assert(sizeof(typename Cfg::Smem) + 1024 <= 227 * 1024, "shared memory");
  const void* k = (const void*)tree_attn8_tc_kernel<T, D, RT, kAlt>;
  if (!prepare_kernel(k)) return 2;
  grid = num_sms();
  rows = Cfg::kRows;
  return launch_with_pdl(k, a, grid, Cfg::kThreads, sizeof(typename Cfg::Smem) + 1024, a.pdl, stream);
}

template <typename T>
int launch_tc8_t(const Attn8Args& a, cudaStream_t stream, int& grid, int& rows) {
  const bool wide = a.max_nodes * a.group > 128;
  if (a.D == 64)
    return wide ? launch_tc8<T, 64, 2, false>(a, stream, grid, rows) : launch_tc8<T, 64, 2, true>(a, stream, grid, rows);
  if (a.D == 128)
    return wide ? launch_tc8<T, 128, 2, false>(a, stream, grid, rows) : launch_tc8<T, 128, 2, true>(a, stream, grid, rows);
  return launch_tc8<T, 256, 1, false>(a, stream, grid, rows);
}

}  // namespace

int launch_tree_attn8_tc(const Attn8Args& a, cudaStream_t stream, int& grid, int& rows) {
  return a.f16 ? launch_tc8_t<__half>(a, stream, grid, rows) : launch_tc8_t<__nv_bfloat16>(a, stream, grid, rows);
}

}  // namespace fnx
