// Tree attention on the 5th-generation tensor cores (tcgen05), for launches with several key tiles an
// SM.  The operator, the split of the work and the partial results are those of tree_attn.cu; here the
// two products run asynchronously with their operands and sums in shared and tensor memory, so loading,
// products and softmax of different key tiles overlap:
//
//   S = Q K^T   A = Q (128 rows x D, shared memory), B = a tile of 64 keys (shared memory)
//   O += P V    A = P (128 x 64, tensor memory, written over S), B = the tile's values as they lie
//               in the cache (N contiguous), D = O (128 x D fp32, tensor memory)
//
// RT row tiles of 128 share every key tile that is loaded (RT = 2: up to 256 rows, D <= 128), each with
// its own group of softmax warps.  Keys and values travel through rings of 64-row chunks, in 64-element
// blocks of 128-byte rows with the 128-byte swizzle: the same layout serves K-major keys and N-major
// values.
//
// Roles: 4 softmax warps a row tile (a thread has a row: its scores come from tensor memory in one
// piece, so the row's maximum and sum need no shuffles), 4 warps that load keys and 4 that load values
// (cp.async, any page size), one warp that issues the first product and one the second.  O is rescaled
// only when a row's maximum has risen by more than 2^8 (or, with fp16, fallen far: tree_attn.cuh): until
// then weights may be larger than one, which costs nothing in floating point.  Every wait is bounded and
// records an error code; roles then fall through to the end.
//
// Measured (B200, both launches, calls in a graph): 24 ragged requests, D = 128 fp16, 357 MB: 104 us, 3.4
// TB/s; 4 requests of 64 nodes over 131,072 keys, 1.48 GB and 171 GFLOP: 400 to 430 us, 3.4 to 3.7 TB/s and
// 400 to 430 TFLOP/s.  Loading alone (the rings emptied at once) takes 234 us at the latter.  What bounds
// it is the softmax warps' chain per tile: about 1,800 cycles from scores to weights, of which the
// exponentials' unit is busy for 512 a row tile.
// A second group on every other key tile of the same rows gained nothing (the rows' quarter of the SM
// has one unit for both groups), nor did deeper rings.
#include <type_traits>

#include "tree_attn.cuh"

namespace fnx {

namespace {

constexpr int kTile = kKeyTile;
constexpr int kBlockBytes = kTile * 128;  // 64 rows of a 64-element block
// Bits by which a row's maximum may rise above its reference's, and a tile's fall below it (fp16), unnoticed.
constexpr float kRise = 8.0f, kFall = 14.0f;
template <typename T> constexpr float kHead = kNarrow<T> ? 7.0f : 0.0f;  // weights are at most 2^(kHead + kRise)

template <int D, int RT>
struct TcAttn {
  static constexpr int kBlocks = D / 64;
  static constexpr int kChunk = kBlocks * kBlockBytes;  // keys or values of a tile
  static constexpr int kQTile = kBlocks * 128 * 128;    // a row tile of queries
  static constexpr int kK = D == 256 ? 2 : D == 128 ? (RT == 2 ? 4 : 5) : 8;  // chunks of the rings
  static constexpr int kV = D == 256 ? 3 : D == 128 ? (RT == 2 ? 5 : 6) : 8;
  static constexpr int kLoad = 4 * RT, kIssue = kLoad + 8;  // first loading, first issuing warp
  static constexpr int kThreads = (kIssue + 4) * 32;  // the issuing warps are the last two of four
  static constexpr int kCols = RT * (D + 2 * kTile) <= 256 ? 256 : 512;
  static_assert(RT * (D + 2 * kTile) <= 512, "tensor memory");
  struct Smem {
    uint8_t q[RT][kQTile];
    uint8_t k[kK][kChunk];
    uint8_t v[kV][kChunk];
    long long before[kAttnMaxBatch + 1];
    unsigned long long kfull[kK], kempty[kK], vfull[kV], vempty[kV];
    unsigned long long sfull[RT][2], pfull[RT][2], odone[RT][2], qfull[RT];
    unsigned long long joined[2];  // softmax warps of the first row tile, of both
    unsigned long long drain;
    // drafted tokens whose values are not all finite, of this segment, the one before and the next
    unsigned long long odd[3];
    uint32_t tmem;
  };
};

__device__ __forceinline__ uint64_t* bar(unsigned long long& b) { return reinterpret_cast<uint64_t*>(&b); }

// Shared-memory descriptors with the 128-byte swizzle (layout type 2 at bits 61-63, version 1 at bits
// 46-47), addresses and distances in 16-byte units.  K-major: 8-row groups SBO apart.  MN-major: 8
// k-rows of 128 bytes each are a group, groups SBO apart, 64-element blocks LBO apart.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46) | (2ull << 61);
}

// Instruction descriptor of kind::f16 with fp32 sums: operand types (0 fp16, 1 bf16) at bits 7 and 10,
// B N-major at bit 16, N / 8 at bit 17, M / 16 at bit 24.
__host__ __device__ constexpr uint32_t attn_idesc(int type, int n_major, int N) {
  return (1u << 4) | ((uint32_t)type << 7) | ((uint32_t)type << 10) | ((uint32_t)n_major << 16) |
         ((uint32_t)(N >> 3) << 17) | (8u << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(0u) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add), "r"(0u) : "memory");
}
__device__ __forceinline__ void commit_to(unsigned long long& b) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(smem_u32(&b)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr) : "memory");
}
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ bool all_wait(unsigned long long& b, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar(b), parity));
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> struct TcType;
template <> struct TcType<__nv_bfloat16> { static constexpr int kCode = 1; static constexpr uint32_t kExp = 0x7F80u; };
template <> struct TcType<__half> { static constexpr int kCode = 0; static constexpr uint32_t kExp = 0x7C00u; };
template <typename T>
__device__ __forceinline__ bool odd_pair(uint32_t w) {
  constexpr uint32_t e = TcType<T>::kExp;
  return (w & e) == e || ((w >> 16) & e) == e;
}

// The softmax warps hold a row's 64 scores and take registers that the others do not need: with one row
// tile 128 * 192 + 384 * 104 are no more than the launch's 512 * 128, with two 256 * 144 + 384 * 56 no
// more than 640 * 96.
template <int RT> __device__ __forceinline__ void give_registers() {
  if (RT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
}
template <int RT> __device__ __forceinline__ void take_registers() {
  if (RT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
  else asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
}

// The CTA's segments, one after the other: the same for every role.
struct Segments {
  const AttnArgs& a;
  const long long* before;
  long long w, end;
  int rows, b;
  AttnReq rq;
  int head, row0, live, t0, t1;
  bool first, last;  // whether the segment has the item's first and last tile

  __device__ __forceinline__ Segments(const AttnArgs& args, const long long* bf, int rows_, long long total, long long G)
      : a(args), before(bf), rows(rows_) {
    w = attn_first(blockIdx.x, total, G);
    end = attn_first(blockIdx.x + 1, total, G);
    b = attn_find(before, a.B, w);
  }
  __device__ __forceinline__ bool next() {
    if (w >= end) return false;
    while (before[b + 1] <= w) ++b;
    rq = attn_request(a, b, false);
    const AttnShape sh = attn_shape(a, rq, rows);
    const int item = (int)((w - before[b]) / sh.key_tiles);
    head = item / sh.row_tiles;
    row0 = (item % sh.row_tiles) * rows;
    live = min(rows, rq.nodes * a.group - row0);
    const long long i0 = before[b] + (long long)item * sh.key_tiles, i1 = i0 + sh.key_tiles;
    const long long w1 = end < i1 ? end : i1;
    t0 = (int)(w - i0);
    t1 = (int)(w1 - i0);
    first = w == i0;
    last = w1 == i1;
    w = w1;
    return true;
  }
};

}  // namespace

template <typename T, int D, int RT>
__global__ void __launch_bounds__((4 * RT + 12) * 32, 1) tree_attn_tc_kernel(const __grid_constant__ AttnArgs a) {
  using Cfg = TcAttn<D, RT>;
  constexpr int NK = Cfg::kK, NV = Cfg::kV, kBlocks = Cfg::kBlocks, kRows = 128 * RT;
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
    mbar_init(bar(s.joined[1]), 8);
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
  Segments sg(a, s.before, kRows, total, G);
  if (warp >= Cfg::kLoad && warp < Cfg::kIssue) {
    // ------------------------------------------------------------------ loading warps
    give_registers<RT>();
    constexpr int kLanesRow = D / 8 < 32 ? D / 8 : 32;  // lanes of a row: 16 bytes each
    constexpr int kRowsPer = 32 / kLanesRow;            // rows of one instruction
    const int pw = warp & 3;                            // rows 16 pw .. + 15 of every chunk
    const int col = lane % kLanesRow;                   // 16-byte unit of the row
    auto run = [&](auto stages, const T* from, uint8_t* ring, unsigned long long* full, unsigned long long* empty,
                   bool values) {
      // chunks in flight behind the last one: few enough that a chunk is not told of only when the one
      // before it has been used up
      constexpr int N = decltype(stages)::value, kLag = N / 2;
      int i = 0;
      bool ok = true;
      auto landed = [&](int chunk) {  // the thread's copies of the chunk are done
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(full[chunk % N]));
      };
      while (ok && sg.next()) {
        const int len = sg.rq.ctx + sg.rq.nodes;
        int64_t place, ahead, unused;
        auto find = [&](int t) {
          const int pos = t * kTile + pw * 16 + (lane & 15);
          if (values) attn_place(a, sg.b, pos, len, sg.head, unused, ahead);
          else attn_place(a, sg.b, pos, len, sg.head, ahead, unused);
        };
        find(sg.t0);
        for (int t = sg.t0; t < sg.t1; ++t) {
          place = ahead;
          if (t + 1 < sg.t1) find(t + 1);
          if (!all_wait(empty[i % N], ((i / N) & 1) ^ 1)) {
            if (lane == 0) record_error(a.err, ERR_WAIT_EMPTY);
            ok = false;
            break;
          }
          const uint32_t to = smem_u32(ring + (i % N) * Cfg::kChunk) + (col >> 3) * kBlockBytes;
#pragma unroll
          for (int j = 0; j < 16 / kRowsPer; ++j) {
            const int rr = j * kRowsPer + lane / kLanesRow;  // row within the warp's 16
            const int64_t at = __shfl_sync(0xffffffffu, place, rr);
            const int r = pw * 16 + rr;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                             to + r * 128 + (((col & 7) ^ (r & 7)) << 4)),
                         "l"(from + col * 8 + (at < 0 ? 0 : at)), "r"(at < 0 ? 0 : 16)
                         : "memory");
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
          ++i;
          if (i > kLag) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
            landed(i - 1 - kLag);
          }
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      for (int j = i > kLag ? i - kLag : 0; j < i; ++j) landed(j);
    };
    if (warp < Cfg::kLoad + 4)
      run(std::integral_constant<int, NK>{}, reinterpret_cast<const T*>(a.k_cache), s.k[0], s.kfull, s.kempty, false);
    else
      run(std::integral_constant<int, NV>{}, reinterpret_cast<const T*>(a.v_cache), s.v[0], s.vfull, s.vempty, true);
  } else if (warp == Cfg::kIssue + 2) {
    // ------------------------------------------------------------------ S = Q K^T
    give_registers<RT>();
    constexpr uint32_t kId = attn_idesc(TcType<T>::kCode, 0, kTile);
    int i = 0;                  // tile of the CTA
    int n[RT], segs[RT];       // tiles and segments of each row tile
#pragma unroll
    for (int r = 0; r < RT; ++r) n[r] = segs[r] = 0;
    int code = 0;
    auto scores = [&](int w, int chunk) {
      // the weights of the buffer's tile before have been used
      if (!all_wait(s.odone[w][n[w] & 1], ((n[w] >> 1) & 1) ^ 1)) { code = ERR_WAIT_RFREE; return; }
      fence_after();
      const uint32_t q = smem_u32(s.q[w]), k = smem_u32(s.k[chunk]);
      const uint32_t d = tm + RT * D + (w * 2 + (n[w] & 1)) * kTile;
#pragma unroll
      for (int x = 0; x < D / 16; ++x)
        mma_ss(d, desc_sw128(q + (x >> 2) * (128 * 128) + (x & 3) * 32, 16, 1024),
               desc_sw128(k + (x >> 2) * kBlockBytes + (x & 3) * 32, 16, 1024), kId, x > 0);
      commit_to(s.sfull[w][n[w] & 1]);
      ++n[w];
    };
    while (code == 0 && sg.next()) {
      const int rts = RT == 1 ? 1 : (sg.live + 127) / 128;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if (r >= rts) break;
        if (!all_wait(s.qfull[r], segs[r] & 1)) code = ERR_WAIT_X;
        ++segs[r];
      }
      for (int t = sg.t0; code == 0 && t < sg.t1; ++t, ++i) {
        const int c = i % NK;
        if (!all_wait(s.kfull[c], (i / NK) & 1)) { code = ERR_WAIT_FULL; break; }
        fence_after();
#pragma unroll
        for (int r = 0; r < RT; ++r)
          if (r < rts && code == 0) scores(r, c);
        commit_to(s.kempty[c]);
      }
    }
    if (code && lane == 0) record_error(a.err, code);
    commit_to(s.drain);  // nothing runs any more when the tensor memory is freed
    if (!all_wait(s.drain, 0) && lane == 0) record_error(a.err, ERR_DRAIN);
  } else if (warp == Cfg::kIssue + 3) {
    // ------------------------------------------------------------------ O += P V
    give_registers<RT>();
    constexpr uint32_t kId = attn_idesc(TcType<T>::kCode, 1, D);
    int i = 0, n[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) n[r] = 0;
    int code = 0;
    auto values = [&](int w, int chunk, bool add) {
      if (!all_wait(s.pfull[w][n[w] & 1], (n[w] >> 1) & 1)) { code = ERR_WAIT_RED; return; }
      fence_after();
      const uint32_t v = smem_u32(s.v[chunk]), p = tm + RT * D + (w * 2 + (n[w] & 1)) * kTile;
#pragma unroll
      for (int x = 0; x < kTile / 16; ++x)
        mma_ts(tm + w * D, p + 8 * x, desc_sw128(v + x * 2048, kBlockBytes, 1024), kId, add || x > 0);
      commit_to(s.odone[w][n[w] & 1]);
      ++n[w];
    };
    while (code == 0 && sg.next()) {
      const int rts = RT == 1 ? 1 : (sg.live + 127) / 128;
      for (int t = sg.t0; code == 0 && t < sg.t1; ++t, ++i) {
        const int c = i % NV;
        if (!all_wait(s.vfull[c], (i / NV) & 1)) { code = ERR_WAIT_FULL; break; }
#pragma unroll
        for (int r = 0; r < RT; ++r)
          if (r < rts && code == 0) values(r, c, t > sg.t0);
        commit_to(s.vempty[c]);
      }
    }
    if (code && lane == 0) record_error(a.err, code);
    commit_to(s.drain);
    if (!all_wait(s.drain, 0) && lane == 0) record_error(a.err, ERR_DRAIN);
  } else if (warp < Cfg::kLoad) {
    // ------------------------------------------------------------------ softmax
    take_registers<RT>();
    const int rt = warp >> 2, quad = warp & 3;
    const int row = quad * 32 + lane;  // of the row tile, and its lane in tensor memory
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const float c2 = a.scale * 1.4426950408889634f;
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
      if (rt * 128 >= sg.live) continue;
      const int who = RT == 2 && sg.live > 128 ? 1 : 0, threads = who ? 256 : 128;
      const int r = rt * 128 + row;
      const bool mine = r < sg.live;
      const bool busy = rt * 128 + quad * 32 < sg.live;  // the warp has a live row
      const int node = mine ? (sg.row0 + r) / a.group : 0;
      const int hq = sg.head * a.group + (sg.row0 + r) % a.group;
      const int64_t qn = sg.rq.n0 + node;
      const unsigned long long mask = mine ? attn_mask(a, sg.rq, node) : 0ull;
      {
        const T* q = reinterpret_cast<const T*>(a.q) + qn * a.q_sn + (int64_t)hq * a.q_sh;
        uint8_t* to = s.q[rt] + row * 128;
#pragma unroll 16
        for (int c = 0; c < D / 8; ++c) {
          const uint4 x = mine ? *reinterpret_cast<const uint4*>(q + c * 8) : make_uint4(0u, 0u, 0u, 0u);
          *reinterpret_cast<uint4*>(to + (c >> 3) * (128 * 128) + (((c & 7) ^ (row & 7)) << 4)) = x;
        }
        if (tid == 0) s.odd[seg % 3] = 0ull;  // the next segment's
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(s.qfull[rt]));
      }
      float ref = -INFINITY, sum = 0.f, peak = -INFINITY;  // reference, weights' sum, highest reference so far
      // held by each thread: the other row tile's warps may be segments ahead of these, or behind
      unsigned long long odd = 0ull;
      const int len = sg.rq.ctx + sg.rq.nodes;
      for (int t = sg.t0; t < sg.t1; ++t, ++n) {
        const int pos0 = t * kTile;
        const bool tail = pos0 + kTile > sg.rq.ctx;
        if (!all_wait(s.sfull[rt][n & 1], (n >> 1) & 1)) {
          if (lane == 0) record_error(a.err, ERR_WAIT_RED);
          ok = false;
          break;
        }
        fence_after();
        if (tail) {
          // A drafted token hidden from a row has weight 0 there, but 0 times an infinite or NaN value is
          // NaN: such tokens' values are cleared here and added at the end for the rows that see them.
          const int chunk = first_tile + t - sg.t0;
          ok = all_wait(s.vfull[chunk % NV], (chunk / NV) & 1) && join(who);
          uint8_t* v = s.v[chunk % NV];
          for (int u = rt * 128 + row; u < kTile * kBlocks * 8; u += threads) {
            const int j = (u >> 3) % kTile;  // unit u: block, row, place
            if (pos0 + j < sg.rq.ctx || pos0 + j >= len) continue;
            const uint4 x = lds128(v + u * 16);
            if (odd_pair<T>(x.x) || odd_pair<T>(x.y) || odd_pair<T>(x.z) || odd_pair<T>(x.w))
              atomicOr(odds, 1ull << (pos0 + j - sg.rq.ctx));
          }
          ok = ok && join(who);
          odd = *reinterpret_cast<volatile unsigned long long*>(odds);  // this tile's and those before
          if (odd) {
            for (int u = rt * 128 + row; u < kTile * kBlocks * 8; u += threads) {
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
        const uint32_t sp = tm + lanes + RT * D + (rt * 2 + (n & 1)) * kTile;
        if (busy) {
          float x[kTile];
          ld32(sp, reinterpret_cast<uint32_t*>(x));
          ld32(sp + 32, reinterpret_cast<uint32_t*>(x) + 32);
          wait_ld();
          if (tail) {
#pragma unroll
            for (int j = 0; j < kTile; ++j) {
              const int d = pos0 + j - sg.rq.ctx;
              if (d >= 0 && (d >= sg.rq.nodes || !(mask >> (d & 63) & 1))) x[j] = -INFINITY;
            }
          }
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < kTile; ++j) m4[j & 3] = fmaxf(m4[j & 3], x[j]);
          const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * c2 - kHead<T>;
          bool move = mx > ref + kRise || (ref == -INFINITY && mx > ref);
          float next = mx;
          if (kNarrow<T>) {
            peak = fmaxf(peak, mx);
            if (mx < ref - kFall && mx > -INFINITY) {
              next = fmaxf(mx, peak - kSpan);
              move = next < ref;
            }
          }
          if (t == sg.t0) {
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
          float s4[4] = {0.f, 0.f, 0.f, 0.f};
          uint32_t p[kTile / 2];
#pragma unroll
          for (int j = 0; j < kTile; j += 2) {
            x[j] = exp2_fast(fmaf(x[j], c2, zero));
            x[j + 1] = exp2_fast(fmaf(x[j + 1], c2, zero));
            s4[j & 2] += x[j];
            s4[(j & 2) + 1] += x[j + 1];
            p[j / 2] = pack2<T>(x[j], x[j + 1]);
          }
          sum += (s4[0] + s4[1]) + (s4[2] + s4[3]);
          st32(sp, p);
          wait_st();
          fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(s.pfull[rt][n & 1]));
      }
      if (!ok) break;
      if (!o_is_done()) {
        if (lane == 0) record_error(a.err, ERR_WAIT_RED);
        break;
      }
      fence_after();
      if (busy) {
        const uint32_t oa = tm + lanes + rt * D;
        while (odd) {  // rare: values that are not finite, for the rows that see them
          const int d = __ffsll((long long)odd) - 1;
          odd &= odd - 1;
          int64_t ko, vo;
          attn_place(a, sg.b, sg.rq.ctx + d, len, sg.head, ko, vo);
          const bool add = mine && (mask >> d & 1) && vo >= 0;
          float wgt = 0.f;
          if (add) {
            const T* q = reinterpret_cast<const T*>(a.q) + qn * a.q_sn + (int64_t)hq * a.q_sh;
            const T* k = reinterpret_cast<const T*>(a.k_cache) + ko;
            float dot = 0.f;
            for (int e = 0; e < D; ++e) dot += to_f32(q[e]) * to_f32(k[e]);
            wgt = exp2_fast(dot * c2 - (ref == -INFINITY ? 0.f : ref));
          }
          const T* v = reinterpret_cast<const T*>(a.v_cache) + (vo >= 0 ? vo : 0);
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            float o[32];
            __syncwarp();
            ld32(oa + c, reinterpret_cast<uint32_t*>(o));
            wait_ld();
            if (add) {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] += wgt * to_f32(v[c + e]);
            }
            __syncwarp();
            st32(oa + c, reinterpret_cast<const uint32_t*>(o));
          }
          wait_st();
        }
        const bool all = sg.first && sg.last, dense = sg.live - rt * 128 - quad * 32 > 8;
        const float inv = all ? (sum > 0.f || sum != sum ? 1.f / sum : 0.f) : 1.f;
        T* out = reinterpret_cast<T*>(a.out) + qn * a.o_sn + (int64_t)hq * a.o_sh;
        float* slot = a.partials + (2ll * blockIdx.x + (sg.first ? 1 : 0)) * attn_slot_floats(kRows, D);
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float o[32];
          __syncwarp();
          ld32(oa + c, reinterpret_cast<uint32_t*>(o));
          wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= inv;
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
          if (mine && !all && !dense) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(slot + (int64_t)r * D + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
          if (!all && dense) {
            // A row a thread would touch 32 lines a store: the warp's 32 rows x 32 columns go through the
            // queries' place of its rows (they have been used), and out four whole lines a store.
            uint8_t* turn = s.q[rt] + quad * 32 * 128;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<float4*>(turn + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                  make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int y = e * 4 + (lane >> 3), k = lane & 7, ry = rt * 128 + quad * 32 + y;
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
    give_registers<RT>();
  }
  fence_before();
  __syncthreads();
  if (warp == Cfg::kIssue) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(Cfg::kCols) : "memory");
  }
}

namespace {

template <typename T, int D, int RT>
int launch_tc(const AttnArgs& a, cudaStream_t stream, int& grid, int& rows) {
  using Cfg = TcAttn<D, RT>;
  const void* k = (const void*)tree_attn_tc_kernel<T, D, RT>;
  if (!prepare_kernel(k)) return 2;
  grid = num_sms();
  rows = 128 * RT;
  return launch_with_pdl(k, a, grid, Cfg::kThreads, sizeof(typename Cfg::Smem) + 1024, a.pdl, stream);
}

template <typename T>
int launch_tc_t(const AttnArgs& a, cudaStream_t stream, int& grid, int& rows) {
  const bool wide = a.max_nodes * a.group > 128;
  if (a.D == 64)
    return wide ? launch_tc<T, 64, 2>(a, stream, grid, rows) : launch_tc<T, 64, 1>(a, stream, grid, rows);
  if (a.D == 128)
    return wide ? launch_tc<T, 128, 2>(a, stream, grid, rows) : launch_tc<T, 128, 1>(a, stream, grid, rows);
  return launch_tc<T, 256, 1>(a, stream, grid, rows);
}

}  // namespace

int launch_tree_attn_tc(const AttnArgs& a, cudaStream_t stream, int& grid, int& rows) {
  return a.f16 ? launch_tc_t<__half>(a, stream, grid, rows) : launch_tc_t<__nv_bfloat16>(a, stream, grid, rows);
}

}  // namespace fnx
