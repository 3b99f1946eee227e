// What the tensor-memory forms of tree attention share: tcgen05 instructions, their descriptors, and a CTA's
// segments.
#pragma once

#include "tree_attn.cuh"

namespace fnx {

namespace {

constexpr int kTile = kKeyTile;
constexpr int kBlockBytes = kTile * 128;  // 64 rows of a 64-element block
// Bits by which a row's maximum may rise above its reference's, and a tile's fall below it (fp16), unnoticed.
constexpr float kRise = 8.0f, kFall = 14.0f;
template <typename T> constexpr float kHead = kNarrow<T> ? 7.0f : 0.0f;  // weights are at most 2^(kHead + kRise)

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

}  // namespace fnx
