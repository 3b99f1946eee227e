// Rotary positions on queries and keys, with keys and values stored in an 8-bit paged cache (cache8.cuh).
//
// The rotation is rotary.cu's: (a cos - b sin, b cos + a sin) for the pairs of a head's first R elements, in fp32
// with each product and sum rounded by itself.  Request b's new tokens go to places context_lens[b] + index.  For
// every block of places and every head that gets new tokens, with amax their largest finite magnitude:
//
//   s' = smallest power of two >= amax / 448 (2^-40 at least), and >= the block's old scale if tokens of the context
//        stay in the block;     new bytes = e4m3(y / s'),     old bytes = e4m3(value s / s')
//
// Bound: memory (each 16-bit element read once, a 16-bit query or an 8-bit key or value written once), or the launch
// and its chain of loads (offsets, page, data) for a few tokens.  A CTA has one block of one request and as many
// (key or value) heads as its 256 threads hold, a thread 16 elements of a token's head, or up to four times that: it
// finds the block's largest element with one exchange and writes the block without reading anything twice.  The
// queries go to CTAs of their own in the same launch.  Measured (B200, calls in a graph): 3.1 us for 8 tokens of 16 + 2
// heads of 256, 25.8 us for 4,097 tokens of 32 + 8 heads of 128 (93 MB, 3.6 TB/s): the queries alone take 14, keys and
// values alone 15 before infinities were looked for once a thread.  Neither is full, at 53 % of the issue slots and 22 % of
// DRAM's rate: a CTA's chain of position, table row and store is exposed once.
#include "cache8.cuh"

namespace fnx {

namespace {

constexpr int kAT = 256;  // threads

__device__ __forceinline__ float one(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float one(__half v) { return __half2float(v); }

// 16 elements of a head: two runs of eight, which hold whole pairs where the sizes allow 16-byte vectors.
struct Unit {
  int o0, o1;
};
template <bool kVec>
__device__ __forceinline__ Unit unit_of(const Append8Args& a, int u) {
  const bool apart = kVec && 16 * u < a.R && !a.interleaved;
  return apart ? Unit{8 * u, a.R / 2 + 8 * u} : Unit{16 * u, 16 * u + 8};
}

// The unit as it lies in memory: elements stay 16 bits until they are used, which leaves registers for more loads.
struct Raw {
  uint32_t w[8];
};
template <typename T, bool kVec>
__device__ __forceinline__ Raw load_raw(const T* src, const Unit& un) {
  Raw r;
  if (kVec) {
    const uint4 v0 = *reinterpret_cast<const uint4*>(src + un.o0), v1 = *reinterpret_cast<const uint4*>(src + un.o1);
    r.w[0] = v0.x, r.w[1] = v0.y, r.w[2] = v0.z, r.w[3] = v0.w;
    r.w[4] = v1.x, r.w[5] = v1.y, r.w[6] = v1.z, r.w[7] = v1.w;
  } else {
    const uint16_t* e = reinterpret_cast<const uint16_t*>(src) + un.o0;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = e[2 * i] | ((uint32_t)e[2 * i + 1] << 16);
  }
  return r;
}

__device__ __forceinline__ float turn_a(float a, float b, float c, float s) { return __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)); }
__device__ __forceinline__ float turn_b(float a, float b, float c, float s) { return __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s)); }

// The unit's elements in 32 bits, turned by row's cosines and sines where `turned`.
template <typename T>
__device__ __forceinline__ void values(const Append8Args& a, const Raw& r, const float* row, int u, bool turned, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 y = two_floats<T>(r.w[i]);
    x[2 * i] = y.x, x[2 * i + 1] = y.y;
  }
  if (!turned) return;
  const int half = a.R / 2;
#pragma unroll
  for (int z = 0; z < 2; ++z) {  // four pairs at a time
    const float4 c4 = __ldg(reinterpret_cast<const float4*>(row + 8 * u + 4 * z));
    const float4 s4 = __ldg(reinterpret_cast<const float4*>(row + half + 8 * u + 4 * z));
    const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 4 * z + e;
      if (a.interleaved) {
        const float p = x[2 * i], q = x[2 * i + 1];
        x[2 * i] = turn_a(p, q, c[e], s[e]);
        x[2 * i + 1] = turn_b(p, q, c[e], s[e]);
      } else {
        const float p = x[i], q = x[8 + i];
        x[i] = turn_a(p, q, c[e], s[e]);
        x[8 + i] = turn_b(p, q, c[e], s[e]);
      }
    }
  }
}
// Any sizes: 16 consecutive elements, each with its partner read by itself.
template <typename T>
__device__ __forceinline__ void turn_any(const Append8Args& a, const T* src, const float* row, int e0, float (&x)[16]) {
  const int half = a.R / 2;
#pragma unroll 1
  for (int i = 0; i < 16; ++i) {
    const int e = e0 + i;
    if (e >= a.R) break;
    const int pair = a.interleaved ? e >> 1 : (e < half ? e : e - half);
    const bool second = a.interleaved ? e & 1 : e >= half;
    const int other = a.interleaved ? e ^ 1 : (second ? e - half : e + half);
    const float c = __ldg(row + pair), s = __ldg(row + half + pair), mine = one(src[e]), its = one(src[other]);
    const float y = second ? turn_b(its, mine, c, s) : turn_a(mine, its, c, s);
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] = k == i ? y : x[k];
  }
}

__device__ __forceinline__ const float* table_row(const Append8Args& a, int64_t t, bool report) {
  int64_t pos = a.positions[t];
  if (pos < 0 || pos >= a.P) {
    if (report) record_error(a.err, ERR_POSITION);
    pos = pos < 0 ? 0 : a.P - 1;
  }
  return a.table + pos * a.table_ld;
}

// The queries of the launch: a CTA takes tokens one after the other, a thread a unit of every `rows`-th head.
template <typename T, bool kVec>
__device__ __forceinline__ void queries(const Append8Args& a, int cta) {
  const int wide = a.D / 16, rows = kAT / wide;
  const int u = threadIdx.x % wide, r = threadIdx.x / wide;
  const int part = cta % a.q_parts, first = cta / a.q_parts, step = a.q_ctas / a.q_parts;
  const Unit un = unit_of<kVec>(a, u);
  const bool turned = 16 * u < a.R;
  for (int t = first; t < a.T; t += step) {
    const float* row = nullptr;
    for (int h0 = part * rows; h0 < a.Hq; h0 += a.q_parts * rows) {
      const int h = h0 + r;
      const bool live = h < a.Hq;
      const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)t * a.q_st + (int64_t)h * a.q_sh;
      T* dst = reinterpret_cast<T*>(a.q_out) + (int64_t)t * a.o_st + (int64_t)h * a.o_sh;
      Raw raw;
      if (live) raw = load_raw<T, kVec>(src, un);  // ahead of the position, which the table waits for
      if (!row) row = table_row(a, t, part == 0 && threadIdx.x == 0);
      float x[16];
      if (live) {
        values<T>(a, raw, row, u, kVec && turned, x);
        if (!kVec && turned) turn_any(a, src, row, un.o0, x);
      }
      if (!kVec) __syncwarp();  // q may be turned in place, and a unit's partners are other lanes'
      if (!live) continue;
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = round_pair<T>(x[2 * i], x[2 * i + 1]);
      if (kVec) {
        *reinterpret_cast<uint4*>(dst + un.o0) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4*>(dst + un.o1) = make_uint4(w[4], w[5], w[6], w[7]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint16_t bits = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
          reinterpret_cast<uint16_t*>(dst)[un.o0 + i] = bits;
        }
      }
    }
  }
}

}  // namespace

// Units of request b: numbers [off[b] / block + 2 b, off[b + 1] / block + 2 (b + 1)), at least as many as the blocks
// that its tokens can touch wherever the context ends.  So a unit's request follows from the offsets alone.
// kItems: 16-element units of a thread, in one block and head.
template <typename T, bool kVec, int kItems>
__global__ void __launch_bounds__(kAT) append8_kernel(const __grid_constant__ Append8Args a) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  const int kv = a.kv_units * a.head_parts;
  if ((int)blockIdx.x >= kv) {
    queries<T, kVec>(a, blockIdx.x - kv);
    pdl_trigger();
    return;
  }
  const int unit = blockIdx.x / a.head_parts, part = blockIdx.x - unit * a.head_parts;
  const int block_shift = 31 - __clz(a.block), wide_shift = 27 - __clz(a.D);  // blocks of 16 to 64, heads of 64 to 256
  int b = -1;
  for (int b0 = 0; b0 < a.B; b0 += kAT) {
    const int i = b0 + tid;
    b += __syncthreads_count(i < a.B && (a.node_offsets[i] >> block_shift) + 2 * i <= unit);
  }
  __shared__ uint32_t amax_of[kAT / 32];
  const int per_shift = kItems == 1 ? block_shift + wide_shift : 8;  // threads of a head: 64 at least
  const int group = tid >> per_shift, at = tid & ((1 << per_shift) - 1), groups = kAT >> per_shift;
  const bool speaks = part == 0 && tid == 0;
  if (b < 0) {  // ahead of the first request's units
    pdl_trigger();
    return;
  }
  const int n0 = a.node_offsets[b], n = a.node_offsets[b + 1] - n0, ctx = a.context_lens[b];
  if (n0 < 0 || n < 0 || n > a.T - n0 || ctx < 0 || (int64_t)ctx + n > (int64_t)a.table_width * a.page_size) {
    if (speaks) record_error(a.err, ERR_LENGTHS);
    pdl_trigger();
    return;
  }
  const int ahead = unit - ((n0 >> block_shift) + 2 * b);  // blocks of the request in front of this one
  const uint32_t start = (uint32_t)((ctx >> block_shift) + ahead) << block_shift, end = (uint32_t)ctx + n;
  if (ahead < 0 || start >= end || n == 0) {
    pdl_trigger();
    return;
  }
  const int kept = (uint32_t)ctx > start ? (int)(ctx - start) : 0;  // places of the block in front of the first new one
  const int64_t to_token = (int64_t)n0 + start - ctx;               // token at the block's first place
  const int last = (int)min((uint32_t)a.block, end - start);
  const uint32_t number = start / (uint32_t)a.page_size;
  const int in_page = (int)(start - number * (uint32_t)a.page_size);
  const int page = a.page_table[(int64_t)b * a.pt_ld + number];
  const int head = part * groups + group;  // keys' heads, then values'
  const bool key = head < a.Hk, mine = head < 2 * a.Hk;
  const int h = key ? head : head - a.Hk;
  const int u = at & ((1 << wide_shift) - 1);  // the same for all of the thread's units
  const Unit un = unit_of<kVec>(a, u);
  const bool turned = key && 16 * u < a.R;
  auto row_of = [&](int i) { return (at + (i << per_shift)) >> wide_shift; };
  auto fresh = [&](int i) { return mine && row_of(i) >= kept && row_of(i) < last; };
  auto source = [&](int i) {
    return reinterpret_cast<const T*>(key ? a.k : a.v) + (to_token + row_of(i)) * (key ? a.k_st : a.v_st) +
           (int64_t)h * (key ? a.k_sh : a.v_sh);
  };
  Raw raw[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i)
    if (fresh(i)) raw[i] = load_raw<T, kVec>(source(i), un);  // ahead of the positions, which the table waits for
  float x[kItems][16];
  uint32_t amax = 0u;  // bits of the largest magnitude, infinities and NaN among them
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    if (!fresh(i)) continue;
    const float* row = turned ? table_row(a, to_token + row_of(i), h == 0 && u == 0) : nullptr;
    values<T>(a, raw[i], row, u, kVec && turned, x[i]);
    if (!kVec && turned) turn_any(a, source(i), row, un.o0, x[i]);
#pragma unroll
    for (int e = 0; e < 16; ++e) amax = max(amax, __float_as_uint(x[i][e]) & 0x7FFFFFFFu);
  }
  const bool odd = amax >= 0x7F800000u;  // rare: an element is not finite
  if (odd) {
    amax = 0u;
#pragma unroll
    for (int i = 0; i < kItems; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t m = fresh(i) ? __float_as_uint(x[i][e]) & 0x7FFFFFFFu : 0u;
        amax = max(amax, m < 0x7F800000u ? m : 0u);
        if (m >= 0x7F800000u) x[i][e] = NAN;
      }
  }
  amax = __reduce_max_sync(0xffffffffu, amax);
  if (lane == 0) amax_of[warp] = amax;
  const bool there = page >= 0 && page < a.num_pages;
  if (!there && speaks) record_error(a.err, ERR_PAGE);
  const bool stores = there && mine;
  float* scale_at = nullptr;
  float old = 0.f;
  if (stores) {
    const int64_t* ss = key ? a.ks_st : a.vs_st;
    scale_at = (key ? a.k_scale : a.v_scale) + (int64_t)page * ss[0] + (int64_t)(in_page >> block_shift) * ss[1] + (int64_t)h * ss[2];
    if (kept > 0) old = *scale_at;
  }
  __syncthreads();
  for (int w = group << (per_shift - 5); w < (group + 1) << (per_shift - 5); ++w) amax = max(amax, amax_of[w]);
  if (stores) {
    const int64_t* st = key ? a.kc_st : a.vc_st;
    uint8_t* rows = reinterpret_cast<uint8_t*>(key ? a.k_cache : a.v_cache) + (int64_t)page * st[0] + (int64_t)in_page * st[1] +
                    (int64_t)h * st[2];
    float now = scale_for(__uint_as_float(amax)), ratio = 1.f;
    if (kept > 0) {
      old = scale_or_least(old);
      now = fmaxf(now, power_above(old));
      ratio = old / now;
    }
    const float inv = 1.f / now;  // exact
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int r = row_of(i);
      if (r >= last) continue;
      uint2* d0 = reinterpret_cast<uint2*>(rows + (int64_t)r * st[1] + un.o0);
      uint2* d1 = reinterpret_cast<uint2*>(rows + (int64_t)r * st[1] + un.o1);
      if (r < kept) {
        if (ratio == 1.f) continue;
        uint2 y0 = *d0, y1 = *d1;
        y0.x = e4m3_scaled(y0.x, ratio), y0.y = e4m3_scaled(y0.y, ratio);
        y1.x = e4m3_scaled(y1.x, ratio), y1.y = e4m3_scaled(y1.y, ratio);
        *d0 = y0, *d1 = y1;
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[i][e] *= inv;
        *d0 = make_uint2(e4m3_four(x[i]), e4m3_four(x[i] + 4));
        *d1 = make_uint2(e4m3_four(x[i] + 8), e4m3_four(x[i] + 12));
      }
    }
    if (at == 0) *scale_at = now;
  }
  pdl_trigger();
}

namespace {

template <typename T, bool kVec>
const void* append8_fn(int items) {
  return items == 1 ? (const void*)append8_kernel<T, kVec, 1> : items == 2 ? (const void*)append8_kernel<T, kVec, 2>
                                                                            : (const void*)append8_kernel<T, kVec, 4>;
}

}  // namespace

int launch_append8(Append8Args a, cudaStream_t stream) {
  const int units = a.block * (a.D / 16);  // 16-element units of a block and head: 64 to 1024
  const int items = units <= kAT ? 1 : units / kAT, heads = units <= kAT ? kAT / units : 1;
  a.kv_units = a.Hk ? a.T / a.block + 2 * a.B : 0;
  a.head_parts = (2 * a.Hk + heads - 1) / heads;
  // Few tokens: a token's query heads spread over CTAs; many: a CTA keeps its cosines and sines over them.
  const int rows = kAT / (a.D / 16), spread = (a.Hq + rows - 1) / rows, want = 4 * num_sms();
  a.q_parts = (want + a.T - 1) / a.T;
  a.q_parts = a.q_parts < 1 ? 1 : a.q_parts > spread ? spread : a.q_parts;
  const int tokens = a.T < 8192 ? a.T : 8192;
  a.q_ctas = a.Hq ? tokens * a.q_parts : 0;
  const void* k = a.f16 ? (a.vectors ? append8_fn<__half, true>(items) : append8_fn<__half, false>(items))
                        : (a.vectors ? append8_fn<__nv_bfloat16, true>(items) : append8_fn<__nv_bfloat16, false>(items));
  return launch_with_pdl(k, a, a.kv_units * a.head_parts + a.q_ctas, kAT, 0, a.pdl, stream);
}

}  // namespace fnx
