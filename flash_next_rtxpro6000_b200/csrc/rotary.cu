// Rotary positions on queries and keys, with keys and values stored in a paged cache:
//
//   y[a] = x[a] cos - x[b] sin,  y[b] = x[b] cos + x[a] sin     for the pairs (a, b) of a head,
//
// (i, i + R/2) in the half layout and (2i, 2i + 1) interleaved, over the first R of D elements;
// the others pass through.  cos and sin come from row positions[t] of an fp32 table [P, R]
// (R/2 cosines, then R/2 sines); products and sums are in fp32 and rounded once.
//
// Bound: memory (each element is read once and written once), or the launch for a few tokens.
// A unit is 16 elements of a head: two 16-byte vectors that hold eight whole pairs in either
// layout, so a unit needs nothing of its neighbours and q may be rotated in place.  A block is
// D/16 units wide; its rows walk the token's heads, so a thread's cosines and sines stay in
// registers over all the heads it turns.  Measured (B200, calls in a graph): 2.3 us for one token of 16 + 2 heads
// of 256 and for 16 of 32 + 8 heads of 128, 21.8 us for 4,097 tokens of 32 + 8 heads of 128 (102 MB, 4.7 TB/s).
#include "fnx_common.cuh"
#include "fnx_kernels.h"

namespace fnx {

namespace {

template <typename T> struct Pair2;
template <> struct Pair2<__nv_bfloat16> {
  using P = __nv_bfloat162;
  static __device__ __forceinline__ float2 get(uint32_t u) { return __bfloat1622float2(*reinterpret_cast<P*>(&u)); }
  static __device__ __forceinline__ uint32_t put(float a, float b) {
    const P p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
  static __device__ __forceinline__ float one(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Pair2<__half> {
  using P = __half2;
  static __device__ __forceinline__ float2 get(uint32_t u) { return __half22float2(*reinterpret_cast<P*>(&u)); }
  static __device__ __forceinline__ uint32_t put(float a, float b) {
    const P p = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
  static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half round(float v) { return __float2half_rn(v); }
};

// Head h of token t's row: queries, then keys, then values.
template <typename T>
struct HeadRow {
  const T* src;
  T* dst;  // nullptr: not stored
  bool turn;
};

template <typename T>
__device__ __forceinline__ HeadRow<T> head_row(const RotaryArgs& a, int t, int h, int64_t page, int64_t in_page) {
  HeadRow<T> r;
  if (h < a.Hq) {
    r.src = reinterpret_cast<const T*>(a.q) + (int64_t)t * a.q_st + (int64_t)h * a.q_sh;
    r.dst = reinterpret_cast<T*>(a.q_out) + (int64_t)t * a.o_st + (int64_t)h * a.o_sh;
    r.turn = true;
    return r;
  }
  h -= a.Hq;
  const bool key = h < a.Hk;
  if (!key) h -= a.Hk;
  r.src = reinterpret_cast<const T*>(key ? a.k : a.v) + (int64_t)t * (key ? a.k_st : a.v_st) +
          (int64_t)h * (key ? a.k_sh : a.v_sh);
  T* base = reinterpret_cast<T*>(key ? a.k_cache : a.v_cache);
  const int64_t* st = key ? a.kc_st : a.vc_st;
  r.dst = page < 0 ? nullptr : base + page * st[0] + in_page * st[1] + (int64_t)h * st[2];
  r.turn = key;
  return r;
}

// The token's table row and cache place; out-of-range ones are recorded, a bad position takes the
// nearest row and a bad slot is not stored.
__device__ __forceinline__ const float* token_place(const RotaryArgs& a, int t, bool report, int64_t& page,
                                                    int64_t& in_page) {
  int64_t pos = a.positions[t];
  if (pos < 0 || pos >= a.P) {
    if (report) record_error(a.err, ERR_POSITION);
    pos = pos < 0 ? 0 : a.P - 1;
  }
  const int64_t slot = a.slots[t];
  page = -1;
  in_page = 0;
  if (slot >= 0 && slot < a.n_slots) {
    page = slot / a.page_size;
    in_page = slot - page * a.page_size;
  } else if (slot != -1 && report) {
    record_error(a.err, ERR_SLOT);
  }
  return a.table + pos * a.table_ld;
}

// 16-byte vectors: D and R multiples of 16 (half of R is then a whole number of vectors), every
// pointer and stride 16-byte aligned.
template <typename T>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  const int u = threadIdx.x;  // unit of the head
  const int H = a.Hq + 2 * a.Hk;
  const int half = a.R / 2;
  const bool turned = 16 * u < a.R;
  pdl_wait();
  for (int t = blockIdx.y; t < a.T; t += gridDim.y) {
    int64_t page, in_page;
    const float* row = token_place(a, t, u == 0 && threadIdx.y == 0 && blockIdx.x == 0, page, in_page);
    float c[8], s[8];
    if (turned) {
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(row + 8 * u + i));
        const float4 y = __ldg(reinterpret_cast<const float4*>(row + half + 8 * u + i));
        c[i] = x.x, c[i + 1] = x.y, c[i + 2] = x.z, c[i + 3] = x.w;
        s[i] = y.x, s[i + 1] = y.y, s[i + 2] = y.z, s[i + 3] = y.w;
      }
    }
    const bool apart = turned && !a.interleaved;  // the pair's elements lie half apart
    const int o0 = apart ? 8 * u : 16 * u, o1 = apart ? half + 8 * u : 16 * u + 8;
    for (int h = blockIdx.x * blockDim.y + threadIdx.y; h < H; h += gridDim.x * blockDim.y) {
      const HeadRow<T> r = head_row<T>(a, t, h, page, in_page);
      if (!r.dst) continue;
      uint4 v0 = *reinterpret_cast<const uint4*>(r.src + o0);
      uint4 v1 = *reinterpret_cast<const uint4*>(r.src + o1);
      if (turned && r.turn) {
        uint32_t* w0 = reinterpret_cast<uint32_t*>(&v0);
        uint32_t* w1 = reinterpret_cast<uint32_t*>(&v1);
        if (apart) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 x = Pair2<T>::get(w0[i]), y = Pair2<T>::get(w1[i]);
            w0[i] = Pair2<T>::put(x.x * c[2 * i] - y.x * s[2 * i], x.y * c[2 * i + 1] - y.y * s[2 * i + 1]);
            w1[i] = Pair2<T>::put(y.x * c[2 * i] + x.x * s[2 * i], y.y * c[2 * i + 1] + x.y * s[2 * i + 1]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 x = Pair2<T>::get(w0[i]), y = Pair2<T>::get(w1[i]);
            w0[i] = Pair2<T>::put(x.x * c[i] - x.y * s[i], x.y * c[i] + x.x * s[i]);
            w1[i] = Pair2<T>::put(y.x * c[4 + i] - y.y * s[4 + i], y.y * c[4 + i] + y.x * s[4 + i]);
          }
        }
      }
      *reinterpret_cast<uint4*>(r.dst + o0) = v0;
      *reinterpret_cast<uint4*>(r.dst + o1) = v1;
    }
  }
  pdl_trigger();
}

// Any sizes and alignment: a unit is one pair, or one element past the rotated ones.
template <typename T>
__global__ void __launch_bounds__(256) rotary_any_kernel(const __grid_constant__ RotaryArgs a) {
  const int H = a.Hq + 2 * a.Hk;
  const int half = a.R / 2, units = half + (a.D - a.R);
  pdl_wait();
  for (int t = blockIdx.y; t < a.T; t += gridDim.y) {
    int64_t page, in_page;
    const float* row = token_place(a, t, threadIdx.x == 0 && threadIdx.y == 0 && blockIdx.x == 0, page, in_page);
    for (int h = blockIdx.x * blockDim.y + threadIdx.y; h < H; h += gridDim.x * blockDim.y) {
      const HeadRow<T> r = head_row<T>(a, t, h, page, in_page);
      if (!r.dst) continue;
      for (int u = threadIdx.x; u < units; u += blockDim.x) {
        if (u >= half) {
          r.dst[u + half] = r.src[u + half];
          continue;
        }
        const int i = a.interleaved ? 2 * u : u, j = a.interleaved ? 2 * u + 1 : u + half;
        const T vi = r.src[i], vj = r.src[j];
        if (r.turn) {
          const float x = Pair2<T>::one(vi), y = Pair2<T>::one(vj);
          const float c = __ldg(row + u), s = __ldg(row + half + u);
          r.dst[i] = Pair2<T>::round(x * c - y * s);
          r.dst[j] = Pair2<T>::round(y * c + x * s);
        } else {
          r.dst[i] = vi;
          r.dst[j] = vj;
        }
      }
    }
  }
  pdl_trigger();
}

}  // namespace

int launch_rotary(const RotaryArgs& a, cudaStream_t stream) {
  const int H = a.Hq + 2 * a.Hk;
  const bool vec = a.vectors != 0;
  const int wide = vec ? a.D / 16 : 32;
  const int rows = 256 / wide < 1 ? 1 : 256 / wide;
  // Few tokens: the heads of one token spread over blocks of one head per row; many tokens: a
  // block's rows walk the heads, which keeps a thread's cosines and sines in registers.
  const int spread = (H + rows - 1) / rows;
  const int want = 4 * num_sms();
  int gx = (want + a.T - 1) / a.T;
  gx = gx < 1 ? 1 : gx > spread ? spread : gx;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(gx, a.T < 65535 ? a.T : 65535);
  cfg.blockDim = dim3(wide, rows);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.pdl ? 1 : 0;
  void* params[1] = {const_cast<RotaryArgs*>(&a)};
  const void* k;
  if (a.f16) k = vec ? (const void*)rotary_kernel<__half> : (const void*)rotary_any_kernel<__half>;
  else k = vec ? (const void*)rotary_kernel<__nv_bfloat16> : (const void*)rotary_any_kernel<__nv_bfloat16>;
  return cudaLaunchKernelExC(&cfg, k, params) == cudaSuccess ? 0 : 2;
}

}  // namespace fnx
