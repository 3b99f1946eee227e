// The probabilities that sampling draws from: which tokens of a row are kept (sample.cuh), then all of its probabilities.
#include "sample.cuh"

namespace fnx {

// The probabilities of a row's tokens: a token's weight over that of all that are kept, 0 for the others.  One read of
// the logits and one write of the probabilities, eight tokens a thread (kVec: in 16-byte vectors).  A launch of its own:
// written by the clusters that find the kept tokens, 128 rows of 248,320 took 240 us, and 184 so, since those have
// few threads and many registers.
namespace {

constexpr int kPT = 256;  // threads

}  // namespace

template <typename T, bool kVec>
__global__ void __launch_bounds__(kPT) token_probs_kernel(const __grid_constant__ SampleArgs a) {
  constexpr int kEach = 8;
  const int row = blockIdx.y, v = (blockIdx.x * kPT + threadIdx.x) * kEach;
  const T* from = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.ldl + v;
  float x[kEach];
  if (v < a.V) {  // given before the launch ahead of this one
    if (kVec) {
      constexpr int kPer = 16 / sizeof(T);
#pragma unroll
      for (int i = 0; i < kEach / kPer; ++i) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4*>(from) + i);
        const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int q = 0; q < kPer; ++q) x[i * kPer + q] = logit(e[q]);
      }
    } else {
#pragma unroll
      for (int q = 0; q < kEach; ++q) x[q] = v + q < a.V ? logit(from[q]) : -INFINITY;
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (v >= a.V) return;
  const KeptTokens k = a.rows[row];
  const Scale sc{k.m, k.T, 0.f, 0.f, 0.f};
  // a weight is e with the bits below 2^-40 taken off; 2^40 over the weight of all, in two parts
  const double by = (double)kOne / (double)k.kept;
  const float hi = (float)by, lo = (float)(by - (double)hi);
  float p[kEach];
#pragma unroll
  for (int q = 0; q < kEach; ++q) {
    bool in;
    if (k.what == KEPT_PREFIX) in = x[q] > k.low || (x[q] == k.low && v + q <= k.last);
    else in = v + q == k.last;
    if (!in) {
      p[q] = 0.f;
    } else if (k.what == KEPT_ONE) {
      p[q] = 1.f;
    } else {
      float e = sc.share(x[q]);
      const int below = (127 + 23 - 40) - (int)(__float_as_uint(e) >> 23);
      if (below > 0) e = below > 23 ? 0.f : __uint_as_float(__float_as_uint(e) & (0xFFFFFFFFu << below));
      p[q] = fmaf(e, hi, e * lo);
    }
  }
  float* to = a.all + (int64_t)row * a.ld_all + v;
  if (kVec) {
    __stcs(reinterpret_cast<float4*>(to), make_float4(p[0], p[1], p[2], p[3]));
    __stcs(reinterpret_cast<float4*>(to) + 1, make_float4(p[4], p[5], p[6], p[7]));
  } else {
#pragma unroll
    for (int q = 0; q < kEach; ++q)
      if (v + q < a.V) to[q] = p[q];
  }
}

namespace {

template <typename T>
const void* probs_fn(bool vec) {
  return vec ? (const void*)token_probs_kernel<T, true> : (const void*)token_probs_kernel<T, false>;
}

}  // namespace

const void* probs_fn_one(int type) { return sample_fn<false, true>(type); }

int launch_token_probs(SampleArgs a, cudaStream_t stream) {
  if (const int rc = launch_rows<true>(a, stream)) return rc;
  const int size = a.type == LOGITS_F32 ? 4 : 2, per = 16 / size;
  const bool vec = a.V % 8 == 0 && a.ldl % per == 0 && a.ld_all % 4 == 0 && reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(a.all) % 16 == 0;
  const void* k = a.type == LOGITS_F32 ? probs_fn<float>(vec) : a.type == LOGITS_F16 ? probs_fn<__half>(vec) : probs_fn<__nv_bfloat16>(vec);
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kPT);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int rows = a.M;
  for (int m = 0; m < rows; m += 32768) {  // rows of one launch
    cfg.gridDim = dim3((a.V + kPT * 8 - 1) / (kPT * 8), rows - m < 32768 ? rows - m : 32768);
    SampleArgs part = a;
    part.logits = static_cast<const char*>(a.logits) + (int64_t)m * a.ldl * size;
    part.all = a.all + (int64_t)m * a.ld_all;
    part.rows = a.rows + m;
    void* params[1] = {&part};
    if (cudaLaunchKernelExC(&cfg, k, params) != cudaSuccess) return 2;
  }
  return 0;
}

}  // namespace fnx
