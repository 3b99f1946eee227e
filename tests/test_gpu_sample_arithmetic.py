"""Arithmetic that sampling and token probabilities take for granted (csrc/sample.cuh), bit for bit, on 2^28 pairs: the
quotient from a reciprocal in two parts gives the weights that the division gives, since one launch uses the first and the
lists and the next launch the second; a weight's parts, split by rounded additions, are those of the shifted significand."""

import ctypes
import subprocess

import pytest
import torch

pytestmark = pytest.mark.gpu

SOURCE = r"""
#include "sample.cuh"

using namespace fnx;

constexpr int kCheck = 256;

__global__ void check(unsigned long long seed, long long pairs, unsigned long long* bad) {
  __shared__ Bins h;
  const int b = threadIdx.x;
  const uint32_t w0 = smem_u32(h.w0) + b * 4;
  for (long long i = blockIdx.x * (long long)kCheck + b; i < pairs; i += (long long)gridDim.x * kCheck) {
    unsigned long long z = (i + seed) * 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull, z = (z ^ (z >> 27)) * 0x94D049BB133111EBull, z ^= z >> 31;
    unsigned long long y = (z + seed) * 0xD1342543DE82EF95ull;
    y = (y ^ (y >> 29)) * 0x94D049BB133111EBull, y ^= y >> 32;
    // T in [2^-60, 2^60): significands anywhere, near 1 and near 2; exponents anywhere, and the two ends
    unsigned te = 67 + (unsigned)(z & 0xFF) % 120, tm = (unsigned)(z >> 8) & 0x7FFFFFu;
    const unsigned kind = (unsigned)(z >> 61);
    if (kind == 0) tm |= 0x7FFF00u;
    if (kind == 1) tm &= 0xFFu;
    if (kind == 2) te = z >> 60 & 1 ? 67 : 186;
    float T = __uint_as_float(te << 23 | tm);
    if (kind == 3) T = z >> 60 & 1 ? 0x1p-60f : 0x1p60f;
    // x - m from 2^-27 T to beyond the clip at -28 T, and next to it
    float d = __uint_as_float((min(254u, te + 5u) - (unsigned)(y & 31)) << 23 | ((unsigned)(y >> 8) & 0x7FFFFFu));
    const unsigned near = (unsigned)(y >> 61);
    if (near == 0) d = __uint_as_float(__float_as_uint(28.0f * T) + (int)(y >> 8 & 15) - 8);
    const float m = near == 1 ? 3.0f * T : near == 2 ? -7.5f * T : near == 3 ? d : 0.0f;
    const float x = near == 4 ? __uint_as_float(__float_as_uint(m)) : near == 5 ? NAN : m - d;
    const Scale sc{m, T, 0.0f, 0.0f, 0.0f};
    if (!sc.plain()) atomicAdd(bad + 2, 1ull);
    const float quick = expf(sc.quotient(x, sc.reciprocal())), slow = x == x ? sc.share(x) : 0.0f;
    if (Scale::weight(quick) != Scale::weight(slow)) atomicAdd(bad, 1ull);
    if (x - m >= -28.0f * T && __float_as_uint(quick) != __float_as_uint(slow)) atomicAdd(bad, 1ull);
    h.w0[b] = h.w1[b] = h.w2[b] = 0u;
    // weights as they come, and of all sizes
    const float e = z >> 40 & 1 ? quick : __uint_as_float((127u - (unsigned)(y >> 40) % 45u) << 23 | (unsigned)(y >> 8 & 0x7FFFFFu));
    add_share(w0, fminf(e, 1.0f));
    if (sum_of(h, b) != Scale::weight(fminf(e, 1.0f))) atomicAdd(bad + 1, 1ull);
  }
}

extern "C" int run(unsigned long long seed, long long pairs, unsigned long long* bad) {
  check<<<1184, kCheck>>>(seed, pairs, bad);
  return cudaDeviceSynchronize();
}
"""


def test_quotients_and_parts_of_weights(tmp_path):
    from flash_next_rtxpro6000_b200 import build

    (tmp_path / "check.cu").write_text(SOURCE)
    made = subprocess.run([build.nvcc(), *build.ARCH, *build.FLAGS, "-I" + str(build.CSRC), "-shared", "-cudart", "static",
                           str(tmp_path / "check.cu"), "-o", str(tmp_path / "check.so")], capture_output=True, text=True)
    assert made.returncode == 0, made.stderr
    lib = ctypes.CDLL(str(tmp_path / "check.so"))
    bad = torch.zeros(3, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    lib.run.argtypes = [ctypes.c_ulonglong, ctypes.c_longlong, ctypes.c_void_p]
    assert lib.run(20260, 2**28, bad.data_ptr()) == 0
    assert bad.tolist() == [0, 0, 0]
