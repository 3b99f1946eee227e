"""Rotary positions and the paged-cache append of a decode, verify or prompt step.

* ``rotary_table(positions, rotated, base, scaling)`` -- the cosines and sines, built once;
* ``rotary_append(q, k, v, positions, slots, table, k_cache, v_cache)`` -- rotates queries and
  keys and stores keys and values in their cache slots, in one launch (csrc/rotary.cu).

No counterpart in the reference's operator modules, whose server does these steps elsewhere.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from ._lib import check, ptr
from .w8a16_gemv import PDL, _stream, _workspace

_TYPES = {torch.bfloat16: _lib.T_BF16, torch.float16: _lib.T_F16}


@dataclass(frozen=True)
class RotaryScaling:
    """Frequencies for contexts ``factor`` times the ``original`` training length.

    ``linear``: every frequency divided by ``factor``.  ``ramp``: pairs that turn fewer than
    ``slow`` times over the original length are divided, those that turn more than ``fast``
    times are kept, with a linear ramp in the number of turns between; cosines and sines are
    multiplied by ``attention`` (default 0.1 ln(factor) + 1)."""

    factor: float
    kind: str = "ramp"
    original: int = 32768
    slow: float = 1.0
    fast: float = 32.0
    attention: Optional[float] = None

    def __post_init__(self):
        if self.kind not in ("linear", "ramp"):
            raise ValueError(f"scaling kind must be 'linear' or 'ramp', got {self.kind!r}")
        if not self.factor >= 1.0:
            raise ValueError(f"scaling factor must be at least 1, got {self.factor}")
        if self.kind == "ramp" and not (self.original > 0 and 0 <= self.slow < self.fast):
            raise ValueError("a ramp needs original > 0 and 0 <= slow < fast")


def rotary_table(positions: int, rotated: int, base: float = 10000.0,
                 scaling: Optional[RotaryScaling] = None, device="cuda") -> torch.Tensor:
    """fp32 [positions, rotated]: rotated / 2 cosines, then rotated / 2 sines, of position *
    frequency; angles are computed in 64 bits, so far positions lose nothing."""
    if positions < 1 or rotated < 2 or rotated % 2:
        raise ValueError(f"need positions >= 1 and an even rotated >= 2, got {positions}, {rotated}")
    if not base > 1.0:
        raise ValueError(f"base must be larger than 1, got {base}")
    half = rotated // 2
    freq = base ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
    gain = 1.0
    if scaling is not None and scaling.kind == "linear":
        freq = freq / scaling.factor
        gain = 1.0 if scaling.attention is None else scaling.attention
    elif scaling is not None:
        turns = scaling.original * freq / (2 * math.pi)
        keep = ((turns - scaling.slow) / (scaling.fast - scaling.slow)).clamp(0, 1)
        freq = freq * keep + freq / scaling.factor * (1 - keep)
        gain = 0.1 * math.log(scaling.factor) + 1.0 if scaling.attention is None else scaling.attention
    table = torch.empty((positions, rotated), dtype=torch.float32, device=device)
    step = 1 << 16  # bounds the 64-bit intermediates
    for p in range(0, positions, step):
        angle = torch.arange(p, min(p + step, positions), dtype=torch.float64, device=device)[:, None] * freq
        table[p:p + step, :half] = angle.cos() * gain
        table[p:p + step, half:] = angle.sin() * gain
    return table


def cache_args(k_cache: torch.Tensor, v_cache: torch.Tensor):
    """Checks a paged cache pair ([pages, page_size, kv_heads, dim], elements of a head contiguous)
    and returns its strides in C form."""
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError("k_cache and v_cache must be [pages, page_size, kv_heads, dim] of one shape; got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    if v_cache.dtype != k_cache.dtype:
        raise ValueError("k_cache and v_cache must have one type")
    ks, vs = k_cache.stride(), v_cache.stride()
    if (ks[3] != 1 or vs[3] != 1) and k_cache.shape[3] > 1:
        raise ValueError("the elements of a cached head must be contiguous")
    return (ctypes.c_int64 * 3)(*ks[:3]), (ctypes.c_int64 * 3)(*vs[:3])


def _heads(t: torch.Tensor, name: str, tokens: int, dim: int, like: torch.Tensor):
    if t.dim() != 3 or t.shape[0] != tokens or t.shape[2] != dim:
        raise ValueError(f"{name} must be [{tokens}, heads, {dim}], got {tuple(t.shape)}")
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
    if t.stride(2) != 1 and dim > 1:
        raise ValueError(f"the elements of a head of {name} must be contiguous")


def _index(t: torch.Tensor, name: str, count: int, dtype: torch.dtype, device) -> None:
    if t.dtype != dtype or t.device != device or t.dim() != 1 or t.shape[0] != count or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} [{count}] tensor on {device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")


def rotary_append(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    positions: torch.Tensor,
    slots: torch.Tensor,
    table: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    interleaved: bool = False,
    out: Optional[torch.Tensor] = None,
    pdl: Optional[bool] = None,
) -> torch.Tensor:
    """q [T, q_heads, dim], k and v [T, kv_heads, dim], bf16 or fp16 (views of one projection's rows
    are fine); positions and slots int64 [T]; table fp32 [P, rotated] from ``rotary_table``; caches
    [pages, page_size, kv_heads, dim] of q's type.

    Rotates the first ``rotated`` elements of each query and key head -- pairs (i, i + rotated/2), or
    (2i, 2i + 1) when ``interleaved`` -- and returns the queries (in ``out``, which may be q).  Rotated
    keys and values are stored at slot = page * page_size + place, or nowhere for slot -1; no two
    tokens may have the same slot.  Positions outside the table and slots outside the cache are
    reported by ``check_device_errors``."""
    if q.dim() != 3:
        raise ValueError(f"q must be [tokens, heads, dim], got {tuple(q.shape)}")
    if q.dtype not in _TYPES:
        raise NotImplementedError(f"rotary_append: bf16 or fp16, got {q.dtype}")
    if not q.is_cuda:
        raise ValueError("rotary_append needs CUDA tensors")
    T, Hq, D = q.shape
    dev = q.device
    _heads(q, "q", T, D, q)
    _heads(k, "k", T, D, q)
    _heads(v, "v", T, D, q)
    Hk = k.shape[1]
    if v.shape[1] != Hk:
        raise ValueError(f"k and v must have one number of heads, got {Hk} and {v.shape[1]}")
    _index(positions, "positions", T, torch.int64, dev)
    _index(slots, "slots", T, torch.int64, dev)
    if table.dim() != 2 or table.dtype != torch.float32 or table.device != dev or table.stride(1) != 1:
        raise ValueError(f"table must be a row-contiguous fp32 [positions, rotated] tensor on {dev}")
    if table.shape[1] > D or table.shape[1] % 2:
        raise ValueError(f"the table's {table.shape[1]} columns must be even and at most dim = {D}")
    ks, vs = cache_args(k_cache, v_cache)
    if tuple(k_cache.shape[2:]) != (Hk, D) or k_cache.dtype != q.dtype or k_cache.device != dev or \
            v_cache.device != dev:
        raise ValueError(f"caches must be [pages, page_size, {Hk}, {D}] {q.dtype} tensors on {dev}")
    if out is None:
        out = torch.empty((T, Hq, D), dtype=q.dtype, device=dev)
    else:
        _heads(out, "out", T, D, q)
        if out.shape[1] != Hq:
            raise ValueError(f"out must have q's {Hq} heads")
    rc = _lib.lib().fnx_rotary_append(
        ptr(q), q.stride(0), q.stride(1), ptr(k), k.stride(0), k.stride(1), ptr(v), v.stride(0), v.stride(1),
        ptr(out), out.stride(0), out.stride(1), ptr(positions), ptr(slots), ptr(table), table.stride(0),
        table.shape[0], ptr(k_cache), ks, ptr(v_cache), vs, k_cache.shape[0], k_cache.shape[1], T, Hq, Hk, D,
        table.shape[1], int(bool(interleaved)), _TYPES[q.dtype], ptr(_workspace(dev).error_flag),
        int(PDL if pdl is None else pdl), _stream(q))
    check(rc, "rotary_append")
    return out
