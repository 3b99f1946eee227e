"""Rotary positions and the paged-cache append of a decode, verify or prompt step.

* ``rotary_table(positions, rotated, base, scaling)`` -- the cosines and sines, built once;
* ``rotary_append(q, k, v, positions, slots, table, k_cache, v_cache)`` -- rotates queries and
  keys and stores keys and values in their cache slots, in one launch (csrc/rotary.cu).

No counterpart in the reference's operator modules, whose server does these steps elsewhere.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .w8a16_gemv import PDL, _flag


@dataclass(frozen=True)
class RotaryScaling:
    """Frequencies for contexts ``factor`` times the ``original`` training length.

    ``linear``: every frequency divided by ``factor``.  ``ramp``: pairs that turn fewer than
    ``slow`` times over the original length are divided, those that turn more than ``fast``
    times are kept, with a linear ramp in the number of turns between; cosines and sines are
    multiplied by ``attention`` (default 0.1 ln(factor) + 1).

    Checkpoints differ in the ramp: some ramp linearly in the pair's index, between the two indices
    (often rounded to whole ones) at which a pair turns ``fast`` and ``slow`` times.  With the same two
    numbers the pairs between then turn at other rates (by up to 40 % at 64 rotated elements, base 1e6,
    factor 4).  For those make the fp32 table of cosines and sines with their own frequencies;
    ``rotary_append`` takes any table."""

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
        # polar, not cos and sin: on the host these go through a vector library that now and then (some 1 in
        # 30 processes) gave a thread's share at half the accuracy, 7e-9 off
        turn = torch.polar(torch.full((1,), gain, dtype=torch.float64, device=device), angle)
        table[p:p + step, :half] = turn.real
        table[p:p + step, half:] = turn.imag
    return table


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
    return _lib.ops().rotary_append(q, k, v, positions, slots, table, k_cache, v_cache, interleaved, out,
                                    _flag(q), PDL if pdl is None else pdl)
