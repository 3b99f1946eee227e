"""tree_attention8 where a CTA's segments alternate between two row tiles and one (more and fewer than 128 query rows a kv
head), with scales that differ from group to group: against 64 bits, and bit for bit over repeated calls.

Tolerance: test_gpu_cache8's, (2^-11 + 2^-12 + 2^-17) of the weighted mean of |v|, half a step of the result and 2^-25, and
what it leaves out, since a key's scale of up to 2 makes rows here lie on few keys: weights w = p s (of the softmax's p and
the value's scale) below 2^-14 are rounded to fp16 by 2^-25 at most, or by all of themselves, in a unit in which the largest
w of the row so far is 2^7 at least (its reference lies 7 bits below the running maximum or lower).  So each key adds
min(w, 2^-32 of the largest w) |v8| / sum p = min(p, 2^-32 max(w) / s) |v| / sum p."""

import pytest
import torch

from tests.gpu_util import dev
from tests.test_gpu_cache8 import UNIT, Attention

pytestmark = pytest.mark.gpu


def _lost(case):
    """The bound of what small weights lose, for each row and element."""
    N, Hq, D = case.q.shape
    G, n = Hq // case.c[0].shape[2], 0
    lost = torch.zeros(N, Hq, D, dtype=torch.float64, device=dev())
    for b, (c, t) in enumerate(zip(case.lens, case.counts)):
        keys, vals = (case.cached(i, b, c + t).repeat_interleave(G, 1) for i in (0, 1))
        p = torch.arange(c + t, device=dev())
        page, at = case.table[b].long()[p // case.page], p % case.page
        scale = case.s[1][page, at // case.block].double().repeat_interleave(G, 1).T
        for i in range(t):
            see = torch.tensor([True] * c + [bool(case.masks[n] >> j & 1) for j in range(t)], device=dev())
            s = torch.einsum("hd,khd->hk", case.q[n].double(), keys) * D**-0.5
            share = torch.softmax(s.masked_fill(~see, -float("inf")), 1)
            least = 2.0**-32 * (share * scale).amax(1, keepdim=True) / scale
            lost[n] = torch.einsum("hk,khd->hd", torch.minimum(share, least), vals.abs())
            n += 1
    return lost


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (64, torch.float16), (128, torch.bfloat16), (128, torch.float16),
                                     (256, torch.bfloat16)])
@pytest.mark.parametrize("lens,counts,Hq,Hk", [
    ([500 + 37 * b for b in range(24)], [60, 3, 60, 2, 33, 1] * 4, 16, 4),   # wide and narrow requests in turn
    ([700 + 11 * b for b in range(8)], [33, 64, 40, 34] * 2, 32, 4),          # 264 to 512 rows: the last row tile is narrow
    ([129, 64, 1000, 63] * 8, [64, 1, 40, 5] * 8, 12, 3),                     # one to three tiles a segment
])
def test_segments_of_one_and_two_row_tiles(lens, counts, Hq, Hk, D, dtype):
    case = Attention(lens, counts, Hq, Hk, D, 32, 16, dtype, seed=D, vary=6)
    out, lse = case.run()
    for _ in range(20):
        a, b = case.run()
        assert torch.equal(a, out) and torch.equal(b, lse)
    want, mean, wlse, big = case.reference()
    err = (out.double() - want).abs()
    tol = (2.0**-11 + 2.0**-12 + 2.0**-17) * mean + UNIT[dtype] * want.abs() + 2.0**-25 + _lost(case)
    assert bool((err <= tol).all()), float((err - tol).max())
    assert bool(((lse.double() - wlse).abs() <= 2.0**-12 * big).all())
