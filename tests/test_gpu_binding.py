"""The native binding of the verify-step operators as a Python extension: errors of its arguments'
conversion, and other threads during its calls."""

import pytest
import torch

from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def _fx():
    import flash_next_rtxpro6000_b200 as fx

    return fx


class Untold:
    def __bool__(self):
        raise KeyError("neither")


def test_an_argument_whose_truth_raises_stops_the_call():
    fx, d = _fx(), dev()
    q = torch.ones(1, 2, 64, dtype=torch.bfloat16, device=d)
    kc, vc = (torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16, device=d) for _ in range(2))
    i = torch.zeros(1, dtype=torch.int64, device=d)
    table = fx.rotary_table(10, 64, device=d)
    with pytest.raises(KeyError):
        fx.rotary_append(q, q, q, i, i, table, kc, vc, interleaved=Untold())
    with pytest.raises(RuntimeError):  # a tensor of two truths
        fx.rotary_append(q, q, q, i, i, table, kc, vc, interleaved=torch.ones(2))
    assert not bool(kc.any()) and not bool(vc.any())
    fx.rotary_append(q, q, q, i, i, table, kc, vc, interleaved=1)
    assert bool(vc.any())
