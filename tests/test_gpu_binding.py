"""The native binding of the verify-step operators as a Python extension: errors of its arguments'
conversion, and other threads during its calls."""

import threading
import time

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


def _calls():
    fx, d = _fx(), dev()
    q = torch.ones(1, 2, 64, dtype=torch.bfloat16, device=d)
    kc, vc = (torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16, device=d) for _ in range(2))
    i = torch.zeros(1, dtype=torch.int64, device=d)
    rot = fx.rotary_table(10, 64, device=d)
    i32 = dict(dtype=torch.int32, device=d)
    pages, ctx, off = torch.tensor([[0, 1]], **i32), torch.tensor([3], **i32), torch.tensor([0, 1], **i32)
    parents = torch.tensor([-1], **i32)
    logits, u = torch.zeros(1, 8, device=d), torch.zeros(1, device=d)
    return dict(
        rotary_append=lambda: fx.rotary_append(q, q, q, i, i, rot, kc, vc),
        tree_layout=lambda: fx.tree_layout(parents, off, ctx, pages, 4, 2),
        tree_attention=lambda: fx.tree_attention(q, kc, vc, pages, ctx, off, max_nodes=1),
        sample_tokens=lambda: fx.sample_tokens(logits, u))


@pytest.mark.parametrize("name", ["rotary_append", "tree_layout", "tree_attention", "sample_tokens"])
def test_other_threads_run_while_a_call_waits(name):
    """Behind a kernel of about a second the launch queue fills up, and the call that finds it full waits; another
    thread's clock goes on ticking meanwhile."""
    call = _calls()[name]
    call()
    torch.cuda.synchronize()
    done, gaps = threading.Event(), []

    def tick():
        last = time.perf_counter()
        while not done.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            gaps.append(now - last)
            last = now

    ticker = threading.Thread(target=tick)
    ticker.start()
    torch.cuda._sleep(2_000_000_000)
    start = time.perf_counter()
    for _ in range(3000):
        call()
    waited = time.perf_counter() - start
    done.set()
    ticker.join()
    torch.cuda.synchronize()
    assert waited > 0.5  # the queue was full
    assert max(gaps) < 0.3
