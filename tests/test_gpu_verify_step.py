"""The verify-step operators together (examples/verify_step.py): accepted tokens are those that decoding
one token at a time gives with the same random numbers, and a captured step follows new trees and lengths."""

import importlib.util
import os

import pytest
import torch

from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def _example():
    path = os.path.join(os.path.dirname(os.path.dirname(__file__)), "examples", "verify_step.py")
    spec = importlib.util.spec_from_file_location("verify_step", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_example_runs():
    assert len(_example().main(["--steps", "3", "--context", "300", "--nodes", "6"])) >= 3


@pytest.mark.parametrize("nodes", [5, 16])
def test_a_tree_gives_what_single_tokens_give(nodes):
    """Every node's logits equal those of a chain that holds only its ancestors, up to the order of sums:
    the same cache, the node's path appended token by token."""
    m = _example()
    step = m.VerifyStep(200, nodes, vocab=4096, room=64, device=dev())
    g = torch.Generator().manual_seed(nodes)
    parents = step.draft(11, g)
    before = [c.clone() for c in (step.k_cache, step.v_cache)]
    step.run()
    tree = step.logits.float().clone()
    tokens = step.tokens.tolist()
    for i in range(nodes):
        path = [i]
        while parents[path[-1]] >= 0:
            path.append(parents[path[-1]])
        path.reverse()
        step.k_cache.copy_(before[0])
        step.v_cache.copy_(before[1])
        one = m.VerifyStep.__new__(m.VerifyStep)
        one.__dict__.update(step.__dict__)
        one.nodes = 1
        one.offsets = torch.tensor([0, 1], dtype=torch.int32, device=dev())
        one.parents = torch.tensor([-1], dtype=torch.int32, device=dev())
        one.temperature, one.top_k, one.top_p = (x[:1] for x in (step.temperature, step.top_k, step.top_p))
        one.uniforms = step.uniforms[i:i + 1]
        for depth, node in enumerate(path):
            one.context = torch.tensor([200 + depth], dtype=torch.int32, device=dev())
            one.tokens = torch.tensor([tokens[node]], device=dev())
            one.run()
        # bf16 logits of a few hundred sums in another order: two roundings of the hidden row and one here
        scale = float(tree[i].abs().max())
        assert float((one.logits[0].float() - tree[i]).abs().max()) <= 3 * 2.0**-8 * scale


def test_accept_moves_the_path_behind_the_context():
    m = _example()
    step = m.VerifyStep(130, 6, vocab=4096, room=64, device=dev())
    step.parents.copy_(torch.tensor([-1, 0, 0, 2, 2, 4], dtype=torch.int32))
    step.tokens.copy_(torch.tensor([9, 1, 2, 3, 4, 5]))
    step.run()
    step.sampled = torch.tensor([2, 0, 4, 0, 5, 77], device=dev())
    keys = step.k_cache.view(-1, step.kv_heads, step.dim)[step.slots].clone()
    accepted, last = step.accept()
    assert accepted == [2, 4, 5] and last == 77 and int(step.context) == 134
    now = step.k_cache.view(-1, step.kv_heads, step.dim)[step.slots]
    assert torch.equal(now[:4], keys[[0, 2, 4, 5]])
