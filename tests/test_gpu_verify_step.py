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


class _Step:
    """layout -> rotation and append -> attention -> GEMV -> sampling, back to back, on a batch."""

    def __init__(self, lens, counts, Hq, Hk, D, max_context):
        import flash_next_rtxpro6000_b200 as fx

        self.fx, d, page = fx, dev(), 16
        g = torch.Generator().manual_seed(len(lens) + D)
        rand = lambda *s: torch.randn(*s, generator=g).bfloat16().to(d)  # noqa: E731
        i32 = dict(dtype=torch.int32, device=d)
        need = [-(-(c + t) // page) for c, t in zip(lens, counts)]
        self.pages, self.page, N = sum(need), page, sum(counts)
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            self.table[b, :n] = order[sum(need[:b]):sum(need[:b]) + n]
        self.table = self.table.to(d)
        self.ctx = torch.tensor(lens, **i32)
        self.offsets = torch.tensor([sum(counts[:b]) for b in range(len(lens) + 1)], **i32)
        self.parents = torch.tensor([i - 1 for t in counts for i in range(t)], **i32)
        self.q, self.k, self.v = rand(N, Hq, D), rand(N, Hk, D), rand(N, Hk, D)
        self.kc, self.vc = rand(self.pages, page, Hk, D), rand(self.pages, page, Hk, D)
        self.rot = fx.rotary_table(max(lens) + max(counts) + 1, D, device=d)
        self.w = torch.randint(-127, 128, (1024, Hq * D), generator=g).to(torch.int8).to(d)
        self.scale = (torch.rand(1024, generator=g) * 0.003).bfloat16().to(d)
        self.u = torch.rand(N, generator=g).to(d)
        self.top_k = (torch.arange(N, device=d) % 3 * 20).int()
        self.max_nodes, self.max_context = max(counts), max_context
        fx.prealloc(d, attention=True)

    def run(self, pdl):
        fx = self.fx
        mask, pos, slots = fx.tree_layout(self.parents, self.offsets, self.ctx, self.table, self.page, self.pages, pdl=pdl)
        q = fx.rotary_append(self.q, self.k, self.v, pos, slots, self.rot, self.kc, self.vc, pdl=pdl)
        out, lse = fx.tree_attention(q, self.kc, self.vc, self.table, self.ctx, self.offsets, mask,
                                     max_nodes=self.max_nodes, max_context=self.max_context, pdl=pdl)
        logits = torch.cat([fx.w8a16_gemv(x, self.w, self.scale, pdl=pdl) for x in out.flatten(1).split(16)])
        tokens, probs = fx.sample_tokens(logits, self.u, top_k=self.top_k, pdl=pdl)
        return mask, pos, slots, q, out, lse, logits, tokens, probs


@pytest.mark.parametrize("lens,counts,Hq,Hk,D,max_context", [
    ([30, 0, 17], [5, 1, 8], 4, 2, 64, 56),                     # one key tile: no joining launch
    ([1000], [16], 8, 2, 128, 1000),                            # mma.sync, partials joined
    ([300, 9, 2000], [3, 1, 4], 4, 1, 256, 2000),
    ([6000, 100, 5000, 64] * 3, [4, 1, 9, 16] * 3, 16, 4, 128, 6000),  # tensor memory
    ([700, 20] * 70, [2, 1] * 70, 4, 2, 64, 700),               # two launches over one scratch, split items
])
def test_early_launches_change_nothing(lens, counts, Hq, Hk, D, max_context):
    """Every operator launched before the one ahead of it has finished (pdl): the same bits, several steps in a
    row, as they come and captured."""
    s = _Step(lens, counts, Hq, Hk, D, max_context)
    want = [x.clone() for x in s.run(False)]
    caches = [c.clone() for c in (s.kc, s.vc)]

    def same(got):
        torch.cuda.synchronize()
        s.fx.check_device_errors()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(s.kc, caches[0]) and torch.equal(s.vc, caches[1])

    steps = [s.run(True) for _ in range(5)]
    for got in steps:
        same(got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps = [s.run(True) for _ in range(3)]
    for _ in range(3):
        for got in steps:
            for x in got:
                x.zero_()
        graph.replay()
        for got in steps:
            same(got)
