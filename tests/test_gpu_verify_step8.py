"""A verify step over an 8-bit cache, its operators one after the other on a batch: tree layout, rotation with the
8-bit append, attention, lm_head, probabilities, verification, compaction.  Launched early (pdl) and captured they give
the bits that they give alone; the cache and lengths they leave are those of the accepted tokens; and a few steps of
decoding with drafts from the model itself accept everything."""

import pytest
import torch

from tests.gpu_util import dev

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


class Step:
    def __init__(self, lens, counts, Hq, Hk, D, page, block, max_context, vocab=1024, seed=0):
        import flash_next_rtxpro6000_b200 as fx

        self.fx, d = fx, dev()
        g = torch.Generator().manual_seed(seed + D)
        rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        i32 = dict(dtype=torch.int32, device=d)
        need = [-(-(c + 3 * t) // page) for c, t in zip(lens, counts)]
        self.pages, self.page, self.block, N = sum(need), page, block, sum(counts)
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            self.table[b, :n] = order[sum(need[:b]):sum(need[:b]) + n]
        self.table = self.table.to(d)
        self.ctx = torch.tensor(lens, **i32)
        self.offsets = torch.tensor([sum(counts[:b]) for b in range(len(lens) + 1)], **i32)
        self.parents = torch.tensor([i if i < 1 else int(torch.randint(0, i, (1,), generator=g)) for t in counts for i in range(t)], **i32)
        self.parents[self.offsets[:-1][torch.tensor(counts, device=d) > 0].long()] = -1
        self.q, self.k, self.v = (rand(N, h, D).bfloat16().to(d) for h in (Hq, Hk, Hk))
        x = [torch.randint(0, 256, (self.pages, page, Hk, D), generator=g, dtype=torch.uint8) for _ in range(2)]
        for y in x:
            y[(y & 0x7F) == 0x7F] = 1
        self.caches = [y.to(d).view(E4M3) for y in x]
        self.scales = [torch.exp2(torch.randint(-8, -5, (self.pages, page // block, Hk), generator=g).float()).to(d) for _ in range(2)]
        self.start = [y.clone() for y in self.caches + self.scales]
        self.rot = fx.rotary_table(max(lens) + 3 * max(counts) + 1, D, device=d)
        self.w = torch.randint(-127, 128, (vocab, Hq * D), generator=g).to(torch.int8).to(d)
        self.ws = (torch.rand(vocab, generator=g) * 0.004).bfloat16().to(d)
        self.tokens = torch.randint(0, vocab, (N,), generator=g).to(d)
        self.u, self.draw = torch.rand(N, generator=g).to(d), torch.rand(len(lens), generator=g).to(d)
        self.temperature, self.top_p = torch.full((N,), 1.5, device=d), torch.full((N,), 0.98, device=d)
        self.top_k = (torch.arange(N, device=d) % 3 * 200).int()
        self.max_nodes, self.max_context = max(counts), max_context
        fx.prealloc(d, attention=True)

    def reset(self):
        for x, y in zip(self.caches + self.scales, self.start):
            x.copy_(y)

    def run(self, pdl):
        fx = self.fx
        mask, pos, _ = fx.tree_layout(self.parents, self.offsets, self.ctx, self.table, self.page, self.pages, pdl=pdl)
        q = fx.rotary_append8(self.q, self.k, self.v, pos, self.ctx, self.offsets, self.table, self.rot, *self.caches,
                              *self.scales, pdl=pdl)
        out, lse = fx.tree_attention8(q, *self.caches, *self.scales, self.table, self.ctx, self.offsets, mask,
                                      max_nodes=self.max_nodes, max_context=self.max_context, pdl=pdl)
        logits = torch.cat([fx.w8a16_gemv(x, self.w, self.ws, pdl=pdl) for x in out.flatten(1).split(16)])
        probs = fx.token_probs(logits, self.temperature, self.top_k, self.top_p, pdl=pdl)
        path, accepted, tokens = fx.verify_tokens(probs, self.draft(probs), self.tokens, self.parents, self.offsets, self.u,
                                                  self.draw, max_nodes=self.max_nodes, pdl=pdl)
        lens = fx.compact_nodes(*self.caches, self.table, self.ctx, path, accepted, *self.scales, pdl=pdl)
        return mask, pos, q, out, lse, logits, probs, path, accepted, tokens, lens

    def draft(self, probs):
        return None

    def stored(self, i, b, n):
        p = torch.arange(n, device=dev())
        page, at = self.table[b].long()[p // self.page], p % self.page
        return self.caches[i].view(torch.uint8)[page, at].view(E4M3).float() * self.scales[i][page, at // self.block][..., None]


CASES = [
    ([30, 0, 17], [5, 1, 8], 4, 2, 64, 32, 16, 56),
    ([1000], [16], 8, 2, 128, 64, 64, 1000),
    ([300, 9, 2000], [3, 1, 4], 4, 1, 256, 32, 32, 2000),
    ([6000, 100, 5000, 64] * 3, [4, 1, 9, 16] * 3, 16, 4, 128, 16, 16, 6000),
    ([700, 20] * 70, [2, 1] * 70, 4, 2, 64, 64, 16, 700),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}x{c[4]}")
def test_early_launches_and_replays_change_nothing(case):
    s = Step(*case)
    want = [x.clone() for x in s.run(False)]
    left = [x.clone() for x in s.caches + s.scales]
    bits = lambda x: x.view(torch.uint8) if x.dtype == E4M3 else x  # noqa: E731

    def same(got):
        torch.cuda.synchronize()
        s.fx.check_device_errors()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(s.caches + s.scales, left))

    for pdl in (True, False, True):
        s.reset()
        same(s.run(pdl))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = s.run(True)
    for _ in range(3):
        s.reset()
        for x in got:
            x.zero_()
        graph.replay()
        same(got)


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}x{c[4]}")
def test_the_cache_holds_the_context_and_the_accepted_tokens(case):
    """Keys and values behind each context are the path's, rounded twice at most: to e4m3 (2^-4, or 2^-10 of the scale they
    have now) and again where their block's scale changed (below 2^-6 of it, 2^-10)."""
    s = Step(*case)
    before = [[s.stored(i, b, int(c)) for b, c in enumerate(s.ctx.tolist())] for i in range(2)]
    pos = s.run(False)
    path, accepted, lens = pos[7], pos[8].tolist(), pos[10].tolist()
    positions = pos[1]
    s.fx.check_device_errors()
    D = s.q.shape[2]
    at = s.rot[positions].double()
    c, sn = at[:, None, : D // 2], at[:, None, D // 2:]
    k = s.k.double()
    keys = torch.cat([k[..., : D // 2] * c - k[..., D // 2:] * sn, k[..., D // 2:] * c + k[..., : D // 2] * sn], -1)
    for i, new in enumerate((keys, s.v.double())):
        for b, ctx in enumerate(s.ctx.tolist()):
            n0 = int(s.offsets[b])
            assert lens[b] == ctx + accepted[b]
            got = s.stored(i, b, lens[b]).double()
            p = torch.arange(lens[b], device=dev())
            scale = s.scales[i][s.table[b].long()[p // s.page], p % s.page // s.block].double()[..., None]
            old = before[i][b].double()
            assert bool(((got[:ctx] - old).abs() <= torch.where(old.abs() >= 2.0**-6 * scale[:ctx], 0.0, 2.0**-10 * scale[:ctx])).all())
            want = new[n0 + path[b, : accepted[b]].long()]
            assert bool(((got[ctx:] - want).abs() <= 2.0**-4 * want.abs() * (1 + 2.0**-16) + 2 * 2.0**-10 * scale[ctx:]).all())


def test_drafts_from_the_target_itself_are_accepted():
    """A chain drawn from the very rows that verify it (p = q) is accepted as a whole, whatever the random numbers."""
    s = Step([40, 7], [6, 4], 4, 2, 64, 32, 16, 64, vocab=512)
    s.parents = torch.tensor([i - 1 for t in (6, 4) for i in range(t)], dtype=torch.int32, device=dev())
    s.draft = lambda probs: probs
    g = torch.Generator(device=dev()).manual_seed(3)
    for _ in range(6):  # the tokens do not enter the model here: rows stay what they are while the chain is drawn
        s.reset()
        probs = s.run(False)[6]
        parents = torch.arange(10, device=dev()) - 1
        drawn = torch.multinomial(probs[parents.clamp(min=0)], 1, generator=g)[:, 0]
        s.tokens.copy_(drawn)
        s.u.copy_(torch.rand(10, generator=g, device=dev()))
        s.reset()
        out = s.run(False)
        assert out[8].tolist() == [6, 4] and out[10].tolist() == [46, 11]
    s.fx.check_device_errors()


def test_another_stream_and_threads_of_their_own_slots():
    """Two steps at once on two streams, each with its own scratch slot, give what they give alone."""
    fx = __import__("flash_next_rtxpro6000_b200")
    steps = [Step(*CASES[1]), Step(*CASES[3], seed=1)]
    want = []
    for s in steps:
        want.append([x.clone() for x in s.run(False)])
        s.reset()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(4):
        got = []
        for slot, (s, stream) in enumerate(zip(steps, streams)):
            s.reset()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream), fx.scratch_slot(slot):
                got.append(s.run(True))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    fx.check_device_errors()
