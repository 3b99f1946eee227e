"""tree_attention and tree_layout on the GPU, against attention in 64 bits that leaves hidden keys out.

Tolerances.  out: the weights are rounded to the type u (2^-8 bf16, 2^-11 fp16) before the second
product and the sums are in fp32, so the error is at most (u + 2^-12) times the weighted mean of
|v|, plus u |out| for the last rounding; 2^-12 covers the fp32 scores' error (D products and scores up
to ~16: 16 * 256 * 2^-24) and that of the sums.  lse: 2^-12 of the largest score or 1, the same
error in the scores."""

import numpy as np
import pytest
import torch

from tests.gpu_util import dev

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _fx():
    import flash_next_rtxpro6000_b200 as fx

    return fx


def _masks(counts, rng, how="tree"):
    out = []
    for t in counts:
        seen = []
        for i in range(t):
            if how == "tree":
                p = int(rng.integers(-1, i)) if i else -1
                seen.append((seen[p] if p >= 0 else 0) | 1 << i)
            elif how == "none":
                seen.append(0)
            else:
                seen.append(int(rng.integers(0, 2**63)) & ((1 << t) - 1))
        out += seen
    return out


def _signed(masks):
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64)


class Case:
    def __init__(self, lens, counts, Hq, Hk, D, page, dtype, seed=0, how="tree", garbage=False, spread=1.0):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        d = dev()
        self.lens, self.counts = lens, counts
        need = [-(-(c + t) // page) for c, t in zip(lens, counts)]
        pages = sum(need) + 2
        order = rng.permutation(pages)
        table = np.full((len(lens), max(max(need), 1) + 1), -12345, np.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        self.table = torch.from_numpy(table).to(d)
        kv = [torch.randn(pages, page, Hk, D, generator=g).to(dtype) for _ in range(2)]
        if garbage:  # places of no token hold anything
            used = torch.zeros(pages * page, dtype=torch.bool)
            for b, (c, t) in enumerate(zip(lens, counts)):
                p = np.arange(c + t)
                used[torch.from_numpy(table[b][p // page] * page + p % page).long()] = True
            for x in kv:
                x.view(-1, Hk, D)[~used] = float("nan")
                x.view(-1, Hk, D)[~used, :, ::3] = float("inf")
        self.k, self.v = (x.to(d) for x in kv)
        N = sum(counts)
        self.q = (torch.randn(N, Hq, D, generator=g) * spread).to(dtype).to(d)
        self.masks = _masks(counts, rng, how)
        self.mask = _signed(self.masks).to(d)
        self.offsets = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=d)
        self.ctx = torch.tensor(lens, dtype=torch.int32, device=d)
        self.page = page

    def run(self, **kw):
        args = dict(max_nodes=max(max(self.counts), 1), max_context=max(self.lens)) | kw
        return _fx().tree_attention(self.q, self.k, self.v, self.table, self.ctx, self.offsets,
                                    args.pop("tree_mask", self.mask), **args)

    def reference(self, scale=None):
        N, Hq, D = self.q.shape
        Hk = self.k.shape[2]
        d = dev()
        out = torch.zeros(N, Hq, D, dtype=torch.float64, device=d)
        mean = torch.zeros_like(out)
        lse = torch.full((N, Hq), -float("inf"), dtype=torch.float64, device=d)
        big = torch.ones(N, Hq, dtype=torch.float64, device=d)
        n = 0
        for b, (c, t) in enumerate(zip(self.lens, self.counts)):
            p = torch.arange(c + t, device=d)
            slots = self.table[b].long()[p // self.page] * self.page + p % self.page
            keys = self.k.reshape(-1, Hk, D)[slots].double()
            vals = self.v.reshape(-1, Hk, D)[slots].double()
            for i in range(t):
                see = torch.tensor([True] * c + [bool(self.masks[n] >> j & 1) for j in range(t)], device=d)
                if bool(see.any()):
                    kk = keys[see].repeat_interleave(Hq // Hk, 1)
                    vv = vals[see].repeat_interleave(Hq // Hk, 1)
                    s = torch.einsum("hd,khd->hk", self.q[n].double(), kk) * (D**-0.5 if scale is None else scale)
                    w = torch.softmax(s, 1)
                    out[n] = torch.einsum("hk,khd->hd", w, vv)
                    mean[n] = torch.einsum("hk,khd->hd", w, vv.abs())
                    lse[n] = torch.logsumexp(s, 1)
                    big[n] = s.abs().amax(1).clamp(min=1)
                n += 1
        return out, mean, lse, big

    def check(self, scale=None, **kw):
        out, lse = self.run(**(kw | ({} if scale is None else {"scale": scale})))
        want, mean, wlse, big = self.reference(scale)
        u = UNIT[self.q.dtype]
        err = (out.double() - want).abs()
        tol = (u + 2.0**-12) * mean + u * want.abs() + 2.0**-25
        ok = (err <= tol) | (want.isnan() & out.isnan()) | (want == out.double())
        assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} off, worst {float((err - tol)[~ok].max())}"
        empty = wlse == -float("inf")
        assert torch.equal(lse == -float("inf"), empty)
        diff = torch.where(empty, 0.0, (lse.double() - wlse).abs())
        assert bool(((diff <= 2.0**-12 * big) | (wlse.isnan() & lse.isnan())).all())
        _fx().check_device_errors()
        return out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hk,T", [(1, 1, 1), (8, 2, 4), (12, 2, 5), (16, 1, 3), (4, 4, 40), (8, 1, 16), (7, 1, 64)])
def test_against_64_bits(D, dtype, Hq, Hk, T):
    Case([0, 1, 63, 64, 65, 300], [T, 1, T, max(1, T - 1), T, T], Hq, Hk, D, 16, dtype, seed=D + T).check()


@pytest.mark.parametrize("page", [1, 7, 64, 100, 4096])
def test_page_sizes(page):
    Case([513, 0, 129, 2000], [3, 2, 1, 7], 8, 2, 128, page, torch.bfloat16, seed=page, garbage=True).check()


@pytest.mark.parametrize("Hq,T,D", [(2, 1, 256), (16, 16, 256), (8, 2, 128), (8, 64, 128), (2, 20, 64)])
def test_long_context_split_over_the_gpu(Hq, T, D):
    Case([20011], [T], Hq, 1, D, 16, torch.bfloat16, seed=T).check()
    Case([9000, 31, 0, 4000, 1], [T, 1, T, T, 2], Hq, 2, D, 32, torch.float16, seed=T + 1).check()


@pytest.mark.parametrize("D,T", [(64, 9), (128, 33), (256, 64)])
@pytest.mark.parametrize("how", ["any", "none"])
def test_masks_that_leave_rows_empty(D, T, how):
    c = Case([0, 70, 0, 5], [T, T, 1, 3], 4, 2, D, 8, torch.bfloat16, seed=7, how=how)
    out, lse = c.check()
    if how == "none":
        assert bool((out[:T] == 0).all()) and bool((lse[:T] == -float("inf")).all())


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,T,ctx", [(2, 5, 0), (8, 20, 100), (4, 64, 3), (8, 33, 700)])
def test_not_finite_where_hidden(D, Hq, T, ctx):
    """A drafted token with infinite or NaN keys and values reaches the rows that see it, no others;
    what lies past the tokens reaches none."""
    c = Case([ctx, 40], [T, 2], Hq, 2, D, 16, torch.bfloat16, seed=11, garbage=True)
    j = T // 2
    slot = int(c.table[0][(ctx + j) // 16]) * 16 + (ctx + j) % 16
    c.v.view(-1, 2, D)[slot, 0, 1] = float("nan")
    c.v.view(-1, 2, D)[slot, 1, D - 1] = -float("inf")
    out, _ = c.check()
    sees = torch.tensor([bool(c.masks[i] >> j & 1) for i in range(T)], device=dev())
    assert torch.equal(out[:T, 0, 1].isnan(), sees) and torch.equal(out[:T, Hq - 1, D - 1].isinf(), sees)
    c.k.view(-1, 2, D)[slot] = float("nan")
    out, lse = c.run()
    assert torch.equal(lse[:T].isnan(), sees[:, None].expand(T, Hq))
    assert bool(out[:T][~sees].isfinite().all()) and bool(out[T:].isfinite().all())


def test_peaked_scores_and_lowest_values():
    c = Case([500, 64], [6, 3], 4, 1, 128, 16, torch.bfloat16, seed=2, spread=30.0)
    c.check()
    c.k.fill_(torch.finfo(torch.bfloat16).min / 1e20)  # scores far below zero, all equal in a row
    c.q.fill_(1.0)
    out, lse = c.run()
    assert bool(out.isfinite().all()) and bool((lse < -1e17).all())


@pytest.mark.parametrize("T", [1, 2, 63, 64])
def test_chain_without_a_mask(T):
    c = Case([77, 0], [T, T], 4, 2, 64, 16, torch.float16, seed=T)
    c.masks = [(2 << i) - 1 for i in range(T)] * 2
    c.check(tree_mask=None)


def test_strides_scale_and_destinations():
    fx = _fx()
    c = Case([300, 20], [5, 9], 8, 2, 128, 16, torch.bfloat16, seed=4)
    ref, rlse = c.check(scale=0.03)
    rows = torch.zeros(14, 3, 8, 128, dtype=torch.bfloat16, device=dev())  # queries within wider rows
    rows[:, 1] = c.q
    kt, vt = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (c.k, c.v))  # head-major pages
    out = torch.zeros(14, 8, 2, 128, dtype=torch.bfloat16, device=dev())[:, :, 1]
    wide = torch.full((2, 99), -1, dtype=torch.int32, device=dev())
    wide[:, : c.table.shape[1]] = c.table
    got, lse = fx.tree_attention(rows[:, 1], kt, vt, wide, c.ctx, c.offsets, c.mask, max_nodes=64, scale=0.03,
                                 out=out, lse=torch.empty(14, 8, device=dev()))
    assert got is out
    # the planned row tiles differ with max_nodes, so sums may round differently
    assert float((got.float() - ref.float()).abs().max()) <= 2 * 2.0**-8 * float(ref.float().abs().max())
    assert float((lse - rlse).abs().max()) <= 2.0**-12
    same, _ = fx.tree_attention(rows[:, 1], kt, vt, c.table, c.ctx, c.offsets, c.mask, max_nodes=9, max_context=300,
                                scale=0.03)
    assert torch.equal(same, ref)


def test_cache_past_32_bit_offsets():
    """Pages whose element offset passes 2^31 (and byte offset 2^32)."""
    d, page, Hk, D = dev(), 64, 8, 128
    pages = (1 << 31) // (page * Hk * D) + 40
    c = Case([500], [4], 16, 8, D, page, torch.bfloat16, seed=5)
    big = torch.empty(pages, page, Hk, D, dtype=torch.bfloat16, device=d)
    n = c.k.shape[0]
    big[-n:] = c.k
    low, llse = c.check()
    far = torch.empty_like(big)
    far[-n:] = c.v
    table = torch.where(c.table >= 0, c.table + (pages - n), c.table)
    out, lse = _fx().tree_attention(c.q, big, far, table, c.ctx, c.offsets, c.mask, max_nodes=4, max_context=500)
    assert torch.equal(out, low) and torch.equal(lse, llse)


def test_many_requests():
    B = 1100
    lens = [(7 * b) % 50 for b in range(B)]
    counts = [b % 4 for b in range(B)]
    Case(lens, counts, 4, 2, 64, 16, torch.bfloat16, seed=6).check()


def test_same_bits_again_on_another_stream_and_in_a_graph():
    fx = _fx()
    c = Case([4000, 9, 700], [16, 3, 8], 16, 2, 256, 64, torch.bfloat16, seed=8)
    ref, rlse = c.check()
    for _ in range(3):
        out, lse = c.run()
        assert torch.equal(out, ref) and torch.equal(lse, rlse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), fx.scratch_slot(1):
        out, lse = c.run()
    side.synchronize()
    assert torch.equal(out, ref) and torch.equal(lse, rlse)
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, lse = c.run()
    for ctx in ([4000, 9, 700], [100, 0, 650]):  # a captured call follows the lengths
        c.ctx.copy_(torch.tensor(ctx, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        c.lens = ctx
        want, wlse = c.run(max_context=4000)
        assert torch.equal(out, want) and torch.equal(lse, wlse)


def test_lengths_and_pages_out_of_range_are_reported():
    fx = _fx()
    d = dev()

    def codes(c, **kw):
        fx.check_device_errors()
        c.run(**kw)
        with pytest.raises(fx.DeviceWaitError) as e:
            fx.check_device_errors()
        return [x for _, x in e.value.codes]

    new = lambda: Case([50, 60], [4, 4], 4, 2, 64, 16, torch.bfloat16, seed=9)  # noqa: E731
    c = new()
    assert codes(c, max_context=59) == [14]
    assert codes(c, max_nodes=3) == [14]
    c.ctx[0] = -1
    assert codes(c) == [14]
    c = new()
    c.ctx[1] = 16 * c.table.shape[1] - 3
    assert codes(c, max_context=10**6) == [14]
    c = new()
    c.offsets[2] = 9  # past q's rows
    assert codes(c) == [14]
    c = new()
    for page in (-1, c.k.shape[0]):
        c.table[1, 2] = page
        assert codes(c) == [15]
    assert d == c.q.device


def test_no_nodes_and_refusals():
    fx = _fx()
    c = Case([30, 9], [3, 2], 4, 2, 64, 16, torch.bfloat16, seed=1)
    out, lse = fx.tree_attention(c.q[:0], c.k, c.v, c.table, c.ctx, torch.zeros_like(c.offsets), c.mask[:0])
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    good = dict(q=c.q, k_cache=c.k, v_cache=c.v, page_table=c.table, context_lens=c.ctx, node_offsets=c.offsets,
                tree_mask=c.mask)
    w = torch.zeros(2, 16, 2, 96, dtype=torch.bfloat16, device=dev())
    bad = [
        (dict(q=c.q.float()), NotImplementedError), (dict(q=c.q[0]), ValueError),
        (dict(q=w[0, :5], k_cache=w, v_cache=w), NotImplementedError),  # head size 96
        (dict(q=c.q[:, :3]), ValueError), (dict(k_cache=c.k.half()), ValueError),
        (dict(v_cache=c.v[:1]), ValueError), (dict(page_table=c.table.long()), ValueError),
        (dict(page_table=c.table[:1]), ValueError), (dict(context_lens=c.ctx.long()), ValueError),
        (dict(node_offsets=c.offsets[:2]), ValueError), (dict(tree_mask=c.mask[:1]), ValueError),
        (dict(tree_mask=c.mask.int()), ValueError), (dict(max_nodes=65), NotImplementedError),
        (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError), (dict(scale=float("nan")), ValueError),
        (dict(scale=float("inf")), ValueError), (dict(max_nodes=0), ValueError), (dict(max_context=-1), ValueError),
        (dict(lse=torch.zeros(5, 4, dtype=torch.float64, device=dev())), ValueError),
        (dict(out=c.q.half()), ValueError), (dict(q=c.q.cpu()), ValueError),
        (dict(q=torch.zeros(5 * 4 * 64 + 1, dtype=torch.bfloat16, device=dev())[1:].view(5, 4, 64)), ValueError),
    ]
    for change, error in bad:
        with pytest.raises(error):
            fx.tree_attention(**(good | change))


def test_tree_layout():
    fx = _fx()
    d = dev()
    rng = np.random.default_rng(3)
    counts, lens, page = [1, 64, 0, 17, 5], [0, 1000, 3, 15, 16], 16
    parents, masks, pos, slots = [], [], [], []
    table = torch.from_numpy(rng.permutation(5 * 70).reshape(5, 70).astype(np.int32))
    for b, t in enumerate(counts):
        m, depth = [], []
        for i in range(t):
            p = int(rng.integers(-1, i)) if i else -1
            parents.append(p)
            m.append((m[p] if p >= 0 else 0) | 1 << i)
            depth.append(depth[p] + 1 if p >= 0 else 0)
            at = lens[b] + i
            slots.append(int(table[b, at // page]) * page + at % page)
        masks += m
        pos += [lens[b] + x for x in depth]
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=d)
    args = [torch.tensor(parents, dtype=torch.int32, device=d), offsets,
            torch.tensor(lens, dtype=torch.int32, device=d), table.to(d), page, 350]
    got = fx.tree_layout(*args)
    fx.check_device_errors()
    for x, want in zip(got, (_signed(masks), torch.tensor(pos), torch.tensor(slots))):
        assert torch.equal(x.cpu(), want)
    # a parent that is not an earlier node, a page outside the cache, a context past the table
    for i, value, code in ((0, 5, 16), (0, -2, 16), (5, 300, 15), (2, 70 * 16, 14)):
        wrong = [x.clone() if torch.is_tensor(x) else x for x in args]
        if i == 5:
            wrong[5] = value
        else:
            wrong[i][0 if i == 0 else 1] = value
        fx.tree_layout(*wrong)
        with pytest.raises(fx.DeviceWaitError) as e:
            fx.check_device_errors()
        assert [c for _, c in e.value.codes] == [code]
    for i, x in ((0, args[0].long()), (1, offsets[:2]), (2, args[2].long()), (3, table.to(d)[:2])):
        with pytest.raises(ValueError):
            fx.tree_layout(*(args[:i] + [x] + args[i + 1:]))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,T", [(4, 9), (4, 30), (8, 64)])
def test_rising_scores(D, Hq, T):
    """Keys whose scores keep rising along the context, so that every tile raises every row's maximum
    far enough for the sums to be rescaled; and falling ones."""
    for sign in (1, -1):
        c = Case([2500, 300], [T, T], Hq, 1, D, 16, torch.bfloat16, seed=D + T)
        c.q = c.q * 0.1
        c.q[:, :, 0] = 1.0
        pos = torch.arange(2500, device=dev())
        for b, n in enumerate((2500, 300)):
            slots = c.table[b].long()[pos[:n] // 16] * 16 + pos[:n] % 16
            c.k.view(-1, 1, D)[slots, 0, 0] = (sign * pos[:n].float() * 0.05 * D**0.5).bfloat16()
        c.check()


@pytest.mark.parametrize("ctx", [1, 60, 61, 64, 65, 127, 128, 129])
def test_trees_across_key_tiles(ctx):
    """64 drafted tokens that lie in one key tile or in two, with values that are not finite in both."""
    c = Case([ctx, ctx + 3], [64, 61], 8, 2, 128, 16, torch.float16, seed=ctx, garbage=True)
    for j in (0, 3, 63):
        slot = int(c.table[0][(ctx + j) // 16]) * 16 + (ctx + j) % 16
        c.v.view(-1, 2, 128)[slot, :, j] = float("nan")
    out, _ = c.check()
    for j in (0, 3, 63):
        sees = torch.tensor([bool(c.masks[i] >> j & 1) for i in range(64)], device=dev())
        assert torch.equal(out[:64, 2, j].isnan(), sees)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,Hq,Hk,T", [(64, 8, 4, 1), (64, 12, 12, 33), (64, 8, 2, 64), (128, 16, 4, 1), (128, 16, 4, 20),
                                       (128, 16, 4, 64), (256, 16, 4, 1), (256, 8, 4, 64), (256, 16, 2, 40)])
def test_batches_that_fill_the_gpu(D, Hq, Hk, T, dtype):
    """Enough key tiles for the tensor-memory form, with short, empty and odd requests among long ones."""
    lens = [5000, 0, 1, 63, 64, 4000, 129, 3000, 7, 4999, 2500, 4095]
    counts = [T, 1, T, T, 0, max(1, T - 1), T, 1, T, T, 2, T]
    counts = [min(c, T) for c in counts]
    big = 12 * Hk * 80 > 8 * 148  # what the launch goes by: requests, kv heads, key tiles of the longest
    assert big
    Case(lens, counts, Hq, Hk, D, 16, dtype, seed=T + D, garbage=True).check()


@pytest.mark.parametrize("D,T", [(64, 40), (128, 20), (128, 64), (256, 24)])
@pytest.mark.parametrize("how", ["any", "none"])
def test_batches_with_any_mask(D, T, how):
    lens = [6000, 0, 0, 70, 5999, 64, 5000, 1]
    c = Case(lens, [T, T, 1, T, T, 3, T, T], 8, 4, D, 24, torch.bfloat16, seed=3, how=how)
    out, lse = c.check()
    if how == "none":
        assert bool((out[T:2 * T] == 0).all()) and bool((lse[T:2 * T] == -float("inf")).all())


@pytest.mark.parametrize("D,T", [(64, 40), (128, 20), (128, 64), (256, 24)])
def test_batches_not_finite_where_hidden(D, T):
    lens = [6000, 3, 64 * 60 - 5, 5999, 5000]
    c = Case(lens, [T] * 5, 8, 4, D, 16, torch.bfloat16, seed=13, garbage=True)
    for b in range(5):
        for j in (T // 2, T - 1):
            slot = int(c.table[b][(lens[b] + j) // 16]) * 16 + (lens[b] + j) % 16
            c.v.view(-1, 4, D)[slot, :, j] = float("nan") if b % 2 else float("inf")
            if b == 3:
                c.k.view(-1, 4, D)[slot] = float("nan")
    out, lse = c.run()
    want, _, wlse, _ = c.reference()
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isinf(), want.isinf())
    assert torch.equal(lse.isnan(), wlse.isnan())
    fine = want.isfinite()
    assert float((out.double() - want)[fine].abs().max()) < 2.0**-6
    _fx().check_device_errors()


@pytest.mark.parametrize("D,Hq,T", [(64, 4, 30), (128, 4, 9), (128, 8, 64), (256, 4, 30)])
def test_batches_with_rising_scores(D, Hq, T):
    c = Case([6000] * 16, [T] * 16, Hq, 1, D, 16, torch.bfloat16, seed=D + T)
    c.q = c.q * 0.1
    c.q[:, :, 0] = 1.0
    pos = torch.arange(6000, device=dev())
    for b in range(16):
        slots = c.table[b].long()[pos // 16] * 16 + pos % 16
        sign = 1 if b % 2 else -1
        c.k.view(-1, 1, D)[slots, 0, 0] = (sign * pos.float() * 0.02 * D**0.5).bfloat16()
    c.check()


def test_batches_not_finite_with_uneven_row_tiles():
    """Requests whose rows fill both row tiles next to ones that fill one, a segment each, all with a
    drafted token that is not finite: no segment takes another's for its own."""
    counts = [64, 3, 40, 64, 1, 33, 64, 9] * 6
    lens = [700 + 13 * b for b in range(len(counts))]
    c = Case(lens, counts, 8, 2, 128, 16, torch.bfloat16, seed=21)
    for b, (ctx, t) in enumerate(zip(lens, counts)):
        j = (t - 1) // 2
        slot = int(c.table[b][(ctx + j) // 16]) * 16 + (ctx + j) % 16
        c.v.view(-1, 2, 128)[slot, b % 2, b] = float("nan")
    out, _ = c.run()
    n = 0
    for b, t in enumerate(counts):
        j = (t - 1) // 2
        sees = torch.tensor([bool(c.masks[n + i] >> j & 1) for i in range(t)], device=dev())
        got = out[n:n + t].view(t, 2, 4, 128).isnan()
        want = torch.zeros_like(got)
        want[:, b % 2, :, b] = sees[:, None]
        assert torch.equal(got, want), b
        n += t


def _sinks(D, Hq, T, n, B, gap, seed):
    """B requests over n keys: every score is a unit normal's but one key's a request, which lies `gap` above and
    has value 0; the others' values lie between 500 and 1,500."""
    c = Case([n] * B, [T] * B, Hq, 1, D, 64, torch.float16, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    c.q.zero_()
    c.q[..., 0] = D**0.5  # the score is the key's first element
    pos = torch.arange(n + T, device=dev())
    slots = c.table.long()[:, pos // 64] * 64 + pos % 64
    c.v.view(-1, D)[slots] = (500 + 1000 * torch.rand(B, n + T, D, generator=g)).half().to(dev())
    c.k.view(-1, D)[slots, 0] = torch.randn(B, n + T, generator=g).half().to(dev())
    c.k.view(-1, D)[slots[:, n // 3], 0] = gap
    c.v.view(-1, D)[slots[:, n // 3]] = 0
    return c, slots


def _whole(c, slots, n, T):
    """(out, weighted mean of |v|) of all rows in 64 bits, for one kv head."""
    N, Hq, D = c.q.shape
    outs, means = [], []
    for b in range(N // T):
        keys, vals = c.k.view(-1, D)[slots[b]].double(), c.v.view(-1, D)[slots[b]].double()
        see = torch.tensor([[True] * n + [bool(m >> j & 1) for j in range(T)] for m in c.masks[b * T:b * T + T]],
                           device=dev())
        s = (c.q[b * T:b * T + T].double() @ keys.T * D**-0.5).masked_fill(~see[:, None], -float("inf"))
        w = torch.softmax(s, -1)
        outs.append(w @ vals)
        means.append(w @ vals.abs())
    return torch.cat(outs), torch.cat(means)


SINKS = [(64, 1, 1, 70000, 1), (64, 4, 1, 500, 100), (128, 4, 8, 500, 100), (256, 2, 5, 500, 100),
         (64, 8, 8, 250, 100), (256, 8, 8, 250, 100),                           # mma.sync, 16 to 64 rows
         (64, 8, 8, 131072, 1), (64, 8, 5, 6000, 20), (64, 8, 32, 3000, 60), (128, 16, 2, 6000, 20),
         (128, 8, 40, 3000, 60), (256, 8, 9, 6000, 20), (256, 8, 20, 3000, 40)]  # tensor memory


@pytest.mark.parametrize("gap", [10.0, 18.0, 20.0, 24.0])
@pytest.mark.parametrize("D,Hq,T,n,B", SINKS)
def test_fp16_weights_far_below_the_largest(D, Hq, T, n, B, gap):
    """Many small weights under one large one whose value is 0: what the row gives is all theirs.

    A weight's rounding is 2^-11 of it, or 2^-25 where fp16 has no smaller step.  A key tile's largest
    weight is at least 2^-7 (the row's reference follows the tiles down), so the second kind costs a tile
    of 64 at most 64 * 2^-25 / 2^-7 = 2^-12 of its weight times the largest |v|, three times the mean here;
    in the large weight's own tile, where that one is at least 2^7, 64 * 2^-32 of the largest |v|."""
    c, slots = _sinks(D, Hq, T, n, B, gap, seed=D + T)
    out, _ = c.run()
    want, mean = _whole(c, slots, n, T)
    u = UNIT[torch.float16]
    tol = (u + 2.0**-12 + 3 * 2.0**-12) * mean + u * want.abs() + 64 * 2.0**-32 * 1500 + 2.0**-25
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), (float((err / want.abs()).max()), float((err - tol).max()))
    _fx().check_device_errors()


@pytest.mark.parametrize("D,Hq,T,n,B", SINKS)
def test_fp16_infinite_value_under_a_small_weight(D, Hq, T, n, B):
    """An infinite value that a row sees makes the row infinite, however small its weight (that of a key
    at its tile's average: within 2^7 of the tile's largest)."""
    c, slots = _sinks(D, Hq, T, n, B, 24.0, seed=D + T)
    c.k.view(-1, D)[slots[:, n - 70], 0] = 0.0
    c.v.view(-1, D)[slots[:, n - 70], 5] = float("inf")
    out, _ = c.run()
    assert bool((out[..., 5] == float("inf")).all())
    assert bool(out[..., 6:].isfinite().all()) and bool(out[..., :5].isfinite().all())


@pytest.mark.parametrize("offsets,bad", [
    ([-3, 2, 6, 8], [0, 1]), ([-70, 2, 6, 8], [0, 1]), ([0, 2, 6, 9], [6, 7]), ([0, 2, 6, 2**31 - 1], [6, 7]),
    ([-2**31, 2, 6, 8], [0, 1]),
])
def test_tree_layout_of_requests_outside_the_arrays(offsets, bad):
    """Offsets below 0 or past the rows are reported and not followed: the request's rows see nothing and are
    stored nowhere, the others' are as ever."""
    fx = _fx()
    i32 = dict(dtype=torch.int32, device=dev())
    parents = torch.tensor([-1, 0, -1, 0, 0, 2, -1, 0], **i32)
    ctx, table = torch.tensor([5, 20, 0], **i32), torch.arange(9, **i32).view(3, 3)
    whole = fx.tree_layout(parents, torch.tensor([0, 2, 6, 8], **i32), ctx, table, 16, 9)
    fx.check_device_errors()
    got = fx.tree_layout(parents, torch.tensor(offsets, **i32), ctx, table, 16, 9)
    with pytest.raises(fx.DeviceWaitError) as e:
        fx.check_device_errors()
    assert [c for _, c in e.value.codes] == [14]
    for x, want, none in zip(got, whole, (0, 0, -1)):
        want = want.clone()
        want[bad] = none
        assert torch.equal(x, want)


def test_tree_layout_of_a_request_with_too_many_nodes():
    fx = _fx()
    i32 = dict(dtype=torch.int32, device=dev())
    parents = torch.arange(-1, 69, **i32)
    parents[65] = -1
    parents[66:] = 0
    mask, pos, slots = fx.tree_layout(parents, torch.tensor([0, 65, 70], **i32), torch.tensor([3, 7], **i32),
                                      torch.arange(12, **i32).view(2, 6), 16, 12)
    with pytest.raises(fx.DeviceWaitError) as e:
        fx.check_device_errors()
    assert [c for _, c in e.value.codes] == [14]
    assert bool((mask[:65] == 0).all()) and bool((pos[:65] == 0).all()) and bool((slots[:65] == -1).all())
    assert mask[65:].tolist() == [1, 3, 5, 9, 17] and slots[65:].tolist() == [96 + 7 + j for j in range(5)]


def _padded(c, ahead, behind):
    """The case with rows of no request ahead of its own and behind them, and destinations that hold NaN."""
    d = c.q.device
    N, Hq, D = c.q.shape
    q = torch.full((ahead + N + behind, Hq, D), float("nan"), dtype=c.q.dtype, device=d)
    q[ahead:ahead + N] = c.q
    mask = torch.full((ahead + N + behind,), -1, dtype=torch.int64, device=d)
    mask[ahead:ahead + N] = c.mask
    out = torch.full_like(q, float("nan"))
    lse = torch.full(q.shape[:2], float("nan"), device=d)
    return q, c.offsets + ahead, mask, out, lse


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,counts,Hq,Hk", [
    ([30], [3], 4, 2), ([50, 60, 0], [4, 9, 1], 4, 2), ([5000, 0, 3000], [16, 4, 9], 4, 1),
    ([5000] * 12, [40, 1, 7] * 4, 8, 4), ([5000] * 12, [64, 1, 7] * 4, 16, 4), ([20, 100] * 100, [2, 3] * 100, 2, 1),
])
def test_rows_of_no_request(lens, counts, Hq, Hk, D):
    """They give 0 and -inf, whatever q holds there, and are no error; the others are as without them."""
    fx = _fx()
    c = Case(lens, counts, Hq, Hk, D, 16, torch.bfloat16, seed=31)
    ref, rlse = c.run()
    N = c.q.shape[0]
    for ahead, behind in ((0, 5), (3, 0), (2, 70)):
        q, offsets, mask, out, lse = _padded(c, ahead, behind)
        fx.tree_attention(q, c.k, c.v, c.table, c.ctx, offsets, mask, max_nodes=max(counts), max_context=max(lens),
                          out=out, lse=lse)
        fx.check_device_errors()
        assert torch.equal(out[ahead:ahead + N], ref) and torch.equal(lse[ahead:ahead + N], rlse)
        for rows in (slice(0, ahead), slice(ahead + N, None)):
            assert bool((out[rows] == 0).all()) and bool((lse[rows] == -float("inf")).all())


@pytest.mark.parametrize("D,Hk,ctx", [(64, 2, 60), (128, 2, 2000), (128, 4, 6000), (256, 4, 6000)])
def test_rows_of_refused_requests(D, Hk, ctx):
    """Requests whose lengths are out of bounds, among them the first and the last of a launch, give 0 and
    -inf and the error; their neighbours are as ever."""
    fx = _fx()
    B = 140 if ctx == 60 else 12
    counts = [3, 8, 1, 5] * (B // 4)
    c = Case([ctx] * B, counts, 2 * Hk, Hk, D, 16, torch.bfloat16, seed=33)
    ref, rlse = c.run()
    refused = [0, 1, 5, B - 1] + ([127, 128] if B > 128 else [])
    good = c.ctx.clone()
    c.ctx[refused] = torch.tensor([-1, ctx + 1] * (len(refused) // 2), dtype=torch.int32, device=dev())
    out, lse = torch.full_like(c.q, float("nan")), torch.full_like(rlse, float("nan"))
    c.run(out=out, lse=lse)
    with pytest.raises(fx.DeviceWaitError) as e:
        fx.check_device_errors()
    assert [x for _, x in e.value.codes] == [14]
    off = c.offsets.tolist()
    for b in range(B):
        rows = slice(off[b], off[b + 1])
        if b in refused:
            assert bool((out[rows] == 0).all()) and bool((lse[rows] == -float("inf")).all()), b
        else:  # the units are spread over the CTAs in another way, so sums may round differently
            assert float((out[rows].float() - ref[rows].float()).abs().max()) <= 2 * 2.0**-8 * float(ref.float().abs().max())
            assert float((lse[rows] - rlse[rows]).abs().max()) <= 2.0**-12, b
    c.ctx.copy_(good)
    again, alse = c.run()
    assert torch.equal(again, ref) and torch.equal(alse, rlse)


def test_a_captured_step_replayed_with_fewer_nodes():
    """Layout, rotation and attention captured at 12 rows, replayed with 12, 5 and 0 nodes: the rest are 0."""
    fx = _fx()
    d, i32 = dev(), dict(dtype=torch.int32, device=dev())
    c = Case([700, 40], [8, 4], 4, 2, 64, 16, torch.bfloat16, seed=35)
    parents = torch.full((12,), -1, **i32)
    table = fx.rotary_table(800, 64, device=d)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(12, 2, 64, generator=g).bfloat16().to(d) for _ in range(2))

    def step():
        mask, pos, slots = fx.tree_layout(parents, c.offsets, c.ctx, c.table, 16, c.k.shape[0])
        q = fx.rotary_append(c.q, k, v, pos, slots, table, c.k, c.v)
        return fx.tree_attention(q, c.k, c.v, c.table, c.ctx, c.offsets, mask, max_nodes=8, max_context=700)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for offsets in ([0, 8, 12], [0, 3, 5], [0, 0, 0], [0, 8, 12]):
        c.offsets.copy_(torch.tensor(offsets))
        out.fill_(float("nan"))
        lse.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        fx.check_device_errors()
        n = offsets[2]
        assert bool(out[:n].isfinite().all()) and bool(lse[:n].isfinite().all())
        assert bool((out[n:] == 0).all()) and bool((lse[n:] == -float("inf")).all())
        want, wlse = step()
        assert torch.equal(out, want) and torch.equal(lse, wlse)
