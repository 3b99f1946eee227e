"""rotary_append8 and tree_attention8 on the GPU, against the rotation, the blocks' scales and the attention in 64
bits.

Tolerances.  Append: y is the rotated element with the error of three fp32 roundings and the table's (8 * 2^-24 of
|x c| + |y s|, as for rotary_append); a block's scale follows from the largest of them, so it has to be that of
amax (1 +- 2^-20); an element is then within half an e4m3 step of y / scale: 2^-4 of it, or 2^-10 (half of the
subnormals' step).  Elements that take another power of two are exact unless they fall below 2^-6, then within 2^-10.

Attention: keys and values are exact, query elements too (down to 2^-28 of their row's largest); weights are rounded
to fp16 (2^-11), the scores' error and the sums' are within 2^-12 (as for tree_attention), the exponent's argument with the
value's scale in it, up to 2^7, adds 2^7 2^-24 ln 2 < 2^-17: (2^-11 + 2^-12 + 2^-17) of the weighted mean of |v|, and half a
step of the result."""

import numpy as np
import pytest
import torch

from tests.gpu_util import dev

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
E4M3 = torch.float8_e4m3fn
NAN = 0x7F


def _fx():
    import flash_next_rtxpro6000_b200 as fx

    return fx


def _power(amax):
    """The smallest power of two, at least 2^-40, by which amax divided is at most 448."""
    amax = np.asarray(amax, np.float64)
    with np.errstate(divide="ignore"):
        e = np.ceil(np.log2(np.maximum(amax, 1e-300) / 448.0))
    e = np.where(np.ldexp(448.0, (e - 1).astype(int)) >= amax, e - 1, e)
    return np.ldexp(1.0, np.maximum(e, -40).astype(int))


def _values(x):
    return x.view(torch.uint8).cpu().view(E4M3).double().numpy()


class Append:
    def __init__(self, lens, counts, Hq, Hk, D, R, page, block, dtype, interleaved=False, seed=0, size=1.0, pad=0, shift=0):
        fx, d = _fx(), dev()
        g = torch.Generator().manual_seed(seed)
        self.__dict__.update(lens=lens, counts=counts, Hq=Hq, Hk=Hk, D=D, R=R, page=page, block=block, dtype=dtype,
                             interleaved=interleaved)
        T, wide = sum(counts), (Hq + 2 * Hk) * D + pad
        rows = (torch.randn(T * wide + shift, generator=g) * size).to(dtype).to(d)[shift:].view(T, wide)[:, : wide - pad]
        self.q, self.k, self.v = (x.unflatten(1, (-1, D)) for x in rows.split([Hq * D, Hk * D, Hk * D], 1))
        self.rot = fx.rotary_table(3000, R, device=d)
        self.pos = torch.randint(0, 3000, (T,), generator=g)
        need = [-(-(c + t) // page) for c, t in zip(lens, counts)]
        self.pages = sum(need) + 2
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(need + [1])), -7, dtype=torch.int32)
        for b, n in enumerate(need):
            self.table[b, :n] = order[sum(need[:b]):sum(need[:b]) + n]
        self.caches = [torch.randint(0, 256, (self.pages, page, Hk, D), generator=g, dtype=torch.uint8) for _ in range(2)]
        for c in self.caches:
            c[(c & 0x7F) == 0x7F] = 5  # no NaN
        self.scales = [torch.exp2(torch.randint(-9, 0, (self.pages, page // block, Hk), generator=g).float()) for _ in range(2)]

    def run(self, out=None, **kw):
        fx, d = _fx(), dev()
        self.c = [x.to(d).view(E4M3) for x in self.caches]
        self.s = [x.to(d) for x in self.scales]
        i32 = dict(dtype=torch.int32, device=d)
        off = np.concatenate([[0], np.cumsum(self.counts)]).tolist()
        args = dict(ctx=torch.tensor(self.lens, **i32), off=torch.tensor(off, **i32)) | kw
        return fx.rotary_append8(self.q, self.k, self.v, self.pos.to(d), args["ctx"], args["off"], self.table.to(d), self.rot,
                                 *self.c, *self.s, interleaved=self.interleaved, out=out)

    def turned(self, x):
        x = x.double().cpu().numpy()
        R = self.R
        angle = self.pos.double().numpy()[:, None] * 10000.0 ** (-np.arange(R // 2) / max(R // 2, 1))
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        y, size = x.copy(), np.abs(x)
        a, b = (slice(0, R, 2), slice(1, R, 2)) if self.interleaved else (slice(0, R // 2), slice(R // 2, R))
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
        size[..., a] = np.abs(x[..., a] * c) + np.abs(x[..., b] * s)
        size[..., b] = np.abs(x[..., b] * c) + np.abs(x[..., a] * s)
        return y, size

    def check_stored(self):
        page, block = self.page, self.block
        untouched = np.ones((self.pages, page), bool)
        blocks_left = np.ones((self.pages, page // block), bool)
        for i, (y, size) in enumerate((self.turned(self.k), (self.v.double().cpu().numpy(), np.abs(self.v.double().cpu().numpy())))):
            got, was = _values(self.c[i]), self.caches[i].view(E4M3).double().numpy()
            now, old = self.s[i].double().cpu().numpy(), self.scales[i].double().numpy()
            n0 = 0
            for b, (c, t) in enumerate(zip(self.lens, self.counts)):
                for j in range(c // block, -(-(c + t) // block) if t else 0):
                    lo, hi = max(c, j * block), min(c + t, (j + 1) * block)
                    p, at = int(self.table[b, j * block // page]), j * block % page
                    new, sz = y[n0 + lo - c:n0 + hi - c], size[n0 + lo - c:n0 + hi - c]
                    amax = np.abs(new).max((0, 2))
                    scale = now[p, at // block]
                    least = [_power(amax * f) for f in (1 - 2.0**-20, 1 + 2.0**-20)]
                    if lo > j * block:
                        least = [np.maximum(x, old[p, at // block]) for x in least]
                    assert ((scale == least[0]) | (scale == least[1])).all(), (scale, least)
                    kept = slice(at, at + lo - j * block)
                    before, after = was[p, kept] * old[p, at // block][:, None], got[p, kept] * scale[:, None]
                    assert (np.abs(before - after) <= np.where(np.abs(before) >= 2.0**-6 * scale[:, None], 0, 2.0**-10 * scale[:, None])).all()
                    stored = got[p, at + lo - j * block:at + hi - j * block] * scale[:, None]
                    err = np.abs(stored - new)
                    assert (err <= np.maximum(2.0**-4 * np.abs(new), 2.0**-10 * scale[:, None]) + 8 * 2.0**-24 * sz).all()
                    untouched[p, at:at + hi - j * block] = False
                    blocks_left[p, at // block] = False
                n0 += t
            assert (self.c[i].view(torch.uint8).cpu().numpy()[untouched] == self.caches[i].numpy()[untouched]).all()
            assert (now[blocks_left] == old[blocks_left]).all()

    def check_queries(self, out):
        want, size = self.turned(self.q)
        tol = UNIT[self.dtype] * np.abs(want) + 8 * 2.0**-24 * size + 2.0**-25
        assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()


APPENDS = [
    ([0], [1], 16, 2, 256, 64, 64, 64, torch.bfloat16, False),
    ([7], [8], 16, 2, 256, 64, 64, 32, torch.bfloat16, False),
    ([63], [2], 4, 2, 256, 256, 64, 64, torch.float16, True),
    ([0, 5, 16, 31, 100], [1, 16, 17, 2, 64], 8, 4, 128, 128, 32, 16, torch.bfloat16, False),
    ([30], [301], 6, 3, 64, 32, 48, 16, torch.float16, True),
    ([0, 0, 40], [0, 70, 0], 12, 12, 64, 64, 64, 64, torch.bfloat16, False),
    ([3], [20], 2, 1, 128, 40, 16, 16, torch.bfloat16, False),   # 20 pairs: no 16-byte vectors
    ([3], [20], 2, 1, 128, 22, 16, 16, torch.float16, True),
    ([9], [40], 2, 1, 64, 2, 32, 32, torch.bfloat16, False),     # one pair
    ([9], [40], 7, 7, 128, 32, 64, 64, torch.float16, False),
]


@pytest.mark.parametrize("args", APPENDS, ids=str)
def test_append(args):
    case = Append(*args)
    out = case.run()
    _fx().check_device_errors()
    case.check_queries(out)
    case.check_stored()


@pytest.mark.parametrize("pad,shift", [(8, 0), (3, 0), (0, 1)])
def test_append_strides_and_alignment(pad, shift):
    case = Append([17, 4], [9, 40], 4, 2, 128, 64, 32, 16, torch.bfloat16, seed=3, pad=pad, shift=shift)
    out = case.run()
    case.check_queries(out)
    case.check_stored()


@pytest.mark.parametrize("rotated", [64, 40])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_in_place(rotated, interleaved):
    case = Append([17], [9], 5, 2, 64, rotated, 32, 16, torch.float16, interleaved, seed=4)
    want = case.run().clone()
    out = case.run(out=case.q)
    assert out is case.q and torch.equal(out, want)


@pytest.mark.parametrize("size", [2.0**-60, 2.0**-20, 300.0, 2.0**40])
def test_append_sizes_of_elements(size):
    """Blocks that grow by many powers of two, shrink not, and elements below the smallest scale's."""
    case = Append([10, 16], [30, 7], 2, 2, 128, 64, 32, 16, torch.bfloat16, seed=5, size=size)
    case.run()
    case.check_stored()


def test_append_zeros_and_elements_that_are_not_finite():
    case = Append([0, 16], [16, 16], 2, 2, 64, 32, 16, 16, torch.float16, seed=6)
    case.k[:16] = 0
    case.v[16:, 0, 3] = float("inf")
    case.v[20, 1, 5] = float("nan")
    case.v[21, 1, 6] = -float("inf")
    case.run()
    p0, p1 = int(case.table[0, 0]), int(case.table[1, 1])
    assert (case.s[0][p0] == 2.0**-40).all() and not case.c[0][p0].float().any()
    finite = case.v[16:].float().clone()
    finite[~finite.isfinite()] = 0
    amax = finite.abs().amax((0, 2)).double().cpu().numpy()
    assert (case.s[1][p1, 0].double().cpu().numpy() == _power(amax)).all()
    got = case.c[1][p1].float()
    assert torch.equal(got.isnan(), ~case.v[16:].isfinite())


def test_append_with_odd_old_scales():
    """Old scales that no append writes: others than powers of two are rounded up, what is no scale counts as the smallest."""
    case = Append([8, 8, 8, 8], [2, 2, 2, 2], 2, 1, 64, 32, 16, 16, torch.float16, seed=7, size=2.0**-14)
    pages = [int(case.table[b, 0]) for b in range(4)]
    for p, s in zip(pages, (3.0, float("nan"), 0.0, -1.0)):
        case.scales[1][p] = s
    case.run()
    assert float(case.s[1][pages[0]]) == 4.0
    old = case.caches[1][pages[0], :8].view(E4M3).float() * 0.75
    assert torch.equal(case.c[1][pages[0], :8].cpu().float(), old.to(E4M3).float())
    for p in pages[1:]:
        assert float(case.s[1][p]) == _power(float(case.v[2 * pages.index(p):][:2].abs().max()))


def test_append_tells_bad_arguments():
    fx = _fx()
    i32 = dict(dtype=torch.int32, device=dev())

    def code():
        with pytest.raises(fx.DeviceWaitError) as e:
            fx.check_device_errors()
        return e.value.codes[0][1]

    def untouched(case):
        return all(torch.equal(a.view(torch.uint8).cpu(), b) for a, b in zip(case.c, case.caches))

    case = Append([5], [4], 2, 1, 64, 32, 16, 16, torch.bfloat16)
    case.run(ctx=torch.tensor([-1], **i32))
    assert code() == 14 and untouched(case)
    case.run(ctx=torch.tensor([13], **i32))
    assert code() == 14 and untouched(case)
    case.run(off=torch.tensor([0, 5], **i32))
    assert code() == 14 and untouched(case)
    case.run(off=torch.tensor([-1, 3], **i32))
    assert code() == 14 and untouched(case)
    case.table[0, 0] = case.pages
    case.run()
    assert code() == 15 and untouched(case)
    case = Append([5], [4], 2, 1, 64, 32, 16, 16, torch.bfloat16)
    case.pos[1] = 3000
    case.run()
    assert code() == 12


def test_append_rows_of_no_request():
    """Rows ahead of the first request and behind the last one are rotated and not stored."""
    case = Append([3], [12], 4, 2, 64, 32, 16, 16, torch.bfloat16, seed=8)
    whole = case.run().clone()
    i32 = dict(dtype=torch.int32, device=dev())
    out = case.run(off=torch.tensor([2, 5], **i32))
    _fx().check_device_errors()
    assert torch.equal(out, whole)
    p = int(case.table[0, 0])
    changed = (case.c[1].view(torch.uint8).cpu() != case.caches[1]).any(-1).any(-1).nonzero().tolist()
    assert all(page == p and at < 6 for page, at in changed)


def test_append_captured_follows_lengths():
    case = Append([3], [12], 4, 2, 64, 32, 64, 16, torch.bfloat16, seed=9)
    fx, d = _fx(), dev()
    i32 = dict(dtype=torch.int32, device=d)
    ctx, off = torch.tensor([3], **i32), torch.tensor([0, 12], **i32)
    pos, table = case.pos.to(d), case.table.to(d)
    caches, scales = [x.to(d).view(E4M3) for x in case.caches], [x.to(d) for x in case.scales]
    fx.prealloc(d)

    def call():
        return fx.rotary_append8(case.q, case.k, case.v, pos, ctx, off, table, case.rot, *caches, *scales)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for c in (3, 0, 16, 50):
        for x, y in zip(caches + scales, case.caches + case.scales):
            x.view(torch.uint8 if x.dtype == E4M3 else torch.float32).copy_(y)
        ctx.fill_(c)
        graph.replay()
        case.lens = [c]
        case.c, case.s = caches, scales
        case.check_stored()


class Attention:
    def __init__(self, lens, counts, Hq, Hk, D, page, block, dtype, seed=0, spread=1.0, vary=2, how="tree"):
        rng, g, d = np.random.default_rng(seed), torch.Generator().manual_seed(seed), dev()
        self.lens, self.counts, self.page, self.block = lens, counts, page, block
        need = [-(-(c + t) // page) for c, t in zip(lens, counts)]
        pages = sum(need) + 2
        order = rng.permutation(pages)
        table = np.full((len(lens), max(max(need), 1) + 1), -12345, np.int32)
        at = 0
        used = torch.zeros(pages, page, dtype=torch.bool)
        for b, (n, c, t) in enumerate(zip(need, lens, counts)):
            table[b, :n] = order[at:at + n]
            at += n
            p = np.arange(c + t)
            used[torch.from_numpy(table[b][p // page]).long(), torch.from_numpy(p % page).long()] = True
        self.table = torch.from_numpy(table).to(d)
        self.c, self.s = [], []
        for _ in range(2):
            x = torch.randint(0, 256, (pages, page, Hk, D), generator=g, dtype=torch.uint8)
            x[(x & 0x7F) == NAN] = 9
            x[~used] = NAN  # places of no token hold anything
            s = torch.exp2(torch.randint(-vary, vary + 1, (pages, page // block, Hk), generator=g).float())
            s *= 2.0**-5 * torch.where(torch.rand(s.shape, generator=g) < 0.5, 1.0, 1.37)  # any scales are read
            s[~used.view(pages, -1, block).any(-1)] = float("nan")
            self.c.append(x.to(d).view(E4M3))
            self.s.append(s.to(d))
        N = sum(counts)
        self.q = (torch.randn(N, Hq, D, generator=g) * spread * 0.3).to(dtype).to(d)
        self.masks = []
        for t in counts:
            seen = []
            for i in range(t):
                parent = int(rng.integers(-1, i)) if i else -1
                seen.append(0 if how == "none" else (seen[parent] if parent >= 0 else 0) | 1 << i)
            self.masks += seen
        self.mask = torch.tensor([m - (1 << 64) if m >> 63 else m for m in self.masks], dtype=torch.int64, device=d)
        self.offsets = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=d)
        self.ctx = torch.tensor(lens, dtype=torch.int32, device=d)

    def run(self, **kw):
        args = dict(max_nodes=max(max(self.counts), 1), max_context=max(self.lens), tree_mask=self.mask) | kw
        return _fx().tree_attention8(self.q, *self.c, *self.s, self.table, self.ctx, self.offsets, **args)

    def cached(self, i, b, n):
        p = torch.arange(n, device=dev())
        page, at = self.table[b].long()[p // self.page], p % self.page
        return self.c[i].view(torch.uint8)[page, at].view(E4M3).double() * self.s[i][page, at // self.block].double()[..., None]

    def reference(self, scale=None):
        N, Hq, D = self.q.shape
        G = Hq // self.c[0].shape[2]
        out = torch.zeros(N, Hq, D, dtype=torch.float64, device=dev())
        mean, lse = torch.zeros_like(out), torch.full((N, Hq), -float("inf"), dtype=torch.float64, device=dev())
        big = torch.ones(N, Hq, dtype=torch.float64, device=dev())
        n = 0
        for b, (c, t) in enumerate(zip(self.lens, self.counts)):
            keys, vals = (self.cached(i, b, c + t) for i in (0, 1))
            for i in range(t):
                see = torch.tensor([True] * c + [bool(self.masks[n] >> j & 1) for j in range(t)], device=dev())
                if bool(see.any()):
                    kk, vv = (x[see].repeat_interleave(G, 1) for x in (keys, vals))
                    s = torch.einsum("hd,khd->hk", self.q[n].double(), kk) * (D**-0.5 if scale is None else scale)
                    w = torch.softmax(s, 1)
                    out[n], mean[n] = torch.einsum("hk,khd->hd", w, vv), torch.einsum("hk,khd->hd", w, vv.abs())
                    lse[n], big[n] = torch.logsumexp(s, 1), s.abs().amax(1).clamp(min=1)
                n += 1
        return out, mean, lse, big

    def check(self, scale=None, **kw):
        out, lse = self.run(**(kw | ({} if scale is None else {"scale": scale})))
        _fx().check_device_errors()
        want, mean, wlse, big = self.reference(scale)
        err = (out.double() - want).abs()
        tol = (2.0**-11 + 2.0**-12 + 2.0**-17) * mean + UNIT[self.q.dtype] * want.abs() + 2.0**-25
        ok = (err <= tol) | (want.isnan() & out.isnan())
        assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} off, worst {float((err - tol)[~ok].max())}"
        empty = wlse == -float("inf")
        assert torch.equal(lse == -float("inf"), empty) and not bool(out[empty].any())
        bad = (lse.double() - wlse).abs()[~empty] > 2.0**-12 * big[~empty]
        assert not bool((bad & ~wlse[~empty].isnan()).any())
        return out, lse


SHAPES = [
    ([1000], [1], 16, 2, 256, 64, 64, torch.bfloat16),
    ([0], [1], 4, 2, 64, 16, 16, torch.float16),
    ([0, 1, 15, 16, 63, 64, 65], [1, 2, 1, 3, 2, 1, 5], 4, 4, 64, 16, 16, torch.bfloat16),
    ([300, 9, 2000], [3, 1, 4], 4, 1, 256, 32, 16, torch.float16),
    ([1000], [16], 8, 2, 128, 64, 32, torch.bfloat16),
    ([517, 64, 1], [17, 64, 33], 12, 12, 64, 48, 16, torch.bfloat16),
    ([130, 700], [40, 7], 8, 1, 256, 96, 32, torch.bfloat16),
    ([5000, 100, 3001, 64], [4, 1, 9, 16], 32, 8, 128, 16, 16, torch.float16),
    ([9000], [64], 16, 4, 128, 256, 64, torch.bfloat16),
    ([20000, 7], [16, 2], 16, 2, 256, 64, 32, torch.bfloat16),
    ([12000, 2], [60, 3], 12, 4, 64, 64, 16, torch.float16),
    ([20000], [1], 16, 2, 256, 64, 64, torch.bfloat16),
    ([9000, 3001], [2, 1], 24, 4, 64, 64, 32, torch.float16),
    ([6000, 129, 2500], [3, 1, 4], 32, 8, 128, 32, 16, torch.bfloat16),
]


@pytest.mark.parametrize("args", SHAPES, ids=str)
def test_attention(args):
    Attention(*args).check()


@pytest.mark.parametrize("args", SHAPES, ids=str)
def test_attention_bounds_far_from_the_lengths(args):
    """Loose bounds take the tensor-memory form whatever the lengths are."""
    Attention(*args, seed=1).check(max_context=10**7, max_nodes=64)


@pytest.mark.parametrize("D,Hq,Hk", [(64, 8, 2), (128, 8, 2), (256, 8, 2)])
@pytest.mark.parametrize("lens,counts", [([200], [8]), ([15000], [40])])
def test_attention_of_rows_that_see_nothing(lens, counts, D, Hq, Hk):
    """Masks without a bit and no context: 0 and -inf; with context: the context alone."""
    Attention(lens, counts, Hq, Hk, D, 32, 16, torch.bfloat16, how="none").check()
    case = Attention([0] + lens, [5] + counts, Hq, Hk, D, 32, 16, torch.bfloat16, how="none")
    out, lse = case.check()
    assert not bool(out[:5].any()) and bool((lse[:5] == -float("inf")).all())


@pytest.mark.parametrize("lens,counts,D", [([120], [12], 128), ([120], [12], 64), ([70], [9], 256), ([16000], [33], 128),
                                           ([9000], [33], 256), ([16000], [20], 64)])
def test_attention_nan_reaches_the_rows_that_see_it(lens, counts, D):
    case = Attention(lens, counts, 8, 2, D, 32, 16, torch.float16, seed=2)
    place = lens[0] + 4
    page, at = int(case.table[0, place // 32]), place % 32
    for x in case.c:
        x.view(torch.uint8)[page, at, 1, 3:7] = NAN
    out, lse = case.run()
    want, mean, wlse, _ = case.reference()
    sees = torch.tensor([bool(m >> 4 & 1) for m in case.masks], device=dev())
    assert torch.equal(lse.isnan(), wlse.isnan()) and bool(lse[sees][:, 4:].isnan().all()) and not bool(lse[~sees].isnan().any())
    assert not bool(out[~sees].isnan().any()) and not bool(out[:, :4].isnan().any())
    ok = (out.double() - want).abs() <= (2.0**-11 + 2.0**-12 + 2.0**-17) * mean + 2.0**-11 * want.abs() + 2.0**-25
    assert bool(ok[~sees].all()) and bool(ok[:, :4].all())
    # a value alone: the row's elements that it has
    case = Attention(lens, counts, 8, 2, D, 32, 16, torch.float16, seed=2)
    case.c[1].view(torch.uint8)[page, at, 1, 3:7] = NAN
    out, _ = case.run()
    assert torch.equal(out.isnan(), case.reference()[0].isnan()) and bool(out[sees][:, 4:, 3:7].isnan().all())


@pytest.mark.parametrize("lens,counts,D", [([400], [4], 128), ([400], [9], 64), ([300], [4], 256), ([30000], [30], 128),
                                           ([30000], [16], 256)])
def test_attention_scales_far_apart(lens, counts, D):
    """Blocks whose values are 2^30 larger have so much smaller weights, and the other way round: each row's result is
    a sum of both, in which neither is lost."""
    case = Attention(lens, counts, 8, 2, D, 64, 16, torch.bfloat16, seed=3, spread=0.05)
    for s in case.s:
        s.copy_(torch.where(s.isnan(), s, 2.0**-6))
    far = torch.rand(case.s[1].shape, generator=torch.Generator().manual_seed(1)).to(dev()) < 0.3
    # keys of those blocks lie against the queries, which all look the same way
    case.q.copy_(case.q.abs() * 12)
    k = case.c[0].view(torch.uint8).unflatten(1, (-1, 16))
    k.copy_(torch.where(far[:, :, None, :, None] & (k != NAN), k | 0x80, k))
    case.s[1].mul_(torch.where(far, 2.0**30, 1.0))
    case.check()
    case.s[1].mul_(torch.where(far, 2.0**-60, 1.0))
    case.check()


def test_attention_tells_bad_scales_and_pages():
    fx = _fx()
    case = Attention([100], [3], 4, 2, 64, 16, 16, torch.bfloat16)
    page = int(case.table[0, 2])
    case.s[1][page, 0, 1] = float("nan")
    case.run()
    with pytest.raises(fx.DeviceWaitError, match="SCALE"):
        fx.check_device_errors()
    case.s[1][page, 0, 1] = 2.0**-40
    case.check()
    case.s[0][page, 0, 0] = 0.0
    case.run()
    with pytest.raises(fx.DeviceWaitError, match="SCALE"):
        fx.check_device_errors()
    case = Attention([100], [3], 4, 2, 64, 16, 16, torch.bfloat16)
    case.table[0, 2] = case.c[0].shape[0]
    case.run()
    with pytest.raises(fx.DeviceWaitError, match="PAGE"):
        fx.check_device_errors()
    case = Attention([100], [3], 4, 2, 64, 16, 16, torch.bfloat16)
    case.ctx.fill_(10**6)
    out, lse = case.run()
    assert not bool(out.any()) and bool((lse == -float("inf")).all())
    with pytest.raises(fx.DeviceWaitError, match="LENGTHS"):
        fx.check_device_errors()


@pytest.mark.parametrize("size", [2.0**-110, 2.0**-30, 2.0**60])
def test_attention_sizes_of_queries(size):
    case = Attention([300, 20000], [5, 17], 8, 2, 128, 32, 16, torch.bfloat16, seed=4)
    case.q.mul_(size)
    case.check(scale=min(max(128**-0.5 / size, 1e-37), 1e37))


def test_attention_strided_arguments_and_destinations():
    case = Attention([200, 31], [6, 3], 4, 2, 128, 32, 16, torch.float16, seed=5)
    want, wlse = case.run()
    N = 9
    case.c = [torch.cat([x.view(torch.uint8), x.view(torch.uint8)], -1).view(E4M3)[..., :128] for x in case.c]
    case.s = [torch.stack([x, x * 0], -1)[..., 0] for x in case.s]
    case.q = torch.cat([case.q, case.q], 1)[:, :4]
    out = torch.zeros(N, 8, 128, dtype=torch.float16, device=dev())[:, ::2]
    lse = torch.empty(N, 4, device=dev())
    got, glse = case.run(out=out, lse=lse)
    assert got is out and glse is lse and torch.equal(out, want) and torch.equal(lse, wlse)


def test_attention_more_requests_than_a_launch_holds():
    lens = [(37 * b) % 211 for b in range(300)]
    Attention(lens, [1 + b % 3 for b in range(300)], 4, 2, 64, 16, 16, torch.bfloat16, seed=6).check()


def test_attention_is_the_same_every_time_and_captured():
    fx = _fx()
    fx.prealloc(dev(), attention=True)
    for args in (SHAPES[4], SHAPES[7], SHAPES[8], SHAPES[9]):
        case = Attention(*args, seed=7)
        out, lse = case.run()
        for _ in range(3):
            a, b = case.run()
            assert torch.equal(a, out) and torch.equal(b, lse)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a, b = case.run()
        for c in case.lens, [max(0, x - 70) for x in case.lens]:
            case.ctx.copy_(torch.tensor(c, dtype=torch.int32))
            graph.replay()
            want = case.run(max_context=max(case.lens))
            assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_argument_errors():
    fx = _fx()
    case = Attention([50], [2], 4, 2, 64, 16, 16, torch.bfloat16)
    good = dict(c=case.c, s=case.s, q=case.q)

    def attend(**kw):
        x = good | kw
        return fx.tree_attention8(x["q"], *x["c"], *x["s"], case.table, case.ctx, case.offsets)

    attend()
    with pytest.raises(ValueError):
        attend(c=[x.view(torch.uint8) for x in case.c])
    with pytest.raises(ValueError):
        attend(c=[x.view(torch.uint8).view(torch.float8_e5m2) for x in case.c])
    with pytest.raises(ValueError):
        attend(s=[x.double() for x in case.s])
    with pytest.raises(ValueError):
        attend(s=[x[:, :, :1] for x in case.s])
    with pytest.raises(ValueError):
        attend(s=[case.s[0], case.s[1][:1]])
    with pytest.raises(NotImplementedError):
        attend(s=[x.repeat(1, 2, 1) for x in case.s])  # blocks of 8
    with pytest.raises(NotImplementedError):
        attend(q=case.q.float())
    with pytest.raises(ValueError):
        attend(q=case.q[:, :3])
    with pytest.raises(ValueError):
        attend(q=torch.cat([case.q, case.q], -1))
    ap = Append([5], [4], 2, 1, 64, 32, 16, 16, torch.bfloat16)
    ap.k = ap.k[:3]
    with pytest.raises(ValueError):
        ap.run()
    ap = Append([5], [4], 2, 1, 64, 32, 16, 16, torch.bfloat16)
    ap.v = ap.v.half()
    with pytest.raises(ValueError):
        ap.run()
    ap = Append([5], [4], 2, 1, 64, 32, 16, 16, torch.bfloat16)
    with pytest.raises(ValueError):
        ap.run(off=torch.zeros(5, dtype=torch.int32, device=dev()))
