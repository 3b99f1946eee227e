"""token_probs, verify_tokens and compact_nodes on the GPU.

token_probs: against the definition in 64 bits.  The weights come from fp32 exponentials (an argument of up to 28 rounded
at 2^-24 moves a weight by less than 28 * 2^-23 + 2^-22 < 2^-18, as for sample_tokens), so probabilities are within
2^-17, relatively, or 2^-40 (a weight's last bit) of those that some top-p within that share of the given one gives.

verify_tokens: against a walk in 64-bit numbers.  An element of what refusals leave is rounded to 32 bits in each
(2^-24 of it, carried through 1 / S of the later ones, S at least 2^-4 in these cases and one after another at most
twice below 2^-1), and sums of whole numbers lose less than V 2^-52: a comparison or a draw that lies within NEAR_CHOICE =
2^-18 of its border may fall either way, and no other.

compact_nodes: exact, but for elements of an 8-bit cache that take another scale: within 2^-10 of it where they fall below
2^-6 of it, exact above (powers of two)."""

import numpy as np
import pytest
import torch

from tests.gpu_util import dev
from tests.test_gpu_sampling import NEAR

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
NEAR_CHOICE = 2.0**-18


def _fx():
    import flash_next_rtxpro6000_b200 as fx

    return fx


# ------------------------------------------------------------------------------------ token_probs


def _kept(x, t, k, p, mp):
    """The probabilities of one float64 row."""
    x = np.where(np.isnan(x), -np.inf, x)
    out = np.zeros(len(x))
    order = np.lexsort((np.arange(len(x)), -x))
    if x.max() == -np.inf:
        return out
    if not t > 0:
        out[order[0]] = 1.0
        return out
    with np.errstate(invalid="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / t))[order]
    n = len(x) if k < 1 else min(k, len(x))
    cum = np.cumsum(w[:n])
    if p < 1:
        n = max(1, int(np.searchsorted(cum - w[:n], p * cum[-1], side="left")))
    if mp > 0:
        n = max(1, min(n, int((w >= min(mp, 1.0)).sum())))
    out[order[:n]] = w[:n] / w[:n].sum()
    return out


def _check_probs(logits, t=None, k=None, p=None, mp=None, **kw):
    fx = _fx()
    got = fx.token_probs(logits, t, k, p, mp, **kw)
    assert got.dtype == torch.float32 and torch.equal(got, fx.token_probs(logits, t, k, p, mp))
    M = logits.shape[0]
    val = lambda x, d: [d] * M if x is None else x.double().cpu().tolist()  # noqa: E731
    rows, mine = logits.double().cpu().numpy(), got.double().cpu().numpy()
    tt, kk, pp, mm = val(t, 1.0), val(k, 0), val(p, 1.0), val(mp, 0.0)
    for m in range(M):
        fit = []
        for dp, dm in ((0, 0), (NEAR, 0), (-NEAR, 0), (0, NEAR), (0, -NEAR)):
            want = _kept(rows[m], tt[m], int(kk[m]), pp[m] + dp if 0 < pp[m] < 1 else pp[m], mm[m] * (1 + dm) if mm[m] < 1 else mm[m])
            fit.append((np.abs(mine[m] - want) <= 2.0**-17 * want + 2.0**-39).all())
        assert any(fit), (m, tt[m], kk[m], pp[m], mm[m])
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,V", [(1, 1), (3, 2), (5, 17), (16, 1000), (33, 4099), (16, 49152), (8, 151936), (24, 60001)])
def test_probs_against_64_bits(dtype, M, V):
    g, d = torch.Generator().manual_seed(M * 37 + V), dev()
    x = torch.randn(M, V, generator=g) * 3
    x[:, torch.randint(0, V, (min(V, 40),), generator=g)] += torch.rand(min(V, 40), generator=g) * 10
    x[torch.rand(M, V, generator=g) < 0.1] = -float("inf")
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (M,), generator=g)].to(d)  # noqa: E731
    x = x.to(dtype).to(d)
    _check_probs(x, pick(0.0, 0.3, 0.7, 1.0, 1.5, 30.0), pick(0, -1, 1, 2, 50, 700, 1500, 10**6).int(),
                 pick(0.0, 0.1, 0.5, 0.9, 0.99, 1.0, 2.0), pick(0.0, 0.0, 0.01, 0.2, 1.0, 3.0))
    _check_probs(x)
    _check_probs(x, mp=pick(0.0, 0.1, 0.9))


def test_probs_ties_and_rows_of_nothing():
    d = dev()
    x = torch.zeros(4, 3000, device=d)
    x[1] = -float("inf")
    x[2] = float("nan")
    x[3, 7] = float("inf")
    got = _check_probs(x, None, torch.tensor([5, 5, 5, 5], dtype=torch.int32, device=d))
    assert got[0].nonzero().flatten().tolist() == [0, 1, 2, 3, 4] and not got[1:3].any()
    assert got[3].nonzero().flatten().tolist() == [7] and float(got[3, 7]) == 1.0
    got = _check_probs(x, p=torch.full((4,), 0.5, device=d))
    assert int((got[0] > 0).sum()) == 1500 and float(got[0, 1499]) > 0


@pytest.mark.parametrize("M", [3, 40])  # few rows, many
@pytest.mark.parametrize("T", [2.0**-70, 2.0**-60, 0.001, 0.9999999, 7.3, 2.0**60, 2.0**70])
def test_probs_at_temperatures_of_any_size(M, T):
    """Logits of the temperature's size, unfiltered and not; some infinite, some NaN."""
    g, d = torch.Generator().manual_seed(M), dev()
    x = torch.randn(M, 20011, generator=g) * 3 * T
    x[torch.rand(M, 20011, generator=g) < 0.05] = -float("inf")
    x[0, 7] = float("inf")
    x[1, 70:90] = float("nan")
    x[2, 5:] = -float("inf")
    x, t = x.to(d), torch.full((M,), T, device=d)
    _check_probs(x, t)
    _check_probs(x, t, p=torch.full((M,), 0.9, device=d))
    _check_probs(x, t, mp=torch.full((M,), 0.05, device=d))


@pytest.mark.parametrize("M", [3, 40])
def test_probs_are_what_sampling_draws_from(M):
    fx, d = _fx(), dev()
    g = torch.Generator().manual_seed(M)
    x = (torch.randn(M, 30011, generator=g) * 4).bfloat16().to(d)
    t, k = torch.full((M,), 0.8, device=d), (torch.arange(M, device=d) % 4 * 30).int()
    p, mp = 0.7 + torch.arange(M, device=d) % 5 * 0.1, (torch.arange(M, device=d) % 3) * 0.01
    probs = fx.token_probs(x, t, k, p, mp)
    for u in (0.0, 0.3, 0.99999):
        tokens, share = fx.sample_tokens(x, torch.full((M,), u, device=d), t, k, p, mp)
        mine = probs.gather(1, tokens[:, None])[:, 0]
        assert bool(((mine - share).abs() <= 2.0**-23 * share).all())  # a product against a division, rounded


def test_probs_strides_and_destinations():
    fx, d = _fx(), dev()
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 2003, generator=g).to(d)
    want = fx.token_probs(x, top_k=torch.full((5,), 40, dtype=torch.int32, device=d))
    wide = torch.full((5, 2100), 9.0, device=d)
    k = torch.full((5,), 40, dtype=torch.int32, device=d)
    got = fx.token_probs(torch.nn.functional.pad(x, (3, 7))[:, 3:-7], top_k=k, out=wide[:, 1:2004])
    assert torch.equal(got, want) and torch.equal(wide[:, 1:2004], want)
    assert bool((wide[:, 0] == 9).all()) and bool((wide[:, 2004:] == 9).all())
    with pytest.raises(ValueError):
        fx.token_probs(x, out=x)
    with pytest.raises(ValueError):
        fx.token_probs(x, out=torch.empty(5, 2002, device=d))
    with pytest.raises(ValueError):
        fx.token_probs(x, out=torch.empty(5, 2003, device=d, dtype=torch.bfloat16))
    with pytest.raises(NotImplementedError):
        fx.token_probs(x.double())
    with pytest.raises(ValueError):
        fx.token_probs(x, torch.ones(4, device=d))


# ---------------------------------------------------------------------------------- verify_tokens


class Drafts:
    def __init__(self, counts, V, seed=0, drafts=True, sharp=3.0, noise=1.0, chain=False, siblings=4, pad=0):
        rng = np.random.default_rng(seed)
        N = sum(counts)
        x = rng.standard_normal((N, V)) * sharp
        soft = lambda z: (lambda e: e / e.sum(1, keepdims=True))(np.exp(z - z.max(1, keepdims=True)))  # noqa: E731
        self.p = soft(x).astype(np.float32)
        q = soft(x + rng.standard_normal((N, V)) * noise).astype(np.float32)
        self.q = q if drafts else None
        self.counts, self.V = counts, V
        self.parents, self.tokens = [], []
        for t in counts:
            n0 = len(self.parents)
            for i in range(t):
                parent = -1 if i == 0 else i - 1 if chain else int(rng.integers(max(0, (i - 1) // siblings), i))
                row = q[n0 + max(parent, 0)].astype(np.float64)
                self.parents.append(parent)
                self.tokens.append(int(rng.choice(V, p=row / row.sum())))
        self.u, self.w = rng.random(N).astype(np.float32), rng.random(len(counts)).astype(np.float32)
        self.off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.pad = pad

    def run(self, **kw):
        d = dev()
        rows = lambda x: None if x is None else torch.nn.functional.pad(torch.from_numpy(x), (0, self.pad)).to(d)[:, : self.V]  # noqa: E731
        to = lambda x, t: torch.tensor(x, dtype=t, device=d)  # noqa: E731
        args = dict(max_nodes=max(max(self.counts), 1)) | kw
        return _fx().verify_tokens(rows(self.p), rows(self.q), to(self.tokens, torch.int64), to(self.parents, torch.int32),
                                   to(self.off, torch.int32), to(self.u, torch.float32), to(self.w, torch.float32), **args)

    def walk(self, b, nudge=0.0):
        """(path, residual) of request b; `nudge` is added to every threshold, relatively."""
        n0, n = int(self.off[b]), int(self.off[b + 1] - self.off[b])
        clean = lambda x: np.clip(np.nan_to_num(x.astype(np.float64), nan=0.0), 0, 1)  # noqa: E731
        path, r, s = [0], clean(self.p[n0]), 1.0
        for i in range(1, n):
            if self.parents[n0 + i] != path[-1]:
                continue
            x, u = self.tokens[n0 + i], float(self.u[n0 + i])
            if self.q is None:
                ok = u * s < r[x] * (1 + nudge)
                if not ok:
                    s = max(s - r[x], 0.0)
                    r = r.copy()
                    r[x] = 0.0
            else:
                q = clean(self.q[n0 + path[-1]])
                ok = u * q[x] < r[x] / s * (1 + nudge)
                if not ok:
                    rest = np.maximum(r / s - q, 0.0)
                    if np.floor(rest * 2.0**52).sum() > 0:
                        r, s = rest, rest.sum()
            if ok:
                path.append(i)
                r, s = clean(self.p[n0 + i]), 1.0
        return path, r

    def check(self, **kw):
        path, accepted, tokens = self.run(**kw)
        again = self.run(**kw)
        assert all(torch.equal(a, b) for a, b in zip((path, accepted, tokens), again))
        for b in range(len(self.counts)):
            got = [x for x in path[b].tolist() if x >= 0]
            assert len(got) == int(accepted[b]) and path[b].tolist()[len(got):] == [-1] * (path.shape[1] - len(got))
            if self.counts[b] == 0:
                assert got == [] and int(tokens[b]) == -1
                continue
            found = [self.walk(b, e) for e in (0.0, NEAR_CHOICE, -NEAR_CHOICE)]
            fit = [r for p, r in found if p == got]
            assert fit, (b, got, [p for p, _ in found])
            t = int(tokens[b])
            right = []
            for r in fit:
                if np.floor(r * 2.0**52).sum() == 0:
                    right.append(t == -1)
                    continue
                cum = np.cumsum(r)
                aim = float(np.clip(self.w[b], 0, 1)) * cum[-1]
                lo = cum[t - 1] if t > 0 else 0.0
                right.append(t >= 0 and r[t] > 0 and lo - NEAR_CHOICE * cum[-1] <= aim <= cum[t] + NEAR_CHOICE * cum[-1])
            assert any(right), (b, t)
        return path, accepted, tokens


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("chain", [True, False])
@pytest.mark.parametrize("counts,V", [([1], 1000), ([6], 151936), ([5, 1, 0, 16, 2], 4096), ([64], 3001), ([9] * 20, 517),
                                      ([4, 4], 1), ([7] * 6, 2), ([33, 64, 12], 250)])
def test_verify_against_64_bits(counts, V, chain, drafts):
    case = Drafts(counts, V, seed=V + len(counts), drafts=drafts, chain=chain)
    case.check()
    _fx().check_device_errors()


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("sharp,noise", [(0.1, 0.0), (0.1, 3.0), (6.0, 6.0)])
def test_verify_drafters_near_and_far(sharp, noise, drafts):
    """The drafter's own distribution (all accepted where tokens are drawn from it), and others."""
    case = Drafts([17] * 12, 700, seed=5, drafts=drafts, sharp=sharp, noise=noise, chain=True)
    _, accepted, _ = case.check()
    if noise == 0.0 and drafts:
        assert bool((accepted == 17).all())


def test_verify_many_siblings():
    """Every node a child of node 0, refused one after the other: one residual on top of the other."""
    case = Drafts([40, 64], 60, seed=6, sharp=2.0, noise=2.0)
    case.parents = [-1] + [0] * 39 + [-1] + [0] * 63
    case.u[:] = 0.9999999
    case.check()
    case.q = None
    case.check()


@pytest.mark.parametrize("pad,V", [(3, 4001), (4, 4000), (1, 4000)])
def test_verify_row_strides(pad, V):
    Drafts([8, 5], V, seed=7, pad=pad).check()


def test_verify_edges_of_random_numbers_and_probabilities():
    case = Drafts([5, 5, 5, 5, 5, 5], 300, seed=8, chain=True)
    case.w[:] = [0.0, 1.0, -3.0, 2.0, float("nan"), 1 - 2.0**-24]
    case.u[:15] = 0.0
    path, accepted, tokens = case.run()
    assert accepted[:3].tolist() == [5, 5, 5]
    for b, r in ((0, "first"), (1, "last"), (2, "first"), (3, "last"), (4, "first")):
        left = case.walk(b)[1]
        some = np.flatnonzero(np.floor(left * 2.0**52) > 0)
        assert int(tokens[b]) == (some[0] if r == "first" else some[-1])
    # zeros, NaN and others than probabilities
    case = Drafts([4, 4, 4], 300, seed=9, chain=True)
    case.p[:4] = 0.0
    case.p[4:8, ::3] = np.nan
    case.p[4:8, 1::3] = -1.0
    case.q[5, 7] = np.nan
    case.check()
    # a token of probability 0 under both is refused whatever its random number
    case = Drafts([2], 300, seed=10)
    case.p[0, case.tokens[1]] = case.q[0, case.tokens[1]] = 0.0
    case.u[:] = 0.0
    _, accepted, _ = case.check()
    assert accepted.tolist() == [1]


@pytest.mark.parametrize("drafts", [True, False])
def test_verify_gives_the_targets_distribution(drafts):
    """The first token after node 0, accepted or drawn, over 40,000 requests with trees of a chain and siblings: its
    frequencies are the target's, within five standard deviations of each."""
    B, V, d = 40000, 12, dev()
    g = torch.Generator().manual_seed(11)
    p = torch.softmax(torch.randn(V, generator=g) * 1.5, 0)
    q = torch.softmax(torch.randn(V, generator=g) * 1.5, 0)
    n = 4  # node 0, two children of it, a child of the first
    if drafts:
        tokens = torch.multinomial(q, B * n, replacement=True, generator=g).view(B, n)
    else:
        tokens = p.topk(4).indices[[3, 1, 0, 2]].expand(B, n).contiguous()
    parents = torch.tensor([-1, 0, 0, 1], dtype=torch.int32).repeat(B)
    path, accepted, last = _fx().verify_tokens(
        p.to(d).expand(B * n, V).contiguous(), q.to(d).expand(B * n, V).contiguous() if drafts else None,
        tokens.flatten().to(d), parents.to(d), torch.arange(0, B * n + 1, n, dtype=torch.int32, device=d),
        torch.rand(B * n, generator=g).to(d), torch.rand(B, generator=g).to(d), max_nodes=n)
    path, accepted, last = path.cpu().long(), accepted.cpu(), last.cpu()
    first = torch.where(accepted > 1, tokens.gather(1, path[:, 1:2].clamp(min=0))[:, 0], last)
    count = torch.bincount(first, minlength=V).double()
    want = p.double() / p.double().sum() * B
    assert bool(((count - want).abs() <= 5 * (want * (1 - want / B)).sqrt() + 1).all())
    # and the second one where the first was accepted by way of node 1
    deep = accepted == 3
    second = torch.bincount(torch.where(deep, tokens[:, 3], last)[path[:, 1] == 1], minlength=V).double()
    total = int((path[:, 1] == 1).sum())
    want = p.double() / p.double().sum() * total
    assert total > 1000 and bool(((second - want).abs() <= 5 * (want * (1 - want / total)).sqrt() + 1).all())


def test_verify_tells_bad_arguments():
    fx = _fx()

    def code(case, **kw):
        out = case.run(**kw)
        with pytest.raises(fx.DeviceWaitError) as e:
            fx.check_device_errors()
        return e.value.codes[0][1], out

    case = Drafts([4, 3], 100, seed=12, chain=True)
    whole = [x.clone() for x in case.run()]
    case.parents[2] = 2
    got, (path, accepted, _) = code(case)
    assert got == 16 and int(accepted[0]) <= 2 and torch.equal(path[1], whole[0][1])
    case = Drafts([4, 3], 100, seed=12, chain=True)
    case.tokens[1] = 100
    got, (path, accepted, tokens) = code(case)
    assert got == 17 and int(accepted[0]) == 1 and 0 <= int(tokens[0]) < 100
    case = Drafts([4, 3], 100, seed=12, chain=True)
    got, (path, accepted, tokens) = code(case, max_nodes=3)
    assert got == 14 and accepted.tolist()[0] == 0 and int(tokens[0]) == -1 and path[0].tolist() == [-1] * 3
    assert torch.equal(path[1], whole[0][1, :3])
    case.off[-1] = 9
    got, (path, accepted, tokens) = code(case)
    assert got == 14 and accepted.tolist()[1] == 0
    with pytest.raises(ValueError):
        fx.verify_tokens(torch.zeros(2, 5, device=dev()), torch.zeros(2, 4, device=dev()), *[torch.zeros(2, device=dev())] * 5)
    with pytest.raises(NotImplementedError):
        Drafts([4], 10, seed=1).run(max_nodes=65)


def test_verify_captured_follows_its_arguments():
    fx, d = _fx(), dev()
    case = Drafts([6, 9, 2], 5003, seed=13)
    to = lambda x, t: torch.tensor(x, dtype=t, device=d)  # noqa: E731
    p, q = torch.from_numpy(case.p).to(d), torch.from_numpy(case.q).to(d)
    args = [to(case.tokens, torch.int64), to(case.parents, torch.int32), to(case.off, torch.int32),
            to(case.u, torch.float32), to(case.w, torch.float32)]
    fx.prealloc(d)
    fx.verify_tokens(p, q, *args, max_nodes=9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fx.verify_tokens(p, q, *args, max_nodes=9)
    for seed in range(14, 18):
        new = Drafts([6, 9, 2], 5003, seed=seed)
        for x, y in zip([p, q] + args, (new.p, new.q, new.tokens, new.parents, new.off, new.u, new.w)):
            x.copy_(torch.as_tensor(np.asarray(y)))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, new.check()))


# ---------------------------------------------------------------------------------- compact_nodes


class Moves:
    def __init__(self, lens, paths, width, layers, Hk, D, page, block, dtype, seed=0):
        g, rng = torch.Generator().manual_seed(seed), np.random.default_rng(seed)
        self.__dict__.update(lens=lens, paths=paths, page=page, block=block, layers=layers, dtype=dtype, Hk=Hk, D=D)
        need = [-(-(c + (max(p) + 1 if p else 0)) // page) for c, p in zip(lens, paths)]
        self.pages = sum(need) + 2
        order = rng.permutation(self.pages)
        self.table = np.full((len(lens), max(max(need), 1)), -5, np.int32)
        for b, n in enumerate(need):
            self.table[b, :n] = order[sum(need[:b]):sum(need[:b]) + n]
        lead = () if layers is None else (layers,)
        self.scales = None
        if block:
            self.caches = [torch.randint(0, 256, (*lead, self.pages, page, Hk, D), generator=g, dtype=torch.uint8) for _ in range(2)]
            for c in self.caches:
                c[(c & 0x7F) == 0x7F] = 3
            self.scales = [torch.exp2(torch.randint(-6, 6, (*lead, self.pages, page // block, Hk), generator=g).float()) for _ in range(2)]
        else:
            self.caches = [torch.randn(*lead, self.pages, page, Hk, D, generator=g).to(dtype) for _ in range(2)]
        self.path = np.full((len(lens), width), -1, np.int32)
        for b, p in enumerate(paths):
            self.path[b, :len(p)] = p
        self.accepted = [len(p) for p in paths]

    def run(self, **kw):
        d = dev()
        i32 = dict(dtype=torch.int32, device=d)
        self.c = [x.to(d).view(E4M3) if self.block else x.to(d) for x in self.caches]
        self.s = [x.to(d) for x in self.scales] if self.block else [None, None]
        args = dict(ctx=self.lens, path=self.path, acc=self.accepted, table=self.table) | kw
        return _fx().compact_nodes(*self.c, torch.tensor(args["table"], **i32), torch.tensor(args["ctx"], **i32),
                                   torch.tensor(args["path"], **i32), torch.tensor(args["acc"], **i32), *self.s)

    def check(self, left=()):
        """`left`: requests that stay as they are."""
        page, block = self.page, self.block
        for i in range(2):
            lead = (lambda x: x if self.layers is not None else x[None])
            if not block:
                want, was = lead(self.caches[i].clone()), lead(self.caches[i])
                for b, (c, p) in enumerate(zip(self.lens, self.paths)):
                    if b in left:
                        continue
                    at = lambda x: (int(self.table[b, x // page]), x % page)  # noqa: E731
                    for d, n in enumerate(p):
                        (p1, o1), (p0, o0) = at(c + d), at(c + n)
                        want[:, p1, o1] = was[:, p0, o0]
                assert torch.equal(lead(self.c[i].cpu()).view(torch.int16), want.view(torch.int16))
                continue
            raw = lead(self.caches[i]).numpy()
            was = lead(self.caches[i]).view(E4M3).double().numpy()
            now = lead(self.c[i].view(torch.uint8).cpu().view(E4M3)).double().numpy()
            old, got = lead(self.scales[i]).double().numpy(), lead(self.s[i].cpu()).double().numpy()
            want, free, vals = old.copy(), np.ones((self.pages, page), bool), {}
            for b, (c, p) in enumerate(zip(self.lens, self.paths)):
                if b in left or all(n == d for d, n in enumerate(p)):
                    continue
                at = lambda x: (int(self.table[b, x // page]), x % page)  # noqa: E731
                for j in range(c // block, (c + len(p) - 1) // block + 1):
                    here = [d for d in range(len(p)) if (c + d) // block == j]
                    p1, o1 = at(j * block)
                    parts = [old[:, at(c + p[d])[0], at(c + p[d])[1] // block] for d in here]
                    if c > j * block:
                        parts.append(old[:, p1, o1 // block])
                    want[:, p1, o1 // block] = np.max(parts, 0)
                    moved = [(at(c + d), at(c + p[d])) for d in here] + [((p1, o1 + z), (p1, o1 + z)) for z in range(max(0, c - j * block))]
                    for (pt, ot), (pf, of) in moved:
                        vals[pt, ot] = was[:, pf, of] * old[:, pf, of // block][..., None]
                        free[pt, ot] = False
            assert (got == want).all()
            for (pt, ot), v in vals.items():
                s = want[:, pt, ot // block][..., None]
                assert (np.abs(now[:, pt, ot] * s - v) <= np.where(np.abs(v) >= 2.0**-6 * s, 0, 2.0**-10 * s)).all()
            same = lead(self.c[i].view(torch.uint8).cpu()).numpy()
            assert (same[:, free] == raw[:, free]).all()


MOVES = [
    ([100], [[0, 2, 3, 7]], 8, 3, 2, 256, 64, 0, torch.bfloat16),
    ([0, 5, 31, 64], [[0, 1, 2], [0, 3], [], [0, 5, 6, 9, 30]], 31, None, 4, 128, 16, 0, torch.float16),
    ([9], [list(range(0, 64, 1))], 64, 2, 3, 64, 24, 0, torch.bfloat16),
    ([9], [[0] + list(range(2, 64))], 64, 1, 12, 256, 24, 0, torch.bfloat16),
    ([1], [[0, 4]], 5, 2, 5, 40, 1, 0, torch.float16),
    ([100], [[0, 2, 3, 7]], 8, 3, 2, 256, 64, 64, None),
    ([0, 5, 31, 64, 14], [[0, 1, 2], [0, 3], [], [0, 5, 6, 9, 30], [0, 1, 2, 17]], 31, None, 4, 128, 16, 16, None),
    ([9], [[0] + list(range(2, 64))], 64, 2, 8, 128, 48, 16, None),
    ([15, 16, 17], [[0, 40, 41], list(range(0, 60, 3)), [1, 2, 3]], 64, 2, 9, 64, 32, 32, None),
    ([3], [[0, 1, 2, 3]], 4, 2, 2, 64, 16, 16, None),
]


@pytest.mark.parametrize("args", MOVES, ids=str)
def test_compact(args):
    case = Moves(*args)
    lens = case.run()
    _fx().check_device_errors()
    assert lens.tolist() == [c + len(p) for c, p in zip(case.lens, case.paths)]
    case.check()


@pytest.mark.parametrize("block,dtype", [(0, torch.bfloat16), (16, None)])
def test_compact_tells_bad_arguments(block, dtype):
    fx = _fx()
    make = lambda: Moves([20, 7], [[0, 2, 5], [0, 1, 3]], 6, 2, 2, 64, 16, block, dtype, seed=3)  # noqa: E731

    def code(case, **kw):
        lens = case.run(**kw)
        with pytest.raises(fx.DeviceWaitError) as e:
            fx.check_device_errors()
        case.check(left=(0,))
        assert lens.tolist()[1] == 10
        return e.value.codes[0][1], lens.tolist()[0]

    for bad in ([0, 2, 2], [0, 5, 2], [0, 0, 5], [-1, 2, 5]):
        case = make()
        path = case.path.copy()
        path[0, :3] = bad
        assert code(case, path=path) == (16, 20)
    case = make()
    path = case.path.copy()
    path[0, 2] = 500
    assert code(case, path=path) == (14, 20)
    assert code(make(), acc=[7, 3]) == (14, 20)
    assert code(make(), acc=[-1, 3]) == (14, 20)
    assert code(make(), ctx=[-4, 7]) == (14, -4)
    case = make()
    table = case.table.copy()
    table[0, 1] = case.pages
    assert code(case, table=table) == (15, 20)


def test_compact_strided_caches():
    case = Moves([20], [[0, 2, 5, 9]], 10, 2, 2, 64, 16, 16, None, seed=4)
    lens = case.run()
    d = dev()
    i32 = dict(dtype=torch.int32, device=d)
    wide = [torch.cat([x, x], -1).to(d).view(E4M3) for x in case.caches]
    both = [torch.stack([x, x * 2], -1).to(d) for x in case.scales]
    got = _fx().compact_nodes(wide[0][..., :64], wide[1][..., :64], torch.tensor(case.table, **i32), torch.tensor(case.lens, **i32),
                              torch.tensor(case.path, **i32), torch.tensor(case.accepted, **i32), both[0][..., 0], both[1][..., 0])
    assert torch.equal(got, lens)
    for i in range(2):
        assert torch.equal(wide[i].view(torch.uint8)[..., :64], case.c[i].view(torch.uint8))
        assert torch.equal(wide[i].view(torch.uint8)[..., 64:].cpu(), case.caches[i])
        assert torch.equal(both[i][..., 0], case.s[i]) and torch.equal(both[i][..., 1].cpu(), case.scales[i] * 2)


def test_compact_argument_errors():
    fx, d = _fx(), dev()
    case = Moves([20], [[0, 2, 5, 9]], 10, None, 2, 64, 16, 16, None)
    case.run()
    i32 = dict(dtype=torch.int32, device=d)
    rest = [torch.tensor(x, **i32) for x in (case.table, case.lens, case.path, case.accepted)]
    with pytest.raises(ValueError):
        fx.compact_nodes(*case.c, *rest)  # 8 bits without scales
    with pytest.raises(ValueError):
        fx.compact_nodes(*case.c, *rest, case.s[0])
    with pytest.raises(ValueError):
        fx.compact_nodes(case.c[0], case.c[1][:1], *rest, *case.s)
    with pytest.raises(ValueError):
        fx.compact_nodes(*case.c, rest[0], rest[1], rest[2].long(), rest[3], *case.s)
    with pytest.raises(NotImplementedError):
        fx.compact_nodes(*[x.float() for x in case.c], *rest)
