"""sample_tokens on the GPU: against the definition in 64 bits, on rows whose answer is known exactly
(ties, equal logits, infinities, empty rows), and its refusals.

Against 64 bits a token may differ only where the random number or a threshold lies within the
rounding of the fp32 exponentials (an argument of up to 28 rounded at 2^-24 moves a weight, and so
any running share, by less than 28 * 2^-23 + 2^-22 < 2^-18): the token has to be the one of some
uniform and top-p within that share of those given, and its probability is then within 2^-17 of it,
relatively."""

import numpy as np
import pytest
import torch

from tests.gpu_util import dev

pytestmark = pytest.mark.gpu

NEAR = 2.0**-18


def _fx():
    import flash_next_rtxpro6000_b200 as fx

    return fx


def _oracle(x, u, t, k, p, mp):
    """(token, probability) of one float64 row."""
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.lexsort((np.arange(len(x)), -x))
    if not np.isfinite(x.max()) and x.max() < 0:
        return -1, 0.0
    if not t > 0:
        return int(order[0]), 1.0
    top = x.max()
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / t))[order]
    n = len(x) if k < 1 else min(k, len(x))
    cum = np.cumsum(w[:n])
    if p < 1:
        n = max(1, int(np.searchsorted(cum[:n] - w[:n], p * cum[-1], side="left")))
    if mp > 0:
        n = max(1, min(n, int((w >= min(mp, 1.0)).sum())))
    total = cum[n - 1]
    i = min(int(np.searchsorted(cum[:n], u * total, side="right")), n - 1)
    return int(order[i]), float(w[i] / total)


def _check(logits, u, t, k, p, mp, **kw):
    tokens, probs = _fx().sample_tokens(logits, u, t, k, p, mp, **kw)
    again = _fx().sample_tokens(logits, u, t, k, p, mp, **kw)
    assert torch.equal(tokens, again[0]) and torch.equal(probs, again[1])
    M = logits.shape[0]
    val = lambda x, d: [d] * M if x is None else x.double().cpu().tolist()  # noqa: E731
    rows = logits.double().cpu().numpy()
    uu, tt, kk, pp, mm = val(u, 0), val(t, 1.0), val(k, 0), val(p, 1.0), val(mp, 0.0)
    for m in range(M):
        got = int(tokens[m])
        found = [_oracle(rows[m], max(0.0, uu[m] + du), tt[m], int(kk[m]), pp[m] + dp, mm[m])
                 for du, dp in ((0, 0), (NEAR, 0), (-NEAR, 0), (0, NEAR), (0, -NEAR))
                 if dp == 0 or 0 < pp[m] < 1]
        fit = [w for tok, w in found if tok == got]
        assert fit, (m, got, found, uu[m], tt[m], kk[m], pp[m], mm[m])
        assert min(abs(float(probs[m]) - w) for w in fit) <= 2.0**-17 * max(fit)
    return tokens, probs


def _params(M, g, d):
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (M,), generator=g)].to(d)  # noqa: E731
    return (torch.rand(M, generator=g).to(d), pick(0.0, 0.3, 0.7, 1.0, 1.5, 30.0),
            pick(0, -1, 1, 2, 50, 700, 1500, 10**6).int(), pick(0.0, 0.1, 0.5, 0.9, 0.99, 1.0, 2.0),
            pick(0.0, 0.0, 0.01, 0.2, 1.0, 3.0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,V", [(1, 1), (3, 2), (5, 17), (16, 1000), (33, 4099), (16, 49152), (8, 151936), (6, 248320)])
def test_against_64_bits(dtype, M, V):
    g = torch.Generator().manual_seed(M * 31 + V)
    x = torch.randn(M, V, generator=g) * 3
    x[:, torch.randint(0, V, (min(V, 40),), generator=g)] += torch.rand(min(V, 40), generator=g) * 10
    _check(x.to(dtype).to(dev()), *_params(M, g, dev()))


@pytest.mark.parametrize("off", ["all", "top_k", "top_p", "min_p", "none"])
def test_each_filter_alone(off):
    g = torch.Generator().manual_seed(5)
    M, V = 24, 30011
    x = (torch.randn(M, V, generator=g) * 2).to(dev())
    u = torch.rand(M, generator=g).to(dev())
    t = torch.full((M,), 0.8, device=dev())
    k = torch.randint(1, 400, (M,), generator=g).int().to(dev()) if off in ("top_k", "none") else None
    p = torch.rand(M, generator=g).to(dev()) if off in ("top_p", "none") else None
    mp = (torch.rand(M, generator=g) * 0.1).to(dev()) if off in ("min_p", "none") else None
    _check(x, u, None if off == "all" else t, k, p, mp)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 7, 2049, 151936])
def test_equal_logits_draw_by_index(dtype, V):
    """All weights are one: the token is the floor of u times what is kept, exactly."""
    M = 12
    u = ((torch.arange(M) + 0.37) / M).float()
    x = torch.full((M, V), -3.25, dtype=dtype, device=dev())
    for k in (0, 5, 3000):
        n = min(k, V) if k else V
        tokens, probs = _fx().sample_tokens(x, u.to(dev()), None, torch.full((M,), k, dtype=torch.int32, device=dev()))
        want = torch.tensor([int(float(v) * n) for v in u])
        assert torch.equal(tokens.cpu(), want)
        assert torch.equal(probs.cpu(), torch.full((M,), 1.0 / n, dtype=torch.float64).float())
    tokens, _ = _fx().sample_tokens(x, u.to(dev()), top_p=torch.full((M,), 0.5, device=dev()))
    n = -(-V // 2)  # the shortest prefix that reaches half
    assert torch.equal(tokens.cpu(), torch.tensor([int(float(v) * n) for v in u]))


def test_ties_at_the_cut_keep_the_lower_tokens():
    x = torch.zeros(4, 5000)
    x[:, 4000] = 2.0
    x[:, 17::100] = 1.0  # 50 ties; top-k 11 keeps token 4000 and the first ten of them
    k = torch.full((4,), 11, dtype=torch.int32, device=dev())
    u = torch.tensor([0.0, 0.5, 0.9, 0.9999999])
    tokens, probs = _check(x.to(dev()), u.to(dev()), None, k, None, None)
    assert int(tokens[0]) == 4000 and int(tokens[3]) == 17 + 900


def test_clusters_of_near_values_are_split():
    """Far outliers put all other tokens into one interval, which is split by key, then by index."""
    g = torch.Generator().manual_seed(2)
    V = 60000
    x = torch.rand(6, V, generator=g)
    x[:, 123] = 300.0
    x[1] = torch.where(torch.arange(V) == 123, 300.0, torch.round(x[1] * 2) / 2)  # long ties
    x[2, 77] = -1e30
    x[3, 78] = torch.finfo(torch.float32).min
    t = torch.tensor([100.0, 100.0, 1000.0, 1000.0, 5000.0, 5000.0])
    u = torch.tensor([0.5, 0.7, 0.2, 0.999, 0.0, 0.9])
    p = torch.tensor([1.0, 0.9, 0.5, 1.0, 1.0, 0.3])
    k = torch.tensor([0, 0, 20000, 0, 2000, 0], dtype=torch.int32)
    d = dev()
    _check(x.to(d), u.to(d), t.to(d), k.to(d), p.to(d), None)


def test_infinities_nan_and_empty_rows():
    V, d = 3001, dev()
    x = torch.randn(8, V, generator=torch.Generator().manual_seed(1))
    x[0] = -float("inf")
    x[1] = float("nan")
    x[2, ::2] = -float("inf")
    x[3, ::3] = float("nan")
    x[4, [5, 900, 2000]] = float("inf")       # draws among the three, whatever else is there
    x[5, 1:] = -float("inf")
    x[6, 1:] = torch.finfo(torch.float32).min
    x[7] = torch.finfo(torch.float32).min
    u = torch.tensor([0.3, 0.3, 0.6, 0.6, 0.5, 0.99, 0.99, 0.5], device=d)
    for t in (None, torch.full((8,), 0.5, device=d), torch.zeros(8, device=d)):
        tokens, probs = _check(x.to(d), u, t, None, None, None)
        assert tokens[:2].tolist() == [-1, -1] and probs[:2].tolist() == [0.0, 0.0]
        assert int(tokens[4]) == (5 if t is not None and float(t[0]) == 0 else 900)
        assert tokens[5:7].tolist() == [0, 0]
    assert int(tokens[7]) == 0


def test_odd_parameters():
    d, V = dev(), 500
    x = torch.randn(7, V, generator=torch.Generator().manual_seed(4)).to(d)
    best = x.argmax(1)
    nan, inf = float("nan"), float("inf")
    f = lambda *v: torch.tensor(v, device=d)  # noqa: E731
    u = f(nan, -1.0, 0.0, 1.0, 2.0, inf, 0.5)
    tokens, _ = _fx().sample_tokens(x, u)
    worst = x.argmin(1)
    assert tokens[:3].tolist() == best[:3].tolist() and tokens[3:6].tolist() == worst[3:6].tolist()
    half = torch.full((7,), 0.5, device=d)
    t = f(nan, 0.0, -1.0, 1e-30, 1.0, 1.0, 1.0)
    p = f(1.0, 1.0, 1.0, 1.0, 0.0, -1.0, 1.0)
    mp = f(0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 5.0)
    tokens, probs = _fx().sample_tokens(x, half, t, None, p, mp)
    assert torch.equal(tokens, best) and probs.tolist() == [1.0] * 7
    none = torch.full((7,), nan, device=d)
    assert torch.equal(_fx().sample_tokens(x, half, None, None, none, none)[0], _fx().sample_tokens(x, half)[0])
    far, _ = _fx().sample_tokens(x, half, torch.full((7,), inf, device=d))  # all alike: by rank
    assert torch.equal(far, x.sort(dim=1, descending=True, stable=True).indices[:, V // 2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype):
    g = torch.Generator().manual_seed(9)
    M, V = 6, 10007
    for pad, off in ((0, 1), (1, 0), (5, 3), (64, 7)):
        flat = (torch.randn(M * (V + pad) + off, generator=g) * 3).to(dtype).to(dev())
        x = flat[off:].view(M, V + pad)[:, :V]
        args = _params(M, g, dev())
        got = _check(x, *args)
        same = _fx().sample_tokens(x.contiguous(), *args)
        assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[1])


def test_rows_wider_than_shared_memory():
    g = torch.Generator().manual_seed(10)
    x = (torch.randn(3, 1 << 20, generator=g) * 2).to(dev())
    u = torch.rand(3, generator=g).to(dev())
    p = torch.tensor([0.9, 1.0, 0.5], device=dev())
    k = torch.tensor([0, 40, 5000], dtype=torch.int32, device=dev())
    _check(x, u, None, k, p, None)


def test_frequencies_follow_the_probabilities():
    """20,000 uniforms spread evenly over a row of 6 tokens: each token's count is its share, to one."""
    x = torch.tensor([0.3, 2.0, -1.0, 1.1, 0.0, 1.9]).expand(20000, 6).contiguous().to(dev())
    u = ((torch.arange(20000) + 0.5) / 20000).to(dev())
    tokens, probs = _fx().sample_tokens(x, u)
    share = torch.softmax(x[0].double(), 0).cpu()
    count = torch.bincount(tokens.cpu(), minlength=6).double()
    assert float((count - share * 20000).abs().max()) <= 1.5
    assert float((probs.double().cpu() - share[tokens.cpu()]).abs().max()) < 1e-6


def test_graph_replay_reads_new_inputs():
    d = dev()
    g = torch.Generator().manual_seed(12)
    x = (torch.randn(4, 49152, generator=g) * 2).to(d)
    u = torch.rand(4, generator=g).to(d)
    _fx().sample_tokens(x, u)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, probs = _fx().sample_tokens(x, u)
    for _ in range(3):
        x.copy_((torch.randn(4, 49152, generator=g) * 2).to(d))
        u.copy_(torch.rand(4, generator=g).to(d))
        graph.replay()
        torch.cuda.synchronize()
        want = _fx().sample_tokens(x, u)
        assert torch.equal(tokens, want[0]) and torch.equal(probs, want[1])


def test_no_rows_and_refusals():
    fx, d = _fx(), dev()
    x = torch.zeros(3, 100, device=d)
    u = torch.zeros(3, device=d)
    assert fx.sample_tokens(x[:0], u[:0])[0].shape == (0,)
    i = torch.zeros(3, dtype=torch.int32, device=d)
    bad = [
        (dict(logits=x.double()), NotImplementedError), (dict(logits=x[0]), ValueError),
        (dict(logits=x.t()), ValueError), (dict(logits=x.cpu()), ValueError),
        (dict(uniforms=u[:2]), ValueError), (dict(uniforms=u.double()), ValueError),
        (dict(uniforms=u.cpu()), ValueError), (dict(temperature=i), ValueError), (dict(top_k=u), ValueError),
        (dict(top_k=i.long()), ValueError), (dict(top_p=u[:1]), ValueError), (dict(min_p=i), ValueError),
        (dict(logits=x[:, :0]), ValueError),
        (dict(logits=torch.zeros(1, (1 << 22) + 1, device=d), uniforms=u[:1]), NotImplementedError),
    ]
    for change, error in bad:
        with pytest.raises(error):
            fx.sample_tokens(**(dict(logits=x, uniforms=u) | change))


@pytest.mark.parametrize("V", [1000, 50021])
def test_many_rows(V):
    """More rows than run at once."""
    g = torch.Generator().manual_seed(14)
    M = 150
    x = torch.randn(M, V, generator=g) * 3
    x[:, torch.randint(0, V, (40,), generator=g)] += torch.rand(40, generator=g) * 10
    _check(x.to(dev()), *_params(M, g, dev()))
    _check(x.half().to(dev()), *_params(M, g, dev()))
