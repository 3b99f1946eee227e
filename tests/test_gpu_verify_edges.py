"""verify_tokens on the GPU where its rules meet their ends, against walks in exact arithmetic.

Siblings that cover a row: probabilities are multiples of 2^-25 and random numbers of 2^-24, so u S and S - r take less
than 53 bits and every comparison of the kernel is exact, as its sums are: paths and tokens are compared for equality."""

from fractions import Fraction

import numpy as np
import pytest
import torch

from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def _fx():
    import flash_next_rtxpro6000_b200 as fx

    return fx


def _call(p, q, tokens, parents, offsets, u, w, max_nodes):
    d = dev()
    to = lambda x, t: torch.as_tensor(np.asarray(x), dtype=t).to(d)  # noqa: E731
    args = (to(p, torch.float32), None if q is None else to(q, torch.float32), to(tokens, torch.int64),
            to(parents, torch.int32), to(offsets, torch.int32), to(u, torch.float32), to(w, torch.float32))
    out = _fx().verify_tokens(*args, max_nodes=max_nodes)
    again = _fx().verify_tokens(*args, max_nodes=max_nodes)
    assert all(torch.equal(a, b) for a, b in zip(out, again))
    return [x.tolist() for x in out]


def _exact_walk(p, tokens, parents, u, w):
    """(path, next token) of one request without drafter probabilities; p {token: Fraction} of each node."""
    path, r, s = [0], dict(p[0]), Fraction(1)
    for i in range(1, len(tokens)):
        if parents[i] != path[-1]:
            continue
        x = tokens[i]
        if Fraction(float(u[i])) * s < r.get(x, 0):
            path.append(i)
            r, s = dict(p[i]), Fraction(1)
        elif sum(v for t, v in r.items() if t != x) > 0:  # else nothing would be left: r stays
            s = max(s - r.get(x, 0), Fraction(0))
            r[x] = Fraction(0)
    total = sum(r.values())
    if total == 0:
        return path, -1
    aim, run = min(Fraction(float(w)) * total, total - Fraction(1, 2**52)), Fraction(0)
    for t in sorted(r):
        run += r[t]
        if aim < run:
            return path, t


def test_siblings_that_cover_a_row_leave_it_a_token():
    """Two tokens share a row whose sum is 1 - 2^-25; both are drafted, and both refused."""
    p = np.zeros((3, 40), np.float32)
    p[:, 7], p[:, 30] = 0.5, 0.5 - 2.0**-25
    u = [0.0, 1 - 2.0**-24, 1 - 2.0**-24]
    path, accepted, tokens = _call(p, None, [1, 7, 30], [-1, 0, 0], [0, 3], u, [0.25], 3)
    assert (path, accepted, tokens) == ([[0, -1, -1]], [1], [30])
    # what stays is asked again by the same token's next sibling: 1 / 4 of 1 / 2 is below it
    p = np.concatenate([p, p[:1]])
    path, accepted, tokens = _call(p, None, [1, 7, 30, 30], [-1, 0, 0, 0], [0, 4], u + [0.25], [0.0], 4)
    assert (path, accepted, tokens) == ([[0, 3, -1, -1]], [2], [7])
    # a row with one token and less than 1 in all
    p = np.zeros((3, 40), np.float32)
    p[:, 39] = 0.25
    path, accepted, tokens = _call(p, None, [1, 39, 5], [-1, 0, 0], [0, 3], [0.0, 0.5, 0.5], [0.5], 3)
    assert (path, accepted, tokens) == ([[0, -1, -1]], [1], [39])
    _fx().check_device_errors()


@pytest.mark.parametrize("V", [2, 3, 50, 4097, 151936])
def test_siblings_over_the_support_of_rows(V):
    """Every token that has probability drafted in some order, some twice, by random numbers near 1 for the most part; rows
    that sum to 1, to 1 - 2^-25 and to less."""
    rng = np.random.default_rng(V)
    p, tokens, parents, u, offsets, want = [], [], [], [], [0], []
    w = rng.integers(0, 2**24, 60) * 2.0**-24
    for b in range(60):
        n = int(rng.integers(2, 9))
        rows = []
        for _ in range(n):
            k = min(int(rng.integers(1, 5)), V)
            cut = np.sort(rng.choice(2**25 - 1, k - 1, replace=False) + 1)
            share = np.diff(np.concatenate([[0], cut, [2**25]]))
            kind = rng.integers(0, 3)
            share = share // 4 if kind == 1 and share.min() >= 4 else share
            share[-1] -= 1 if kind == 2 and share[-1] > 1 else 0
            share = np.array([s if s < 2**24 else s // 2 * 2 for s in share])  # 24 bits
            at = rng.choice(min(V, 300), k, replace=False) * max(V // 300, 1)
            rows.append({int(t): Fraction(int(s), 2**25) for t, s in zip(at, share)})
        par = [-1] + [int(rng.integers(0, 2)) if i > 1 and rng.random() < 0.3 else 0 for i in range(1, n)]
        tok, seen = [0], {}
        for i in range(1, n):  # the parent's support in turn
            support = sorted(rows[par[i]])
            tok.append(support[seen.get(par[i], 0) % len(support)])
            seen[par[i]] = seen.get(par[i], 0) + 1
        uu = np.where(rng.random(n) < 0.85, 2**24 - 1 - rng.integers(0, 2, n), rng.integers(0, 2**24, n)) * 2.0**-24
        want.append(_exact_walk(rows, tok, par, uu, w[b]))
        for row in rows:
            x = np.zeros(V, np.float32)
            for t, s in row.items():
                x[t] = float(s)
            p.append(x)
        tokens += tok
        parents += par
        u += uu.tolist()
        offsets.append(offsets[-1] + n)
    path, accepted, drawn = _call(np.stack(p), None, tokens, parents, offsets, u, w, 8)
    for b, (right, token) in enumerate(want):
        assert [x for x in path[b] if x >= 0] == right and accepted[b] == len(right) and drawn[b] == token, b
    assert min(drawn) >= 0
    _fx().check_device_errors()


# A refusal's residual in 64 bits: each element is rounded at 2^-53 of r / S, and S, a sum of V truncations, is off by
# V 2^-52 of 1 at most.  Relative to an r(x) that is at least 2^-8 of the r(x) / S it came from (children with less are not
# drafted here) and S of 2^-4 at least, ten refusals at V = 700 stay below 10 * 2^8 * (2^-53 + 700 * 2^-52 * 2^4) < 2^-26:
# random numbers 2^-25.5 above a refusal's border, or as far below an acceptance's, decide as the formula does.
MARGIN = 2.0**-25.5


def _bordering(p, q, rng, refusals):
    """Tokens and random numbers of one node's children: `refusals` that are just refused, then one that is just accepted;
    and what is left of the row."""
    tokens, u, r, s = [], [], p.astype(np.longdouble), np.longdouble(1)
    p, q = p.astype(np.longdouble), q.astype(np.longdouble)
    for k in range(refusals + 1):
        share = r / s
        last = k == refusals
        # borders r(x) / (S q(x)) inside (0, 1), without much cancellation in what made r(x)
        border = np.where(q > 0, share / np.maximum(q, np.longdouble(1e-30)), 0)
        fit = np.flatnonzero((border > 2.0**-8) & (border < 0.99) & (share > 2.0**-8 * p))
        x = int(rng.choice(fit))
        at = np.float32(border[x])
        if last:
            while np.longdouble(at) * q[x] >= share[x] * (1 - np.longdouble(MARGIN)):
                at = np.nextafter(at, np.float32(0))
        else:
            while np.longdouble(at) * q[x] < share[x] * (1 + np.longdouble(MARGIN)):
                at = np.nextafter(at, np.float32(1))
            r = np.maximum(share - q, 0)
            s = r.sum()
            assert s > 2.0**-4
        tokens.append(x)
        u.append(float(at))
    return tokens, u


def test_residuals_keep_the_bits_that_choices_need():
    """Up to ten refusals one after the other at random numbers that are the next or next but one above their borders, then
    one acceptance as near below its border."""
    rng = np.random.default_rng(21)
    B, V = 200, 700
    soft = lambda z: (np.exp(z) / np.exp(z).sum(1, keepdims=True)).astype(np.float32)  # noqa: E731
    x = rng.standard_normal((B, V)) * 2
    p, q = soft(x), soft(x + rng.standard_normal((B, V)) * 1.5)
    rows, draft, tokens, parents, u, offsets, want = [], [], [], [], [], [0], []
    for b in range(B):
        k = int(rng.integers(0, 11))
        t, v = _bordering(p[b], q[b], rng, k)
        tokens += [0] + t
        u += [0.0] + v
        parents += [-1] + [0] * (k + 1)
        rows += [p[b]] * (k + 2)
        draft += [q[b]] * (k + 2)
        offsets.append(offsets[-1] + k + 2)
        want.append([0, k + 1] + [-1] * 10)
    path, accepted, _ = _call(np.stack(rows), np.stack(draft), tokens, parents, offsets, u, np.full(B, 0.5), 12)
    wrong = [b for b in range(B) if path[b] != want[b]]
    assert not wrong, (len(wrong), wrong[:5], [path[b] for b in wrong[:5]])
    _fx().check_device_errors()


def test_rows_of_ones_up_to_63():
    """Elements are clamped to [0, 1], rows are not: a row of 63 ones is drawn from in equal shares."""
    V, w = 4000, np.array([0.0, 0.25, 0.3, 1 - 2.0**-24], np.float32)
    p = np.zeros((4, V), np.float32)
    p[:, 1 : 63 * 63 : 63] = 1.0
    at = [1 + 63 * min(int(Fraction(float(x)) * 63), 62) for x in w]
    assert _call(p, None, [0] * 4, [-1] * 4, range(5), [0.0] * 4, w, 1) == [[[0]] * 4, [1] * 4, at]
    _fx().check_device_errors()


@pytest.mark.parametrize("V", [64, 4095, 4096, 4099, 30000, 2**21])
def test_rows_of_ones_are_no_distributions(V):
    """What sums to 64 or more is told, whatever 64 bits hold, and such a request is as one without nodes; others are not
    affected."""
    fx = _fx()

    def told(*args):
        out = _call(*args)
        with pytest.raises(fx.DeviceWaitError, match="PROBS") as e:
            fx.check_device_errors()
        assert "wait" not in str(e.value)
        return out

    p = np.ones((3, V), np.float32)
    p[1] = 0.0
    p[1, V - 1] = 0.75
    out = told(p, None, [0] * 3, [-1] * 3, range(4), [0.0] * 3, [0.5] * 3, 2)
    assert out == [[[-1, -1], [0, -1], [-1, -1]], [0, 1, 0], [-1, V - 1, -1]]
    # the row of the path's end, and what refusals leave: with and without drafter probabilities
    p = np.ones((4, V), np.float32)
    p[2:] = 0.0
    p[0, 5] = 0.5
    p[2:, 7] = 1.0
    q = np.zeros((4, V), np.float32)
    q[:, 5] = 1.0
    for draft in (None, q):
        args = (p, draft, [0, 5, 0, 5], [-1, 0, -1, 0], [0, 2, 4], [0.0, 0.75, 0.0, 0.75], [0.5, 0.5], 2)
        if V > 64:
            assert told(*args) == [[[-1, -1], [0, -1]], [0, 1], [-1, 7]]
        else:  # 63 are left: the 32nd of them is token 32, behind token 5
            assert _call(*args) == [[[0, -1], [0, -1]], [1, 1], [32, 7]]
    # a refusal's sum is told although the path goes on from there
    if V > 64:
        p = np.ones((3, V), np.float32)
        p[0, 5] = 0.5
        p[2] = 0.0
        p[2, 7] = 1.0
        q[:, 9] = 0.25
        out = told(p[:3], q[:3], [0, 5, 9], [-1, 0, 0], [0, 3], [0.0, 0.75, 0.0], [0.5], 3)
        assert out == [[[-1, -1, -1]], [0], [-1]]


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("chain", [True, False])
@pytest.mark.parametrize("counts,V", [([6], 151936), ([5, 1, 0, 16, 2], 4096), ([64], 3001), ([9] * 20, 517), ([33, 64, 12], 250)])
def test_walks_in_64_bits_at_a_border_of_2_to_the_minus_28(monkeypatch, counts, V, chain, drafts):
    """Residuals are rounded at 2^-53, and sums lose V 2^-52 < 2^-34 of 1; over an S of 2^-4 at least, a few refusals one
    after the other stay below 2^-28 of what is compared and drawn from."""
    from tests import test_gpu_verification as other

    monkeypatch.setattr(other, "NEAR_CHOICE", 2.0**-28)
    for seed in range(4):
        other.Drafts(counts, V, seed=100 * seed + V, drafts=drafts, chain=chain, noise=2.0).check()
    _fx().check_device_errors()
