"""rotary_append and rotary_table on the GPU, against the rotation in 64 bits.

Tolerance: products and one sum in fp32 (three roundings of at most 2^-24 of |x c| + |y s|, with the
table's own 2^-24), then one rounding to the type (2^-8 bf16, 2^-11 fp16, or half the smallest fp16
step 2^-25)."""

import math

import numpy as np
import pytest
import torch

from tests.gpu_util import dev

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _fx():
    import flash_next_rtxpro6000_b200 as fx

    return fx


def _turn64(x, angle, gain, interleaved):
    """x [T, H, D] float64 numpy, angle [T, R/2]; returns the rotated heads and |x c| + |y s|."""
    R = 2 * angle.shape[1]
    c, s = np.cos(angle)[:, None] * gain, np.sin(angle)[:, None] * gain
    y, size = x.copy(), np.abs(x)
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    size[..., a] = np.abs(x[..., a] * c) + np.abs(x[..., b] * s)
    size[..., b] = np.abs(x[..., b] * c) + np.abs(x[..., a] * s)
    return y, size


def _check(got, want, size, dtype):
    got = got.double().cpu().numpy()
    tol = UNIT[dtype] * np.abs(want) + 8 * 2.0**-24 * size + 2.0**-25
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) - tol).max())


def _case(T, Hq, Hk, D, R, dtype, interleaved, page, seed=0, P=5000, base=10000.0, pad=0, offset=0):
    fx = _fx()
    g = torch.Generator().manual_seed(seed)
    width = (Hq + 2 * Hk) * D + pad
    rows = torch.randn(T * width + offset, generator=g).to(dtype).to(dev())
    rows = rows[offset:].view(T, width)[:, : width - pad]
    q, k, v = (x.unflatten(1, (-1, D)) for x in rows.split([Hq * D, Hk * D, Hk * D], 1))
    table = fx.rotary_table(P, R, base, device=dev())
    pos = torch.randint(0, P, (T,), generator=g)
    pages = T // page + 2
    slots = torch.randperm(pages * page, generator=g)[:T]
    kc, vc = (torch.full((pages, page, Hk, D), 7.0, dtype=dtype, device=dev()) for _ in range(2))
    out = fx.rotary_append(q, k, v, pos.to(dev()), slots.to(dev()), table, kc, vc, interleaved=interleaved)
    freq = base ** (-np.arange(R // 2) / (R // 2))
    angle = pos.double().numpy()[:, None] * freq
    _check(out, *_turn64(q.double().cpu().numpy(), angle, 1.0, interleaved), dtype)
    flat = kc.view(-1, Hk, D)
    _check(flat[slots.to(dev())], *_turn64(k.double().cpu().numpy(), angle, 1.0, interleaved), dtype)
    assert torch.equal(vc.view(-1, Hk, D)[slots.to(dev())], v)
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots] = False
    for c in (kc, vc):  # no other place is touched
        assert bool((c.view(-1, Hk, D)[rest.to(dev())] == 7.0).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,Hq,Hk,D,R,page", [
    (1, 16, 2, 256, 64, 64), (16, 32, 8, 128, 128, 16), (3, 5, 1, 64, 32, 1), (257, 4, 4, 64, 64, 24),
    (700, 2, 1, 16, 16, 7), (9, 3, 1, 80, 48, 16),
])
def test_against_64_bits(T, Hq, Hk, D, R, page, dtype, interleaved):
    _case(T, Hq, Hk, D, R, dtype, interleaved, page, seed=T)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,D,R,pad,offset", [
    (5, 3, 1, 24, 24, 0, 0),     # half a rotation is no whole vector
    (5, 3, 2, 7, 2, 0, 0),       # an odd head
    (6, 2, 1, 64, 8, 0, 0),      # few rotated
    (4, 2, 1, 64, 64, 3, 0),     # rows that break 16-byte alignment
    (4, 2, 1, 64, 64, 0, 1),     # a base that does
    (2, 2, 1, 8192, 8192, 0, 0),  # a head wider than a block of vectors
])
def test_any_alignment(T, Hq, Hk, D, R, pad, offset, interleaved):
    _case(T, Hq, Hk, D, R, torch.bfloat16, interleaved, 4, seed=D, pad=pad, offset=offset)


def test_many_tokens():
    _case(70001, 1, 1, 16, 16, torch.float16, False, 64, seed=3)  # past the grid's second dimension


def test_table_far_positions_and_scaling():
    fx = _fx()
    for scaling in (None, fx.RotaryScaling(4.0, "linear"), fx.RotaryScaling(8.0, original=4096)):
        t = fx.rotary_table(300000, 64, 1e6, scaling, device=dev()).double().cpu().numpy()
        f = 1e6 ** (-np.arange(32) / 32)
        gain = 1.0
        if scaling is not None and scaling.kind == "linear":
            f = f / 4
        elif scaling is not None:
            turns = 4096 * f / (2 * math.pi)
            keep = np.clip((turns - 1) / 31, 0, 1)
            f = f * keep + f / 8 * (1 - keep)
            gain = 0.1 * math.log(8) + 1
        for p in (0, 1, 65535, 65536, 299999):
            # 64-bit angles of up to 3e5 carry 3e5 * 2^-52; the table rounds to fp32
            assert np.abs(t[p, :32] - np.cos(p * f) * gain).max() < 2.0**-23
            assert np.abs(t[p, 32:] - np.sin(p * f) * gain).max() < 2.0**-23


def test_in_place_skipped_slots_and_strided_cache():
    fx = _fx()
    d, T, Hq, Hk, D = dev(), 6, 4, 2, 64
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(T, h, D, generator=g).bfloat16().to(d) for h in (Hq, Hk, Hk))
    table = fx.rotary_table(100, D, device=d)
    pos = torch.arange(T, device=d) * 3
    slots = torch.tensor([5, -1, 0, 31, -1, 17], device=d)
    kc, vc = (torch.zeros(4, 8, Hk, D, dtype=torch.bfloat16, device=d) for _ in range(2))
    ref = fx.rotary_append(q, k, v, pos, slots, table, kc, vc)
    # head-major pages, seen through a transpose
    kt, vt = (torch.zeros(4, Hk, 8, D, dtype=torch.bfloat16, device=d).transpose(1, 2) for _ in range(2))
    q2 = q.clone()
    out = fx.rotary_append(q2, k, v, pos, slots, table, kt, vt, out=q2)
    assert out is q2 and torch.equal(out, ref) and torch.equal(kt, kc) and torch.equal(vt, vc)
    assert int((kc.view(32, -1) != 0).any(1).sum()) == 4
    fx.check_device_errors()


def test_positions_and_slots_out_of_range_are_reported():
    fx = _fx()
    d = dev()
    fx.check_device_errors()
    q = torch.ones(1, 2, 64, dtype=torch.bfloat16, device=d)
    kc, vc = (torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16, device=d) for _ in range(2))
    table = fx.rotary_table(10, 64, device=d)
    one = lambda x: torch.tensor([x], device=d)  # noqa: E731
    for pos, slot, code in ((10, 0, 12), (-1, 0, 12), (3, 8, 13), (3, -2, 13)):
        fx.rotary_append(q, q, q, one(pos), one(slot), table, kc, vc)
        with pytest.raises(fx.DeviceWaitError) as e:
            fx.check_device_errors()
        assert [c for _, c in e.value.codes] == [code]
    assert bool((kc.view(8, -1)[1:] == 0).all())


def test_no_tokens_and_refusals():
    fx = _fx()
    d = dev()
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=d)
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=d)
    kc, vc = (torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16, device=d) for _ in range(2))
    i = torch.zeros(2, dtype=torch.int64, device=d)
    table = fx.rotary_table(10, 64, device=d)
    assert fx.rotary_append(q[:0], k[:0], k[:0], i[:0], i[:0], table, kc, vc).shape == (0, 4, 64)
    bad = [
        (dict(q=q.float(), k=k.float(), v=k.float()), NotImplementedError),
        (dict(k=k[:1]), ValueError), (dict(k=k.half()), ValueError), (dict(v=k[:, :1]), ValueError),
        (dict(positions=i.int()), ValueError), (dict(slots=i[:1]), ValueError),
        (dict(positions=i.cpu()), ValueError), (dict(table=table.double()), ValueError),
        (dict(table=fx.rotary_table(10, 66, device=d)), ValueError), (dict(table=table[:, :31]), ValueError),
        (dict(k_cache=kc.half()), ValueError), (dict(v_cache=vc[:1]), ValueError),
        (dict(k_cache=kc[:, :, :1], v_cache=vc[:, :, :1]), ValueError),
        (dict(k_cache=kc.transpose(2, 3).contiguous().transpose(2, 3)), ValueError),
        (dict(out=torch.zeros(2, 3, 64, dtype=torch.bfloat16, device=d)), ValueError),
        (dict(out=q.half()), ValueError),
    ]
    for change, error in bad:
        args = dict(q=q, k=k, v=k, positions=i, slots=i, table=table, k_cache=kc, v_cache=vc) | change
        with pytest.raises(error):
            fx.rotary_append(**args)
    for args in ((0, 64), (10, 63), (10, 0), (10, 64, 1.0)):
        with pytest.raises(ValueError):
            fx.rotary_table(*args)
    for args in (dict(factor=0.5), dict(factor=2.0, kind="other"), dict(factor=2.0, slow=3.0, fast=2.0)):
        with pytest.raises(ValueError):
            fx.RotaryScaling(**args)
