"""The C entry points of the verify-step operators refuse bad arguments before any launch, and the
Python ones refuse tensors that are not on a GPU."""

import ctypes

import pytest
import torch

import flash_next_rtxpro6000_b200 as fx
from flash_next_rtxpro6000_b200 import _lib

S3 = ctypes.c_int64 * 3


def _call(name, args, kw):
    assert set(kw) <= set(args), kw
    return getattr(_lib.lib(), name)(*(args | kw).values())


def _rotary(**kw):
    return _call("fnx_rotary_append", dict(
        q=16, q_st=256, q_sh=64, k=16, k_st=128, k_sh=64, v=16, v_st=128, v_sh=64, out=16, o_st=256, o_sh=64,
        pos=16, slots=16, table=16, table_ld=64, P=100, kc=16, ks=S3(2048, 128, 64), vc=16, vs=S3(2048, 128, 64),
        pages=4, page=16, T=2, Hq=4, Hk=2, D=64, R=64, inter=0, dtype=0, err=None, pdl=0, stream=None), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(T=0), _lib.FNX_OK), (dict(dtype=2), _lib.FNX_EUNSUPPORTED), (dict(T=-1), _lib.FNX_EINVAL),
    (dict(R=65), _lib.FNX_EINVAL), (dict(R=66), _lib.FNX_EINVAL), (dict(R=63), _lib.FNX_EINVAL),
    (dict(page=0), _lib.FNX_EINVAL), (dict(P=0), _lib.FNX_EINVAL), (dict(table_ld=32), _lib.FNX_EINVAL),
    (dict(q=None), _lib.FNX_EINVAL), (dict(vc=None), _lib.FNX_EINVAL), (dict(pos=None), _lib.FNX_EINVAL),
    (dict(ks=None), _lib.FNX_EINVAL), (dict(Hq=0, Hk=0), _lib.FNX_EINVAL),
])
def test_rotary_append(kw, code):
    assert _rotary(**kw) == code
    assert bool(_lib.last_error()) == (code != _lib.FNX_OK)


def _attention(**kw):
    return _call("fnx_tree_attention", dict(
        q=16, q_sn=256, q_sh=64, kc=16, ks=S3(2048, 128, 64), vc=16, vs=S3(2048, 128, 64), pages=4, page=16,
        table=16, table_ld=4, width=4, ctx=16, off=16, mask=None, out=16, o_sn=256, o_sh=64, lse=None, B=1, N=2,
        Hq=4, Hk=2, D=64, max_nodes=2, max_context=60, scale=0.125, dtype=0, part=16, err=None, pdl=0,
        stream=None), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(N=0), _lib.FNX_OK), (dict(dtype=2), _lib.FNX_EUNSUPPORTED), (dict(D=96), _lib.FNX_EUNSUPPORTED),
    (dict(Hq=3), _lib.FNX_EINVAL), (dict(Hk=0), _lib.FNX_EINVAL), (dict(B=0), _lib.FNX_EINVAL),
    (dict(max_nodes=0), _lib.FNX_EINVAL), (dict(max_nodes=65), _lib.FNX_EUNSUPPORTED),
    (dict(max_context=-1), _lib.FNX_EINVAL), (dict(max_context=2**31), _lib.FNX_EUNSUPPORTED),
    (dict(page=0), _lib.FNX_EINVAL), (dict(q=None), _lib.FNX_EINVAL), (dict(part=None), _lib.FNX_EINVAL),
    (dict(table=None), _lib.FNX_EINVAL), (dict(q=8), _lib.FNX_EINVAL), (dict(q_sh=65), _lib.FNX_EINVAL),
    (dict(ks=S3(2048, 128, 65)), _lib.FNX_EINVAL), (dict(vs=None), _lib.FNX_EINVAL),
])
def test_tree_attention(kw, code):
    assert _attention(**kw) == code
    assert bool(_lib.last_error()) == (code != _lib.FNX_OK)


def _layout(**kw):
    return _call("fnx_tree_layout", dict(
        parents=16, off=16, ctx=16, table=16, table_ld=4, width=4, pages=4, page=16, B=1, N=2, mask=16, pos=16,
        slots=16, err=None, pdl=0, stream=None), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(N=0), _lib.FNX_OK), (dict(B=0), _lib.FNX_EINVAL), (dict(parents=None), _lib.FNX_EINVAL),
    (dict(table=None), _lib.FNX_EINVAL), (dict(ctx=None), _lib.FNX_EINVAL), (dict(page=0), _lib.FNX_EINVAL),
    (dict(N=-1), _lib.FNX_EINVAL),
])
def test_tree_layout(kw, code):
    assert _layout(**kw) == code


def _sample(**kw):
    return _call("fnx_sample", dict(
        logits=16, ldl=100, dtype=2, M=2, V=100, u=16, t=None, k=None, p=None, mp=None, tokens=16, probs=16, pdl=0,
        stream=None), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(M=0), _lib.FNX_OK), (dict(dtype=3), _lib.FNX_EUNSUPPORTED), (dict(V=0), _lib.FNX_EINVAL),
    (dict(ldl=99), _lib.FNX_EINVAL), (dict(V=2**22 + 1, ldl=2**23), _lib.FNX_EUNSUPPORTED),
    (dict(M=2**25), _lib.FNX_EUNSUPPORTED), (dict(logits=None), _lib.FNX_EINVAL), (dict(u=None), _lib.FNX_EINVAL),
    (dict(tokens=None), _lib.FNX_EINVAL), (dict(probs=None), _lib.FNX_EINVAL), (dict(M=-1), _lib.FNX_EINVAL),
])
def test_sample(kw, code):
    assert _sample(**kw) == code
    assert bool(_lib.last_error()) == (code != _lib.FNX_OK)


def test_tensors_on_the_host_are_refused():
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    c = torch.zeros(2, 4, 4, 64, dtype=torch.bfloat16)
    i, i32 = torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        fx.rotary_append(x, x, x, i, i, torch.zeros(9, 64), c, c)
    with pytest.raises(ValueError):
        fx.tree_attention(x, c, c, i32.view(2, 1), i32, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        fx.tree_layout(i32, i32, i32[:1], i32.view(2, 1), 4, 2)
    with pytest.raises(ValueError):
        fx.sample_tokens(torch.zeros(2, 9), torch.zeros(2))


def test_rotary_table_on_the_host():
    """The table is built wherever it is asked for: rows are cosines, then sines, of unit radius."""
    t = fx.rotary_table(70000, 8, device="cpu").double()
    assert t.shape == (70000, 8)
    assert float((t[:, :4] ** 2 + t[:, 4:] ** 2 - 1).abs().max()) < 2.0**-21
    assert t[0].tolist() == [1.0] * 4 + [0.0] * 4
    scaled = fx.rotary_table(10, 8, scaling=fx.RotaryScaling(2.0, "linear"), device="cpu")
    assert torch.equal(scaled[2], t[1].float())


def test_device_errors_say_what_happened():
    wait, slot = ("a", 3), ("b", 13)
    assert str(fx.DeviceWaitError([wait])).startswith("device-side wait expired, ")
    text = str(fx.DeviceWaitError([slot]))
    assert "wait" not in text and "out of bounds" in text and "SLOT" in text
    text = str(fx.DeviceWaitError([wait, slot]))
    assert "wait expired and argument out of bounds" in text


@pytest.mark.parametrize("n", [2**30 + 1, 2**31 - 1])
def test_more_tokens_than_the_kernels_count(n):
    """Their 32-bit token numbers would pass 2^31 in the last stride."""
    assert _rotary(T=n) == _lib.FNX_EUNSUPPORTED
    assert _layout(N=n) == _lib.FNX_EUNSUPPORTED
