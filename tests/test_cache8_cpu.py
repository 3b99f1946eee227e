"""The C entry points of the operators around the 8-bit cache and of verification refuse bad arguments before any
launch, and the Python ones refuse tensors that are not on a GPU."""

import ctypes

import pytest
import torch

import flash_next_rtxpro6000_b200 as fx
from flash_next_rtxpro6000_b200 import _lib

S3 = ctypes.c_int64 * 3


def _call(name, args, kw):
    assert set(kw) <= set(args), kw
    return getattr(_lib.lib(), name)(*(args | kw).values())


def _append(**kw):
    return _call("fnx_rotary_append8", dict(
        q=16, q_st=256, q_sh=64, k=16, k_st=128, k_sh=64, v=16, v_st=128, v_sh=64, out=16, o_st=256, o_sh=64, pos=16,
        ctx=16, off=16, pt=16, pt_ld=4, width=4, table=16, table_ld=64, P=100, kc=16, kcs=S3(4096, 128, 64), vc=16,
        vcs=S3(4096, 128, 64), ks=16, kss=S3(4, 2, 1), vs=16, vss=S3(4, 2, 1), pages=4, page=32, block=16, B=1, T=2,
        Hq=4, Hk=2, D=64, R=64, inter=0, dtype=0, err=None, pdl=0, stream=None), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(T=0), _lib.FNX_OK), (dict(dtype=2), _lib.FNX_EUNSUPPORTED), (dict(T=-1), _lib.FNX_EINVAL),
    (dict(D=96), _lib.FNX_EUNSUPPORTED), (dict(block=8), _lib.FNX_EUNSUPPORTED), (dict(block=24), _lib.FNX_EUNSUPPORTED),
    (dict(page=24), _lib.FNX_EINVAL), (dict(page=0), _lib.FNX_EINVAL), (dict(R=66), _lib.FNX_EINVAL),
    (dict(R=63), _lib.FNX_EINVAL), (dict(P=0), _lib.FNX_EINVAL), (dict(table_ld=32), _lib.FNX_EINVAL),
    (dict(q=None), _lib.FNX_EINVAL), (dict(v=None), _lib.FNX_EINVAL), (dict(ks=None), _lib.FNX_EINVAL),
    (dict(vss=None), _lib.FNX_EINVAL), (dict(pt=None), _lib.FNX_EINVAL), (dict(B=0), _lib.FNX_EINVAL),
    (dict(kc=8), _lib.FNX_EINVAL), (dict(kcs=S3(4096, 136, 64)), _lib.FNX_EINVAL), (dict(Hk=0), _lib.FNX_EINVAL),
    (dict(T=2**24 + 1), _lib.FNX_EUNSUPPORTED), (dict(B=2**16 + 1), _lib.FNX_EUNSUPPORTED),
])
def test_rotary_append8(kw, code):
    assert _append(**kw) == code
    assert bool(_lib.last_error()) == (code != _lib.FNX_OK)


def _attention(**kw):
    return _call("fnx_tree_attention8", dict(
        q=16, q_sn=256, q_sh=64, kc=16, kcs=S3(4096, 128, 64), vc=16, vcs=S3(4096, 128, 64), ks=16, kss=S3(4, 2, 1),
        vs=16, vss=S3(4, 2, 1), pages=4, page=32, block=16, table=16, table_ld=4, width=4, ctx=16, off=16, mask=None,
        out=16, o_sn=256, o_sh=64, lse=None, B=1, N=2, Hq=4, Hk=2, D=64, max_nodes=2, max_context=60, scale=0.125,
        dtype=0, part=16, err=None, pdl=0, stream=None), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(N=0), _lib.FNX_OK), (dict(dtype=2), _lib.FNX_EUNSUPPORTED), (dict(D=96), _lib.FNX_EUNSUPPORTED),
    (dict(Hq=3), _lib.FNX_EINVAL), (dict(B=0), _lib.FNX_EINVAL), (dict(max_nodes=65), _lib.FNX_EUNSUPPORTED),
    (dict(max_context=-1), _lib.FNX_EINVAL), (dict(block=128), _lib.FNX_EUNSUPPORTED), (dict(page=40), _lib.FNX_EINVAL),
    (dict(ks=None), _lib.FNX_EINVAL), (dict(kss=None), _lib.FNX_EINVAL), (dict(part=None), _lib.FNX_EINVAL),
    (dict(q=8), _lib.FNX_EINVAL), (dict(kcs=S3(4096, 128, 72)), _lib.FNX_EINVAL), (dict(scale=0.0), _lib.FNX_EINVAL),
])
def test_tree_attention8(kw, code):
    assert _attention(**kw) == code
    assert bool(_lib.last_error()) == (code != _lib.FNX_OK)


def _probs(**kw):
    return _call("fnx_token_probs", dict(logits=16, ldl=100, dtype=2, M=2, V=100, t=None, k=None, p=None, mp=None,
                                         probs=16, ldp=100, scratch=16, pdl=0, stream=None), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(M=0), _lib.FNX_OK), (dict(dtype=3), _lib.FNX_EUNSUPPORTED), (dict(V=0), _lib.FNX_EINVAL),
    (dict(ldl=99), _lib.FNX_EINVAL), (dict(ldp=99), _lib.FNX_EINVAL), (dict(V=2**22, ldl=2**23, ldp=2**23), _lib.FNX_EUNSUPPORTED),
    (dict(logits=None), _lib.FNX_EINVAL), (dict(probs=None), _lib.FNX_EINVAL), (dict(scratch=None), _lib.FNX_EINVAL),
    (dict(scratch=12), _lib.FNX_EINVAL),
])
def test_token_probs(kw, code):
    assert _probs(**kw) == code
    assert bool(_lib.last_error()) == (code != _lib.FNX_OK)


def _verify(**kw):
    return _call("fnx_verify_tokens", dict(
        target=16, ldt=100, draft=16, ldd=100, tokens=16, parents=16, off=16, nu=16, du=16, B=1, N=3, V=100, max_nodes=4,
        path=16, accepted=16, next=16, err=None, pdl=0, stream=None), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(B=0), _lib.FNX_OK), (dict(V=0), _lib.FNX_EINVAL), (dict(ldt=99), _lib.FNX_EINVAL), (dict(ldd=99), _lib.FNX_EINVAL),
    (dict(max_nodes=0), _lib.FNX_EINVAL), (dict(max_nodes=65), _lib.FNX_EUNSUPPORTED), (dict(N=-1), _lib.FNX_EINVAL),
    (dict(V=2**21 + 1, ldt=2**22, ldd=2**22), _lib.FNX_EUNSUPPORTED), (dict(target=None), _lib.FNX_EINVAL),
    (dict(tokens=None), _lib.FNX_EINVAL), (dict(du=None), _lib.FNX_EINVAL), (dict(path=None), _lib.FNX_EINVAL),
])
def test_verify_tokens(kw, code):
    assert _verify(**kw) == code
    assert bool(_lib.last_error()) == (code != _lib.FNX_OK)


def _compact(**kw):
    return _call("fnx_compact_nodes", dict(
        kc=16, kcs=S3(4096, 128, 64), kl=0, vc=16, vcs=S3(4096, 128, 64), vl=0, ks=16, kss=S3(4, 2, 1), ksl=0, vs=16,
        vss=S3(4, 2, 1), vsl=0, pages=4, page=32, block=16, elem=1, layers=1, Hk=2, D=64, pt=16, pt_ld=4, width=4, ctx=16,
        path=16, path_ld=8, acc=16, B=1, W=8, lens=None, err=None, pdl=0, stream=None), kw)


@pytest.mark.parametrize("kw,code", [
    (dict(B=0), _lib.FNX_OK), (dict(elem=4), _lib.FNX_EUNSUPPORTED), (dict(D=32), _lib.FNX_EUNSUPPORTED),
    (dict(page=24), _lib.FNX_EINVAL), (dict(W=65, path_ld=65), _lib.FNX_EUNSUPPORTED), (dict(path_ld=7), _lib.FNX_EINVAL),
    (dict(layers=0), _lib.FNX_EINVAL), (dict(kc=None), _lib.FNX_EINVAL), (dict(ks=None), _lib.FNX_EINVAL),
    (dict(kl=8), _lib.FNX_EINVAL), (dict(vcs=S3(4096, 128, 60)), _lib.FNX_EINVAL), (dict(path=None), _lib.FNX_EINVAL),
    (dict(elem=2, D=4), _lib.FNX_EINVAL), (dict(Hk=2**15), _lib.FNX_EUNSUPPORTED), (dict(layers=2**30), _lib.FNX_EUNSUPPORTED),
])
def test_compact_nodes(kw, code):
    assert _compact(**kw) == code
    assert bool(_lib.last_error()) == (code != _lib.FNX_OK)


def test_tensors_on_the_host_are_refused():
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    c = torch.zeros(2, 16, 4, 64, dtype=torch.bfloat16).to(torch.float8_e4m3fn)
    s = torch.ones(2, 1, 4)
    i, i32 = torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    off, u = torch.zeros(3, dtype=torch.int32), torch.zeros(2)
    with pytest.raises(ValueError):
        fx.rotary_append8(x, x, x, i, i32, off, i32.view(2, 1), torch.zeros(9, 64), c, c, s, s)
    with pytest.raises(ValueError):
        fx.tree_attention8(x, c, c, s, s, i32.view(2, 1), i32, off)
    with pytest.raises(ValueError):
        fx.token_probs(torch.zeros(2, 9))
    with pytest.raises(ValueError):
        fx.verify_tokens(torch.zeros(2, 9), None, i, i32, off, u, u)
    with pytest.raises(ValueError):
        fx.compact_nodes(c, c, i32.view(2, 1), i32, i32.view(2, 1), i32, s, s)


def test_new_device_errors_are_arguments():
    for code, text in ((17, "TOKEN"), (18, "SCALE")):
        message = str(fx.DeviceWaitError([("a", code)]))
        assert text in message and "out of bounds" in message and "wait" not in message
