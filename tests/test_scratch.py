"""The scratch slots on the host: what first calls allocate, and that the raw addresses handed to the
native binding belong to tensors that stay alive.  Device tensors are stood in for by host ones."""

import importlib
import threading
import time

import pytest
import torch

from flash_next_rtxpro6000_b200 import _lib

w8a16_gemv = importlib.import_module("flash_next_rtxpro6000_b200.w8a16_gemv")  # the package has a function of that name


class FakeLib:
    """The attention scratch's size goes by the device that is current when it is asked for."""

    current = 0
    floats = {0: 1000, 1: 1600}

    def fnx_tree_attention_workspace_floats(self, n):
        time.sleep(0.02)  # lets the other threads get here too
        n._obj.value = self.floats[self.current]
        return 0


class FakeWorkspace:
    def __init__(self, device):
        time.sleep(0.02)
        self.device = torch.device("cpu")
        self.error_flag = torch.zeros(1, dtype=torch.int32)
        self.attention = None


class On:
    """A tensor's place, as far as the scratch looks at it."""

    is_cuda = True

    def __init__(self, index=0):
        self.index = index

    def get_device(self):
        return self.index


@pytest.fixture
def slots(monkeypatch):
    monkeypatch.setattr(w8a16_gemv, "Workspace", FakeWorkspace)
    for name in ("_WS", "_ADDRESSES", "_FLAGS"):
        monkeypatch.setattr(w8a16_gemv, name, {})
    monkeypatch.setattr(w8a16_gemv, "_ONES", {torch.device("cuda", i): None for i in range(2)})
    fake = FakeLib()
    monkeypatch.setattr(_lib, "_lib", fake)

    class Device:  # torch.cuda.device
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, fake.current = fake.current, self.index

        def __exit__(self, *exc):
            fake.current = self.before

    monkeypatch.setattr(torch.cuda, "device", Device)
    return fake


def test_first_calls_of_many_threads_share_one_live_scratch(slots):
    got, start = [], threading.Barrier(8)

    def call():
        start.wait()
        got.append(tuple(w8a16_gemv._scratch(On())[:2]))

    threads = [threading.Thread(target=call) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    (ws,) = w8a16_gemv._WS.values()
    live = (ws.error_flag.data_ptr(), ws.attention.data_ptr())
    assert set(got) == {live} and tuple(w8a16_gemv._scratch(On())[:2]) == live


def test_the_scratch_is_sized_for_its_own_device(slots):
    w8a16_gemv.prealloc("cuda:1", attention=True)  # while device 0 is current
    assert slots.current == 0
    for slot in (0, 1):
        assert w8a16_gemv._WS[(torch.device("cuda", 1), slot)].attention.numel() == slots.floats[1]
    w8a16_gemv._scratch(On(0))
    assert w8a16_gemv._WS[(torch.device("cuda", 0), 0)].attention.numel() == slots.floats[0]


def test_only_the_attention_makes_its_scratch(slots):
    w8a16_gemv.prealloc("cuda:0")
    flag = w8a16_gemv._flag(On())
    (ws, other) = w8a16_gemv._WS.values()
    assert flag == ws.error_flag.data_ptr() and ws.attention is None and other.attention is None
    assert w8a16_gemv._scratch(On())[:2] == (flag, ws.attention.data_ptr())
    assert other.attention is None
    w8a16_gemv.prealloc("cuda:0", attention=True)
    assert other.attention is not None and w8a16_gemv._scratch(On())[1] == ws.attention.data_ptr()
