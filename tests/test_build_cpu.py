"""The build on the host: when the native binding is made anew, with the compiler stood in for."""

import importlib

import pytest
import torch

from flash_next_rtxpro6000_b200 import _lib

build = importlib.import_module("flash_next_rtxpro6000_b200.build")


def test_the_binding_in_the_tree_is_of_this_torch():
    _lib.ops()
    assert build.binding_fits() and torch.__version__ in _lib.ops().__doc__


@pytest.mark.parametrize("there", ["another torch", "none"])
def test_a_binding_of_another_torch_is_built_again(there, tmp_path, monkeypatch):
    _lib.ops()
    path = tmp_path / build.OPS_PATH.name
    whole = build.OPS_PATH.read_bytes()
    if there != "none":
        path.write_bytes(whole.replace(build.binding_build().encode(), b"x" * len(build.binding_build())))
    monkeypatch.setattr(build, "OPS_PATH", path)
    monkeypatch.setattr(_lib, "OPS_PATH", path)
    assert not build.binding_fits() and not build.up_to_date()
    built = []

    def compiler():
        built.append(1)
        path.write_bytes(whole)

    monkeypatch.setattr(build, "build_binding", compiler)
    loaded = []
    monkeypatch.setattr(importlib.machinery, "ExtensionFileLoader", lambda name, at: loaded.append(at) or Loader())
    monkeypatch.setattr(_lib, "_ops", None)
    _lib.ops()
    assert built == [1] and loaded == [str(path)] and build.binding_fits()


class Loader:  # what is loaded is not the point here, and a second copy of the extension is not wanted
    def create_module(self, spec):
        return None

    def exec_module(self, module):
        pass


def test_the_library_needs_no_binding(tmp_path, monkeypatch):
    """Where torch's or Python's headers are missing the GEMVs, MoE and router load as ever."""
    path = tmp_path / build.LIB_PATH.name
    monkeypatch.setattr(build, "LIB_PATH", path)
    monkeypatch.setattr(_lib, "LIB_PATH", path)
    monkeypatch.setattr(build, "OBJ_DIR", tmp_path / "objects")
    monkeypatch.setattr(build, "nvcc", lambda: "nvcc")

    class Done:
        returncode, stdout, stderr = 0, "", ""

    def compiler(cmd, **kw):
        assert cmd[0] == "nvcc"
        out = cmd[cmd.index("-o") + 1]
        with open(out, "w") as f:
            f.write("made")
        return Done

    def no_headers():
        raise RuntimeError("Python.h: no such file")

    monkeypatch.setattr(build.subprocess, "run", compiler)
    monkeypatch.setattr(build, "build_binding", no_headers)
    monkeypatch.setattr(_lib, "_declare", lambda handle: None)
    monkeypatch.setattr(_lib.ctypes, "CDLL", lambda at: at)
    monkeypatch.setattr(_lib, "_lib", None)
    assert _lib.lib() == str(path) and path.read_text() == "made"
    with pytest.raises(RuntimeError):  # the command still says so
        build.build(force=True)
