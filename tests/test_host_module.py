"""The serving calls' host module: absent, or built for another torch, the calls
go the whole way in Python; and it is rebuilt when torch is another one."""
import sys
import types

import pytest
import torch

import heliopause_b200
from heliopause_b200 import _lib, build, kernels as hk


def _refused():
    """A call that the Python form refuses, on a machine without a device too."""
    with pytest.raises(hk.CudaKernelError):
        hk.logits_topk(torch.zeros((2, 100)), 4)


@pytest.fixture
def fresh(monkeypatch):
    monkeypatch.setattr(hk, "_host", None)
    monkeypatch.delattr(heliopause_b200, "_host", raising=False)
    return monkeypatch


def test_absent_module(fresh):
    fresh.setitem(sys.modules, "heliopause_b200._host", None)
    with pytest.warns(RuntimeWarning, match="_host does not load"):
        _refused()
    _refused()  # and says so once


@pytest.mark.parametrize("built_for", ["torch 1.0, python 3.12", None])
def test_module_of_another_torch_is_not_called(fresh, built_for):
    class Module(types.ModuleType):
        def __getattr__(self, name):
            if name == "built_for" or name.startswith("__"):
                raise AttributeError(name)
            pytest.fail(f"{name} was called")

    m = Module("heliopause_b200._host")
    if built_for:
        m.built_for = built_for
    fresh.setitem(sys.modules, "heliopause_b200._host", m)
    with pytest.warns(RuntimeWarning, match="built for"):
        _refused()


def test_built_module_is_of_this_torch(fresh):
    assert hk._load_host().built_for == _lib.host_built_for() and torch.__version__ in _lib.host_built_for()


def test_module_is_rebuilt_for_another_torch(monkeypatch, tmp_path):
    lib, ran = tmp_path / "_host.so", []

    class Done:
        returncode, stdout, stderr = 0, "", ""

    def run(cmd, **kw):
        ran.append(cmd)
        lib.write_bytes(b"")
        return Done

    monkeypatch.setattr(build, "HOST_LIB", lib)
    monkeypatch.setattr(build, "OBJ", tmp_path)
    monkeypatch.setattr(build.subprocess, "run", run)
    build._build_host(False)
    build._build_host(False)
    assert len(ran) == 1
    monkeypatch.setattr(_lib, "host_built_for", lambda: "torch 99, python 3.12")
    build._build_host(False)
    build._build_host(False)
    assert len(ran) == 2 and any("torch 99" in x for x in ran[1])
