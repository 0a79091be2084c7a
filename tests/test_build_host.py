"""The build where torch is missing, was built without CUDA, or is another
version than the binding was built for."""
import builtins
import types

import pytest

from witchcraft_b200 import build as b


@pytest.fixture
def binding(tmp_path, monkeypatch):
    """The binding's file and stamp in a folder of their own; compiler calls are
    recorded in place of being made."""
    runs = []
    monkeypatch.setattr(b, "BUILD_DIR", str(tmp_path))
    monkeypatch.setattr(b, "TORCH_BINDING", str(tmp_path / "_fp8_torch.so"))

    def run(cmd):
        runs.append(cmd)
        open(b.TORCH_BINDING, "w").close()
    monkeypatch.setattr(b, "_run", run)
    return runs


def without_torch(monkeypatch, replacement=None):
    real = builtins.__import__

    def fake(name, *args, **kw):
        if name == "torch" or name.startswith("torch."):
            if replacement is None:
                raise ImportError(name)
            return replacement
        return real(name, *args, **kw)
    monkeypatch.setattr(builtins, "__import__", fake)


def test_no_torch_is_no_binding(binding, monkeypatch):
    without_torch(monkeypatch)
    assert b.build_torch_binding(force=True) is None and not binding


def test_torch_without_cuda_is_no_binding(binding, monkeypatch):
    without_torch(monkeypatch, types.SimpleNamespace(version=types.SimpleNamespace(cuda=None), __version__="2"))
    assert b.build_torch_binding(force=True) is None and not binding


def test_library_builds_without_torch(binding, monkeypatch):
    monkeypatch.setattr(b, "_nvcc", lambda: "nvcc")
    monkeypatch.setattr(b, "_stale", lambda target, deps: target == b.TORCH_BINDING)  # all else is up to date
    without_torch(monkeypatch)
    assert b.build() == b.LIB and not binding


def test_binding_follows_torch(binding, monkeypatch):
    import torch
    assert b.build_torch_binding() == b.TORCH_BINDING and len(binding) == 1
    b.build_torch_binding()
    assert len(binding) == 1               # up to date
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    b.build_torch_binding()
    assert len(binding) == 2               # another torch
