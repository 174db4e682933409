"""What the build makes, and beside which torch: nothing is compiled here."""
import importlib.machinery
import importlib.util
import os

import pytest

from ecahlang_b200 import build as B


@pytest.fixture
def steps(monkeypatch, tmp_path):
    """The build's steps, recorded: sources compiled, the link, the binding."""
    done = []
    monkeypatch.setattr(B, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(B, "BINDING", str(tmp_path / "binding.so"))
    monkeypatch.setattr(B, "OBJ_DIR", str(tmp_path / "build"))
    monkeypatch.setattr(B, "_object", lambda source, force, verbose: done.append(source) or source)

    def run(cmd, check):
        out = cmd[cmd.index("-o") + 1]
        done.append("binding" if out.startswith(B.BINDING) else "library")
        open(out, "w").close()
    monkeypatch.setattr(B.subprocess, "run", run)
    return done


def _torch_at(monkeypatch, origin):
    spec = None if origin is None else importlib.machinery.ModuleSpec("torch", None, origin=origin)
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: spec if name == "torch" else find(name, *a))


@pytest.mark.parametrize("torch", ["none", "namespace", "cpu"])
def test_the_library_builds_without_a_cuda_torch(monkeypatch, tmp_path, steps, torch):
    os.makedirs(tmp_path / "torch" / "lib")
    _torch_at(monkeypatch, str(tmp_path / "torch" / "__init__.py") if torch == "cpu" else None)
    if torch == "namespace":
        find = importlib.util.find_spec
        monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a:
                            importlib.machinery.ModuleSpec("torch", None) if name == "torch" else find(name, *a))
    assert B.build(force=True) == B.LIB
    assert sorted(steps) == sorted([*B.SOURCES, "library"])


def test_the_binding_builds_beside_a_cuda_torch(monkeypatch, tmp_path, steps):
    os.makedirs(tmp_path / "torch" / "lib")
    (tmp_path / "torch" / "lib" / "libtorch_cuda.so").write_bytes(b"")
    _torch_at(monkeypatch, str(tmp_path / "torch" / "__init__.py"))
    B.build(force=True)
    assert sorted(steps) == sorted([*B.SOURCES, "library", "binding"])


def test_a_binding_of_another_torch_or_interpreter_is_not_taken(monkeypatch):
    """Its file name holds both versions, and loading looks for the one that building makes."""
    import torch
    from ecahlang_b200 import _abi
    B.build()
    assert B.BINDING == B.binding_path() and not B._stale(B.BINDING)
    here = os.path.basename(B.BINDING)
    assert B.sysconfig.get_config_var("SOABI") in here and torch.__version__ in here
    monkeypatch.setattr(B.importlib.metadata, "version", lambda name: "9.9.9")
    other = B.binding_path()
    assert other != B.BINDING and B._stale(other)
    monkeypatch.setattr(_abi, "_binding", None)
    with pytest.raises(_abi.EcahError, match="torch-9.9.9.so is missing"):
        _abi.binding()
