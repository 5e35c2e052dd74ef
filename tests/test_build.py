"""The C library builds where torch is not installed: only the binding for torch tensors is left out."""
import importlib.metadata
import importlib.util
import os

from spinn_b200 import build


def test_build_without_torch(monkeypatch, capsys):
    find, version = importlib.util.find_spec, importlib.metadata.version

    def no_torch(name, *a):
        if name == "torch":
            raise importlib.metadata.PackageNotFoundError(name)
        return version(name, *a)

    stamp = os.path.getmtime(build.TORCH_OPS) if os.path.exists(build.TORCH_OPS) else None
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    monkeypatch.setattr(importlib.metadata, "version", no_torch)
    assert build.build() == build.LIB
    assert "torch is not installed" in capsys.readouterr().err
    assert stamp is None or os.path.getmtime(build.TORCH_OPS) == stamp
