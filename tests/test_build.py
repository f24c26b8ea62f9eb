"""What the build makes where torch is missing or changed (CPU; nothing is compiled)."""
import importlib.util
import subprocess
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

from moba_hip.ops import _lib

SOURCE = Path(__file__).resolve().parents[1] / "moba-merge-cuda_amd" / "build.py"


@pytest.fixture
def recorded(monkeypatch, tmp_path):
    """build.py with its outputs in a folder of the test's, and the commands it
    would run (each leaves an empty file as its output)."""
    spec = importlib.util.spec_from_file_location("build_under_test", SOURCE)
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    ran = []

    def run(cmd, **kw):
        out = Path(cmd[cmd.index("-o") + 1])
        assert tmp_path in out.parents
        out.write_bytes(b"")
        ran.append([str(c) for c in cmd])
        return SimpleNamespace(returncode=0, stdout="", stderr="")
    monkeypatch.setattr(subprocess, "run", run)
    monkeypatch.setattr(subprocess, "check_call", run)
    monkeypatch.setattr(build, "OUT_DIR", tmp_path / "obj")
    monkeypatch.setattr(build, "LIB", tmp_path / "libmoba_hip.so")
    monkeypatch.setattr(build, "CALLS", tmp_path / "_calls.so")
    return build, ran


def test_the_library_is_built_without_torch(recorded, monkeypatch, capsys):
    build, ran = recorded
    for name in [m for m in sys.modules if m == "torch" or m.startswith("torch.")]:
        monkeypatch.setitem(sys.modules, name, None)    # import raises ImportError
    assert build.build() == build.LIB and build.LIB.exists()
    assert not build.CALLS.exists() and not any("calls.cpp" in " ".join(c) for c in ran)
    assert "no torch" in capsys.readouterr().err


def test_another_torch_rebuilds_the_extension(recorded, monkeypatch):
    build, ran = recorded
    build.build()
    assert build.CALLS.exists() and sum("calls.cpp" in " ".join(c) for c in ran) == 2   # compiled, linked
    ran.clear()
    build.build()
    assert not ran
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    build.build()
    assert len(ran) == 2 and all("calls.cpp" in " ".join(c) for c in ran)
    assert any("torch 9.9.9" in x for x in ran[0])


def test_an_extension_of_another_torch_is_refused(monkeypatch):
    _lib.calls()
    monkeypatch.setattr(_lib, "_calls", None)
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    with pytest.raises(_lib.MobaHipError, match="build it again"):
        _lib.calls()
