"""The module of the paged cache's calls is there for speed alone: what keeps it from
being built is noted, and the calls go by ctypes (no GPU)."""
import importlib
from types import SimpleNamespace

import pytest

pytest.importorskip("torch")


@pytest.fixture
def build(tmp_path, monkeypatch):
    b = importlib.import_module("firepit_b200.build")
    monkeypatch.setattr(b, "CALLS", tmp_path / "_calls.so")
    monkeypatch.setattr(b, "BUILD", tmp_path)
    return b


@pytest.mark.parametrize("failure", ["no compiler", "no header", "no nvcc"])
def test_a_module_that_does_not_build_is_noted(build, monkeypatch, failure):
    build.CALLS.write_text("an older one, for other entry points")

    def run(cmd, **kw):
        if failure == "no compiler":
            raise FileNotFoundError("g++")
        return SimpleNamespace(returncode=1, stdout="", stderr="c10_cuda: no such file")

    monkeypatch.setattr(build.subprocess, "run", run)
    if failure == "no nvcc":
        monkeypatch.setattr(build, "nvcc", lambda: (_ for _ in ()).throw(RuntimeError("nvcc not found")))
    with pytest.warns(UserWarning, match="ctypes"):
        build._build_calls(True)
    assert not build.CALLS.exists()
