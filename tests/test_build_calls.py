"""The module of the paged cache's calls is there for speed alone: what keeps it from
being built or loaded is noted, and the calls go by ctypes (no GPU)."""
import importlib
import subprocess
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest

pytest.importorskip("torch")
ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture
def build(tmp_path, monkeypatch):
    b = importlib.import_module("firepit_b200.build")
    monkeypatch.setattr(b, "CALLS", tmp_path / "_calls.so")
    monkeypatch.setattr(b, "BUILD", tmp_path)
    return b


@pytest.mark.parametrize("failure", ["no compiler", "no header", "no nvcc", "no version"])
def test_a_module_that_does_not_build_is_noted(build, monkeypatch, failure):
    build.CALLS.write_text("an older one, for other entry points")

    def run(cmd, **kw):
        if failure == "no compiler":
            raise FileNotFoundError("g++")
        return SimpleNamespace(returncode=1, stdout="", stderr="c10_cuda: no such file")

    monkeypatch.setattr(build.subprocess, "run", run)
    if failure == "no nvcc":
        monkeypatch.setattr(build, "nvcc", lambda: (_ for _ in ()).throw(RuntimeError("nvcc not found")))
    if failure == "no version":
        monkeypatch.setattr(build.runpy, "run_path", lambda p: {})
    with pytest.warns(UserWarning, match="ctypes"):
        build._build_calls(True)
    assert not build.CALLS.exists()


def test_the_module_is_made_again_for_another_torch(build, monkeypatch):
    made = []

    def run(cmd, **kw):
        made.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_text("module")
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(build.subprocess, "run", run)
    build._build_calls(False)
    build._build_calls(False)
    assert len(made) == 1 and build.CALLS.exists()
    monkeypatch.setattr(build.runpy, "run_path", lambda p: {"__version__": "9.9"})
    build._build_calls(False)
    build._build_calls(False)
    assert len(made) == 2 and any("9.9" in word for word in made[1])
    monkeypatch.setattr(build.sys, "implementation", SimpleNamespace(cache_tag="cpython-999"))
    build._build_calls(False)
    assert len(made) == 3


def test_a_module_for_another_torch_is_not_loaded():
    if not (ROOT / "firepit_b200" / "_calls.so").exists():
        pytest.skip("_calls.so is not built")
    code = ("import torch, warnings; torch.__version__ = '9.9'\n"
            "from firepit_b200.speculative import _Torch\n"
            "with warnings.catch_warnings(record=True) as seen:\n"
            "    warnings.simplefilter('always')\n"
            "    _Torch.load()\n"
            "assert _Torch.calls is None and _Torch.module is torch\n"
            "assert any('9.9' in str(w.message) and 'ctypes' in str(w.message) for w in seen), seen\n")
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True, timeout=300)
