"""The module of the short way (mantle_cuda/_launch) is built beside the library and bound to one torch and
one Python; where it cannot be built the build goes on without it."""
import importlib
import importlib.util
import subprocess
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest

import mantle_cuda as M

ROOT = Path(__file__).resolve().parent.parent
torch = pytest.importorskip("torch")


@pytest.fixture
def b(tmp_path, monkeypatch):
    """build.py with its outputs in a folder of the test's, and a compiler that writes down what it is asked."""
    spec = importlib.util.spec_from_file_location("build_under_test", ROOT / "mantle.jl_b200" / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    build.OBJ, build.LAUNCH_OUT, build.calls = tmp_path, tmp_path / build.LAUNCH_OUT.name, []

    def run(cmd, **kw):
        build.calls.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_bytes(b"built")
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    return build


with_cuda = pytest.mark.skipif(not torch.version.cuda, reason="a torch without CUDA")


@with_cuda
def test_the_module_is_there_and_loads():
    # a build that lost it would only be slower, and its other tests skipped
    importlib.import_module("mantle_cuda._launch")
    M._with_torch()
    assert M._short_launch is not None


@with_cuda
def test_it_is_built_once_and_again_for_another_torch_or_python(b, monkeypatch):
    b.build_launch()
    b.build_launch()
    assert len(b.calls) == 1 and b.LAUNCH_OUT.name.endswith(importlib.machinery.EXTENSION_SUFFIXES[0])
    stamp = b.OBJ / "launch.stamp"
    stamp.write_text(stamp.read_text().replace(torch.__version__, "1.0"))  # as an upgrade leaves it
    b.build_launch()
    assert len(b.calls) == 2
    monkeypatch.setattr(b.sys, "version", "3.99")
    b.build_launch()
    assert len(b.calls) == 3
    b.LAUNCH_OUT.unlink()
    b.build_launch()
    assert len(b.calls) == 4
    b.build_launch(force=True)
    assert len(b.calls) == 5


@with_cuda
@pytest.mark.parametrize("how", ["no compiler", "no headers"])
def test_a_build_without_it_goes_on_and_leaves_no_old_one(b, monkeypatch, capsys, how):
    b.build_launch()
    old = b.LAUNCH_OUT.with_name("_launch.so")  # of a build before names had a tag
    old.write_bytes(b"old")

    def run(cmd, **kw):
        if how == "no compiler":
            raise FileNotFoundError("g++")
        return SimpleNamespace(returncode=1, stdout="", stderr="Python.h: No such file")

    monkeypatch.setattr(b.subprocess, "run", run)
    b.build_launch(force=True)
    assert "was not built" in capsys.readouterr().err
    assert not b.LAUNCH_OUT.exists() and not old.exists() and not (b.OBJ / "launch.stamp").exists()


@pytest.mark.parametrize("spec", [None, SimpleNamespace(origin=None)])
def test_without_torch_there_is_nothing_to_build(b, monkeypatch, spec):
    monkeypatch.setattr(b.importlib.util, "find_spec", lambda name: spec)
    b.build_launch()
    assert b.calls == []


@with_cuda
def test_another_torch_takes_the_long_way():
    code = ("import sys; sys.path.insert(0, 'mantle.jl_b200')\nimport torch\ntorch.__version__ = '0.1'\nimport mantle_cuda as M\nM._with_torch()\n"
            "assert M._short_launch is None\ntry:\n    import mantle_cuda._launch\nexcept ImportError as e:\n    print(e)")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert r.returncode == 0, r.stderr
    assert r.stdout.strip() == f"_launch was built for torch {torch.__version__}, not 0.1"
