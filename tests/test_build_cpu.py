"""The build step: what a failing binding costs, and when it is built again.  No compiler runs here."""
import importlib.util
import subprocess
from pathlib import Path

import pytest
import torch

from conftest import PKG
from speech_serving import _native as N


@pytest.fixture
def build(monkeypatch, tmp_path):
    """csrc/build.py with its outputs under tmp_path and compilers that only write their output file."""
    spec = importlib.util.spec_from_file_location("spd_build", PKG / "csrc" / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    monkeypatch.setattr(mod, "OBJ_DIR", tmp_path / "_build")
    monkeypatch.setattr(mod, "LIB", tmp_path / "lib" / "libspd_b200.so")
    monkeypatch.setattr(mod, "BINDING", tmp_path / "lib" / "spd_torch.so")
    monkeypatch.setattr(mod, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    mod.ran, mod.broken = [], set()

    def run(cmd, **kw):
        tool = Path(cmd[0]).name
        mod.ran.append(tool)
        if tool in mod.broken:
            return subprocess.CompletedProcess(cmd, 1, "", "")
        Path(cmd[cmd.index("-o") + 1]).write_text(tool)
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(mod.subprocess, "run", run)
    return mod


def test_a_binding_that_does_not_compile_leaves_the_library_built(build):
    build.broken.add("g++")
    with pytest.raises(RuntimeError, match="torch_binding.cpp"):
        build.build()
    assert build.LIB.exists() and not build.BINDING.exists()
    build.broken.clear()
    build.ran.clear()
    assert build.build() == build.LIB and build.BINDING.exists()
    assert build.ran == ["g++"]  # nothing else was left to do


def test_a_binding_that_no_longer_fits_is_not_left_behind(build, monkeypatch):
    build.build()
    monkeypatch.setattr(torch, "__version__", "0.0.0+other")
    build.broken.add("g++")
    with pytest.raises(RuntimeError, match="torch_binding.cpp"):
        build.build()
    assert not build.BINDING.exists()


def test_the_binding_is_built_again_for_another_torch_only(build, monkeypatch):
    build.build()
    build.ran.clear()
    build.build()
    assert build.ran == []
    monkeypatch.setattr(torch, "__version__", "0.0.0+other")
    build.build()
    assert build.ran == ["g++"]


def test_a_binding_that_does_not_load_says_what_to_do(monkeypatch, tmp_path):
    bad = tmp_path / "spd_torch.so"
    bad.write_text("not a library")
    monkeypatch.setattr(N, "BINDING_PATH", bad)
    monkeypatch.setattr(N, "_binding", None)
    with pytest.raises(RuntimeError, match="build it again"):
        N.binding()
