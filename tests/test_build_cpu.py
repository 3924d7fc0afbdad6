"""What the build makes of which tools (the compilers replaced by a recorder)."""

import importlib.util
import os
import subprocess
import sys
from types import SimpleNamespace

import pytest

BUILD_PY = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nki-moe-7013_amd", "build.py")


@pytest.fixture
def build(tmp_path, monkeypatch):
    """The build module with its outputs under tmp_path; ``ran`` collects the commands."""
    spec = importlib.util.spec_from_file_location("qmoe_build", BUILD_PY)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    for name in ("OUT_DIR", "LIB", "NATIVE", "PROBE_LIB", "BUILD_INFO"):
        monkeypatch.setattr(mod, name, str(tmp_path / os.path.basename(getattr(mod, name))))
    mod.ran, mod.native_fails = [], False

    def run(cmd, **kw):
        mod.ran.append(cmd)
        if cmd[0] != "git":
            if mod.native_fails and mod.NATIVE_SRC in cmd:
                return SimpleNamespace(returncode=1, stdout="", stderr="no torch/headers.h")
            with open(cmd[cmd.index("-o") + 1], "w"):
                pass
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(subprocess, "run", run)
    return mod


def test_build_makes_everything(build):
    assert build.build(2) == build.LIB
    assert all(os.path.exists(p) for p in (build.LIB, build.PROBE_LIB, build.BUILD_INFO, build.NATIVE))


def test_libraries_need_no_torch(build, monkeypatch, capsys):
    build.build(2)
    monkeypatch.setitem(sys.modules, "torch", None)  # import torch: ImportError
    for p in (build.LIB, build.PROBE_LIB, build.BUILD_INFO):
        os.remove(p)
    assert build.build(2) == build.LIB
    assert all(os.path.exists(p) for p in (build.LIB, build.PROBE_LIB, build.BUILD_INFO))
    assert not os.path.exists(build.NATIVE)  # not that of an earlier library
    assert "_native.so" in capsys.readouterr().err


def test_a_module_that_does_not_compile_fails_after_the_libraries(build):
    build.native_fails = True
    with pytest.raises(RuntimeError, match="native module failed"):
        build.build(2)
    assert all(os.path.exists(p) for p in (build.LIB, build.PROBE_LIB, build.BUILD_INFO))


def test_module_without_gxx(build, monkeypatch):
    monkeypatch.setattr(build.shutil, "which", lambda name: None)
    build.build(2)
    cmd = next(c for c in build.ran if build.NATIVE_SRC in c)
    assert cmd[0].endswith("llvm/bin/clang++")
