"""build.py: what it builds where, and from what.  Nothing is compiled here: the compilers' command lines are recorded."""
from __future__ import annotations

import subprocess
import sys
import sysconfig

import pytest


@pytest.fixture
def recorded(monkeypatch, tmp_path):
    """The build module with an empty output folder, and the command lines that it runs."""
    import build

    commands = []

    def run(cmd, **_):
        commands.append([str(x) for x in cmd])
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "BUILD", tmp_path / "_build")
    monkeypatch.setattr(build, "LIB", tmp_path / "lib" / "libb2g.so")
    return build, commands


def test_the_c_library_needs_no_torch(recorded, monkeypatch, capsys):
    build, commands = recorded
    monkeypatch.setitem(sys.modules, "torch", None)  # (import torch raises)
    assert build.build(force=True) == build.LIB
    assert any(str(build.LIB) in c for c in commands) and not any("calls.cpp" in x for c in commands for x in c)
    assert "no torch" in capsys.readouterr().err


def test_the_c_library_needs_no_python_headers(recorded, monkeypatch, tmp_path, capsys):
    build, commands = recorded
    paths = sysconfig.get_paths()
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda *a, **k: {**paths, "include": str(tmp_path)})
    assert build.build(force=True) == build.LIB
    assert any(str(build.LIB) in c for c in commands) and not any("calls.cpp" in x for c in commands for x in c)
    assert "no Python.h" in capsys.readouterr().err


def test_both_libraries_are_built(recorded):
    build, commands = recorded
    build.build(force=True)
    assert any(str(build.LIB) in c for c in commands) and any(x.endswith("calls.cpp") for c in commands for x in c)


def test_the_python_side_belongs_to_one_torch_and_interpreter(recorded, monkeypatch, tmp_path):
    """Their versions are in its name, and a file of another name does not pass for it, however new."""
    import torch

    import b2g

    build, commands = recorded
    assert torch.__version__ in b2g.CALLS_PATH.name and sysconfig.get_config_var("SOABI") in b2g.CALLS_PATH.name
    other = tmp_path / b2g.CALLS_PATH.name.replace(torch.__version__, "0.0.1")
    monkeypatch.setattr(b2g, "CALLS_PATH", other)
    assert build.build_calls() == other
    assert [c for c in commands if str(other) in c and any(x.endswith("calls.cpp") for x in c)]
    assert f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}" in commands[0]
    with pytest.raises(b2g.B2GError, match="is missing: build it"):
        monkeypatch.setattr(b2g, "_calls", None)
        b2g.gemm_s8(torch.zeros(1, 16), torch.zeros(1, 16, dtype=torch.int8), torch.ones(1))
