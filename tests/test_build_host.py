"""CPU: the build's own logic, with the compilers replaced by writers of small files."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

from cugo_b200 import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """Empty library folders, and a `run` that writes what a compiler would."""
    monkeypatch.setattr(build, "LIB_DIR", tmp_path)
    monkeypatch.setattr(build, "LIB", tmp_path / build.LIB.name)
    monkeypatch.setattr(build, "BINDING", tmp_path / build.BINDING.name)
    if hasattr(build, "BUILT_FOR"):
        monkeypatch.setattr(build, "BUILT_FOR", tmp_path / build.BUILT_FOR.name)
    commands = []

    def run(command, check):
        assert check
        commands.append(command)
        Path(command[command.index("-o") + 1]).write_text("built")

    monkeypatch.setattr(build.subprocess, "run", run)
    return commands


def test_the_library_is_built_without_torch(tree, monkeypatch, capsys):
    """No torch, no host compiler, or a binding that does not compile: the library is there and
    the call ends well; what is missing is said."""
    monkeypatch.setitem(sys.modules, "torch", None)  # an ImportError
    assert build.build(force=True) == build.LIB and build.LIB.exists() and not build.BINDING.exists()
    assert "was not built" in capsys.readouterr().err


@pytest.mark.parametrize("error", [FileNotFoundError("g++"), subprocess.CalledProcessError(1, "g++")])
def test_the_library_is_built_without_a_host_compiler(tree, monkeypatch, capsys, error):
    written = build.subprocess.run

    def run(command, check):
        if str(build.BINDING_SOURCE) in command:
            raise error
        written(command, check)

    monkeypatch.setattr(build.subprocess, "run", run)
    assert build.build(force=True) == build.LIB and build.LIB.exists() and not build.BINDING.exists()
    assert "was not built" in capsys.readouterr().err
    with pytest.raises(type(error)):
        build.build_binding()
