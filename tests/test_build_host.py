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
    commands = []

    def run(command, check):
        assert check
        commands.append(command)
        Path(command[command.index("-o") + 1]).write_text(" ".join(command))

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


def test_a_binding_of_another_torch_is_built_again(tree, monkeypatch):
    """The binding goes by the torch and Python it was built against, not by its date alone."""
    from cugo_b200 import ext
    build.build(force=True)
    count = len(tree)
    build.build_binding()
    assert build.binding_fits() and len(tree) == count
    import torch
    version = torch.__version__
    monkeypatch.setattr(torch, "__version__", version + ".other")
    assert not build.binding_fits()
    monkeypatch.setattr(ext, "_UPDATE", None)
    monkeypatch.setattr(ext, "load_library", lambda build_if_missing=True: None)
    with pytest.raises(RuntimeError, match="not of this torch"):
        ext.load_update(build_if_missing=False)
    with pytest.raises(ImportError):  # built, and then no module: a small text file
        ext.load_update()
    assert len(tree) == count + 1 and build.binding_fits()
    monkeypatch.setattr(torch, "__version__", version)
    build.build_binding()
    assert len(tree) == count + 2
    # One whose build is not known.
    build.BINDING.write_text("built")
    build.build_binding()
    assert len(tree) == count + 3


def test_builds_that_start_together(tree, monkeypatch):
    """Two ranks without a library: one builds, the other waits and finds it."""
    import threading
    import time
    written, inside, most = build.subprocess.run, [], []

    def run(command, check):
        name = command[command.index("-o") + 1]
        inside.append(name)
        most.append(inside.count(name))
        time.sleep(0.05)
        written(command, check)
        inside.remove(name)

    monkeypatch.setattr(build.subprocess, "run", run)
    for call, commands in ((build.build, len(build.SOURCES) + 2), (build.build_binding, 1)):
        for f in (build.LIB, build.BINDING) if call is build.build else (build.BINDING,):
            f.unlink(missing_ok=True)
        before = len(tree)
        threads = [threading.Thread(target=call) for _ in range(3)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert len(tree) - before == commands and max(most) == 1, call.__name__
        assert build.LIB.exists() and build.binding_fits()
