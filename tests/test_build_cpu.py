"""The build itself, with a stand-in for nvcc: what it makes, and with what it has to make do."""
import importlib.metadata
import importlib.util
import stat

import pytest

from sys1_b200 import build


@pytest.fixture
def sandbox(tmp_path, monkeypatch):
    """The build's outputs in a folder of their own; nvcc and g++ only write the file that `-o` names, and note their calls."""
    tool = tmp_path / "compiler"
    tool.write_text(f'#!/bin/sh\necho "$0 $*" >> {tmp_path}/calls\nwhile [ $# -gt 1 ]; do [ "$1" = "-o" ] && echo made > "$2"; shift; done\n')
    tool.chmod(tool.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("NVCC", str(tool))
    monkeypatch.setenv("CXX", str(tool))
    for name, at in (("LIB", "lib.so"), ("BINDING", "binding.so"), ("STAMP", "stamp"), ("OBJ", "obj")):
        monkeypatch.setattr(build, name, tmp_path / at)
    return tmp_path


def _hide_pytorch(monkeypatch):
    find, version = importlib.util.find_spec, importlib.metadata.version

    def no_version(name):
        if name == "torch":
            raise importlib.metadata.PackageNotFoundError(name)
        return version(name)

    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    monkeypatch.setattr(importlib.metadata, "version", no_version)


def test_the_library_builds_without_pytorch(sandbox, monkeypatch, capsys):
    """The C ABI needs nvcc alone. The Python side is left out and said to be, and made once PyTorch is there."""
    with monkeypatch.context() as m:
        _hide_pytorch(m)
        assert build.build() == build.LIB
        assert build.LIB.exists() and not build.BINDING.exists() and "PyTorch" in capsys.readouterr().err
        calls = (sandbox / "calls").read_text()
        assert build.build() == build.LIB and (sandbox / "calls").read_text() == calls  # up to date: nothing is made again
    build.build()
    assert build.BINDING.exists() and "binding.cpp" in (sandbox / "calls").read_text()


def test_the_build_makes_both(sandbox):
    build.build()
    assert build.LIB.exists() and build.BINDING.exists()
    calls = (sandbox / "calls").read_text()
    build.build()
    assert (sandbox / "calls").read_text() == calls
    build.BINDING.unlink()  # one of the two is gone
    build.build()
    assert build.BINDING.exists()
