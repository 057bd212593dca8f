"""When the native library is built again (the compiler is replaced by one that only writes its output's name)."""
import os
import types
from pathlib import Path

import pytest


@pytest.fixture
def tree(tmp_path, monkeypatch):
    from aether_amd import build
    csrc = tmp_path / "aether_amd" / "csrc"
    csrc.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    for f in (csrc / "a.hip", csrc / "b.hip", csrc / "c.hpp", tmp_path / "include" / "aether_hip.h"):
        f.write_text("// " + f.name)
        os.utime(f, (1000, 1000))
    calls = []

    def run(cmd, **_):
        calls.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_text(" ".join(map(str, cmd)))
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(build, "CSRC", csrc)
    monkeypatch.setattr(build, "LIB", csrc / "libaether_hip.so")
    monkeypatch.setattr(build.subprocess, "run", run)
    return types.SimpleNamespace(build=build, csrc=csrc, calls=calls)


def _built(tree):
    n = len(tree.calls)
    assert tree.build.build_native() == tree.build.LIB
    return len(tree.calls) - n


def test_built_once(tree):
    assert _built(tree) == 3 and _built(tree) == 0
    assert tree.build.build_native(force=True) and len(tree.calls) == 6


@pytest.mark.parametrize("name", ["a.hip", "c.hpp"])
def test_a_changed_source_builds_again(tree, name):
    _built(tree)
    os.utime(tree.csrc / name)
    later = (tree.csrc / "libaether_hip.so").stat().st_mtime + 10
    os.utime(tree.csrc / name, (later, later))
    assert _built(tree) == 3


def test_other_flags_build_again(tree, monkeypatch):
    _built(tree)
    monkeypatch.setattr(tree.build, "FLAGS", [*tree.build.FLAGS, "-DOTHER"])
    assert _built(tree) == 3 and "-DOTHER" in tree.calls[-2] and _built(tree) == 0
    monkeypatch.setattr(tree.build, "HIPCC", "/elsewhere/hipcc")
    assert _built(tree) == 3 and _built(tree) == 0


def test_a_source_less_builds_again(tree):
    _built(tree)
    (tree.csrc / "b.hip").unlink()
    assert _built(tree) == 2 and _built(tree) == 0
