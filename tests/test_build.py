"""When the build is done again."""
from __future__ import annotations

import os

import pytest

from conftest import pkg


@pytest.fixture
def build(tmp_path, monkeypatch):
    """The build with its outputs in a folder of their own; compilers only leave their output files."""
    b = pkg("build")
    monkeypatch.setattr(b, "BUILD", str(tmp_path))
    for name in ("BIND_LIB", "BIND_STAMP"):
        monkeypatch.setattr(b, name, str(tmp_path / name))
    runs = []

    def run(cmd, **kw):
        runs.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return type("Done", (), dict(returncode=0, stdout="", stderr=""))

    monkeypatch.setattr(b.subprocess, "run", run)
    b.runs = runs
    return b


def test_torch_calls_are_rebuilt_for_another_torch(build, monkeypatch):
    assert build._bind_stale()
    build._build_bind(False)
    assert len(build.runs) == 1 and not build._bind_stale()
    with monkeypatch.context() as m:
        m.setattr(build.importlib.metadata, "version", lambda name: "0.0")
        assert build._bind_stale()
        build._build_bind(False)
        assert not build._bind_stale()
    assert build._bind_stale()
    build._build_bind(False)
    os.utime(build.BIND_LIB, (0, 0))  # older than its sources
    assert build._bind_stale()
