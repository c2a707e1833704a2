"""What helios_b200.build runs: the compilers are not started here, their commands are looked at."""
import sys

import pytest

from helios_b200 import build as B


@pytest.fixture
def ran(monkeypatch):
    """The commands of a build that compiles everything."""
    cmds = []
    monkeypatch.setattr(B.subprocess, "run", lambda cmd, check: cmds.append(cmd))
    return cmds


def module_commands(cmds):
    return [c for c in cmds if str(B.TORCH_SRC) in c]


def test_the_library_builds_without_torch(ran, monkeypatch, capfd):
    monkeypatch.setitem(sys.modules, "torch", None)           # import torch raises ImportError
    assert B.build(force=True) == B.LIB
    assert not module_commands(ran)
    sources = [c[c.index("-c") + 1] for c in ran if "-c" in c]
    assert sorted(sources) == sorted(str(B.CSRC / s) for s in B.SOURCES)
    assert str(B.LIB) in ran[-1] and "-shared" in ran[-1]
    assert "torch" in capfd.readouterr().err


def test_the_library_is_linked_before_a_module_that_fails_is_reported(ran, monkeypatch):
    def run(cmd, check):
        if str(B.TORCH_SRC) in cmd:
            raise RuntimeError("no such header")
        ran.append(cmd)

    monkeypatch.setattr(B.subprocess, "run", run)
    with pytest.raises(RuntimeError, match="no such header"):
        B.build(force=True)
    assert str(B.LIB) in ran[-1]


def test_the_module_is_built_where_torch_is(ran):
    B.build(force=True)
    assert len(module_commands(ran)) == 1
