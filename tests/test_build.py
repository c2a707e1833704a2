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


def test_another_torch_has_a_module_of_its_own(ran, monkeypatch):
    """The module is bound to the ABI of one torch and one Python: after an upgrade it is neither loaded nor up to date."""
    import sysconfig

    import torch

    from helios_b200 import _lib
    B.build()
    path = _lib.torch_module_path(torch.__version__)
    assert not module_commands(ran) and path.exists() and _lib.torch_ops()       # this one's is there
    assert path.name.endswith(sysconfig.get_config_var("EXT_SUFFIX"))
    monkeypatch.setattr(torch, "__version__", "99.1")
    monkeypatch.setattr(_lib, "_torch_ops", None)
    with pytest.raises(_lib.G4qUnavailable, match="99.1.*helios_b200.build"):
        _lib.torch_ops()
    B.build()
    (cmd,) = module_commands(ran)
    assert cmd[cmd.index("-o") + 1] == str(_lib.torch_module_path("99.1")) != str(path)
