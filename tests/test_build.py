"""When papr_amd/build.py compiles again: a source, a header, the command line or the torch it builds against has changed."""
import os

import pytest
import torch

from papr_amd import build


@pytest.fixture
def recorded(tmp_path, monkeypatch):
    """build.py in an empty folder with a compiler that writes empty files; -> the commands that ran since last asked."""
    ran = []

    def compiles(cmd, **kw):
        ran.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return 0

    class Done:
        def __init__(self, cmd):
            compiles(cmd)

        def wait(self):
            return 0
    monkeypatch.setattr(build, "PKG", str(tmp_path / "papr_amd"))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "papr_amd" / "lib.so"))
    monkeypatch.setattr(build, "GLUE", str(tmp_path / "papr_amd" / "glue.so"))
    monkeypatch.setattr(build, "NO_ACCVGPR", [])
    monkeypatch.setattr(build.subprocess, "Popen", Done)
    monkeypatch.setattr(build.subprocess, "check_call", compiles)
    os.makedirs(tmp_path / "papr_amd")
    os.makedirs(tmp_path / "include")
    (tmp_path / "include" / "papr_hip.h").write_text("")

    def go():
        del ran[:]
        build.build_library(verbose=False)
        build.build_glue(verbose=False)
        return [os.path.basename(c[c.index("-o") + 1]) for c in ran]
    return go


def test_a_second_build_compiles_nothing_and_another_command_everything_it_concerns(recorded, monkeypatch):
    everything = [s.replace(".hip", ".o") for s in build.SOURCES] + ["lib.so", "glue.so"]
    assert recorded() == everything and recorded() == []
    monkeypatch.setattr(build, "FLAGS", build.FLAGS + ["-DX"])
    assert recorded() == everything[:-1] and recorded() == []
    monkeypatch.setitem(build.EXTRA_FLAGS, "knn.hip", ["-DY"])
    assert recorded() == ["knn.o", "lib.so"] and recorded() == []
    monkeypatch.setattr(torch, "__version__", "0.0")
    assert recorded() == ["glue.so"] and recorded() == []


def test_what_was_built_without_a_record_of_its_command_is_built_again(recorded):
    recorded()
    os.remove(os.path.join(build.PKG, "build", "adam.o.cmd"))
    os.remove(build.GLUE + ".cmd")
    assert recorded() == ["adam.o", "lib.so", "glue.so"]


def test_a_newer_header_reaches_its_sources(recorded):
    recorded()
    header = os.path.join(os.path.dirname(build.PKG), "include", "papr_hip.h")
    t = os.path.getmtime(build.LIB) + 10
    os.utime(header, (t, t))
    assert recorded() == [s.replace(".hip", ".o") for s in build.SOURCES] + ["lib.so", "glue.so"]
