"""Building: the C library needs no torch; the Python binding is rebuilt for another torch."""
import os
import subprocess
import sys

import pytest

from tests.conftest import ROOT
from wisp_b200 import build as b


def test_the_library_builds_without_torch():
    """The build itself (nothing of it is stale here), and the step that would compile against torch's headers."""
    code = ("import sys; sys.modules['torch'] = None\n"
            "from wisp_b200 import build as b\n"
            "assert b.build() == b.LIB\n"
            "assert b.build_bind(force=True) is None\n")
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    assert "binding" in done.stderr and "not built" in done.stderr


@pytest.fixture()
def tree(tmp_path, monkeypatch):
    """A tree of its own; the compiler only leaves its output."""
    src, inc = tmp_path / "bind.cpp", tmp_path / "wisp_b200.h"
    for p in (src, inc):
        p.write_text("")
    monkeypatch.setattr(b, "BIND_SRC", str(src))
    monkeypatch.setattr(b, "INCLUDE", str(tmp_path))
    monkeypatch.setattr(b, "BIND", str(tmp_path / "bind.so"))
    monkeypatch.setattr(b, "BIND_STAMP", str(tmp_path / "bind.stamp"))
    runs = []

    def run(cmd, **kwargs):
        runs.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
    monkeypatch.setattr(b.subprocess, "run", run)
    return src, runs


def test_binding_is_rebuilt_for_another_torch(tree, monkeypatch):
    src, runs = tree
    assert b.build_bind() == b.BIND and len(runs) == 1
    assert b.build_bind() == b.BIND and len(runs) == 1                  # nothing changed
    monkeypatch.setattr(b.importlib.metadata, "version", lambda name: "0.0.1")
    assert b.build_bind() == b.BIND and len(runs) == 2
    assert b.build_bind() == b.BIND and len(runs) == 2
    os.utime(src, (os.path.getmtime(b.BIND) + 5,) * 2)
    b.build_bind()
    assert len(runs) == 3
    os.remove(b.BIND_STAMP)                                             # one from before there were stamps
    b.build_bind()
    assert len(runs) == 4
