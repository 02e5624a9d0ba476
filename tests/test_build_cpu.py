"""s2t_amd.build: what is compiled and linked again, with a compiler that only writes down its command."""
import os
import types

import pytest

from s2t_amd import build as b


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """Two sources and a header, all older than anything built from them; ``ran``: the commands since it was last emptied."""
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    for name in ("one.hip", "two.hip", "common.h"):
        (csrc / name).write_text("")
        os.utime(csrc / name, (1e9, 1e9))
    monkeypatch.setattr(b, "CSRC", str(csrc))
    monkeypatch.setattr(b, "LIBDIR", str(tmp_path / "lib"))
    monkeypatch.setattr(b, "LIB", str(tmp_path / "lib" / "lib.so"))
    monkeypatch.setattr(b, "HIPCC", "hipcc")
    monkeypatch.setattr(b, "FLAGS", ["-O3"])
    monkeypatch.setattr(b, "FILE_FLAGS", {})
    monkeypatch.setattr(b, "_deps_mtime", lambda: os.path.getmtime(csrc / "common.h"))
    t = types.SimpleNamespace(csrc=csrc, ran=[], fails=False, set=lambda name, value: monkeypatch.setattr(b, name, value))

    def run(cmd, **kw):
        out = cmd[cmd.index("-o") + 1]
        t.ran.append(os.path.basename(out))
        if not t.fails:
            with open(out, "w") as f:
                f.write(" ".join(cmd))
        return types.SimpleNamespace(returncode=int(t.fails), stderr="no")
    monkeypatch.setattr(b.subprocess, "run", run)

    def built():
        t.ran.clear()
        b.build(verbose=False)
        return sorted(t.ran)
    t.built = built
    return t


ALL = ["lib.so", "one.o", "two.o"]


def test_what_is_there_is_not_built_again(tree):
    assert tree.built() == ALL and tree.built() == []
    os.utime(tree.csrc / "two.hip")
    os.utime(os.path.join(b.LIBDIR, "obj", "two.o"), (1e9 - 1, 1e9 - 1))
    assert tree.built() == ["lib.so", "two.o"] and tree.built() == []


def test_other_flags_build_again(tree):
    """All of them, one file's, another compiler; and back again."""
    tree.built()
    tree.set("FLAGS", ["-O3", "-Xclang", "-target-feature"])
    assert tree.built() == ALL and tree.built() == []
    tree.set("FILE_FLAGS", {"two.hip": ["-mllvm"]})
    assert tree.built() == ["lib.so", "two.o"] and tree.built() == []
    tree.set("FILE_FLAGS", {})
    assert tree.built() == ["lib.so", "two.o"]
    tree.set("HIPCC", "/other/hipcc")
    assert tree.built() == ALL and tree.built() == []


def test_objects_whose_command_is_not_known_are_built_again(tree):
    """As an earlier version of the build left them."""
    tree.built()
    os.remove(os.path.join(b.LIBDIR, "obj", "one.o.cmd"))
    assert tree.built() == ["lib.so", "one.o"]
    os.remove(b.LIB + ".cmd")
    assert tree.built() == ["lib.so"]


def test_a_failed_build_and_a_source_that_is_gone_leave_nothing_that_passes(tree):
    tree.built()
    tree.set("FLAGS", ["-O2"])
    tree.fails = True
    with pytest.raises(RuntimeError, match="hipcc failed"):
        tree.built()
    tree.fails = False
    assert tree.built() == ALL
    os.remove(tree.csrc / "two.hip")
    assert tree.built() == ["lib.so"] and "two.o" not in open(b.LIB).read()
