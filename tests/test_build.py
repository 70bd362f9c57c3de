"""What makes the native library's objects stale.  The compiler is a stand-in that notes its calls."""
import os
import stat

import pytest

from conformer_amd import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    for name in ("a.hip", "b.hip", "c.h"):
        (csrc / name).write_text("")
        os.utime(csrc / name, (1, 1))
    log, cc = tmp_path / "calls", tmp_path / "cc"
    cc.write_text(f"""#!/bin/sh
echo "$@" >> {log}
for a; do last=$a; done
echo made > "$last"
""")
    cc.chmod(cc.stat().st_mode | stat.S_IEXEC)
    for name, value in (("CSRC", str(csrc)), ("OBJ", str(csrc / "build")), ("LIB", str(tmp_path / "lib.so")), ("SOURCES", ["a.hip", "b.hip"]),
                        ("FLAGS", ["-O3"]), ("EXTRA_FLAGS", {}), ("_hipcc", lambda: str(cc))):
        monkeypatch.setattr(build, name, value)

    def calls(**k):
        log.write_text("")
        build.build_native(**k)
        return log.read_text().split("\n")[:-1]

    calls.csrc = csrc
    return calls


def test_changed_flags_compile_again(tree, monkeypatch):
    assert len(tree()) == 3 and tree() == []                  # two objects and the library, then nothing
    monkeypatch.setattr(build, "FLAGS", ["-O3", "-g"])
    again = tree()
    assert len(again) == 3 and sum("-g" in c for c in again) == 2 and tree() == []
    monkeypatch.setattr(build, "EXTRA_FLAGS", {"b.hip": ["-x"]})
    again = tree()
    assert [c for c in again if "-x" in c and "b.hip" in c] and len(again) == 2 and tree() == []


def test_changed_sources_compile_again(tree):
    tree()
    os.utime(tree.csrc / "a.hip", (2 ** 32, 2 ** 32))
    assert sum("a.hip" in c for c in tree()) == 1
    os.utime(tree.csrc / "a.hip", (1, 1))
    assert len(tree(force=True)) == 3


def test_the_entry_point_always_compiles(monkeypatch):
    import __graft_entry__
    seen = []
    monkeypatch.setattr(build, "build_native", lambda **k: seen.append(k) or build.LIB)
    __graft_entry__.build()
    assert seen == [{"force": True}]
