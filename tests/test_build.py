"""build_library() compiles again what was compiled by another command line (a compiler that only notes its calls stands in for hipcc)."""
import os
import stat

import pytest

from asr_amd import _lib


@pytest.fixture
def tree(tmp_path, monkeypatch):
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    for name in ("a.hip", "b.hip", "asr_common.h", "asr_hip.h"):
        (csrc / name).write_text("")
        os.utime(csrc / name, (1000, 1000))
    cc, log = tmp_path / "cc", tmp_path / "log"
    cc.write_text('#!/bin/sh\necho "$@" >> %s\nwhile [ $# -gt 0 ]; do [ "$1" = -o ] && echo x > "$2"; shift; done\n[ ! -e %s ]\n' % (log, tmp_path / "broken"))
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("HIPCC", str(cc))
    monkeypatch.delenv("ASR_AMD_EXTRA_HIPCC_FLAGS", raising=False)
    for name, value in (("CSRC", str(csrc)), ("SOURCES", ["a.hip", "b.hip"]), ("HEADER", str(csrc / "asr_hip.h")), ("LIB_PATH", str(csrc / "lib.so"))):
        monkeypatch.setattr(_lib, name, value)

    def build(force=False):
        """-> the sources compiled, whether the library was linked"""
        if log.exists():
            log.unlink()
        _lib.build_library(force=force)
        calls = log.read_text().splitlines() if log.exists() else []
        return sorted(s for s in ("a.hip", "b.hip") if any(" -c " in c and s in c.split()[c.split().index("-c") + 1] for c in calls)), any("-shared" in c for c in calls)
    build.tmp, build.csrc = tmp_path, csrc
    return build


def test_nothing_is_compiled_twice(tree):
    assert tree() == (["a.hip", "b.hip"], True)
    assert tree() == ([], False)
    os.utime(tree.csrc / "a.hip")
    for f in ("build/a.hip.o", "lib.so"):
        os.utime(tree.csrc / f, (2000, 2000))
    assert tree() == (["a.hip"], True)
    assert tree(force=True) == (["a.hip", "b.hip"], True)


def test_other_flags_compile_again(tree, monkeypatch):
    tree()
    monkeypatch.setenv("ASR_AMD_EXTRA_HIPCC_FLAGS", "-DPROBE")
    assert tree() == (["a.hip", "b.hip"], True)
    assert tree() == ([], False)
    monkeypatch.delenv("ASR_AMD_EXTRA_HIPCC_FLAGS")
    assert tree() == (["a.hip", "b.hip"], True)
    monkeypatch.setattr(_lib, "NO_PACKED_F32", [])
    assert tree() == (["a.hip", "b.hip"], True)
    monkeypatch.setattr(_lib, "EXTRA_FLAGS", {"b.hip": ["-ffp-contract=off"]})
    assert tree() == (["b.hip"], True)


def test_objects_of_an_unknown_command_are_compiled_again(tree):
    """a tree that was built before the commands were kept, or whose library came without them"""
    for f in ("build/a.hip.o", "build/b.hip.o", "lib.so"):
        (tree.csrc / f).parent.mkdir(exist_ok=True)
        (tree.csrc / f).write_text("x")
    assert tree() == (["a.hip", "b.hip"], True)


def test_a_failed_compile_is_not_taken_for_done(tree):
    tree()
    os.utime(tree.csrc / "a.hip")
    for f in ("build/a.hip.o", "lib.so"):
        os.utime(tree.csrc / f, (2000, 2000))
    (tree.tmp / "broken").write_text("")
    with pytest.raises(RuntimeError, match="hipcc failed"):
        tree()
    (tree.tmp / "broken").unlink()
    assert tree() == (["a.hip"], True)      # (the compiler had written its output before it failed)


def test_a_library_elsewhere_is_left_alone_while_it_is_newer(tree, monkeypatch, tmp_path):
    """ASR_AMD_LIB names another build for comparisons: its flags are its own business, and this tree's record is not its"""
    tree()
    other = tmp_path / "other.so"
    other.write_text("another build")
    monkeypatch.setattr(_lib, "LIB_PATH", str(other))
    assert tree() == ([], False) and other.read_text() == "another build"
    os.utime(other, (1, 1))
    assert tree() == ([], True)                        # (older than the sources: linked anew, as ever)
    monkeypatch.setattr(_lib, "LIB_PATH", str(tree.csrc / "lib.so"))
    assert tree() == ([], False)
