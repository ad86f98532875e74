"""The build of _paged_ext.so: when it is made again, and what is left when it cannot be made (CPU)."""

import os
import sys

import pytest

from locals_b200 import _lib, build


@pytest.fixture
def elsewhere(tmp_path, monkeypatch):
    monkeypatch.setattr(build, "EXT", str(tmp_path / "_paged_ext.so"))
    monkeypatch.setattr(build, "EXT_HASH", str(tmp_path / "_paged_ext.so.srchash"))
    return tmp_path


def _compiler(tmp_path, name, line):
    p = tmp_path / name
    p.write_text("#!/bin/sh\n" + line + "\n")
    p.chmod(0o755)
    return str(p)


def test_made_again_for_another_interpreter_compiler_or_flags(elsewhere, monkeypatch):
    log = elsewhere / "calls"
    cc = 'if [ "$1" = --version ]; then echo one; else echo x >> %s; touch %s.tmp; fi' % (log, build.EXT)
    monkeypatch.setenv("CXX", _compiler(elsewhere, "cc", cc))

    def calls():
        build.build_ext()
        return len(log.read_text())

    first = calls()
    assert calls() == first  # nothing has changed
    monkeypatch.setattr(sys.implementation, "cache_tag", "cpython-0")
    second = calls()
    assert second > first and calls() == second
    _compiler(elsewhere, "cc", cc.replace("echo one", "echo two"))
    third = calls()
    assert third > second and calls() == third
    command = build._ext_command
    monkeypatch.setattr(build, "_ext_command", lambda out: [*command(out), "-DANOTHER"])
    assert calls() > third


def test_the_library_does_not_need_it(elsewhere, monkeypatch, capsys):
    for cxx in (_compiler(elsewhere, "cc", "echo no headers >&2; exit 1"), str(elsewhere / "none")):
        monkeypatch.setenv("CXX", cxx)
        for f in (build.EXT, build.EXT_HASH):
            with open(f, "w") as old:
                old.write("an older one")
        assert build.build() == build.LIB and os.path.exists(build.LIB)
        assert "paged.py and rotary.py will not run" in capsys.readouterr().err
        assert not os.path.exists(build.EXT)  # none, rather than an older one
        with pytest.raises(RuntimeError):
            build.build_ext()


def test_what_needs_it_says_so(monkeypatch):
    monkeypatch.setattr(_lib, "_ext", None)
    monkeypatch.setitem(sys.modules, "locals_b200._paged_ext", None)
    monkeypatch.delattr(sys.modules["locals_b200"], "_paged_ext", raising=False)
    with pytest.raises(RuntimeError, match="locals_b200.build"):
        _lib.ext()
