"""Which host compiler builds the torch extension (deltagrid_b200/build.py)."""
import shutil

import pytest

from deltagrid_b200 import build


def _wrapper(tmp_path, name, *flags):
    p = tmp_path / name
    p.write_text(f"#!/bin/sh\nexec {shutil.which('g++')} \"$@\" {' '.join(flags)}\n")
    p.chmod(0o755)
    return str(p)


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_the_compiler_that_was_asked_for(tmp_path, monkeypatch):
    mine = _wrapper(tmp_path, "mine")
    monkeypatch.setenv("CXX", mine)
    assert build.host_compiler() == mine
    monkeypatch.setenv("CXX", f"{mine} -g")
    assert build.host_compiler() == f"{mine} -g"
    monkeypatch.delenv("CXX")
    assert build.host_compiler() == shutil.which("g++")


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_a_compiler_with_a_static_library_of_its_own_is_passed_over(tmp_path, monkeypatch):
    monkeypatch.setenv("CXX", _wrapper(tmp_path, "static", "-static-libstdc++"))
    assert build.host_compiler() == shutil.which("g++")
    monkeypatch.setenv("CXX", str(tmp_path / "absent"))
    assert build.host_compiler() == shutil.which("g++")
