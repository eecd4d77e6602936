"""When the HIP library is compiled: by `__graft_entry__.build()` always, by the test session only where a source is younger than the library."""
import os
import types

import pytest

from legommenders_amd import _lib


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """a source folder of its own, and what is run there instead of make"""
    ran = []
    for name, age in [("a.hip", 30), ("b.hpp", 20), ("Makefile", 40), ("lego_hip.h", 25), ("liblego_hip.so", 10)]:
        (tmp_path / name).write_text("")
        os.utime(tmp_path / name, (1e9 - age, 1e9 - age))
    monkeypatch.setattr(_lib, "CSRC", str(tmp_path))
    monkeypatch.setattr(_lib, "HEADER", str(tmp_path / "lego_hip.h"))
    monkeypatch.setattr(_lib, "LIB_PATH", str(tmp_path / "liblego_hip.so"))
    monkeypatch.setattr(_lib.subprocess, "run", lambda cmd, **kw: ran.append(cmd) or types.SimpleNamespace(returncode=0, stdout="", stderr=""))
    return tmp_path, ran


def test_an_up_to_date_library_is_loaded_as_it_is(tree):
    _lib.build()                                                                             # there are no objects beside it
    assert tree[1] == []


@pytest.mark.parametrize("name", ["a.hip", "b.hpp", "Makefile", "lego_hip.h"])
def test_a_younger_source_is_compiled(tree, name):
    os.utime(tree[0] / name, (1e9, 1e9))
    _lib.build()
    assert len(tree[1]) == 1 and "-B" not in tree[1][0]


def test_a_missing_library_is_built(tree):
    os.remove(tree[0] / "liblego_hip.so")
    _lib.build()
    assert len(tree[1]) == 1


def test_the_entry_point_compiles_every_source(tree, monkeypatch):
    import __graft_entry__ as entry
    monkeypatch.setattr(_lib, "lib", lambda: types.SimpleNamespace(present=1))
    monkeypatch.setattr(_lib, "declared_symbols", lambda: ["present"])
    entry.build()
    assert len(tree[1]) == 1 and "-B" in tree[1][0]
