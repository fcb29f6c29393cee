"""What the build needs: the Python calls of the operators are left out where they cannot be built."""

import importlib
import os

import pytest

import llm_b200
from llm_b200 import build as b


@pytest.fixture(autouse=True)
def library_as_it_is(monkeypatch):
    """The library is there; its sources are not compiled again."""
    assert os.path.exists(b.LIB)
    monkeypatch.setattr(b, "SOURCES", [])


def test_the_library_is_built_without_a_c_compiler(monkeypatch, tmp_path, capsys):
    monkeypatch.setattr(b, "CALL", str(tmp_path / "_native.abi3.so"))
    monkeypatch.setenv("CC", "no-such-compiler -O1")
    assert b.build() == b.LIB and os.path.exists(b.LIB)
    assert not os.path.exists(b.CALL)
    assert "no C compiler" in capsys.readouterr().err


def test_the_library_is_built_without_pythons_headers(monkeypatch, tmp_path, capsys):
    monkeypatch.setattr(b, "CALL", str(tmp_path / "_native.abi3.so"))
    monkeypatch.setattr(b.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    assert b.build() == b.LIB and not os.path.exists(b.CALL)
    assert "no Python.h" in capsys.readouterr().err


def test_the_python_calls_say_what_they_need(monkeypatch):
    def missing(name, package=None):
        raise ImportError("No module named 'llm_b200._native'")

    monkeypatch.setattr(llm_b200, "_native_calls", None)
    monkeypatch.setattr(importlib, "import_module", missing)
    with pytest.raises(ImportError, match="C compiler"):
        llm_b200._calls()


def test_a_compiler_with_arguments(monkeypatch, tmp_path):
    monkeypatch.setattr(b, "CALL", str(tmp_path / "_native.abi3.so"))
    monkeypatch.setenv("CC", "gcc -g0")
    b.build()
    assert os.path.exists(b.CALL)
