"""What the build makes, and for whom."""
import os
import re
import shutil
import subprocess

import pytest

from sparseflow_b200 import _lib, build


def test_python_calls_use_the_stable_interface_only(lib):
    """One build of the module serves every CPython from 3.10 on: nothing that it takes from the interpreter changes between versions."""
    source = open(build.CALLS_SRC).read()
    assert re.search(r"#define Py_LIMITED_API 0x030A0000\b.*#include <Python.h>", source, re.S)
    if shutil.which("nm") is None:
        pytest.skip("no nm")
    _lib.calls()
    names = subprocess.run(["nm", "-D", "--undefined-only", build.CALLS], capture_output=True, text=True, check=True).stdout.split()
    stable = {"PyErr_Format", "PyErr_Occurred", "PyEval_RestoreThread", "PyEval_SaveThread", "PyExc_OverflowError", "PyExc_TypeError", "PyFloat_AsDouble",
              "PyLong_AsLongLong", "PyLong_AsVoidPtr", "PyLong_FromLong", "PyLong_FromSize_t", "PyModule_Create2", "_Py_NoneStruct"}
    assert {n for n in names if re.match(r"_?Py", n)} <= stable


def test_build_without_python_headers(monkeypatch, tmp_path, capsys):
    """The library is built alone, a module of another build goes, and the operators that need it say so."""
    made = []
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build, "CALLS", str(tmp_path / "_calls.so"))
    monkeypatch.setattr(build, "OBJ_DIR", str(tmp_path))
    monkeypatch.setattr(build, "sources", lambda: [])
    monkeypatch.setattr(build, "_nvcc", lambda: "nvcc")
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: made.append(cmd[cmd.index("-o") + 1]))
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    (tmp_path / "_calls.so").write_text("")
    assert build.build(force=True) == build.LIB
    assert made == [build.LIB] and not os.path.exists(build.CALLS) and "Python.h" in capsys.readouterr().err
    monkeypatch.setattr(build, "_deps", lambda: [])
    (tmp_path / "lib.so").write_text("")
    assert build.up_to_date()                       # nothing to make again
    (tmp_path / "Python.h").write_text("")
    assert not build.up_to_date()                   # now there is
    build.build()
    assert made == [build.LIB, build.LIB, build.CALLS]


def test_calls_without_the_module(monkeypatch, tmp_path, lib):
    monkeypatch.setattr(_lib, "_calls", None)
    monkeypatch.setattr(_lib, "CALLS_PATH", str(tmp_path / "_calls.so"))
    with pytest.raises(ImportError, match="headers"):
        _lib.calls()
