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
