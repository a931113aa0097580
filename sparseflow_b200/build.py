"""Build libsparseflow_b200.so, and _calls.so (its Python calls without ctypes), in-tree with nvcc for sm_100a.

    python -m sparseflow_b200.build [--force]

The library is the product: every compute entry point of the package goes through it, and the
package refuses to work without it.  ``_calls.so`` needs Python's headers; where there are none the library is built
alone, and the operators around the gated FFN, which go through that module, say what they miss.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libsparseflow_b200.so")
CALLS_SRC = os.path.join(CSRC, "python", "calls.cpp")
CALLS = os.path.join(HERE, "_calls.so")
OBJ_DIR = os.path.join(HERE, "csrc", "build")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC,-fvisibility=hidden",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources() -> list[str]:
    return sorted(
        os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cpp"))
    )


def _deps() -> list[str]:
    out = sources()
    out += [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    out.append(os.path.join(HERE, "..", "include", "sparseflow_b200.h"))
    out += [CALLS_SRC, os.path.abspath(__file__)]
    return out


def _python_include() -> str | None:
    """The folder of Python.h, or None."""
    path = sysconfig.get_paths()["include"]
    return path if os.path.exists(os.path.join(path, "Python.h")) else None


def up_to_date() -> bool:
    made = [LIB, CALLS] if _python_include() else [LIB]
    if not all(os.path.exists(f) for f in made):
        return False
    t = min(os.path.getmtime(f) for f in made)
    return all(os.path.getmtime(d) <= t for d in _deps())


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB
    nvcc = _nvcc()
    os.makedirs(OBJ_DIR, exist_ok=True)
    objs = []
    procs = []
    for src in sources():
        obj = os.path.join(OBJ_DIR, os.path.basename(src) + ".o")
        objs.append(obj)
        cmd = [nvcc, *NVCC_FLAGS, "-x", "cu", "-c", src, "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    for src, p in procs:
        out, _ = p.communicate()
        if verbose or p.returncode:
            sys.stderr.write(out.decode())
        if p.returncode:
            raise RuntimeError(f"nvcc failed on {src}")
    cmd = [nvcc, "-shared", "-o", LIB, *objs, "-gencode", "arch=compute_100a,code=sm_100a", "-ldl"]
    subprocess.run(cmd, check=True)
    include = _python_include()
    if include is None:
        if os.path.exists(CALLS):      # of another library than this one
            os.remove(CALLS)
        sys.stderr.write("Python.h not found: the library is built, _calls.so (calls of the operators around the gated FFN) is not\n")
        return LIB
    # found beside the library whatever the working directory
    subprocess.run([nvcc, "-shared", "-cudart", "none", "-Wno-deprecated-gpu-targets", "-O2", "-std=c++17", "-Xcompiler", "-fPIC,-fvisibility=hidden", "-I", include,
                    CALLS_SRC, "-o", CALLS, "-L", HERE, "-lsparseflow_b200", "-Xlinker", "-rpath,$ORIGIN"], check=True)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
