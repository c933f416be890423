"""Build libforgetune_b200.so in-tree with nvcc for sm_100a.

    python -m forgetune_b200.build_native [--force]

The library holds the engine (graph blob, fusion, arena planner), every CUDA
kernel and the C ABI declared in include/forgetune_b200.h.  It is written to
forgetune_b200/lib/ and linked (with an rpath) by every per-model shim and by
_torch_ops.so, the extension behind the operators on torch tensors.  The
library needs nvcc alone; where the extension cannot be built (no torch
headers, Python headers or host compiler), the rest still is.
"""

from __future__ import annotations

import argparse
import importlib.util
import os
import re
import shlex
import shutil
import subprocess
import sys
import sysconfig
import time
import warnings
from concurrent.futures import ThreadPoolExecutor
from typing import Optional

PKG = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(REPO, "include")
LIB_DIR = os.path.join(PKG, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libforgetune_b200.so")
TORCH_OPS_PATH = os.path.join(LIB_DIR, "_torch_ops.so")
OBJ_DIR = os.path.join(LIB_DIR, "obj")

SOURCES = ["runtime.cu", "fp8.cu", "engine.cpp"]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.isfile(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC or put CUDA on PATH)")


def _inputs(source=None):
    """The source (default: all sources) and every project header it includes, transitively."""
    todo = [os.path.join(CSRC, s) for s in ([source] if source else SOURCES)]
    files = []
    while todo:
        path = todo.pop()
        if path in files:
            continue
        files.append(path)
        with open(path, encoding="utf-8") as f:
            for name in re.findall(r'^\s*#include\s+"([^"]+)"', f.read(), re.M):
                for d in (CSRC, INCLUDE):
                    if os.path.isfile(os.path.join(d, name)):
                        todo.append(os.path.join(d, name))
    return files


def _newer(target, files) -> bool:
    if not os.path.isfile(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(f) <= t for f in files)


def _torch_dir() -> Optional[str]:
    spec = importlib.util.find_spec("torch")
    return os.path.dirname(spec.origin) if spec and spec.origin else None


def torch_ops_target() -> str:
    """What an extension built now is for: the installed torch (the file it takes its version from) and the
    interpreter's ABI, whose headers' layouts it compiles in."""
    version = {"__version__": "", "git_version": ""}
    path = os.path.join(_torch_dir() or "", "version.py")
    if os.path.isfile(path):
        with open(path, encoding="utf-8") as f:
            version.update(re.findall(r"^(__version__|git_version)\b[^=\n]*=\s*['\"]([^'\"]*)", f.read(), re.M))
    return "torch %s %s, %s" % (version["__version__"], version["git_version"], sysconfig.get_config_var("SOABI"))


def torch_ops_built_for(path: str) -> Optional[str]:
    """The same of an extension file, from the line it carries (csrc/torch_ops.cpp); None without one."""
    try:
        with open(path, "rb") as f:
            found = re.search(rb"_torch_ops built for: ([^\0]*)\0", f.read())
    except OSError:
        return None
    return found.group(1).decode() if found else None


def _torch_ops_current() -> bool:
    return _newer(TORCH_OPS_PATH, _inputs("torch_ops.cpp")) and torch_ops_built_for(TORCH_OPS_PATH) == torch_ops_target()


def host_compiler() -> Optional[str]:
    for c in (os.environ.get("CXX"), shutil.which("g++"), shutil.which("c++"), shutil.which("clang++")):
        if c:
            return c
    return None


def torch_ops_lacks() -> Optional[str]:
    """What the extension needs and this machine does not have, or None."""
    torch_dir = _torch_dir()
    if not torch_dir or not os.path.isfile(os.path.join(torch_dir, "include", "torch", "csrc", "Dtype.h")):
        return "torch's C++ headers"
    if not os.path.isfile(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "Python.h"
    if not host_compiler():
        return "a host C++ compiler (g++, c++, clang++ or $CXX)"
    try:
        nvcc()
    except RuntimeError:
        return "nvcc, beside CUDA's headers"
    return None


def up_to_date() -> bool:
    """Whether build() has nothing to do here."""
    return _newer(LIB_PATH, _inputs()) and (_torch_ops_current() or torch_ops_lacks() is not None)


def _run(cmd, target, verbose) -> None:
    """Run ``cmd`` + ["-o", file] and put the file in place of ``target``, dated when the command began: an
    input edited meanwhile stays newer."""
    began = time.time()
    tmp = target + ".tmp%d" % os.getpid()
    cmd = cmd + ["-o", tmp]
    if verbose:
        print(" ".join(cmd), flush=True)
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        raise RuntimeError("cannot run %s: %s" % (cmd[0], e)) from e
    if r.returncode != 0:
        raise RuntimeError("%s failed (%d):\n%s\n%s" % (os.path.basename(cmd[0]), r.returncode, r.stdout[-4000:], r.stderr[-8000:]))
    os.utime(tmp, (began, began))
    os.replace(tmp, target)


def _compile(source, force, verbose) -> str:
    obj = os.path.join(OBJ_DIR, source + ".o")
    if force or not _newer(obj, _inputs(source)):
        _run([nvcc(), "-std=c++17", "-O3", "-lineinfo"] + ARCH_FLAGS + [
            "-I", INCLUDE, "-Xcompiler", "-fPIC,-fvisibility=hidden", "-c", os.path.join(CSRC, source)], obj, verbose)
    return obj


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile what changed (the sources side by side), link the library and build the torch extension."""
    if force or not _newer(LIB_PATH, _inputs()):
        os.makedirs(OBJ_DIR, exist_ok=True)
        with ThreadPoolExecutor(len(SOURCES)) as pool:
            objs = list(pool.map(lambda s: _compile(s, force, verbose), SOURCES))
        if force or not _newer(LIB_PATH, objs):
            _run([nvcc()] + ARCH_FLAGS + ["-shared"] + objs, LIB_PATH, verbose)
    if force or not _torch_ops_current():
        lacks = torch_ops_lacks()
        if lacks:
            warnings.warn("_torch_ops.so is not built: this machine has not %s (the operators on torch tensors need it; "
                          "compiled models do not)" % lacks)
        else:
            _build_torch_ops(verbose)
    return LIB_PATH


def _build_torch_ops(verbose) -> None:
    """The CPython extension behind fp8.py, against the installed torch and the engine library."""
    torch_dir = _torch_dir()
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    include = [os.path.join(torch_dir, "include"), os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
               os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    torch_lib = os.path.join(torch_dir, "lib")
    cxx = host_compiler()
    cxx = [cxx] if os.path.isfile(cxx) else shlex.split(cxx)  # $CXX may be a command with arguments
    _run(cxx + ["-std=c++17", "-O2", "-fPIC", "-fvisibility=hidden", "-shared", "-I", INCLUDE,
          '-DFTB_TORCH_OPS_TARGET="%s"' % torch_ops_target()]
         + [a for d in include for a in ("-isystem", d)] + [os.path.join(CSRC, "torch_ops.cpp"), "-L", torch_lib]
         + ["-l" + n for n in ("c10", "c10_cuda", "torch_cpu", "torch_cuda", "torch", "torch_python")]
         + ["-L", LIB_DIR, "-l:" + os.path.basename(LIB_PATH), "-Wl,-rpath,$ORIGIN"], TORCH_OPS_PATH, verbose)


def main() -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=True))
    return 0


if __name__ == "__main__":
    sys.exit(main())
