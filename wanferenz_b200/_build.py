"""Builds the in-tree CUDA library ``wanferenz_b200/lib/libwfb200.so`` for sm_100a.

Usage: ``python -m wanferenz_b200._build`` (or ``__graft_entry__.build()``).
The library is plain nvcc output with a C ABI (``include/wfb200.h``); it
statically links the CUDA runtime and is loaded with ctypes.  Beside it goes
``lib/_wfb200_torch.so``, the compiled Python entry of the operators of
``csrc/wf_torch.cpp`` (host code, linked to the library and to torch).
"""

from __future__ import annotations

import glob
import hashlib
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIBDIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIBDIR, "libwfb200.so")
EXT = os.path.join(LIBDIR, "_wfb200_torch.so")
EXT_KEY = EXT + ".key"
EXT_SRC = os.path.join(CSRC, "wf_torch.cpp")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
    "-I", os.path.join(ROOT, "include"),
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def deps():
    return sources() + sorted(glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h"))) + [
        os.path.join(ROOT, "include", "wfb200.h")]


def ext_deps():
    return [EXT_SRC, os.path.join(ROOT, "include", "wfb200.h")]


def up_to_date() -> bool:
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(p) <= t for p in deps())


def ext_key():
    """What the Python entry module is compiled against (torch, the interpreter's ABI) and from (its sources; empty in
    a package without them), a line each."""
    import sysconfig

    import torch

    against = f"{torch.__version__} {sysconfig.get_config_var('SOABI')}"
    if not all(os.path.exists(p) for p in ext_deps()):
        return against, ""
    source = hashlib.sha256()
    for p in ext_deps():
        with open(p, "rb") as f:
            source.update(f.read())
    return against, source.hexdigest()


def ext_current() -> bool:
    """Whether the module in place is of this torch, interpreter and source (by the key written beside it)."""
    try:
        with open(EXT_KEY) as f:
            has = f.read().split("\n")
    except FileNotFoundError:
        return False
    against, source = ext_key()
    return os.path.exists(EXT) and has[0] == against and (not source or has[1:] == [source])


def _run(cmd, target, verbose):
    tmp = target + f".tmp{os.getpid()}"
    cmd = [tmp if c is None else c for c in cmd]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({r.returncode}):\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, target)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(LIBDIR, exist_ok=True)
    if force or not up_to_date():
        _run([nvcc(), *NVCC_FLAGS, "--threads", "0", "-o", None, *sources()], LIB, verbose)
    return LIB


def build_ext(force: bool = False, verbose: bool = False) -> str:
    """The Python entry module; links ``build()``'s library, which must exist."""
    if not force and ext_current():
        return EXT
    key = ext_key()
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    flags = ["-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-Wall", "-Wno-unknown-pragmas",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}"]
    for d in cpp_extension.include_paths(device_type="cuda") + [sysconfig.get_paths()["include"]]:
        flags += ["-isystem", d]
    libs = ["-L" + d for d in cpp_extension.library_paths(device_type="cuda")]
    libs += ["-ltorch_python", "-ltorch", "-ltorch_cuda", "-ltorch_cpu", "-lc10_cuda", "-lc10",
             "-L" + LIBDIR, "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN"]
    _run([cxx(), *flags, EXT_SRC, "-o", None, *libs], EXT, verbose)
    tmp = EXT_KEY + f".tmp{os.getpid()}"
    with open(tmp, "w") as f:
        f.write("\n".join(key))
    os.replace(tmp, EXT_KEY)
    return EXT


def cxx() -> str:
    return os.environ.get("CXX", "g++")


def ext_lacks():
    """What this machine lacks to compile the Python entry module (None: nothing)."""
    import sysconfig

    if shutil.which(cxx()) is None:
        return f"a C++ compiler ({cxx()})"
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "Python's headers"
    try:
        import torch  # noqa: F401
    except ImportError:
        return "torch"
    return None


def main(argv) -> None:
    """The library always; the Python entry module where it can be compiled, since a host of the C ABI needs neither
    torch nor Python's headers."""
    force = "--force" in argv
    print(build(force=force, verbose=True))
    lacks = ext_lacks()
    if lacks:
        print(f"not built: {EXT}, the Python entry of the layer operators; this machine lacks {lacks}", file=sys.stderr)
    else:
        print(build_ext(force=force, verbose=True))


if __name__ == "__main__":
    main(sys.argv)
