"""In-tree build of liblutgemm_b200.so (sm_100a only) and of lutgemm_torch.so, the PyTorch operators over it.

    python appmult-aware-retraining_b200/build_ext.py [--force] [--verbose] [--library-only]

Each .cu under csrc/ is compiled with nvcc for compute_100a/sm_100a and linked into one shared
library next to this file; lutgemm_torch.cpp is compiled against the installed PyTorch and linked to that library, and again when
another PyTorch or Python is installed.  C callers need the library alone: --library-only, and where PyTorch is not installed, leaves
the module out.  nvcc cross-compiles without a GPU, so this also runs on a CPU-only box.
"""
from __future__ import annotations

import importlib.metadata
import os
import subprocess
import sys
import threading
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
OBJ_DIR = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "liblutgemm_b200.so")
TORCH_SRC = os.path.join(CSRC, "lutgemm_torch.cpp")
TORCH_LIB = os.path.join(HERE, "lutgemm_torch.so")
TORCH_STAMP = os.path.join(OBJ_DIR, "torch_module.version")  # what the module was compiled against

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC",
    "-Xptxas", "-v", "--expt-relaxed-constexpr",
    "-I", INCLUDE, "-I", CSRC,
]


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _deps_mtime():
    files = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE)]
    return max(os.path.getmtime(f) for f in files)


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(OBJ_DIR, src.replace(".cu", ".o"))
    cmd = ["nvcc", *NVCC_FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
    res = subprocess.run(cmd, capture_output=True, text=True)
    log = os.path.join(OBJ_DIR, src.replace(".cu", ".ptxas.log"))
    with open(log, "w") as f:
        f.write(res.stderr)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"nvcc failed on {src}")
    if verbose:
        sys.stderr.write(res.stderr)
    return obj


def _torch_version():
    """The PyTorch and Python that the extension module has to fit; None without PyTorch."""
    try:
        return f"torch {importlib.metadata.version('torch')} {sys.implementation.cache_tag}"
    except importlib.metadata.PackageNotFoundError:
        return None


def _built_for() -> str:
    try:
        with open(TORCH_STAMP) as f:
            return f.read()
    except OSError:
        return ""


def _compile_torch(lib_ready) -> None:
    """The extension module: compiled while the library's sources are, linked when it is there (`lib_ready`: waits for that)."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    obj = os.path.join(OBJ_DIR, "torch_module.obj")  # (not .o: it is no part of the library)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    includes = [INCLUDE, sysconfig.get_paths()["include"], os.path.join(cuda, "include"), *include_paths()]
    flags = ["-O2", "-std=c++17", "-fPIC", "-DTORCH_EXTENSION_NAME=lutgemm_torch", "-DTORCH_API_INCLUDE_EXTENSION_H",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    res = subprocess.run(["g++", *flags, *(x for i in includes for x in ("-isystem", i)), "-c", TORCH_SRC, "-o", obj], capture_output=True,
                         text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("g++ failed on lutgemm_torch.cpp")
    lib_ready()
    dirs = [HERE, *library_paths()]
    subprocess.run(["g++", "-shared", "-o", TORCH_LIB + ".tmp", obj, *(f"-L{d}" for d in dirs), "-l:liblutgemm_b200.so", "-lc10", "-lc10_cuda",
                    "-ltorch_cpu", "-ltorch", "-ltorch_python", "-Wl,-rpath,$ORIGIN"], check=True)
    os.replace(TORCH_LIB + ".tmp", TORCH_LIB)


def build(force: bool = False, verbose: bool = False, module: bool = True) -> str:
    """Builds what is older than its sources (`force`: all) and returns the library's path; `module`: lutgemm_torch.so too, if PyTorch is
    installed."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    newest = _deps_mtime()

    def fresh(path):
        return not force and os.path.exists(path) and os.path.getmtime(path) >= newest

    version = _torch_version() if module else None
    make_library, make_module = not fresh(LIB), version is not None and not (fresh(TORCH_LIB) and _built_for() == version)
    srcs = _sources()
    linked = threading.Event()
    with ThreadPoolExecutor(max_workers=min(8, len(srcs)) + 1) as ex:
        compiled = ex.submit(_compile_torch, linked.wait) if make_module else None
        try:
            if make_library:
                objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
                subprocess.run(["nvcc", "-shared", "-o", LIB + ".tmp", *objs, "-lcudart"], check=True)
                os.replace(LIB + ".tmp", LIB)
        finally:
            linked.set()
        if compiled is not None:
            try:
                compiled.result()
            except Exception as e:
                raise RuntimeError(f"{LIB} is built, but not its PyTorch module; --library-only leaves that out") from e
            with open(TORCH_STAMP, "w") as f:
                f.write(version)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv, module="--library-only" not in sys.argv))
    if "--library-only" not in sys.argv and _torch_version() is None:
        print("PyTorch is not installed: lutgemm_torch.so was left out")
