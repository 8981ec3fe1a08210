"""What a build makes and leaves alone, with the compilers replaced by stand-ins: the library for C callers needs no PyTorch, and its PyTorch
module follows the installed version."""
import os

import pytest


@pytest.fixture
def build(tmp_path, monkeypatch):
    import build_ext
    made = []
    for name in ("csrc", "include", "build"):
        (tmp_path / name).mkdir()
    for name in ("csrc/a.cu", "csrc/b.cu", "csrc/lutgemm_torch.cpp", "include/x.h"):
        (tmp_path / name).write_text("")
        os.utime(tmp_path / name, (1000, 1000))
    for name, path in (("CSRC", "csrc"), ("INCLUDE", "include"), ("OBJ_DIR", "build"), ("LIB", "lib.so"), ("TORCH_LIB", "module.so"),
                       ("TORCH_STAMP", "build/torch_module.version")):
        monkeypatch.setattr(build_ext, name, str(tmp_path / path))

    def compile_(src, verbose):
        made.append(src)
        return src

    def link(cmd, **kw):
        made.append("library")
        open(cmd[cmd.index("-o") + 1], "w").close()

    def module(lib_ready):
        lib_ready()
        assert os.path.exists(build_ext.LIB)
        made.append("module")
        open(build_ext.TORCH_LIB, "w").close()
    monkeypatch.setattr(build_ext, "_compile", compile_)
    monkeypatch.setattr(build_ext.subprocess, "run", link)
    monkeypatch.setattr(build_ext, "_compile_torch", module)
    monkeypatch.setattr(build_ext, "_torch_version", lambda: "torch 1")

    def run(**kw):
        made.clear()
        assert build_ext.build(**kw) == build_ext.LIB
        return sorted(made)
    run.ext, run.patch, run.path = build_ext, monkeypatch.setattr, tmp_path
    return run


EVERYTHING = ["a.cu", "b.cu", "library", "module"]


def test_what_is_fresh_is_left_alone(build):
    assert build() == EVERYTHING
    assert build() == []
    assert build(force=True) == EVERYTHING
    os.utime(build.path / "csrc/a.cu")  # (newer than both)
    for lib in ("lib.so", "module.so"):
        os.utime(build.path / lib, (2000, 2000))
    assert build() == EVERYTHING


def test_the_library_needs_no_pytorch(build):
    build.patch(build.ext, "_torch_version", lambda: None)
    assert build() == EVERYTHING[:3]
    assert build() == []
    build.patch(build.ext, "_torch_version", lambda: "torch 1")
    assert build(module=False) == []
    assert build() == ["module"]


def test_another_pytorch_makes_the_module_anew(build):
    build()
    build.patch(build.ext, "_torch_version", lambda: "torch 2")
    assert build() == ["module"]
    assert build() == []
    os.remove(build.path / "build/torch_module.version")  # (of a build that did not say)
    assert build() == ["module"]


def test_a_module_that_fails_leaves_the_library(build):
    def fails(lib_ready):
        raise RuntimeError("no compiler")
    compile_module = build.ext._compile_torch
    build.patch(build.ext, "_compile_torch", fails)
    with pytest.raises(RuntimeError, match="library-only"):
        build()
    assert (build.path / "lib.so").exists() and not (build.path / "module.so").exists()
    build.patch(build.ext, "_compile_torch", compile_module)
    assert build() == ["module"]


def test_the_installed_version():
    import build_ext
    import torch
    assert build_ext._torch_version().split()[1].split("+")[0] == torch.__version__.split("+")[0]
