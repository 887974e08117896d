"""What the build makes anew, and in which order (no compiler runs)."""
import os
import subprocess

import pytest

from lazy_compiler_b200 import build as B


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A build tree of one kernel source, and the commands that were run: each writes its output file."""
    for name in ("csrc", "include", "_build"):
        (tmp_path / name).mkdir()
    for name in ("one.cu", "serving_ext.cpp"):
        (tmp_path / "csrc" / name).write_text("")
    (tmp_path / "include" / "lazyb200.h").write_text("")
    for name, path in (("CSRC", "csrc"), ("INCLUDE", "include"), ("BUILD", "_build"), ("LIBRARY", "lib.so"), ("EXTENSION", "_serving.so")):
        monkeypatch.setattr(B, name, tmp_path / path)
    commands = []

    def run(cmd, **kwargs):
        commands.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write(" ".join(map(str, cmd)))
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(B.subprocess, "run", run)
    monkeypatch.setattr(B, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setenv("CXX", "g++")
    return tmp_path, commands


def extensions(commands):
    return sum("serving_ext.cpp" in " ".join(map(str, c)) for c in commands)


def test_the_library_does_not_wait_for_the_extension(tree, monkeypatch):
    """Without torch, or a compiler that can build against it, the package path's library is linked all the same."""
    path, commands = tree

    def no_torch(name):
        raise B.metadata.PackageNotFoundError(name)

    monkeypatch.setattr(B.metadata, "version", no_torch)
    with pytest.raises(RuntimeError, match="needs torch"):
        B.build()
    assert (path / "lib.so").exists() and not (path / "_serving.so").exists() and extensions(commands) == 0


def test_the_extension_is_built_again_for_another_torch(tree, monkeypatch):
    path, commands = tree
    B.build()
    assert (path / "lib.so").exists() and (path / "_serving.so").exists() and extensions(commands) == 1
    for name in ("_serving.so", "_build/one.o", "lib.so"):  # newer than this repository's build.py
        os.utime(path / name)
    B.build()
    assert extensions(commands) == 1
    version = B.metadata.version("torch")
    monkeypatch.setattr(B.metadata, "version", lambda name: version + ".other")
    B.build()
    assert extensions(commands) == 2
    B.build()
    assert extensions(commands) == 2
    B.build(force=True)
    assert extensions(commands) == 3
