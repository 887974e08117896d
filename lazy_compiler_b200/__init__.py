"""lazy_compiler_b200: a B200 (sm_100a) operator backend for Emmy Kernel IR packages.

Host side: :mod:`.ir` (IR loader), :mod:`.recognize` (operation classes),
:mod:`.compiler` (``compile_file``), :mod:`.runtime` (ctypes C-ABI launcher
over ``liblazyb200.so``), :mod:`.runner` (meta.json-driven package runner).
Beside the packages: :mod:`.serving` (prompt and paged attention and the
key-value cache's pages on torch tensors).
"""
from .ir import CompileError  # noqa: F401

__all__ = ["CompileError"]
