"""Loads the in-tree native extension. The CUDA path must never be replaced by a silent fallback:
if the extension is missing it is built once (nvcc is part of the image); if that fails the import
fails loudly."""
from __future__ import annotations

import importlib
import os

from . import _build

_C = None
_A = None
_testk = None


def _autobuild() -> bool:
    return os.environ.get("ROCSHMEM_B200_NO_AUTOBUILD") != "1"


def load():
    """Return the ``_C`` extension module, building it on first use if it is absent."""
    global _C
    if _C is None:
        if not _build.is_built(with_attention=False) and _autobuild():
            _build.build(with_tests=False)
        _C = importlib.import_module("rocshmem_b200._C")
    return _C


def load_attention():
    """Return the extension with the attention operators (its functions take torch tensors), building it on first use if
    it is absent or was compiled against another version of torch. Never loaded into another torch than its own."""
    global _A
    if _A is None:
        load()
        if not _build.is_built() and _autobuild():
            _build.build(with_tests=False)
        torch = importlib.import_module("torch")     # whose libraries the extension resolves its symbols from
        built = _build.attention_torch()
        if built != str(torch.__version__):
            raise ImportError(f"the attention operators were compiled against torch {built}, this is torch "
                              f"{torch.__version__}: run `python -m rocshmem_b200._build` with it")
        _A = importlib.import_module("rocshmem_b200._A")
    return _A


def load_test_kernels():
    """Return the extension with the functional-test kernels (device API exercised from user code)."""
    global _testk
    load()
    if _testk is None:
        if not _build.is_built(with_tests=True, with_attention=False):
            _build.build(with_tests=True)
        _testk = importlib.import_module("rocshmem_b200._testk")
    return _testk
