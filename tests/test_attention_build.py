"""The extension with the attention operators is compiled against torch's headers: it is rebuilt when torch changes, and
never loaded into another torch than its own. No GPU."""
import os
import subprocess
import sys

import pytest
import torch

from rocshmem_b200 import _build, _native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_extension_names_the_torch_it_was_compiled_against():
    assert _build._torch_version() == str(torch.__version__)
    _native.load_attention()
    assert _build.attention_torch() == str(torch.__version__)
    assert _native.load_attention().built_for == f"rocshmem_b200._A for torch {torch.__version__}"


def test_another_torch_changes_the_command_of_the_objects_that_include_its_headers(monkeypatch):
    """System headers are not among ninja's dependencies: without the version an upgrade in place rebuilt nothing."""
    now = _build._ninja_text(with_tests=False)
    monkeypatch.setattr(_build, "_torch_version", lambda: "99.0.1+cu777")
    then = _build._ninja_text(with_tests=False)
    differ = [(a, b) for a, b in zip(now.splitlines(), then.splitlines()) if a != b]
    assert len(differ) == len(_build.TORCH_CPP) and all("ROCSHMEM_TORCH_VERSION=99.0.1+cu777" in b for _, b in differ)
    assert not _build.is_built() and _build.is_built(with_attention=False)


@pytest.mark.parametrize("content,version", [(None, None), (b"\0\1 something else", None),
                                             (b"\0rocshmem_b200._A for torch 2.99.0a0+git12ab\0x", "2.99.0a0+git12ab")])
def test_the_version_in_a_file(tmp_path, monkeypatch, content, version):
    monkeypatch.setattr(_build, "PKG", tmp_path)
    if content is not None:
        (tmp_path / f"_A{_build.EXT}").write_bytes(content)
    assert _build.attention_torch() == version


def test_a_build_for_another_torch_is_refused_and_the_rest_still_loads():
    code = """
from rocshmem_b200 import _build, _native
_build.attention_torch = lambda: "1.0.0+other"
_native.load()
try:
    _native.load_attention()
except ImportError as e:
    assert "compiled against torch 1.0.0+other" in str(e), e
else:
    raise AssertionError("loaded")
import sys
assert "rocshmem_b200._A" not in sys.modules
print("refused")
"""
    env = dict(os.environ, ROCSHMEM_B200_NO_AUTOBUILD="1", PYTHONPATH=ROOT)
    out = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "refused", out.stderr


def test_an_isolated_build_is_refused(monkeypatch):
    """It would compile against a torch of its own, in a folder that is deleted afterwards."""
    import importlib.util
    import tomllib
    with open(os.path.join(ROOT, "pyproject.toml"), "rb") as f:
        assert not any(r.startswith("torch") for r in tomllib.load(f)["build-system"]["requires"])
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    with pytest.raises(RuntimeError, match="no-build-isolation"):
        _build._ninja_text(with_tests=False)


def test_the_extension_has_no_run_path_to_a_torch():
    text = _build._ninja_text(with_tests=False)
    libs = [line for line in text.splitlines() if line.lstrip().startswith("libs =")]
    assert len(libs) == 1 and "rpath" not in libs[0]
