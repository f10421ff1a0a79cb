"""What the build needs, and when the extension module of ops.py is built again (no GPU needed, nothing is compiled but by the first test)."""
import subprocess
import sys

import pytest
import torch

from lemonade_burn_b200 import build


@pytest.fixture
def quiet(monkeypatch, tmp_path):
    """build() that notes what it would compile, in a tree without anything built."""
    done = []
    monkeypatch.setattr(build, "LIB", tmp_path / "liblbk.so")
    monkeypatch.setattr(build, "PKG", tmp_path)
    monkeypatch.setattr(build, "TORCH_OPS", tmp_path / "_torch_ops.so")
    monkeypatch.setattr(build, "_build_library", lambda force, verbose, lib, sources: done.append(lib.name))
    real, build_module = build.build_torch_ops, lambda force=False: done.append("_torch_ops.so") if force or build.torch_ops_stale() else None
    monkeypatch.setattr(build, "build_torch_ops", build_module)
    assert callable(real)
    return done


def test_the_module_is_what_this_torch_needs():
    build.build()
    assert not build.torch_ops_stale() and torch.__version__ in build.torch_ops_target()


def test_a_module_of_another_torch_is_stale_and_refused(monkeypatch):
    from lemonade_burn_b200 import ops
    build.build()
    monkeypatch.setattr(build, "torch_ops_target", lambda: "lbk torch ops: torch 9.9, cpython-312")
    assert build.torch_ops_stale()
    monkeypatch.setattr(ops, "_native", None)
    with pytest.raises(RuntimeError, match="another torch"):
        ops.advance_pos_by(torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_a_file_that_is_no_module_is_refused(monkeypatch, tmp_path):
    from lemonade_burn_b200 import _lib, ops
    (tmp_path / "_torch_ops.so").write_bytes(b"not a library")
    monkeypatch.setattr(_lib, "LIB_PATH", tmp_path / "liblbk.so")
    monkeypatch.setattr(ops, "_native", None)
    with pytest.raises(RuntimeError, match="build it with"):
        ops.advance_pos_by(torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_the_library_is_built_without_torch():
    """liblbk.so has no torch in it: a host in C or Rust builds it with nvcc alone."""
    code = """
import sys
sys.modules["torch"] = None
from pathlib import Path
from lemonade_burn_b200 import build
built = []
build.LIB, build.TORCH_OPS = Path("/nowhere/liblbk.so"), Path("/nowhere/_torch_ops.so")
build._build_library = lambda force, verbose, lib, sources: built.append(lib.name)
build.build()
build.build(force=True)
print(built)
"""
    out = subprocess.run([sys.executable, "-W", "error", "-c", code], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "['liblbk.so', 'liblbk.so']", out.stderr


def test_without_pythons_headers_the_library_is_built_and_the_rest_is_said(quiet, monkeypatch, tmp_path):
    monkeypatch.setattr(build.sysconfig, "get_path", lambda name: str(tmp_path))
    with pytest.warns(UserWarning, match="Python.h"):
        build.build()
    assert quiet == ["liblbk.so"]


def test_one_familys_part_comes_with_the_module(quiet):
    """It has log probabilities, which ops.py calls."""
    assert build.library_for("Pefolix").name == "liblbk-Pefolix.so"
    assert quiet == ["liblbk-Pefolix.so", "_torch_ops.so"]
