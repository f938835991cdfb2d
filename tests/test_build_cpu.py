"""The build script with a stand-in for nvcc: what it builds where torch or the host compiler is missing."""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

import pytest

from conftest import PKG_NAME, ROOT

NVCC = """#!/bin/sh
while [ $# -gt 0 ]; do if [ "$1" = -o ]; then echo made > "$2"; fi; shift; done
"""


@pytest.fixture
def tree(tmp_path):
    """A copy of the package's sources; (run, library, binding): run(...) builds it and returns the finished process."""
    pkg = tmp_path / PKG_NAME
    pkg.mkdir()
    shutil.copy(ROOT / PKG_NAME / "build.py", pkg)
    shutil.copytree(ROOT / PKG_NAME / "csrc", pkg / "csrc")
    shutil.copytree(ROOT / "include", tmp_path / "include")
    nvcc = tmp_path / "cuda" / "bin" / "nvcc"
    nvcc.parent.mkdir(parents=True)
    nvcc.write_text(NVCC)
    nvcc.chmod(0o755)
    no_torch = tmp_path / "no_torch" / "torch"
    no_torch.mkdir(parents=True)
    (no_torch / "__init__.py").write_text("raise ImportError('no torch here')\n")

    def run(torch, **env):
        env = {**os.environ, "NVCC": str(nvcc), **env}
        if not torch:
            env["PYTHONPATH"] = str(no_torch.parent)
        return subprocess.run([sys.executable, str(pkg / "build.py")], env=env, capture_output=True, text=True, timeout=300)

    return run, pkg / "libfqkv_b200.so", pkg / "_torch_binding.so"


def test_the_library_needs_no_torch(tree):
    run, lib, binding = tree
    r = run(torch=False)
    assert r.returncode == 0, r.stderr
    assert lib.exists() and not binding.exists()
    assert "_torch_binding.so" in r.stderr  # and it says what is missing
    before = lib.stat().st_mtime_ns
    assert run(torch=False).returncode == 0 and lib.stat().st_mtime_ns == before  # nothing to do the second time


def test_a_failing_binding_leaves_a_whole_library(tree):
    run, lib, binding = tree
    r = run(torch=True, CXX="false")
    assert r.returncode != 0 and "torch_binding.cpp" in r.stderr
    assert lib.exists() and not binding.exists()
