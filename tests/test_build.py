"""What `make` needs: the C ABI builds without torch and Python's headers, the
Python host path follows the installed torch. No GPU."""
import os
import shutil
import subprocess
import sys

import pytest

from conftest import ROOT

PKG = os.path.join(ROOT, "sm_120__gemm_b200")


def dry_run(where, *args):
    return subprocess.run(["make", "-C", str(where), "-n", *args], capture_output=True, text=True)


@pytest.mark.skipif(shutil.which("make") is None, reason="no make")
def test_library_needs_no_python():
    out = dry_run(PKG, "-B", "PYTHON=/nowhere/python3")
    assert out.returncode == 0, out.stderr
    assert "libi4g.so" in out.stdout and "_binding.so" not in out.stdout
    assert "/nowhere" not in out.stdout + out.stderr


@pytest.mark.skipif(shutil.which("make") is None, reason="no make")
def test_python_part_follows_torch(tmp_path):
    """The binding is built once, and again when another torch is installed; the library
    is not built for it. In a copy whose compiler only notes that it was called."""
    tree = tmp_path / "pkg"
    (tree / "_build").mkdir(parents=True)
    shutil.copytree(os.path.join(PKG, "csrc"), tree / "csrc")
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    shutil.copy(os.path.join(PKG, "Makefile"), tree)
    for n in os.listdir(tree / "csrc"):
        if n.endswith(".cu"):
            (tree / "_build" / (n[:-3] + ".o")).touch()
    (tree / "libi4g.so").touch()
    cxx = tmp_path / "cxx"
    cxx.write_text(f"#!/bin/sh\necho $* >> {tmp_path}/calls\ntouch {tree}/_binding.so\n")
    cxx.chmod(0o755)

    def calls():
        subprocess.run(["make", "-C", str(tree), "python", f"PYTHON={sys.executable}",
                        f"CXX={cxx}", "NVCC=/nowhere/nvcc"], check=True, capture_output=True)
        return (tmp_path / "calls").read_text().splitlines()
    import torch
    first = calls()
    assert len(first) == 1
    assert f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}" in first[0]
    assert len(calls()) == 1
    (tree / "_build" / "torch.id").write_text("another torch\n")
    assert len(calls()) == 2 and len(calls()) == 2


def test_binding_names_the_torch_it_was_built_against():
    import torch
    from sm_120__gemm_b200 import launching
    module = launching.binding()
    assert torch.__version__.startswith(module.torch_version) and module.torch_version


def test_binding_of_another_torch_is_refused(monkeypatch):
    import torch
    from sm_120__gemm_b200 import launching
    module = launching.binding()
    for version, fits in (("2.11.0+cu128", True), ("2.11.0.dev20260101", True),
                          ("2.12.0+cu128", False)):
        monkeypatch.setattr(module, "torch_version", "2.11.0")
        monkeypatch.setattr(torch, "__version__", version)
        monkeypatch.setattr(launching, "_binding", None)
        if fits:
            launching.binding()
        else:
            with pytest.raises(ImportError):
                launching.binding()
