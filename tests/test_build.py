"""What a build asks for."""
import os
import shutil
import subprocess
import sys

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "genllm_amd", "csrc")
pytestmark = pytest.mark.skipif(shutil.which("make") is None, reason="make")


def dry(*args):
    return subprocess.run(["make", "-n", "-B", "-C", CSRC, *args], capture_output=True, text=True, timeout=60)


def test_the_c_library_needs_no_python():
    r = dry("PYTHON=/bin/false")
    assert r.returncode == 0 and "libgenllm_hip.so" in r.stdout
    assert "_calls.so" not in r.stdout and "torch" not in r.stdout and "Python" not in r.stdout


def test_the_python_calls_are_built_for_this_torch():
    import torch

    r = dry("calls", f"PYTHON={sys.executable}")
    assert r.returncode == 0 and os.path.dirname(torch.__file__) + "/include" in r.stdout and "_calls.so" in r.stdout


def test_the_python_calls_without_torch(tmp_path):
    """A message that says what is missing, in a copy of the folder."""
    copy = tmp_path / "genllm_amd" / "csrc"
    copy.mkdir(parents=True)
    for f in ("Makefile", "calls.cpp"):
        shutil.copy(os.path.join(CSRC, f), copy)
    shutil.copytree(os.path.join(CSRC, "..", "..", "include"), tmp_path / "include")
    r = subprocess.run(["make", "-C", str(copy), "calls", "PYTHON=/bin/false"], capture_output=True, text=True, timeout=60)
    assert r.returncode != 0 and "importable torch" in r.stderr and not (tmp_path / "genllm_amd" / "_calls.so").exists()
