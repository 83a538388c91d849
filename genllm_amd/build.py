"""Build step for libgenllm_hip.so (gfx950) and _calls.so -- see genllm_amd/csrc/Makefile."""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libgenllm_hip.so")
CALLS = os.path.join(HERE, "_calls.so")


def build_library(clean: bool = True, jobs: int = 8) -> str:
    """Compile every HIP source for gfx950 and link libgenllm_hip.so; the Python calls on tensors into _calls.so."""
    if clean:
        subprocess.run(["make", "-s", "-C", CSRC, "clean"], check=True)
    subprocess.run(["make", "-s", "-C", CSRC, f"-j{jobs}", f"PYTHON={sys.executable}", "all", "calls"], check=True)
    for path in (LIB, CALLS):
        if not os.path.exists(path):
            raise RuntimeError("build did not produce " + path)
    return LIB
