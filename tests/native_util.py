"""Compiles a file of tests/native for the host, with the kernels' own headers: what they compute apart
from the GPU's instructions can be tested without one."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("MCB_NVCC", "/usr/local/cuda/bin/nvcc")


def compile_native(name, folder):
    if not os.path.exists(NVCC):
        pytest.skip("no nvcc")
    out = str(folder / name)
    subprocess.run(
        [NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-O1", "-std=c++17",
         "--expt-relaxed-constexpr", "-ccbin", "/usr/bin/g++", "-I", os.path.join(ROOT, "include"),
         "-I", os.path.join(ROOT, "matcoredsl_b200", "csrc"),
         os.path.join(ROOT, "tests", "native", name + ".cu"), "-o", out],
        check=True, capture_output=True, text=True)
    return out
