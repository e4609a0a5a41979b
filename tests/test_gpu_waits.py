"""GPU test of the bounded wait that the tile kernel's roles use: on a barrier that nobody completes it ends by its
limit."""
from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "wzy-flash-serve_b200", "csrc")


def test_wait_that_runs_out(wz, tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    so = str(tmp_path / "wait_probe.so")
    subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", CSRC, "-shared", "-Xcompiler", "-fPIC",
                    os.path.join(HERE, "wait_probe.cu"), "-o", so], check=True)
    ended, took, faults = (ctypes.c_int * 2)(), (ctypes.c_ulonglong * 2)(), ctypes.c_uint()
    assert ctypes.CDLL(so).wait_probe(ended, took, ctypes.byref(faults)) == 0
    # a barrier that nobody completes, then one that is complete
    assert list(ended) == [2, 2]
    # the limit is 1 s, the polls sleep for 0.1 ms at most
    assert all(0.99e9 <= t <= 1.2e9 for t in took), list(took)
    assert faults.value == wz.FAULT_WAIT_TIMEOUT
