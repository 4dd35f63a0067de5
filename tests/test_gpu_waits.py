"""Bounded waits of the tensor-core kernels: a thread that gives one up marks it for the whole block, so
that warps whose own waits end well, on what it left undone, write no results either."""
import ctypes
import os
import shutil
import subprocess

import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.join(HERE, "..", "spiking-affine-lazy-training_b200")
FEW = 200  # looks of some 4 us


@pytest.fixture(scope="module")
def waits(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    lib = str(tmp_path_factory.mktemp("waits") / "waits.so")
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17",
                    "--expt-relaxed-constexpr", "-I", os.path.join(ROOT, "csrc"), "-shared",
                    "-Xcompiler", "-fPIC", "-o", lib, os.path.join(HERE, "waits.cu")], check=True)
    run = ctypes.CDLL(lib).run_waits

    def call(arrives, limit):
        out = (ctypes.c_int * 5)()
        assert run(ctypes.c_int(arrives), ctypes.c_uint(limit), out) == 0
        return list(out)

    return call


def test_a_wait_that_is_given_up_is_seen_by_those_whose_waits_end_well(waits):
    first_left, second_left, second_sees, left, sees = waits(False, FEW)
    assert not first_left and second_left and second_sees
    assert not left and sees


def test_waits_that_end_leave_no_mark(waits):
    first_left, second_left, second_sees, *_ = waits(True, FEW)
    assert first_left and second_left and not second_sees
