"""Layer norm when a wait for a row's copies runs out: the rows of the threads that gave up are NaN, mean, deviation and column
sums included, the others as ever, and the kernel ends after one limit, not one for every row that is left."""
import os
import subprocess
import time

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


def test_a_row_that_does_not_come_is_told(tmp_path):
    program = str(tmp_path / "norm_waits")
    subprocess.check_call(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-I", os.path.join(HERE, "..", "include"),
                           "-o", program, os.path.join(HERE, "norm_waits.cu")])
    start = time.time()
    r = subprocess.run([program], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    # six launches lose a row, ten milliseconds each; the rest is the program's start
    assert time.time() - start < 60
