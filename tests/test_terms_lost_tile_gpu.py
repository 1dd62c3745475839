"""A tile whose wait ran out leaves its score gradients unfinished: the table's gradient of its head is NaN, not a sum of whatever was
there.  No wait is made to run out: a program calls the sums with a tile that says so."""
import os
import subprocess

import pytest

from helpers import ROOT
from custom_op_benchmark_b200 import build

pytestmark = pytest.mark.gpu


def test_sums_by_bucket_with_a_lost_tile(tmp_path):
    exe = tmp_path / "terms_lost_tile"
    res = subprocess.run([build._nvcc(), "-std=c++17", "-O2", "-gencode", "arch=compute_100a,code=sm_100a", "-I" + build.CSRC,
                          os.path.join(ROOT, "tests", "terms_lost_tile.cu"), "-o", str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and res.stdout.strip() == "fine", res.stdout + res.stderr
