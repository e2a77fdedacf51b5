"""The host refuses a kv_attention call whose requests could pass 2^31 places on the
kernels' line (their prefix sums are 32-bit), so its bound on a request's places must hold
for every shape.  tests/cpp/line_bound.cu compares it with the line's own formula on the
CPU, over calls drawn evenly in the logarithms of their sizes."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_no_line_passes_the_hosts_bound(tmp_path):
    nvcc = shutil.which("nvcc")
    if nvcc is None:
        pytest.skip("no nvcc")
    out = str(tmp_path / "line_bound")
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O2", "-std=c++17", "--expt-relaxed-constexpr",
                    "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(ROOT, "qgemm-mx_b200", "csrc"), "-o", out,
                    os.path.join(ROOT, "tests", "cpp", "line_bound.cu")], check=True)
    r = subprocess.run([out], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
