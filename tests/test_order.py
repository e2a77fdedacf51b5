"""A run that stops at the first failure still reaches every test that can run."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DRIVER = os.path.join(ROOT, "oracle", "_ref", "time_graphed_w4a16")


def test_what_needs_the_reference_driver_runs_last_without_it():
    r = subprocess.run([sys.executable, "-m", "pytest", "tests", "--collect-only", "-q", "-m", "gpu", "-p", "no:cacheprovider"],
                       cwd=ROOT, capture_output=True, text=True)
    files = [line.split("::")[0] for line in r.stdout.splitlines() if "::" in line]
    order = [f for i, f in enumerate(files) if i == 0 or files[i - 1] != f]
    assert len(order) == len(set(order)) > 10, r.stdout[-2000:]
    others = [f for f in order if not f.endswith("test_gpu_cpp_driver.py")]
    assert others == sorted(others)
    if not os.path.exists(DRIVER):
        assert order[-1].endswith("test_gpu_cpp_driver.py")
