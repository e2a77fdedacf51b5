"""The products need the library alone: the package imports, and `make` builds, without
what the serving operators' Python calls need beside it."""
import os
import shutil
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "qgemm-mx_b200")


def test_package_imports_without_the_binding(tmp_path):
    copy = tmp_path / "qgemm-mx_b200"
    copy.mkdir()
    for f in ("__init__.py", "serving.py"):
        shutil.copy(os.path.join(PACKAGE, f), copy / f)
    os.symlink(os.path.join(PACKAGE, "libqgemm_b200.so"), copy / "libqgemm_b200.so")
    code = """
import importlib
qg = importlib.import_module("qgemm-mx_b200")
assert qg.bytes_per_weight(qg.MXFP4) == 0.53125 and callable(qg.gemm_w4a16)
assert "qgemm_kv_plan" in qg.EXPORTED and "kv_plan" in dir(qg)
assert qg.lib().qgemm_kv_max_runs(3, 100, 16) == 12  # the C-ABI is whole
for name in ("kv_plan", "KVCache", "residual_norm", "serving"):
    try:
        getattr(qg, name)
    except ImportError as e:
        assert "make" in str(e) and "binding" in str(e), e
    else:
        raise AssertionError(name)
try:
    qg.no_such_name
except AttributeError:
    print("fine")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=tmp_path, capture_output=True, text=True,
                       env={**os.environ, "PYTHONPATH": str(tmp_path)})
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stderr[-2000:]


def test_make_builds_the_library_without_python(qg):
    def planned(*targets):
        r = subprocess.run(["make", "-n", "-B", "-C", os.path.join(PACKAGE, "csrc"), "PYTHON=/no/such/python", *targets],
                           capture_output=True, text=True)
        return r.stdout + r.stderr

    text = planned()
    assert "libqgemm_b200.so" in text and "kv_plan.cu" in text
    assert "binding" not in text and "no/such" not in text
    assert "_binding.so" in planned("binding")


def test_serving_names_are_the_packages(qg):
    for name in ("KV_E4M3", "KV_INT8", "KVCache", "KVPlan", "kv_append", "kv_attention", "kv_attention_workspace", "kv_plan",
                 "make_kv_cache", "make_kv_workspace", "residual_norm"):
        assert getattr(qg, name) is getattr(qg.serving, name) and name in dir(qg)
