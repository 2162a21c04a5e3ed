"""How the work of the attention weights is split, on the CPU (tests/cpp/weights_work_check.cpp runs
csrc/weights_work.hpp)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_shape_has_its_launches():
    exe = os.path.join(ROOT, "tests", "cpp", "weights_work_check")
    assert os.path.exists(exe), "tests/cpp/weights_work_check is built by __graft_entry__.build()"
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "weights_work_check: OK" in r.stdout, r.stdout + r.stderr
