"""How paged attention numbers its work, on the CPU (tests/cpp/attention_work_check.cpp
runs csrc/attention_work.hpp): every tile of rows answered once over all of its keys,
and no entry written outside the table of ranges."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_number_has_its_work():
    exe = os.path.join(ROOT, "tests", "cpp", "attention_work_check")
    assert os.path.exists(exe), "tests/cpp/attention_work_check is built by __graft_entry__.build()"
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "attention_work_check: OK" in r.stdout, r.stdout + r.stderr
