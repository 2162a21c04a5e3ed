"""Loads to LDS have arrived before the waves of a workgroup meet, as the built library says of the attention weights'
kernel for many rows: between such a load and the next barrier behind it stands a wait for all loads."""
import os
import re
import subprocess

import curoaring as cr
from test_attention_registers import READELF, _code_objects

OBJDUMP = os.path.join(os.path.dirname(READELF), "llvm-objdump")


def test_loads_to_lds_are_waited_for(tmp_path):
    with open(cr.LIB_PATH, "rb") as f:
        data = f.read()
    seen = {}
    for i, code in enumerate(_code_objects(data)):
        if b"wt_tiles" not in code:
            continue
        path = tmp_path / f"{i}.elf"
        path.write_bytes(code)
        text = subprocess.run([OBJDUMP, "-d", str(path)], capture_output=True, text=True, check=True, timeout=60).stdout
        for kernel in re.split(r"\n(?=[0-9a-f]+ <)", text):
            name = re.match(r"[0-9a-f]+ <(\S*wt_tiles\S*)>:", kernel)
            if not name:
                continue
            pending, loads, early = False, 0, 0
            for line in kernel.split("\n"):
                if "global_load_lds" in line:
                    pending, loads = True, loads + 1
                elif "s_waitcnt" in line and "vmcnt(0)" in line:
                    pending = False
                elif "s_barrier" in line:
                    early += pending
            seen[name.group(1)] = loads, early
    assert len(seen) == 18 and all(loads and not early for loads, early in seen.values()), seen
