"""The kernels of the operators for long and speculative answers keep their work in registers, as the built library
says of them: none has scratch memory or spilled vector registers."""
import re
import subprocess

import curoaring as cr
from test_attention_registers import READELF, _code_objects


def test_no_kernel_spills(tmp_path):
    with open(cr.LIB_PATH, "rb") as f:
        data = f.read()
    seen = {}
    for i, code in enumerate(_code_objects(data)):
        path = tmp_path / f"{i}.elf"
        path.write_bytes(code)
        notes = subprocess.run([READELF, "--notes", str(path)], capture_output=True, text=True, check=True, timeout=60).stdout
        for kernel in notes.split("- .agpr_count:")[1:]:
            value = lambda key: re.search(rf"\.{key}:\s*(\S+)", kernel).group(1)  # noqa: E731
            name = value("symbol")
            if re.search(r"\d(ro|wt|ev|sg|dv)_[a-z]+", name):
                seen[name] = int(value("private_segment_fixed_size")), int(value("vgpr_spill_count"))
    assert any("wt_tiles" in k for k in seen) and any("dv_sums" in k for k in seen), sorted(seen)
    assert set(seen.values()) == {(0, 0)}, {k: v for k, v in seen.items() if v != (0, 0)}
