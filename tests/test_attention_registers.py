"""The attention kernels keep their work in registers, as the built library says of
them: none has scratch memory or spilled vector registers.  (An instance that
spilled has given wrong f16 results, and each would be slow.)"""
import os
import re
import subprocess

import curoaring as cr

READELF = os.path.join(os.environ.get("ROCM", "/opt/rocm"), "llvm", "bin", "llvm-readelf")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def _code_objects(data):
    """The gfx950 code objects of the library's bundles: count, then (offset, size, name) of each entry."""
    at = data.find(MAGIC)
    while at >= 0:
        word = lambda p: int.from_bytes(data[p:p + 8], "little")  # noqa: E731
        p = at + len(MAGIC) + 8
        for _ in range(word(at + len(MAGIC))):
            offset, size, n = word(p), word(p + 8), word(p + 16)
            if size and b"gfx950" in data[p + 24:p + 24 + n]:
                yield data[at + offset:at + offset + size]
            p += 24 + n
        at = data.find(MAGIC, at + len(MAGIC))


def test_no_attention_kernel_spills(tmp_path):
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
            if re.search(r"at_rows|at_tiles", name):
                seen[name] = int(value("private_segment_fixed_size")), int(value("vgpr_spill_count"))
    # two types; at_tiles and at_rows for five lengths of rows, and two blocks a wave for three of them
    assert len(seen) == 2 * (5 + 5 + 3), sorted(seen)
    assert set(seen.values()) == {(0, 0)}, {k: v for k, v in seen.items() if v != (0, 0)}
