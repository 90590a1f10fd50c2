"""Range checks of the built gfx950 code (CPU only).

A buffer load's range check covers the lane's offset and the instruction's; the
scalar offset is not promised to be part of it.  The kernels that run down a
matrix' rows and count on the check to drop those past its end (k_w4_vec,
k_moe_vec_up, k_moe_vec_down: include/hipgemm/detail/w4_vec.hpp, Vec::load) must
therefore step rows by the lane's offset alone; this test disassembles the built
library and looks at the scalar offset of each of their buffer loads."""
import os
import re
import shutil
import subprocess

import pytest

from test_isa_hazards import LIB, OBJDUMP, code_objects

ENTRY = re.compile(r"^[0-9a-f]+ <(\S+)>:")
KERNELS = ("k_w4_vec", "k_moe_vec_up", "k_moe_vec_down")
LOAD = re.compile(r"^\s*buffer_load_\w+\s+(?:v\d+|v\[\d+:\d+\]),\s*\w+,\s*s\[\d+:\d+\],\s*(\w+)")


def scalar_offsets(lines, kernels=KERNELS):
    """(loads seen by kernel, loads with a scalar offset)."""
    seen, found, name = dict.fromkeys(kernels, 0), [], None
    for line in lines:
        m = ENTRY.match(line)
        if m:
            name = next((k for k in kernels if k in m[1]), None)
        elif name and "buffer_load" in line:
            m = LOAD.match(line)
            assert m, f"not understood: {line}"
            seen[name] += 1
            if m[1] != "0":
                found.append(f"{name}: {line.strip()}")
    return seen, found


@pytest.mark.skipif(not os.path.exists(LIB), reason="library not built")
@pytest.mark.skipif(not os.path.exists(OBJDUMP) or not shutil.which("objcopy"),
                    reason="llvm-objdump / objcopy not available")
def test_rows_are_stepped_inside_the_range_check(tmp_path):
    total, found = dict.fromkeys(KERNELS, 0), []
    for i, co in enumerate(code_objects(LIB)):
        if not any(k.encode() in co for k in KERNELS):
            continue
        f = tmp_path / f"co{i}.o"
        f.write_bytes(co)
        asm = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(f)], check=True,
                             capture_output=True, text=True).stdout
        seen, bad = scalar_offsets(asm.splitlines())
        found += bad
        for k, n in seen.items():
            total[k] += n
    assert all(total.values()), f"kernels without buffer loads: {total}"
    assert not found, f"{len(found)} loads, e.g.:\n" + "\n".join(found[:5])


def test_scanner_tells_the_forms_apart():
    head = ["0000000000001900 <_ZN7hipgemm6detail8k_w4_vecILi1EEEvNS0_6W4ArgsE>:"]
    good = head + ["\tbuffer_load_dwordx4 v[2:5], v40, s[4:7], 0 offen nt",
                   "\tbuffer_load_ushort v6, v41, s[8:11], 0 offen offset:2"]
    bad = head + ["\tbuffer_load_ubyte v6, v41, s[8:11], s33 offen"]
    assert scalar_offsets(good) == ({"k_w4_vec": 2, "k_moe_vec_up": 0, "k_moe_vec_down": 0}, [])
    assert len(scalar_offsets(bad)[1]) == 1
    assert scalar_offsets(["0 <other>:"] + bad[1:])[1] == []
