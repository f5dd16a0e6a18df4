"""The instructions that this library's own kernels were compiled to: what the compiler is known to get wrong is not in them."""
import os
import re
import shutil
import subprocess

import pytest

from tokenstation5_amd import ts5hip

OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")


def empty_branches(asm):
    """Kernels with a divergent branch around nothing: lanes are chosen and at once all are back. That is what is left
    where the compiler took a vector's element (free, so it is moved before the branch) out of a block that lanes reach in
    two ways, as in `a || b ? x[i] : y`, and gave those that come by b the other value."""
    found, kernel, saved = [], None, None
    for line in asm.splitlines():
        line = line.split("//")[0].strip()
        name = re.match(r"[0-9a-f]+ <(\w+)>:", line)
        if name:
            kernel, saved = name[1], None
        elif saved and re.match(rf"s_or_b64 exec, exec, {re.escape(saved)}$", line):
            found.append(kernel)
            saved = None
        elif not re.match(r"(s_cbranch_execz|s_waitcnt|s_nop)\b", line):
            m = re.match(r"s_and_saveexec_b64 (s\[\d+:\d+\]), ", line)
            saved = m[1] if m else None
    return found


def test_the_pattern_is_found():
    asm = """0000000000001000 <k_some>:
\ts_and_saveexec_b64 s[0:1], vcc           // 000000001000
\ts_cbranch_execz 3                        // 000000001004
\tv_add_f32_e32 v0, v1, v0                 // 000000001008
\ts_or_b64 exec, exec, s[0:1]              // 00000000100C
0000000000002000 <k_other>:
\ts_and_saveexec_b64 s[2:3], s[4:5]        // 000000002000
\ts_or_b64 exec, exec, s[2:3]              // 000000002004
"""
    assert empty_branches(asm) == ["k_other"]


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")
def test_no_branch_lost_its_values(tmp_path):
    lib = shutil.copy(ts5hip.lib()._name, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", str(lib)], cwd=tmp_path, check=True, capture_output=True)
    objects = [f for f in os.listdir(tmp_path) if f.endswith("gfx950")]
    assert len(objects) >= 10
    kernels = 0
    for f in objects:
        asm = subprocess.run([OBJDUMP, "-d", f], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        kernels += len(re.findall(r"^[0-9a-f]+ <_Z", asm, re.M))
        assert empty_branches(asm) == [], f
    assert kernels > 100
