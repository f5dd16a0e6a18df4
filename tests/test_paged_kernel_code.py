"""What the kernels of a paged cache and of the drafts' verification were compiled to: no registers in memory, and no load that
loops over the lanes of a wave for a buffer that all of them share."""
import os
import re
import shutil
import subprocess

import pytest

from tokenstation5_amd import ts5hip

LLVM = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")
KERNELS = re.compile(r"k_(attn_paged|paged_merge|append_paged|read_paged|verify_rows|verify_pick)")


def lane_loops(asm):
    """Kernels with a loop that picks one lane's buffer after another for a load."""
    found, kernel, picked = [], None, 0
    for line in asm.splitlines():
        line = line.split("//")[0].strip()
        name = re.match(r"[0-9a-f]+ <(\w+)>:", line)
        if name:
            kernel, picked = name[1], 0
        elif line.startswith("v_readfirstlane_b32"):
            picked += 1
        elif picked >= 4 and line.startswith("s_and_saveexec_b64"):
            picked = -1
        elif picked == -1 and line.startswith("buffer_load"):
            found.append(kernel)
            picked = 0
        elif not re.match(r"(v_cmp|s_and|s_nop|s_waitcnt)", line):
            picked = 0
    return found


def test_the_pattern_is_found():
    asm = """0000000000001000 <k_some>:
\tv_readfirstlane_b32 s8, v6
\tv_readfirstlane_b32 s9, v7
\tv_readfirstlane_b32 s10, v8
\tv_readfirstlane_b32 s11, v9
\tv_cmp_eq_u64_e64 s[4:5], s[8:9], v[6:7]
\ts_nop 0
\tv_cmp_eq_u64_e64 s[6:7], s[10:11], v[8:9]
\ts_and_b64 s[4:5], s[4:5], s[6:7]
\ts_and_saveexec_b64 s[4:5], s[4:5]
\tbuffer_load_dwordx2 v[130:131], v101, s[8:11], 0 offen
0000000000002000 <k_other>:
\tv_readfirstlane_b32 s8, v6
\ts_and_saveexec_b64 s[4:5], s[4:5]
\tbuffer_load_dwordx2 v[130:131], v101, s[8:11], 0 offen
"""
    assert lane_loops(asm) == ["k_some"]


@pytest.mark.skipif(not os.path.exists(os.path.join(LLVM, "llvm-objdump")), reason="no llvm-objdump")
def test_registers_and_buffers(tmp_path):
    lib = shutil.copy(ts5hip.lib()._name, tmp_path / "lib.so")

    def run(tool, *args):
        return subprocess.run([os.path.join(LLVM, tool), *args], cwd=tmp_path, check=True, capture_output=True, text=True).stdout

    run("llvm-objdump", "--offloading", str(lib))
    seen = 0
    for f in os.listdir(tmp_path):
        if not f.endswith("gfx950"):
            continue
        notes = run("llvm-readelf", "--notes", f)
        for m in re.finditer(r"\.name:\s+(\S+).*?\.private_segment_fixed_size:\s+(\d+).*?\.vgpr_spill_count:\s+(\d+)", notes, re.S):
            if KERNELS.search(m[1]):
                seen += 1
                assert (m[2], m[3]) == ("0", "0"), m.groups()
        if KERNELS.search(notes):
            assert [k for k in lane_loops(run("llvm-objdump", "-d", f)) if KERNELS.search(k)] == [], f
    assert seen > 40
