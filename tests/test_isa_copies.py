"""CPU: properties of the generated gfx950 code of the attention over the paged cache that the compiler does not check
for inline asm.

Its HBM -> LDS copies take a 64-bit address from vector registers and the place in LDS from M0, set in the same asm. Checked
for every copy: the address is a pair of VGPRs (an SGPR base would need the wait states that test_isa_hazards.py counts); M0 was
last written by an SALU move at least 3 wait states earlier; and no VGPR of an inline-asm load is touched before the
first wait. The kernels use no scratch memory: a spilled vector register's reload would stand among the counted copies,
whose waits say how many loads may still be on their way.
"""
import os
import re
import subprocess

import pytest

from test_isa_hazards import CSRC, HIPCC, ROOT, copy_base_hazards, inflight_register_uses

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
M0_WAIT_STATES = 3


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("isa") / "attend.s")
    cmd = [HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-ffp-contract=off", "-Xclang", "-target-feature", "-Xclang",
           "-packed-fp32-ops", "-mllvm", "-amdgpu-kernarg-preload-count=10", "--cuda-device-only", "-S", "-I",
           os.path.join(ROOT, "include"), os.path.join(CSRC, "attend.hip"), "-o", out]
    subprocess.run(cmd, check=True, capture_output=True, timeout=600)
    return open(out).read()


def m0_hazards(text: str):
    """(number of copies, descriptions of those without an SALU write of M0 at least M0_WAIT_STATES before)."""
    lines = [x.split(";")[0].strip() for x in text.splitlines()]
    n, bad = 0, []
    for i, line in enumerate(lines):
        if not line.startswith("global_load_lds"):
            continue
        n += 1
        states = 0
        for t in reversed(lines[:i]):
            if t.endswith(":"):
                bad.append(f"line {i + 1}: M0 is not written in this block")
                break
            if not t or t.startswith("."):
                continue
            if re.match(r"s_mov_b32\s+m0\s*,", t):
                if states < M0_WAIT_STATES:
                    bad.append(f"line {i + 1}: `{t}` {states} wait states before")
                break
            if re.match(r"\w+\s+m0\s*,", t):
                bad.append(f"line {i + 1}: M0 written by `{t}`")
                break
            m = re.match(r"s_nop\s+(\w+)", t)
            states += int(m[1], 0) + 1 if m else 1
    return n, bad


def test_copies_take_vector_addresses(asm):
    copies = [x.split(";")[0].strip() for x in asm.splitlines() if x.strip().startswith("global_load_lds")]
    assert len(copies) > 100, "the scan no longer matches the code"
    assert all(re.match(r"global_load_lds_dwordx4\s+v\[\d+:\d+\], off", x) for x in copies)
    assert copy_base_hazards(asm) == (0, [])


def test_m0_is_set_before_copies(asm):
    n, bad = m0_hazards(asm)
    assert n > 100 and not bad, "\n".join(bad[:10])


def test_no_register_of_an_asm_load_touched_early(asm):
    assert not inflight_register_uses(asm)


def test_no_scratch_memory(asm):
    sizes = re.findall(r"\.private_segment_fixed_size:\s*(\d+)", asm)
    assert len(sizes) >= 6 and not any(map(int, sizes))
    assert not re.search(r"^\s*scratch_(load|store)", asm, re.M)


def test_scan_on_small_cases():
    late = "_Zk:\n s_mov_b32 m0, s3\n s_nop 2\n global_load_lds_dwordx4 v[0:1], off\n"
    assert m0_hazards(late) == (1, [])
    assert m0_hazards(late + " global_load_lds_dwordx4 v[2:3], off offset:1024\n") == (2, [])
    assert len(m0_hazards(late.replace("s_nop 2", "s_nop 1"))[1]) == 1
    assert len(m0_hazards(late.replace("s_mov_b32 m0, s3", "v_readfirstlane_b32 m0, v3"))[1]) == 1
    assert len(m0_hazards("_Zk:\n global_load_lds_dwordx4 v[0:1], off\n")[1]) == 1
