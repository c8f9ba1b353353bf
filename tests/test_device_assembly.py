"""What the compiler makes of decoding over 4 bits, on the CPU.  Where lanes that left a branch come
back, their execution mask is restored by an instruction at the block's beginning; the register
allocator has put copies of registers in front of it (f16, head dim 256, when addresses were
chosen in a branch), which the lanes that had left then do not have."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "go-darwinml_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

COPY = re.compile(r"v_(mov_b32|mov_b64|accvgpr_read|accvgpr_write|accvgpr_mov)\S* [va]\S*, [va][\[\d]")
SMALL = re.compile(r"(v_mov|v_accvgpr|s_mov|s_nop|v_readlane|v_writelane|s_waitcnt)")


def lost_copies(assembly):
    """(kernel, label) of each block that copies vector registers and then takes its lanes back."""
    found, kernel, label, copies = [], None, None, None
    for line in assembly.splitlines():
        name = re.match(r"(_Z\S+):", line)
        if name:
            kernel = name[1]
        if line.startswith((".LBB", "; %bb.")):
            label = line.split()[0]
            copies = 0 if line.startswith(".LBB") else None
            continue
        op = line.split(";")[0].strip()
        if not op or op.startswith(".") or copies is None:
            continue
        if op.startswith("s_or_b64 exec, exec"):
            if copies:
                found.append((kernel, label))
            copies = None
        elif SMALL.match(op):
            copies += bool(COPY.match(op))
        else:
            copies = None
    return found


def test_the_search_finds_one():
    bad = "_Zkernel:\n; %bb.1:\n\tv_add_u32 v1, v2, v3\n.LBB0_2:\n\tv_accvgpr_write_b32 a80, v78\n\ts_mov_b32 s4, s5\n\ts_or_b64 exec, exec, s[4:5]\n"
    assert lost_copies(bad) == [("_Zkernel", ".LBB0_2:")]
    good = "_Zkernel:\n.LBB0_2:\n\ts_or_b64 exec, exec, s[4:5]\n\tv_accvgpr_write_b32 a80, v78\n.LBB0_3:\n\tv_mov_b32_e32 v1, 0\n\ts_or_b64 exec, exec, s[4:5]\n"
    assert lost_copies(good) == []


@pytest.mark.parametrize("source", ["k_attn_paged_kv4"])
def test_no_copies_are_lost(tmp_path, source):
    out = tmp_path / "kernels.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-fPIC", "-std=c++17", "-I", os.path.join(ROOT, "include"), "-I", CSRC,
                    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "--offload-device-only", "-S",
                    os.path.join(CSRC, source + ".hip"), "-o", str(out)], check=True, capture_output=True)
    text = out.read_text()
    assert text.count("attend4_kernel") > 0
    assert lost_copies(text) == []
