"""Where lanes that left a branch come back, on the CPU: nothing that they need is copied, or loaded back
from where registers are spilled, in front of the instruction that restores their execution mask
(lanes that had left would not have it).  The search reads over scalar instructions."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "go-darwinml_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
KERNELS = {"k_attn_paged_kv4": "attend4_kernel", "k_attn_paged": "attend_kernel", "k_rope": "rope_kernel",
           "k_logprobs": "stream_kernel", "k_attn_window": "kernel", "k_attn_window_bwd": "kernel"}

COPY = re.compile(r"v_(mov_b32|mov_b64|accvgpr_read|accvgpr_write|accvgpr_mov)\S* [va]\S*, [va][\[\d]")
# What may stand in front of the mask's return without ending the search: scalar instructions that do not
# change the mask or the path, and vector moves.
OVER = re.compile(r"(v_mov|v_accvgpr|v_readlane|v_writelane|s_(?!c?branch|setpc|swappc|endpgm|barrier))")


def lost_values(assembly):
    """(kernel, label) of each block that copies or reloads vector registers, then takes its lanes back."""
    found, kernel, label, lost = [], None, None, None
    for line in assembly.splitlines():
        name = re.match(r"(_Z\S+):", line)
        if name:
            kernel = name[1]
        if line.startswith((".LBB", "; %bb.")):
            label = line.split()[0]
            lost = 0 if line.startswith(".LBB") else None
            continue
        op = line.split(";")[0].strip()
        if not op or op.startswith(".") or lost is None:
            continue
        if op.startswith("s_or_b64 exec, exec"):
            if lost:
                found.append((kernel, label))
            lost = None
        elif "Folded Reload" in line or COPY.match(op):
            lost += 1
        elif not OVER.match(op) or re.match(r"\S+ exec", op):
            lost = None
    return found


def test_the_search_finds_them():
    head, back = "_Zkernel:\n; %bb.1:\n\tv_add_u32 v1, v2, v3\n.LBB0_2:\n", "\ts_or_b64 exec, exec, s[4:5]\n"
    for bad in ("\tv_accvgpr_write_b32 a80, v78\n\ts_mov_b32 s4, s5\n", "\ts_add_u32 s4, s5, 1\n\tv_mov_b32_e32 v3, v7\n\ts_cmp_eq_u32 s4, 0\n",
                "\tscratch_load_dword v1, off, off offset:8 ; 4-byte Folded Reload\n\ts_waitcnt vmcnt(0)\n"):
        assert lost_values(head + bad + back) == [("_Zkernel", ".LBB0_2:")]
    for good in ("", "\tv_mov_b32_e32 v1, 0\n", "\tv_mov_b32_e32 v1, v2\n\tv_add_u32 v1, v1, v3\n", "\tv_mov_b32_e32 v1, v2\n\ts_branch .LBB0_2\n",
                 "\tv_mov_b32_e32 v1, v2\n\ts_mov_b64 exec, s[0:1]\n"):
        assert lost_values(head + good + back) == []
    assert lost_values(head + back + "\tv_accvgpr_write_b32 a80, v78\n") == []


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    """The sources' assembly, compiled side by side."""
    at = tmp_path_factory.mktemp("assembly")
    runs = {k: subprocess.Popen([HIPCC, "--offload-arch=gfx950", "-O3", "-fPIC", "-std=c++17", "-I", os.path.join(ROOT, "include"), "-I", CSRC,
                                 "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "--offload-device-only", "-S",
                                 os.path.join(CSRC, k + ".hip"), "-o", str(at / (k + ".s"))], stderr=subprocess.DEVNULL) for k in KERNELS}
    assert all([r.wait() == 0 for r in runs.values()])
    return {k: (at / (k + ".s")).read_text() for k in KERNELS}


@pytest.mark.parametrize("source", KERNELS)
def test_nothing_is_lost(assembly, source):
    assert KERNELS[source] in assembly[source]
    assert lost_values(assembly[source]) == []


def test_nothing_spills_where_logits_stream(assembly):
    """Log probabilities and the rotation keep their registers."""
    for source in ("k_logprobs", "k_rope"):
        sizes = re.findall(r"\.amdhsa_private_segment_fixed_size (\d+)", assembly[source])
        assert len(sizes) > 10 and set(sizes) == {"0"}
