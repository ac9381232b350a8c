"""Lane exchanges (v_permlane16_swap, v_permlane32_swap, DPP operands) read a vector register two wait states after a vector
instruction wrote it at the earliest.  The compiler keeps them for what it sees; a write inside inline assembly it does not
see.  Compile the kernels that exchange lanes to ISA and count."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
DPP = re.compile(r"_dpp\b|quad_perm:|row_(?:shl|shr|ror|mirror|half_mirror|newbcast|bcast)|wave_(?:shl|shr|rol|ror)")


def registers(text):
    out = set()
    for lo, hi, one in re.findall(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", text):
        out.update([int(one)] if one else range(int(lo), int(hi) + 1))
    return out


def violations(isa):
    """(instruction, wait states) of every lane exchange that reads too early.  A label starts anew: nothing is known of
    what ran before it."""
    written, clock, found, exchanges = {}, 0, [], 0
    for line in isa.splitlines():
        line = line.split(";")[0].strip()
        if not line or line.startswith("."):
            if line.endswith(":"):
                written = {}
            continue
        if line.endswith(":"):
            written = {}
            continue
        op, _, rest = line.partition(" ")
        op = op.strip()
        if op == "s_nop":
            clock += int(rest, 0) + 1
            continue
        if op.startswith("v_"):
            parts = rest.split(",")
            swap = op.startswith("v_permlane")
            if swap or DPP.search(line):
                exchanges += 1
                # a swap reads both of its registers; of a DPP instruction the first source is the one that is exchanged
                for r in registers(rest) if swap else registers(parts[1]):
                    if clock - written.get(r, -8) - 1 < 2:
                        found.append((line, clock - written[r] - 1))
            for part in parts[:2] if swap else parts[:1]:
                for r in registers(part):
                    written[r] = clock
        clock += 1
    return exchanges, found


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
@pytest.mark.parametrize("src", ["bf16_pk.hip", "scan.hip"])
def test_lane_exchanges_wait(src, tmp_path):
    out = tmp_path / (src + ".s")
    subprocess.check_call([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                           "-S", "--cuda-device-only", os.path.join(ROOT, "superresolution_amd", "csrc", src), "-o", str(out)],
                          stderr=subprocess.DEVNULL)
    exchanges, found = violations(out.read_text())
    assert exchanges > 20
    assert not found, found[:5]


def test_counting_of_wait_states():
    early = "\tv_cvt_pk_bf16_f32 v1, v2, v3\n\ts_nop 0\n\tv_permlane16_swap_b32_e32 v0, v1\n"
    late = early.replace("s_nop 0", "s_nop 1")
    dpp = "\tv_add_f32_e32 v1, v2, v3\n\tv_mov_b32_dpp v4, v1 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
    assert violations(early) == (1, [("v_permlane16_swap_b32_e32 v0, v1", 1)])
    assert violations(late) == (1, [])
    assert len(violations(dpp)[1]) == 1 and not violations(dpp.replace("\tv_mov", "\ts_nop 1\n\tv_mov"))[1]
