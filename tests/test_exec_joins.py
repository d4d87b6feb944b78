"""The assembly of the 8-bit cache's kernels, searched for vector instructions that run
while no lane is switched on.

Where lanes of a wave part, the compiler lets some of them wait: a branch or a loop is
left with no lane on (exec is 0), and the block behind it switches them on again
(s_or_b64 exec). A copy that saves a register and stands before that does nothing, and
what is read back later is whatever lay there. The compiler has put such copies behind a
loop of `f8_rows` (heads of 256), whose form was changed; this notices it where another
compiler, or another form, brings them back.
"""

from __future__ import annotations

import importlib.util
import re
import subprocess
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parent.parent
_spec = importlib.util.spec_from_file_location("pth_build", REPO / "pth-flash-attn_amd" / "build.py")
build = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(build)


def joins(text):
    """(number of places where a wave goes on with exec possibly 0, [(kernel, line,
    instruction)] of vector instructions there before exec is set again)."""
    lines = text.splitlines()
    targets = {x.split(";")[0].split()[-1] for x in lines if "s_cbranch_execz" in x}
    kernel, number, found, pending, empty = "", 0, [], [], False
    for i, line in enumerate(lines, 1):
        if m := re.match(r"(_Z\w+):", line):
            kernel, empty = m.group(1), False
            continue
        if m := re.match(r"(\.LBB\w+):", line):
            if m.group(1) in targets:
                number, pending, empty = number + 1, [], True
            continue
        t = line.split(";")[0].strip()
        if not t or t.startswith(".") or t.endswith(":"):
            continue
        if empty and ("exec" in t or t.startswith(("s_cbranch", "s_branch", "s_endpgm"))):
            if t.startswith("s_or_b64 exec"):
                found += pending
            empty = False
        elif empty and not t.startswith(("s_", "v_readlane", "v_writelane", "v_readfirstlane")):
            pending.append((kernel, i, t))
        if t.startswith("s_cbranch_execnz"):  # the loop's end
            number, pending, empty = number + 1, [], True
    return number, found


def test_the_search():
    """Copies behind a loop, and in a block that a branch without lanes goes to, are
    found; those behind the restored exec are not."""
    planted = """_Z6kernelv:
.LBB0_1:
    v_add_u32_e32 v1, 1, v1
    s_andn2_b64 exec, exec, s[2:3]
    s_cbranch_execnz .LBB0_1
    v_accvgpr_write_b32 a3, v5
    s_or_b64 exec, exec, s[4:5]
    v_accvgpr_write_b32 a4, v6
    s_cbranch_execz .LBB0_2
    ds_read_b32 v7, v8
.LBB0_2:
    v_writelane_b32 v9, s1, 0
    v_mov_b32_e32 v2, v3
    s_or_b64 exec, exec, s[6:7]
"""
    number, found = joins(planted)
    assert number == 2
    assert [t.split()[0] for _, _, t in found] == ["v_accvgpr_write_b32", "v_mov_b32_e32"]
    clean = "\n".join(x for x in planted.splitlines() if "a3" not in x and "v_mov" not in x)
    assert joins(clean) == (2, [])


@pytest.mark.skipif(not Path(build.HIPCC).is_file(), reason="needs hipcc")
@pytest.mark.parametrize("source", ["fp8_rows.hip", "fp8_wide.hip", "fp8_writer.hip", "p16_combine.hip",
                                    "rotary.hip"])
def test_kernels(source, tmp_path):
    out = tmp_path / "kernels.s"
    subprocess.run([build.HIPCC, *build.DEVICE_FLAGS, f"-I{build.INCLUDE}", f"-I{build.CSRC}", "-S",
                    "--cuda-device-only", str(build.CSRC / source), "-o", str(out)],
                   check=True, capture_output=True, timeout=600)
    number, found = joins(out.read_text())
    assert number > 0
    assert not found, found[:4]
