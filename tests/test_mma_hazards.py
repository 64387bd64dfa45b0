"""The built code of the 8-bit products keeps the distance between a matrix instruction and the
use of its result (CPU: compiles to assembly, runs nothing).

The vector unit may read the result of v_mfma_f32_16x16x128_f8f6f4 12 wait states after it was
issued (16x16x32 in bf16: 8). The compiler fills up with s_nop inside a block of
instructions; across a branch it was seen to leave too few. So every block has to keep the
distance by itself: each read of a result by another than a matrix instruction, and the end
of the block, come late enough after it."""

from __future__ import annotations

import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "reframework_amd",
                    "csrc")
WAIT = {"v_mfma_f32_16x16x128_f8f6f4": 12, "v_mfma_f32_16x16x32_bf16": 8}


def assembly(source, tmp_path):
    out = tmp_path / (source + ".s")
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    subprocess.run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Xclang",
                    "-target-feature", "-Xclang", "-packed-fp32-ops", "-S", "--cuda-device-only",
                    os.path.join(CSRC, source), "-o", str(out)], check=True, capture_output=True)
    return out.read_text()


def registers(text):
    found = set()
    for k, a, b in re.findall(r"\b([va])\[(\d+):(\d+)\]", text):
        found.update((k, r) for r in range(int(a), int(b) + 1))
    found.update((k, int(r)) for k, r in re.findall(r"\b([va])(\d+)\b", text))
    return found


def broken(text):
    """Lines that come too early after a matrix instruction."""
    bad, pending, mmas = [], {}, 0  # register -> wait states that are still missing
    for line in text.splitlines():
        code = line.split(";")[0].strip()
        if not code or (code.startswith(".") and not code.endswith(":")):
            continue
        if code.endswith(":") or code.startswith(("s_cbranch", "s_branch", "s_endpgm", "s_setpc")):
            # the branch itself is one wait state
            if any(n > 1 for n in pending.values()):
                bad.append(line)
            pending = {}
            continue
        name, _, rest = code.partition(" ")
        mma = name.startswith("v_mfma")
        if not mma and any(r in pending for r in registers(rest)):
            bad.append(line)
        step = int(rest, 0) + 1 if name == "s_nop" else 1
        pending = {r: n - step for r, n in pending.items() if n > step}
        if mma:
            mmas += 1
            pending.update({r: WAIT[name] for r in registers(rest.split(",")[0])})
    return bad, mmas


@pytest.mark.parametrize("source", ["fp8_stream.hip", "fp8_tiled.hip"])
def test_results_are_read_late_enough(source, tmp_path):
    bad, mmas = broken(assembly(source, tmp_path))
    assert mmas > 16 and not bad, bad[:5]


def test_the_check_finds_an_early_read():
    mma = "\tv_mfma_f32_16x16x128_f8f6f4 v[56:59], v[16:23], v[8:15], 0"
    read = "\tv_fmac_f32_e32 v40, v56, v106"
    assert not broken("\n".join([mma, "\ts_nop 11", read]))[0]
    assert broken("\n".join([mma, "\ts_nop 10", read]))[0]
    assert broken("\n".join([mma, "\ts_cbranch_vccnz .L1", "\ts_nop 11", read]))[0]
    assert broken("\n".join([mma, "\ts_nop 4", ".L1:", "\ts_nop 11", read]))[0]
