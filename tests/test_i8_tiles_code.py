"""More of the machine code that hipcc makes of the large tiles of products of 8-bit integers, the gathered ones past 2 GiB
among them: the order of LDS between a wave's lanes, which the compiler is told at each hand-over."""

import re
import subprocess

import pytest

from minicompiler_amd import build

@pytest.fixture(scope="module")
def bodies(tmp_path_factory):
    out = tmp_path_factory.mktemp("code") / "gemm_i8.s"
    cmd = [str(build.ROCM / "bin" / "hipcc"), *build.HIPFLAGS, "--offload-device-only", "-S",
           str(build.CSRC / "hip" / "gemm_i8.hip"), "-o", str(out)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=600)
    found = dict(re.findall(r"^(_Z\w*(?:i8_tiles|i8_far_rows)\w*):[^\n]*\n(.*?)^\.Lfunc_end", out.read_text(), re.M | re.S))
    # Dense and up: three types, gated or not; down: fp32; each with large and small tiles. Past 2 GiB: up, large ones.
    assert len(found) == 2 * (2 * 3 * 2 + 1) + 6
    return {name: body.splitlines() for name, body in found.items()}


def test_lanes_hand_over_in_order(bodies):
    """Behind the products, what a lane writes to LDS is read by others: the compiler has to be told at every turn."""
    for name, lines in bodies.items():
        last, told, turns = "", True, 0
        products = [i for i, line in enumerate(lines) if re.match(r"\s+v_mfma", line)]
        for i, line in enumerate(lines):
            if i and i in products:
                last, told = "", True
            elif re.match(r"\s+; wave barrier|\s+s_barrier", line):
                told = True
            elif m := re.match(r"\s+ds_(read|write)_b(32|64|128)\b", line):
                if last == "write" and m[1] == "read":
                    assert told, (name, i, line)
                    turns += 1
                if m[1] == "write":
                    told = False
                last = m[1]
        assert turns > 0, name
