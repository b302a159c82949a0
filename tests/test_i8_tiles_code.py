"""More of the machine code that hipcc makes of the large tiles of products of 8-bit integers, the gathered ones past 2 GiB
among them: what the waits that are counted by hand count, no spilled registers, and the order of LDS between a wave's
lanes, which the compiler is told at each hand-over."""

import re
import subprocess

import pytest

from minicompiler_amd import build
from test_mx4_product_code import Code, faults, is_product, operands

FETCH = re.compile(r"^(buffer_load_dword\w*|global_load_lds_dword\w*)$")
MEMORY = re.compile(r"^(global|buffer|scratch|flat)_")


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


def is_fetch(name, rest):
    return bool(FETCH.match(name)) and ("lds" in name or rest.split()[-1] == "lds")


def loops(code):
    """(first, last) instruction of each loop that multiplies."""
    found = []
    for at, back in enumerate(code.back):
        for end in back:
            if end >= at and any(is_product(code.ops[i][0]) for i in range(at, end + 1)):
                found.append((at, end))
    return found


def of_tile(code, first, last):
    """Fetches of A and of B that a wave issues for each stage, by the loop's products: 4 x 16, 4 x 8 or 4 x 4."""
    products = sum(is_product(code.ops[i][0]) for i in range(first, last + 1))
    return {64: (8, 8), 32: (4, 8), 16: (4, 4)}[products]


def test_the_tiles_spill_nothing(bodies):
    for name, lines in bodies.items():
        assert not any("scratch_" in line for line in lines), name


def test_a_stage_fetches_what_its_wait_counts(bodies):
    for name, lines in bodies.items():
        code = Code(lines)
        found = loops(code)
        assert len(found) == (1 if re.search(r"ELi128EEEv", name) else 2), name
        for first, last in found:
            a, b = of_tile(code, first, last)
            ops = code.ops[first:last + 1]
            assert sum(is_fetch(*op) for op in ops) == a + b, name
            assert all(is_fetch(*op) for op in ops if MEMORY.match(op[0])), name
            waits = [m[1] for op, rest in ops if op == "s_waitcnt" for m in [re.search(r"vmcnt\((\d+)\)", rest)] if m]
            assert waits == [str(b)], name
            # Before the loop: all but B's second stage and the half of what comes after that.
            start = first
            while not (code.ops[start][0] == "s_waitcnt" and "vmcnt" in code.ops[start][1]):
                start -= 1
            assert f"vmcnt({b + (a + b) // 2})" in code.ops[start][1], name
            fetched, at = 0, start - 1
            while fetched < a + 2 * b + (a + b) // 2:
                if MEMORY.match(code.ops[at][0]):
                    assert is_fetch(*code.ops[at]), (name, code.ops[at])
                    fetched += 1
                at -= 1


def test_products_past_2_gib_have_their_operands_and_time(bodies):
    far = {name: Code(lines) for name, lines in bodies.items() if "i8_far_rows" in name}
    assert len(far) == 6
    for name, code in far.items():
        products = [rest for op, rest in code.ops if is_product(op)]
        assert len(products) == 4 * (4 * 4 + 2 * 4), name
        assert all(operands(rest)[0] == operands(rest)[3] for rest in products), name
        assert not faults(code), (name, faults(code)[:5])
        # A's by addresses, B's through a resource in scalar registers.
        assert sum(op.startswith("global_load_lds") for op, _ in code.ops) == 3 * (8 + 4), name  # two stages ahead, one in the loop
        assert not any(op.startswith("v_cmp_eq_u64") for op, _ in code.ops), name


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
