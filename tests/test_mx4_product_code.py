"""The machine code that hipcc makes of the large-tile product of two mx4 operands. Its products are written out as
assembly, so the compiler does not know what they need around them: a vector instruction's result is there for a
product two instructions later at the earliest, and a product's for another instruction after its passes. The file is
compiled as the library is, and every path of the kernels' code looked through."""

import re
import subprocess

import pytest

from minicompiler_amd import build

BEFORE = 2   # wait states between a vector instruction that writes a register and a product that reads it
AFTER = 18   # ... between a product and anything else that touches its sums


class Code:
    """One kernel's instructions: (mnemonic, operands), and the instructions that each may follow."""

    def __init__(self, lines):
        self.ops, self.back, labels, jumps = [], [], {}, []
        for line in lines:
            line = re.split(r";|//", line)[0].strip()
            if re.match(r"^[.\w$]+:$", line):
                labels[line[:-1]] = len(self.ops)
            elif line and not line.startswith("."):
                name, _, rest = line.partition(" ") if " " in line else line.partition("\t")
                for op in (name + " " + rest).split("\n"):
                    self.ops.append((name, rest.strip()))
                if name.startswith(("s_branch", "s_cbranch")):
                    jumps.append((len(self.ops) - 1, rest.strip()))
        ends = ("s_branch", "s_endpgm", "s_setpc")
        self.back = [[i - 1] if i and not self.ops[i - 1][0].startswith(ends) else [] for i in range(len(self.ops))]
        for at, label in jumps:
            self.back[labels[label]].append(at)

    def earlier(self, i, states):
        """Instructions that run fewer than `states` wait states before instruction i, on any path."""
        found, todo = set(), [(p, 0) for p in self.back[i]]
        least = {}
        while todo:
            p, passed = todo.pop()
            if passed >= states or least.get(p, states) <= passed:
                continue
            least[p] = passed
            found.add(p)
            name, rest = self.ops[p]
            here = int(rest, 0) + 1 if name == "s_nop" else 1
            todo += [(q, passed + here) for q in self.back[p]]
        return found


def registers(operand):
    """{"v12", ...} of one operand."""
    m = re.match(r"^-?\|?([va])(?:(\d+)|\[(\d+):(\d+)\])", operand.strip())
    if not m:
        return set()
    lo = int(m[2] or m[3])
    return {m[1] + str(r) for r in range(lo, int(m[2] or m[4]) + 1)}


def operands(rest):
    return re.findall(r"-?\|?[\w.]+(?:\[[^\]]*\])?(?::\[[^\]]*\])?\|?", rest)


def is_product(name):
    return name.startswith(("v_mfma", "v_smfma"))


def written(name, rest):
    """Registers that a vector instruction (of no memory) writes."""
    if not name.startswith("v_") or is_product(name):
        return set()
    parts = operands(rest)
    two = "swap" in name
    return set().union(*(registers(p) for p in parts[:2 if two else 1]))


def faults(code):
    """What comes too early, as text."""
    out = []
    for i, (name, rest) in enumerate(code.ops):
        parts = operands(rest)
        if is_product(name):
            read = set().union(*(registers(p) for p in parts[1:6]))
            for p in code.earlier(i, BEFORE):
                if written(*code.ops[p]) & read:
                    out.append(f"{code.ops[p]} before {code.ops[i]}")
        else:
            touched = {r for p in parts for r in registers(p) if r[0] == "a"}
            if not touched:
                continue
            for p in code.earlier(i, AFTER):
                if is_product(code.ops[p][0]) and registers(operands(code.ops[p][1])[0]) & touched:
                    out.append(f"{code.ops[i]} after {code.ops[p]}")
    return out


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    out = tmp_path_factory.mktemp("code") / "gemm_mx4.s"
    cmd = [str(build.ROCM / "bin" / "hipcc"), *build.HIPFLAGS, "--offload-device-only", "-S",
           str(build.CSRC / "hip" / "gemm_mx4.hip"), "-o", str(out)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=300)
    text = out.read_text()
    bodies = re.findall(r"^(_Z\w*product_tiles\w*):[^\n]*\n(.*?)^\.Lfunc_end", text, re.M | re.S)
    return {name: Code(body.splitlines()) for name, body in bodies}


def test_products_have_their_operands_and_time(kernels):
    assert len(kernels) == 3
    for name, code in kernels.items():
        products = [rest for op, rest in code.ops if is_product(op)]
        # Two tile heights, two stages of two steps, and every one adds in place.
        assert len(products) == 4 * 8 * 8 + 4 * 4 * 8, name
        assert all(operands(rest)[0] == operands(rest)[3] for rest in products), name
        assert not faults(code), (name, faults(code)[:5])


HEAD = "\tv_mfma_scale_f32_16x16x128_f8f6f4 a[4:7], v[8:11], v[12:15], a[4:7], v20, v21 op_sel_hi:[0,0,0] cbsz:4 blgp:4"


@pytest.mark.parametrize("lines,count", [
    (["\tv_mov_b32_e32 v20, v1", "\ts_nop 1", HEAD], 0),
    (["\tv_mov_b32_e32 v20, v1", "\ts_nop 0", HEAD], 1),
    (["\tv_mov_b32_e32 v20, v1", HEAD], 1),
    (["\tv_mov_b32_e32 v22, v20", HEAD], 0),
    (["\tv_permlane16_swap_b32 v1, v9", HEAD], 1),
    (["\tds_read_b128 v[8:11], v1", "\ts_waitcnt lgkmcnt(0)", HEAD], 0),
    ([".LBB0_1:", HEAD, "\tv_add_u32_e32 v21, 1, v21", "\ts_cbranch_scc1 .LBB0_1", "\ts_endpgm"], 1),
    ([HEAD, "\ts_nop 15", "\ts_nop 0", "\tv_accvgpr_read_b32 v0, a5"], 1),
    ([HEAD, "\ts_nop 15", "\ts_nop 1", "\tv_accvgpr_read_b32 v0, a5"], 0),
    ([HEAD, "\tv_accvgpr_read_b32 v0, a8"], 0),
    (["\tv_accvgpr_write_b32 a4, 0", HEAD], 1)])
def test_the_search_finds_what_is_too_early(lines, count):
    assert len(faults(Code(lines))) == count
