"""What the sources of the 4-bit and mixture-of-experts kernels have to say for their machine code to be right."""

import re
from pathlib import Path

import pytest

HIP = Path(__file__).resolve().parent.parent / "minicompiler_amd" / "csrc" / "hip"


@pytest.mark.parametrize("path", sorted([*HIP.glob("*.hip"), *HIP.glob("*.h")]), ids=lambda p: p.name)
def test_dynamic_lds_is_aligned_to_its_widest_access(path):
    """The dynamic part lies behind the static variables, at its own type's alignment: for floats 4 bytes, where the
    compiler takes a vector of four to lie at a multiple of 16."""
    for declaration in re.findall(r"extern\s+__shared__[^;]*;", path.read_text()):
        assert "__attribute__((aligned(16)))" in declaration, declaration
