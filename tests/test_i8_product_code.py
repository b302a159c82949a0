"""The machine code that hipcc makes of the large tiles of products of 8-bit integers. As in the tiles of 4-bit products,
their matrix instructions are written out as assembly, so the compiler does not know what they need around them; and
their fetches have to come from scalar registers, or the compiler tries each lane's resource in a loop."""

import re
import subprocess

import pytest

from minicompiler_amd import build
from test_mx4_product_code import Code, faults, is_product, operands


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    out = tmp_path_factory.mktemp("code") / "gemm_i8.s"
    cmd = [str(build.ROCM / "bin" / "hipcc"), *build.HIPFLAGS, "--offload-device-only", "-S",
           str(build.CSRC / "hip" / "gemm_i8.hip"), "-o", str(out)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=600)
    bodies = re.findall(r"^(_Z\w*i8_tiles\w*):[^\n]*\n(.*?)^\.Lfunc_end", out.read_text(), re.M | re.S)
    return {name: Code(body.splitlines()) for name, body in bodies}


def test_products_have_their_operands_and_time(kernels):
    # Dense and up: three types, gated or not; down: fp32; each with large and small tiles.
    assert len(kernels) == 2 * (2 * 3 * 2 + 1)
    for name, code in kernels.items():
        products = [rest for op, rest in code.ops if is_product(op)]
        # Four steps: of 256x256 and of 128x256, or of 128x128; every product adds in place.
        assert len(products) in (4 * (4 * 4 + 2 * 4), 4 * 2 * 2), name
        assert all(operands(rest)[0] == operands(rest)[3] for rest in products), name
        assert not faults(code), (name, faults(code)[:5])


def test_fetches_need_no_loop_over_lanes(kernels):
    """A resource in vector registers is compared with the first lane's, in a loop, around every use."""
    for name, code in kernels.items():
        assert any(op.startswith("buffer_load") and "lds" in rest for op, rest in code.ops), name
        assert not any(op.startswith("v_cmp_eq_u64") for op, _ in code.ops), name
