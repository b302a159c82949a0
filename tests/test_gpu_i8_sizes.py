"""8-bit integer operators on the GPU against float64 at sizes that change how they work: many rows of every length, more
rows and columns than one launch takes, rows of C of which 256 pass 2 GiB, and a part of the experts' products each rank
would run."""

import numpy as np
import pytest

import i8_oracle as ref
from test_gpu_experts_i8 import check_up
from test_gpu_i8 import check_quantize, compare, operand, random_operand
from test_gpu_mx4 import Out

pytestmark = pytest.mark.gpu


# 1024 rows and more take as few lanes each as hold one: a wave for up to 2048 numbers, a block for up to 8192.
@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("rows,k,pad", [(1030, 500, 0), (1030, 520, 3), (1100, 1024, 0), (1027, 1025, 1), (1030, 2048, 0),
                                        (1026, 2050, 0), (1025, 4090, 6), (1030, 4097, 0), (1024, 8192, 8), (1025, 8200, 0)])
def test_many_rows_of_every_length(device, mc, kind, rows, k, pad):
    print(f"case many rows {kind} {rows}x{k}", flush=True)
    rng = np.random.default_rng(k)
    check_quantize(mc, rng.standard_normal((rows, k)) * np.exp(rng.standard_normal((rows, 1)) * 3), ref.TYPES[kind], pad=pad)


@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("rows", [(1 << 21) + 3, (1 << 22) + 5])
def test_more_rows_than_a_launch_takes(device, mc, rows, columns):
    print(f"case rows {rows} columns {columns}", flush=True)
    rng = np.random.default_rng(rows)
    k = 3
    bits = rng.integers(0, 1 << 16, (rows, k), dtype=np.uint16)
    bits[(bits & 0x7C00) == 0x7C00] = 0x3C01  # numbers all
    x = mc.DeviceBuffer.from_array(np.ascontiguousarray(bits.T) if columns else bits)
    codes, scales, values = Out(mc, mc.i8_code_bytes(rows, k)), Out(mc, rows * 4), Out(mc, rows * k * 2)
    if columns:
        mc.quantize_i8_columns(ref.F16, x.ptr, rows, codes.ptr, scales.ptr, k, rows, values.ptr)
    else:
        mc.quantize_i8(ref.F16, x.ptr, k, codes.ptr, scales.ptr, rows, k, values.ptr)
    mc.synchronize()
    got = codes.get(np.int8, (rows, 128))
    want = ref.quantize(ref.from_type(bits, ref.F16))
    assert np.array_equal(scales.get(np.float32, rows), want[1])
    assert np.array_equal(got[:, :k], want[0][:, :k]) and not got[:, k:].any()
    back = values.get(np.uint16, (k, rows) if columns else (rows, k))
    # Codes of 0 stand for +0, whatever the sign was.
    assert np.array_equal(back.T if columns else back, ref.values(*want, k, ref.F16))


@pytest.mark.parametrize("k", [100, 256])  # on tiles of 128x128 and of 256x256
@pytest.mark.parametrize("act", [None, "swiglu"])
def test_long_rows_of_c(device, mc, k, act):
    print(f"case long rows {k} {act}", flush=True)
    rng = np.random.default_rng(k)
    m, n = 140, (1 << 21) + 8
    rows = 2 * n if act else n
    a, sa = random_operand(rng, m, k)
    b = np.zeros((rows, ref.padded(k)), dtype=np.int8)
    b[:, :k] = np.frombuffer(rng.bytes(rows * k), dtype=np.int8).reshape(rows, k)
    sb = (rng.uniform(0.5, 2.0, rows) * 4 / 127 / np.sqrt(k)).astype(np.float32)
    da, db = operand(mc, a, sa), operand(mc, b, sb)
    c = Out(mc, m * n * 4)
    mc.launch_matmul_i8(da[0].ptr, da[1].ptr, db[0].ptr, db[1].ptr, None, act, ref.F32, c.ptr, m, n, k)
    mc.synchronize()
    got = c.get(np.float32, (m, n))
    # All of the ends, and parts between them.
    for at in (0, 1 << 18, n // 2 - 999, n - 70000):
        part = np.r_[at:at + 70000]
        part = np.r_[part, part + n] if act else part
        want, err = ref.activate(*ref.scaled(a, sa, b[part], sb[part], None), act)
        compare(got[:, at:at + 70000], want, ref.rounded(want, err, ref.F32), ref.F32)


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("tokens", [5, 130, 2100])
def test_each_ranks_part_of_the_first_product(device, mc, kind, tokens):
    """Experts by twos, as four ranks would hold them: each call's slots right, and the others' left alone."""
    for first in range(0, 8, 2):
        check_up(mc, tokens, tokens, 8, 3, 264, 384, kind, "swiglu", part=(first, first + 2))
