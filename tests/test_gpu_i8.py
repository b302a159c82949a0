"""8-bit integer operands on the GPU against float64 numpy: quantisation bit for bit (codes, scales, values), products
within the bound of their roundings, at sizes off every tile, strides, types and special values; bytes around the outputs
stay untouched."""

import numpy as np
import pytest

import i8_oracle as ref
from test_gpu_mx4 import Out, bits_type, device_rows, spread

pytestmark = pytest.mark.gpu


def run_quantize(mc, bits, dtype, columns=False, pad=0, values=True, stream=None):
    """codes, scales, values (or None) of bits [rows, k], stored [k, rows] for the column form."""
    rows, k = bits.shape
    stored = np.ascontiguousarray(bits.T) if columns else bits
    x = device_rows(mc, stored, stored.shape[1] + pad)
    codes, scales = Out(mc, mc.i8_code_bytes(rows, k)), Out(mc, rows * 4)
    v = Out(mc, rows * k * (4 if dtype == ref.F32 else 2)) if values else None
    where = v.ptr if v else None
    if columns:
        mc.quantize_i8_columns(dtype, x.ptr, stored.shape[1] + pad, codes.ptr, scales.ptr, k, rows, where, stream)
    else:
        mc.quantize_i8(dtype, x.ptr, k + pad, codes.ptr, scales.ptr, rows, k, where, stream)
    mc.synchronize()
    got = None
    if v:
        got = v.get(bits_type(dtype), stored.shape)
        got = got.T if columns else got
    return codes.get(np.int8, (rows, ref.padded(k))), scales.get(np.float32, rows), got


def check_quantize(mc, x, dtype, **kw):
    bits = ref.to_type(x, dtype)
    k = x.shape[1]
    want = ref.quantize(ref.from_type(bits, dtype))
    codes, scales, values = run_quantize(mc, bits, dtype, **kw)
    assert np.array_equal(scales, want[1], equal_nan=True)
    assert np.array_equal(codes, want[0])
    if values is not None:
        assert np.array_equal(ref.from_type(np.ascontiguousarray(values), dtype),
                              ref.from_type(ref.values(*want, k, dtype), dtype), equal_nan=True)


SIZES = [(1, 1, 0), (1, 4096, 0), (3, 31, 1), (2, 33, 8), (17, 128, 4), (65, 130, 0), (64, 257, 7), (130, 1000, 24),
         (5, 2048, 3), (7, 5000, 1), (3, 14336, 0), (2, 20001, 5), (300, 64, 0), (1, 140000, 0), (1001, 513, 2)]


@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("rows,k,pad", SIZES)
def test_quantize_gives_the_nearest_codes(device, mc, kind, rows, k, pad, columns):
    print(f"case quantize {kind} {rows}x{k} pad {pad} columns {columns}", flush=True)
    rng = np.random.default_rng(rows * 1000 + k)
    low, high = {"f32": (-126, 120), "bf16": (-126, 120), "f16": (-18, 10)}[kind]
    check_quantize(mc, spread(rng, rows, k, low, high), ref.TYPES[kind], columns=columns, pad=pad)


@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("kind", sorted(ref.TYPES))
def test_quantize_ties_zeros_subnormals_and_the_largest(device, mc, kind, columns):
    dtype = ref.TYPES[kind]
    largest = {"f32": np.finfo(np.float32).max, "bf16": float(np.uint32(0x7F7F0000).view(np.float32)), "f16": 65504.0}[kind]
    least = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}[kind]
    n = np.arange(-127, 128)
    # Quotients that are halves exactly (the scale is a power of two), and next to halves.
    ties = [np.r_[127.0, n + 0.5][:256].clip(-127, 127), np.r_[127.0, (n + 0.5) * (1 - 2.0 ** -12)].clip(-127, 127),
            np.r_[127.0, (n + 0.5) * (1 + 2.0 ** -12)].clip(-127, 127)]
    rows = [*ties, ties[0] * 2.0 ** -9, np.zeros(256), np.full(256, -0.0), np.arange(256) * least,
            np.arange(256) * -least * 3, np.r_[np.full(255, 0.0), least], np.r_[np.full(255, 0.0), 50 * least],
            np.r_[np.full(255, least), 63 * least], np.linspace(-1, 1, 256) * largest,
            np.r_[largest, np.full(255, least)], np.r_[np.nan, np.ones(255)], np.r_[np.ones(254), -np.inf, 2.0],
            np.r_[np.full(255, np.inf), np.nan], np.full(256, 3.0)]
    if kind != "f16":
        rows += [np.linspace(-1, 1, 256) * 2.0 ** e for e in (-90, -93, -94, -100, -119, -120, -126, -130)]
    if kind == "f32":
        # Every scale's mantissa rounds, and a quotient lies as near to a half as one may.
        for a in (1.1, 1.7, 1.999999, 1.0000001):
            s = np.float64(np.float32(np.float32(a) / np.float32(127)))
            h = (n[:255] + 0.5) * s
            rows += [np.r_[a, h].clip(-a, a), np.r_[a, np.nextafter(h.astype(np.float32), np.float32(9))].clip(-a, a),
                     np.r_[a, np.nextafter(h.astype(np.float32), np.float32(-9))].clip(-a, a)]
    with np.errstate(over="ignore", invalid="ignore"):
        check_quantize(mc, np.array([r[:256] for r in rows]), dtype, columns=columns)


def test_quantize_without_values_and_on_a_stream(device, mc):
    rng = np.random.default_rng(5)
    s = mc.Stream()
    for columns in (False, True):
        check_quantize(mc, rng.standard_normal((33, 300)), ref.BF16, values=False, columns=columns, stream=s)


# ---------------------------------------------------------------- products


def operand(mc, codes, scales):
    return mc.DeviceBuffer.from_array(np.ascontiguousarray(codes)), mc.DeviceBuffer.from_array(np.asarray(scales, np.float32))


def random_operand(rng, rows, k, most=127):
    codes = np.zeros((rows, ref.padded(k)), dtype=np.int8)
    codes[:, :k] = rng.integers(-most, most + 1, (rows, k))
    return codes, (rng.uniform(0.5, 2.0, rows) / 127 / np.sqrt(k)).astype(np.float32)


def compare(got_bits, want, bound, dtype):
    got = ref.from_type(got_bits, dtype)
    if not got.size:
        return
    off = np.abs(got - want)
    worst = np.unravel_index(np.argmax(off - bound), off.shape)
    assert np.all(off <= bound), f"at {worst}: {got[worst]} for {want[worst]}, bound {bound[worst]}"


def check_product(mc, seed, m, n, k, kind="f32", act=None, bias=False, stream=None):
    rng = np.random.default_rng(seed)
    dtype = ref.TYPES[kind]
    rows = 2 * n if act == "swiglu" else n
    a, sa = random_operand(rng, m, k)
    b, sb = random_operand(rng, rows, k)
    sb *= np.float32(4.0)
    v = rng.standard_normal(rows).astype(np.float32) if bias else None
    want, err = ref.activate(*ref.scaled(a, sa, b, sb, v), act)
    da, db = operand(mc, a, sa), operand(mc, b, sb)
    dv = mc.DeviceBuffer.from_array(v) if bias else None
    c = Out(mc, m * n * (4 if dtype == ref.F32 else 2))
    mc.launch_matmul_i8(da[0].ptr, da[1].ptr, db[0].ptr, db[1].ptr, dv.ptr if bias else None, act, dtype, c.ptr, m, n, k,
                        stream)
    mc.synchronize()
    compare(c.get(bits_type(dtype), (m, n)), want, ref.rounded(want, err, dtype), dtype)


PRODUCTS = [(1, 1, 1), (1, 16, 64), (1, 17, 129), (2, 300, 4096), (3, 100, 8192), (5, 33, 1000), (8, 512, 512),
            (9, 65, 257), (16, 64, 128), (17, 48, 300), (31, 1000, 640), (33, 40, 2000), (64, 129, 384), (65, 64, 1023),
            (100, 1001, 130), (200, 72, 1536), (257, 300, 520), (300, 257, 1025)]


@pytest.mark.parametrize("act", ref.ACTS)
@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(device, mc, kind, m, n, k, act):
    print(f"case product {kind} {m}x{n}x{k} {act}", flush=True)
    check_product(mc, m + n + k, m, n, k, kind, act, bias=(m + n) % 2 == 0)


@pytest.mark.parametrize("m,n,k,act", [(512, 1024, 512, None), (777, 1500, 1000, "swiglu"), (1025, 513, 600, "relu"),
                                       (2048, 2056, 256, None), (1030, 4104, 384, "gelu"), (2100, 1100, 640, "swiglu")])
@pytest.mark.parametrize("kind", sorted(ref.TYPES))
def test_product_of_many_tiles(device, mc, kind, m, n, k, act):
    print(f"case product {kind} {m}x{n}x{k} {act}", flush=True)
    check_product(mc, m + n, m, n, k, kind, act, bias=act is not None)


# Each kernel by sizes that its rule gives it: blocks of 16x32, 32x32 and 32x64, tiles of 128x128 and of 256x256 (whole
# rounds, halves, short last rows), every activation and type, columns that are and are not eights, short k.
VARIANTS = [(16, 1056, 512), (32, 4104, 200), (60, 4099, 300), (128, 4096, 130), (250, 4090, 260), (600, 4104, 384),
            (640, 4100, 129), (1025, 2056, 256), (1100, 2049, 1100), (4000, 4090, 128), (3850, 4096, 600), (6100, 4096, 1000)]


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("m,n,k", VARIANTS)
def test_product_by_every_kernel(device, mc, kind, m, n, k):
    for act in (ref.ACTS[(m + sorted(ref.TYPES).index(kind)) % 3], "swiglu"):
        print(f"case kernel {kind} {m}x{n}x{k} {act}", flush=True)
        check_product(mc, m + n + k, m, n // 2 if act == "swiglu" else n, k, kind, act, bias=n % 2 == 0)


def test_columns_of_b_past_32_bits(device, mc):
    """B of 2.2 GB: the last columns' offsets pass 2^31."""
    m, n, k = 20, 17500, 131000
    kp = ref.padded(k)
    rng = np.random.default_rng(2)
    b = mc.DeviceBuffer(n * kp)
    b.fill_bytes(0)
    mc.synchronize()
    last = rng.integers(-127, 128, (64, kp)).astype(np.int8)
    last[:, k:] = 0
    assert mc.library().mc_memcpy_htod(b.ptr + (n - 64) * kp, last.ctypes.data, last.nbytes) == 0
    sb = np.ones(n, dtype=np.float32)
    a, sa = random_operand(rng, m, k, 20)
    da, ds = operand(mc, a, sa), mc.DeviceBuffer.from_array(sb)
    c = Out(mc, m * n * 4)
    mc.launch_matmul_i8(da[0].ptr, da[1].ptr, b.ptr, ds.ptr, None, None, 0, c.ptr, m, n, k)
    mc.synchronize()
    got = c.get(np.float32, (m, n))
    want, err = ref.scaled(a, sa, last, sb[-64:], None)
    assert np.all(got[:, :-64] == 0)
    assert np.all(np.abs(got[:, -64:] - want) <= ref.rounded(want, err, ref.F32))


@pytest.mark.parametrize("m", [1, 20, 300])
def test_sums_at_the_end_of_32_bits(device, mc, m):
    """k = 131071 codes of -128 (never quantised, but codes) and 127: sums up to 2147467264."""
    k, n = 131071, 24
    a = np.zeros((m, ref.padded(k)), dtype=np.int8)
    b = np.zeros((n, ref.padded(k)), dtype=np.int8)
    a[:, :k] = -128
    a[::2, :k] = 127
    b[:, :k] = -128
    b[1::2, :k] = 127
    one = np.float32(1.0)
    da, db = operand(mc, a, np.full(m, one)), operand(mc, b, np.full(n, one))
    c = Out(mc, m * n * 4)
    mc.launch_matmul_i8(da[0].ptr, da[1].ptr, db[0].ptr, db[1].ptr, None, None, 0, c.ptr, m, n, k)
    mc.synchronize()
    line_a, line_b = a[:, 0].astype(np.int64), b[:, 0].astype(np.int64)
    want = (np.outer(line_a, line_b) * k).astype(np.float32)
    assert np.array_equal(c.get(np.float32, (m, n)), want)


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("act", ref.ACTS)
def test_rows_and_columns_that_are_no_numbers(device, mc, m, act):
    """A NaN scale (a row with an infinity) makes its row or column of C NaN and nothing else."""
    rng = np.random.default_rng(m)
    n, k = 50, 300
    rows = 2 * n if act == "swiglu" else n
    a, sa = random_operand(rng, m, k)
    b, sb = random_operand(rng, rows, k)
    sa[m // 2], sb[7] = np.nan, np.nan
    da, db = operand(mc, a, sa), operand(mc, b, sb)
    c = Out(mc, m * n * 4)
    mc.launch_matmul_i8(da[0].ptr, da[1].ptr, db[0].ptr, db[1].ptr, None, act, 0, c.ptr, m, n, k)
    mc.synchronize()
    want = np.zeros((m, n), dtype=bool)
    want[m // 2], want[:, 7] = True, True
    assert np.array_equal(np.isnan(c.get(np.float32, (m, n))), want)
