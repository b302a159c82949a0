"""Microscaled 4-bit operands on the GPU against float64 numpy: quantisation bit for bit (codes, scales, values),
products within the bound of fp32 sums of exact products, at sizes off every tile, strides, types, special values and
offsets past 32 bits; bytes around the outputs stay untouched."""

import numpy as np
import pytest

import mx4_oracle as ref

pytestmark = pytest.mark.gpu

GUARD = 256
FILL = 0xAB


class Out:
    """A device array of `nbytes` bytes between two guards."""

    def __init__(self, mc, nbytes):
        self.mc, self.nbytes = mc, nbytes
        self.buf = mc.DeviceBuffer(nbytes + 2 * GUARD)
        self.buf.fill_bytes(FILL)
        self.ptr = self.buf.ptr + GUARD

    def get(self, dtype, shape):
        raw = self.buf.download(np.uint8)
        assert np.all(raw[:GUARD] == FILL) and np.all(raw[GUARD + self.nbytes:] == FILL), "a write outside the output"
        return raw[GUARD:GUARD + self.nbytes].view(dtype).reshape(shape)


def bits_type(dtype):
    return np.float32 if dtype == ref.F32 else np.uint16


def device_rows(mc, bits, ld):
    """The rows in a buffer with ld elements between them, NaN in the gaps."""
    rows, k = bits.shape
    wide = np.full((rows, ld), np.nan if bits.dtype == np.float32 else 0x7FFF, dtype=bits.dtype)
    wide[:, :k] = bits
    return mc.DeviceBuffer.from_array(wide.reshape(-1)[:(rows - 1) * ld + k])


def run_quantize(mc, bits, dtype, columns=False, pad=0, values=True, stream=None):
    """codes, scales, values (or None) of bits [rows, k], stored [k, rows] for the column form."""
    rows, k = bits.shape
    stored = np.ascontiguousarray(bits.T) if columns else bits
    x = device_rows(mc, stored, stored.shape[1] + pad)
    size = 4 if dtype == ref.F32 else 2
    codes, scales = Out(mc, mc.mx4_code_bytes(rows, k)), Out(mc, mc.mx4_scale_bytes(rows, k))
    v = Out(mc, rows * k * size) if values else None
    where = v.ptr if v else None
    if columns:
        mc.quantize_mx4_columns(dtype, x.ptr, stored.shape[1] + pad, codes.ptr, scales.ptr, k, rows, where, stream)
    else:
        mc.quantize_mx4(dtype, x.ptr, k + pad, codes.ptr, scales.ptr, rows, k, where, stream)
    mc.synchronize()
    kp = ref.padded(k)
    got_v = None
    if v:
        got_v = v.get(bits_type(dtype), stored.shape)
        got_v = got_v.T if columns else got_v
    return codes.get(np.uint8, (rows, kp // 2)), scales.get(np.uint8, (rows, kp // 32)), got_v


def check_quantize(mc, x, dtype, **kw):
    bits = ref.to_type(x, dtype)
    want = ref.quantize(ref.from_type(bits, dtype))
    codes, scales, values = run_quantize(mc, bits, dtype, **kw)
    assert np.array_equal(scales, want[1])
    assert np.array_equal(codes, want[0])
    if values is not None:
        assert np.array_equal(ref.from_type(np.ascontiguousarray(values), dtype), want[2], equal_nan=True)


def spread(rng, rows, k, low, high):
    """Values over many binary orders, blocks of very different size."""
    x = rng.standard_normal((rows, k)) * 2.0 ** rng.integers(-3, 4, (rows, k))
    return x * 2.0 ** rng.integers(low, high, (rows, 1))


@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("rows,k,pad", [(1, 1, 0), (1, 4096, 0), (3, 31, 1), (2, 33, 8), (17, 128, 4), (65, 130, 0),
                                        (64, 257, 7), (130, 1000, 24), (5, 2048, 3)])
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
    halves = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 6.0, 4.0, 3.0, 2.0, 1.5, 1.0, 0.5, 0.0])
    rows = [np.concatenate([halves, -halves]), np.concatenate([halves, -halves]) * 2.0 ** -9, np.zeros(32),
            np.full(32, -0.0), np.arange(32) * least, np.arange(32) * -least * 3, np.linspace(-1, 1, 32) * largest,
            np.r_[largest, np.full(31, least)], np.r_[np.nan, np.ones(31)], np.r_[np.ones(30), -np.inf, 2.0],
            np.r_[np.full(31, 1.0), np.nextafter(np.float32(8), 0)]]
    if kind != "f16":
        rows += [np.linspace(-1, 1, 32) * 2.0 ** e for e in (-126, -125, -124, -123, -127, -130)]
    with np.errstate(over="ignore", invalid="ignore"):
        check_quantize(mc, np.array(rows), dtype, columns=columns)


def test_quantize_without_values_and_on_a_stream(device, mc):
    rng = np.random.default_rng(5)
    s = mc.Stream()
    check_quantize(mc, rng.standard_normal((33, 300)), ref.BF16, values=False, stream=s)
    check_quantize(mc, rng.standard_normal((33, 300)), ref.BF16, values=False, columns=True, stream=s)


def upload_at(mc, buf, offset, a):
    a = np.ascontiguousarray(a)
    rc = mc.library().mc_memcpy_htod(buf.ptr + offset, a.ctypes.data, a.nbytes)
    assert rc == 0


def test_quantize_rows_more_than_4_gib_apart(device, mc):
    rows, k, ld = 3, 200, (1 << 31) + 40
    rng = np.random.default_rng(6)
    bits = ref.to_type(rng.standard_normal((rows, k)), ref.BF16)
    x = mc.DeviceBuffer(2 * ((rows - 1) * ld + k))
    for i in range(rows):
        upload_at(mc, x, 2 * i * ld, bits[i])
    codes, scales = Out(mc, mc.mx4_code_bytes(rows, k)), Out(mc, mc.mx4_scale_bytes(rows, k))
    mc.quantize_mx4(ref.BF16, x.ptr, ld, codes.ptr, scales.ptr, rows, k)
    mc.synchronize()
    want = ref.quantize(ref.from_type(bits, ref.BF16))
    assert np.array_equal(codes.get(np.uint8, want[0].shape), want[0])
    assert np.array_equal(scales.get(np.uint8, want[1].shape), want[1])
    # The column form: its input's rows are as far apart.
    codes, scales = Out(mc, mc.mx4_code_bytes(k, rows)), Out(mc, mc.mx4_scale_bytes(k, rows))
    mc.quantize_mx4_columns(ref.BF16, x.ptr, ld, codes.ptr, scales.ptr, rows, k)
    mc.synchronize()
    want = ref.quantize(ref.from_type(bits, ref.BF16).T)
    assert np.array_equal(codes.get(np.uint8, want[0].shape), want[0])
    assert np.array_equal(scales.get(np.uint8, want[1].shape), want[1])


def download_at(mc, buf, offset, dtype, shape):
    out = np.empty(shape, dtype=dtype)
    assert mc.library().mc_memcpy_dtoh(out.ctypes.data, buf.ptr + offset, out.nbytes) == 0
    return out


@pytest.mark.parametrize("rows,k", [(1, (1 << 29) + 300), ((1 << 24) + 3, 2048)])
def test_quantize_more_than_one_launch(device, mc, rows, k):
    """2^29 rows of one column, 2^35 elements by rows: more threads than a launch has. The ends of both."""
    columns = rows == 1
    most = 4096  # elements at each end
    rng = np.random.default_rng(9)
    bits = ref.to_type(rng.standard_normal((2, most)), ref.BF16)
    x = mc.DeviceBuffer(2 * rows * k)
    x.fill_bytes(0)
    # From an element that starts a row, and a step of one.
    last = (k - most) // 128 * 128 if columns else rows * k - most
    upload_at(mc, x, 0, bits[0])
    upload_at(mc, x, 2 * last, bits[1])
    codes, scales = mc.DeviceBuffer(mc.mx4_code_bytes(rows, k)), mc.DeviceBuffer(mc.mx4_scale_bytes(rows, k))
    codes.fill_bytes(255)
    scales.fill_bytes(255)
    if columns:
        mc.quantize_mx4_columns(ref.BF16, x.ptr, 1, codes.ptr, scales.ptr, k, 1)
    else:
        mc.quantize_mx4(ref.BF16, x.ptr, k, codes.ptr, scales.ptr, rows, k)
    mc.synchronize()
    for at, end in ((0, bits[0]), (last, bits[1])):
        want = ref.quantize(ref.from_type(end, ref.BF16).reshape(1, -1))
        assert np.array_equal(download_at(mc, codes, at // 2, np.uint8, want[0].shape), want[0])
        assert np.array_equal(download_at(mc, scales, at // 32, np.uint8, want[1].shape), want[1])
    middle = rows * k // 2 // 4096 * 4096
    assert not download_at(mc, codes, middle // 2, np.uint8, (1 << 20,)).any()
    assert not download_at(mc, scales, middle // 32, np.uint8, (1 << 16,)).any()


# ---------------------------------------------------------------- products


def operand(mc, rng, rows, k, std=1.0):
    """A quantised random operand: (device codes, device scales, float64 values)."""
    codes, scales, values = ref.quantize(rng.standard_normal((rows, k)) * std * np.exp(0.5 * rng.standard_normal(k)))
    return mc.DeviceBuffer.from_array(codes), mc.DeviceBuffer.from_array(scales), values


def within(got, exact, bound):
    off = np.abs(got - exact)
    bad = ~(off <= bound)
    assert not bad.any(), f"{bad.sum()} of {bad.size} outside the bound; worst {np.nanmax(off / bound):.3g} of it"


PRODUCTS = [(1, 1, 1), (1, 16, 128), (1, 300, 4096), (2, 17, 129), (16, 64, 1000), (16, 4096, 256), (17, 33, 511),
            (31, 1000, 640), (32, 128, 2048), (40, 100, 33), (64, 64, 128), (65, 129, 1023), (100, 1001, 300),
            (128, 256, 512), (255, 257, 385), (256, 256, 256), (300, 70, 8192), (513, 300, 130), (700, 1030, 900)]


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product_of_quantised_operands(device, mc, kind, m, n, k):
    print(f"case mx4 product {kind} {m}x{n}x{k}", flush=True)
    dtype = ref.TYPES[kind]
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    ac, as_, a = operand(mc, rng, m, k)
    bc, bs, b = operand(mc, rng, n, k, k ** -0.5)
    c = Out(mc, m * n * (4 if dtype == ref.F32 else 2))
    mc.launch_matmul_mx4(ac.ptr, as_.ptr, bc.ptr, bs.ptr, dtype, c.ptr, m, n, k)
    mc.synchronize()
    exact, bound = ref.product_bound(a, b, k, dtype)
    within(ref.from_type(c.get(bits_type(dtype), (m, n)), dtype), exact, bound)


@pytest.mark.parametrize("kind,m,n,k", [("f32", 1500, 2100, 1100), ("f32", 1024, 4096, 1536), ("f32", 2300, 2049, 129),
                                        ("f32", 3000, 3001, 520), ("f32", 2900, 2820, 1290), ("bf16", 2817, 2952, 640),
                                        ("f16", 2900, 2948, 513), ("bf16", 2900, 2950, 2049), ("f16", 4200, 2090, 898),
                                        ("f32", 300, 40000, 1100)])
def test_product_of_many_tiles(device, mc, kind, m, n, k):
    print(f"case mx4 product {kind} {m}x{n}x{k}", flush=True)
    dtype = ref.TYPES[kind]
    rng = np.random.default_rng(m)
    ac, as_, a = operand(mc, rng, m, k)
    bc, bs, b = operand(mc, rng, n, k, k ** -0.5)
    c = Out(mc, m * n * (4 if dtype == ref.F32 else 2))
    mc.launch_matmul_mx4(ac.ptr, as_.ptr, bc.ptr, bs.ptr, dtype, c.ptr, m, n, k)
    mc.synchronize()
    exact, bound = ref.product_bound(a, b, k, dtype)
    within(ref.from_type(c.get(bits_type(dtype), (m, n)), dtype), exact, bound)


@pytest.mark.parametrize("m,n", [(3, 40), (300, 700), (1300, 2100), (2900, 3000)])
def test_a_block_without_a_scale_reaches_its_rows_alone(device, mc, m, n):
    k = 600
    rng = np.random.default_rng(9)
    x, w = rng.standard_normal((m, k)), rng.standard_normal((n, k))
    x[m // 2, 100] = np.nan
    w[n // 3, 599] = np.inf
    (xc, xs, _), (wc, ws, _) = ref.quantize(x), ref.quantize(w)
    bufs = [mc.DeviceBuffer.from_array(t) for t in (xc, xs, wc, ws)]
    c = Out(mc, m * n * 4)
    mc.launch_matmul_mx4(*(b.ptr for b in bufs), ref.F32, c.ptr, m, n, k)
    mc.synchronize()
    nan = np.zeros((m, n), dtype=bool)
    nan[m // 2, :] = True
    nan[:, n // 3] = True
    assert np.array_equal(np.isnan(c.get(np.float32, (m, n))), nan)


WEIGHTS = [(1, 1, 1, 0), (1, 14, 130, 0), (1, 1000, 4096, 0), (2, 33, 77, 3), (5, 128, 512, 8), (16, 257, 1023, 0),
           (17, 64, 257, 1), (32, 500, 640, 0), (33, 100, 128, 4), (64, 129, 300, 0), (65, 300, 1000, 0),
           (128, 256, 256, 0), (200, 77, 2048, 8), (300, 513, 129, 5), (700, 600, 520, 0),
           (8, 5000, 384, 1), (9, 4100, 250, 0), (40, 4097, 700, 2), (130, 4500, 200, 0), (2050, 2060, 390, 0),
           (2200, 2201, 640, 3)]


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("m,n,k,pad", WEIGHTS)
def test_product_with_quantised_weights(device, mc, kind, m, n, k, pad):
    print(f"case mx4 weights {kind} {m}x{n}x{k} pad {pad}", flush=True)
    dtype = ref.TYPES[kind]
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    bits = ref.to_type(rng.standard_normal((m, k)) * np.exp(rng.standard_normal(k)), dtype)
    a = device_rows(mc, bits, k + pad)
    bc, bs, b = operand(mc, rng, n, k, k ** -0.5)
    for out in (dtype, (dtype + 1) % 3):
        c = Out(mc, m * n * (4 if out == ref.F32 else 2))
        workspace = mc.DeviceBuffer(mc.matmul_mx4_weights_workspace_bytes(dtype, m, n, k))
        mc.launch_matmul_mx4_weights(dtype, a.ptr, k + pad, bc.ptr, bs.ptr, out, c.ptr, m, n, k, None, workspace.ptr)
        mc.synchronize()
        # Up to three pieces of A per product.
        exact, bound = ref.product_bound(ref.from_type(bits, dtype), b, 3 * k, out)
        within(ref.from_type(c.get(bits_type(out), (m, n)), out), exact, bound)


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("m", [3, 200])
def test_infinities_and_nans_of_unquantised_rows(device, mc, kind, m):
    dtype, n, k = ref.TYPES[kind], 50, 200
    rng = np.random.default_rng(4)
    x = rng.standard_normal((m, k))
    x[0, 7], x[2, 190] = np.inf, np.nan
    w = np.abs(rng.standard_normal((n, k))) + 0.5  # no zero among the codes that meet the infinity
    w[::2] *= -1.0
    bits = ref.to_type(x, dtype)
    wc, ws, _ = ref.quantize(w)
    a, bc, bs = device_rows(mc, bits, k), mc.DeviceBuffer.from_array(wc), mc.DeviceBuffer.from_array(ws)
    c = Out(mc, m * n * 4)
    workspace = mc.DeviceBuffer(mc.matmul_mx4_weights_workspace_bytes(dtype, m, n, k))
    mc.launch_matmul_mx4_weights(dtype, a.ptr, k, bc.ptr, bs.ptr, ref.F32, c.ptr, m, n, k, None, workspace.ptr)
    mc.synchronize()
    got = c.get(np.float32, (m, n))
    assert np.array_equal(got[0], np.where(np.arange(n) % 2 == 0, -np.inf, np.inf))
    assert np.all(np.isnan(got[2])) and np.all(np.isfinite(got[1])) and np.all(np.isfinite(got[3:]))


def test_few_rows_more_than_2_gib_apart(device, mc):
    m, n, k, lda = 3, 40, 200, (1 << 30) + 24
    rng = np.random.default_rng(31)
    bits = ref.to_type(rng.standard_normal((m, k)), ref.BF16)
    a = mc.DeviceBuffer(2 * ((m - 1) * lda + k))
    for i in range(m):
        upload_at(mc, a, 2 * i * lda, bits[i])
    bc, bs, b = operand(mc, rng, n, k)
    c = Out(mc, m * n * 4)
    mc.launch_matmul_mx4_weights(ref.BF16, a.ptr, lda, bc.ptr, bs.ptr, ref.F32, c.ptr, m, n, k)
    mc.synchronize()
    exact, bound = ref.product_bound(ref.from_type(bits, ref.BF16), b, k, ref.F32)
    within(c.get(np.float32, (m, n)).astype(np.float64), exact, bound)


def test_operands_of_more_than_4_gib(device, mc):
    """The last rows of a weight operand whose codes and scales lie past 2^32 and 2^28 bytes."""
    n, k, last = 540000, 16384, 48
    codes, scales = mc.DeviceBuffer(mc.mx4_code_bytes(n, k)), mc.DeviceBuffer(mc.mx4_scale_bytes(n, k))
    codes.fill_bytes(0x22)  # every code 1
    scales.fill_bytes(127)
    rng = np.random.default_rng(8)
    tc, ts, tail = ref.quantize(rng.standard_normal((last, k)))
    upload_at(mc, codes, (n - last) * (k // 2), tc)
    upload_at(mc, scales, (n - last) * (k // 32), ts)
    bits = ref.to_type(rng.standard_normal((1, k)), ref.BF16)
    a = mc.DeviceBuffer.from_array(bits)
    ac, as_, av = ref.quantize(ref.from_type(bits, ref.BF16))
    dac, das = mc.DeviceBuffer.from_array(ac), mc.DeviceBuffer.from_array(as_)
    for quantised in (False, True):
        c = mc.DeviceBuffer(4 * n)
        if quantised:
            mc.launch_matmul_mx4(dac.ptr, das.ptr, codes.ptr, scales.ptr, ref.F32, c.ptr, 1, n, k)
        else:
            mc.launch_matmul_mx4_weights(ref.BF16, a.ptr, k, codes.ptr, scales.ptr, ref.F32, c.ptr, 1, n, k)
        mc.synchronize()
        got = c.download()
        left = av if quantised else ref.from_type(bits, ref.BF16)
        exact, bound = ref.product_bound(left, np.concatenate([np.ones((1, k)), tail]), k, ref.F32)
        within(got[n - last:], exact[0, 1:], bound[0, 1:])
        within(got[:n - last], exact[0, 0], bound[0, 0])


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k,pad", [(17, 16, 128, 0), (18, 40, 2050, 0), (31, 100, 4099, 1), (32, 4130, 300, 2),
                                       (25, 5000, 2333, 3), (29, 33, 77, 5), (32, 8200, 130, 64)])
def test_rows_of_16_bits_that_start_at_dwords(device, mc, kind, m, n, k, pad):
    """Even distances between rows: read as they are, up to 32 of them; block scales over the whole range."""
    print(f"case mx4 weights {kind} {m}x{n}x{k} pad {pad}", flush=True)
    dtype = ref.TYPES[kind]
    rng = np.random.default_rng(m * 11 + n + k)
    bits = ref.to_type(rng.standard_normal((m, k)) * np.exp(rng.standard_normal(k)), dtype)
    a = device_rows(mc, bits, k + pad)
    bc, bs, b = operand(mc, rng, n, k, k ** -0.5)
    c = Out(mc, m * n * 4)
    workspace = mc.DeviceBuffer(mc.matmul_mx4_weights_workspace_bytes(dtype, m, n, k))
    mc.launch_matmul_mx4_weights(dtype, a.ptr, k + pad, bc.ptr, bs.ptr, ref.F32, c.ptr, m, n, k, None, workspace.ptr)
    mc.synchronize()
    exact, bound = ref.product_bound(ref.from_type(bits, dtype), b, 3 * k, ref.F32)
    within(c.get(np.float32, (m, n)).astype(np.float64), exact, bound)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("n", [40, 4200])
def test_scales_at_the_ends_and_of_no_number(device, mc, kind, n):
    """Rows of powers of two meet columns of one scale each, from 2^-127 to 2^120: exact in fp32 down to 2^-126;
    255 makes its columns NaN, whatever their codes."""
    m, k, dtype = 32, 300, ref.TYPES[kind]
    kp = ref.padded(k)
    a_bits = ref.to_type(np.tile(2.0 ** (np.arange(m) % 4).reshape(m, 1), (1, k)), dtype)
    codes, scales = np.zeros((n, kp // 2), np.uint8), np.zeros((n, kp // 32), np.uint8)
    codes[:, 60] = 0x42  # elements 120 and 121: 1 and 2
    scales[:, 3] = np.arange(n) * 31 % 248
    bad = np.arange(n) % 7 == 3
    scales[bad, 3] = 255
    codes[np.arange(n) % 14 == 3, 60] = 0
    a, bc, bs = device_rows(mc, a_bits, k), mc.DeviceBuffer.from_array(codes), mc.DeviceBuffer.from_array(scales)
    c = Out(mc, m * n * 4)
    workspace = mc.DeviceBuffer(mc.matmul_mx4_weights_workspace_bytes(dtype, m, n, k))
    mc.launch_matmul_mx4_weights(dtype, a.ptr, k, bc.ptr, bs.ptr, ref.F32, c.ptr, m, n, k, None, workspace.ptr)
    mc.synchronize()
    got = c.get(np.float32, (m, n)).astype(np.float64)
    assert np.all(np.isnan(got[:, bad]))
    want = 3.0 * 2.0 ** (np.arange(m) % 4).reshape(m, 1) * 2.0 ** (scales[~bad, 3].astype(np.float64) - 127)
    normal = want >= 2.0 ** -126
    assert normal.mean() > 0.95 and np.array_equal(got[:, ~bad][normal], want[normal])
    assert np.all(got[:, ~bad][~normal] <= 2.0 ** -126)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k,pad", [(1, 30, 2050, 0), (3, 100, 4097, 1), (9, 1000, 2200, 6), (16, 4096, 2052, 0),
                                       (32, 70, 9000, 0)])
def test_few_rows_of_16_bits_and_a_long_k(device, mc, kind, m, n, k, pad):
    test_rows_of_16_bits_that_start_at_dwords(device, mc, kind, m, n, k, pad)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k,pad", [(33, 16, 128, 0), (49, 100, 2050, 2), (64, 4200, 1100, 0), (63, 9000, 333, 1),
                                       (64, 40, 4100, 0)])
def test_up_to_64_rows_of_16_bits(device, mc, kind, m, n, k, pad):
    test_rows_of_16_bits_that_start_at_dwords(device, mc, kind, m, n, k, pad)
