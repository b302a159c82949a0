"""Products with 4-bit weights on the GPU where the numbers end: the largest and smallest scales, small fp32 rows,
infinities and NaNs in the rows, for every kernel that a number of rows leads to. Expected values are exact: each
result is one product, or a sum whose every partial sum fp32 holds."""

import numpy as np
import pytest

import mx4_oracle as ref
from test_gpu_mx4 import Out, bits_type, device_rows

pytestmark = pytest.mark.gpu

# Rows, columns and k: few rows at a short and at a long k, up to 32 and 64 rows at once, pieces, large tiles.
SHAPES = [(3, 70, 300), (16, 70, 2300), (20, 70, 300), (32, 70, 300), (40, 70, 300), (64, 70, 300), (64, 70, 2300),
          (200, 70, 300), (2050, 2060, 300)]


def multiply(mc, dtype, bits, codes, scales, n, k):
    """[m, n] fp32 results of rows `bits` and weights given by their codes and scales, on guarded memory."""
    m = bits.shape[0]
    a, bc, bs = device_rows(mc, bits, k), mc.DeviceBuffer.from_array(codes), mc.DeviceBuffer.from_array(scales)
    c = Out(mc, m * n * 4)
    workspace = mc.DeviceBuffer(max(1, mc.matmul_mx4_weights_workspace_bytes(dtype, m, n, k)))
    mc.launch_matmul_mx4_weights(dtype, a.ptr, k, bc.ptr, bs.ptr, ref.F32, c.ptr, m, n, k, None, workspace.ptr)
    mc.synchronize()
    return c.get(np.float32, (m, n)).astype(np.float64)


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_the_largest_scales(device, mc, kind, m, n, k):
    """One code per column at each scale byte from 248 to 254, met by small rows: exact up to fp32's largest number;
    a weight past it makes no finite product, in any kernel."""
    print(f"case largest scales {kind} {m}x{n}x{k}", flush=True)
    kp = ref.padded(k)
    codes, scales = np.zeros((n, kp // 2), np.uint8), np.full((n, kp // 32), 127, np.uint8)
    column = np.arange(n)
    code = column % 8 | (column // 16 % 2) << 3
    byte = 248 + column // 8 % 7
    at = np.array([0, 100, 299])[column % 3]
    codes[column, at // 2] = code << (4 * (at % 2))
    scales[column, at // 32] = byte
    weight = ref.MAGNITUDES[code & 7] * np.where(code & 8, -1.0, 1.0) * 2.0 ** (byte.astype(np.float64) - 127)
    finite = np.abs(weight) <= np.finfo(np.float32).max
    assert (~finite).sum() >= 6
    row = 2.0 ** -20 * (1 + np.arange(m) % 4)
    bits = ref.to_type(np.tile(row.reshape(m, 1), (1, k)), ref.TYPES[kind])
    got = multiply(mc, ref.TYPES[kind], bits, codes, scales, n, k)
    want = row.reshape(m, 1) * weight
    assert np.array_equal(got[:, finite], want[:, finite])
    assert not np.isfinite(got[:, ~finite]).any()


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_small_fp32_rows(device, mc, m, n, k):
    """fp32 rows of one number each, down to the smallest subnormal, against a weight of 2^100: whole from 2^-110 up,
    below that the multiple of 2^-133 towards zero."""
    print(f"case small rows {m}x{n}x{k}", flush=True)
    kp = ref.padded(k)
    codes, scales = np.zeros((n, kp // 2), np.uint8), np.full((n, kp // 32), 227, np.uint8)
    at = np.arange(n) * 37 % k
    codes[np.arange(n), at // 2] = 2 << (4 * (at % 2))  # 1
    rng = np.random.default_rng(m + k)
    x = (rng.integers(1 << 23, 1 << 24, m) * 2.0 ** (-149 + np.arange(m) * 5 % 45)).astype(np.float32)
    x[::3] *= -1.0
    x[1] = 2.0 ** -149
    got = multiply(mc, ref.F32, np.tile(x.reshape(m, 1), (1, k)), codes, scales, n, k)
    kept = np.where(np.abs(x) < 2.0 ** -110, np.trunc(x.astype(np.float64) * 2.0 ** 133) * 2.0 ** -133, x.astype(np.float64))
    assert np.array_equal(got, np.tile((kept * 2.0 ** 100).reshape(m, 1), (1, n)))


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_the_smallest_scales_and_none(device, mc, kind, m, n, k):
    """One code per column at the scale bytes 0 to 6, and 255: exact products, those below fp32's normal numbers exact or
    zero; a column with a scale of no number is none, whatever its code."""
    print(f"case smallest scales {kind} {m}x{n}x{k}", flush=True)
    kp = ref.padded(k)
    codes, scales = np.zeros((n, kp // 2), np.uint8), np.full((n, kp // 32), 127, np.uint8)
    column = np.arange(n)
    code, byte = column % 8, column // 8 % 8
    byte = np.where(byte == 7, 255, byte)
    at = np.array([3, 130, 287])[column % 3]
    codes[column, at // 2] = code << (4 * (at % 2))
    scales[column, at // 32] = byte
    none = byte == 255
    assert none.sum() >= 6
    weight = ref.MAGNITUDES[code] * 2.0 ** (np.where(none, 0, byte).astype(np.float64) - 127)
    row = 2.0 ** (np.arange(m) % 4)
    bits = ref.to_type(np.tile(row.reshape(m, 1), (1, k)), ref.TYPES[kind])
    got = multiply(mc, ref.TYPES[kind], bits, codes, scales, n, k)
    want = row.reshape(m, 1) * weight
    assert np.isnan(got[:, none]).all()
    normal = want >= 2.0 ** -126
    equal = got == want
    assert equal[:, ~none][normal[:, ~none]].all()
    assert (equal | (got == 0.0))[:, ~none].all()


@pytest.mark.parametrize("kind", sorted(ref.TYPES))
@pytest.mark.parametrize("m,n,k", [s for s in SHAPES if s[0] >= 3])
@pytest.mark.parametrize("pad", [1, 2])
def test_rows_of_infinities_and_nans(device, mc, kind, m, n, k, pad):
    """An infinity makes its row's results infinite and a NaN makes them NaN, the last element of an odd row among them;
    the other rows, and what lies between rows (NaN), reach nothing."""
    k, dtype = k + 1, ref.TYPES[kind]
    print(f"case rows of no numbers {kind} {m}x{n}x{k} pad {pad}", flush=True)
    rng = np.random.default_rng(m + k)
    x = rng.standard_normal((m, k))
    x[0, 7], x[1, k - 1], x[2, 190], x[m - 1, k - 1] = np.inf, np.nan, np.nan, -np.inf
    w = np.abs(rng.standard_normal((n, k))) + 0.5  # no zero among the codes that meet an infinity
    w[::2] *= -1.0
    bits = ref.to_type(x, dtype)
    wc, ws, values = ref.quantize(w)
    a, bc, bs = device_rows(mc, bits, k + pad), mc.DeviceBuffer.from_array(wc), mc.DeviceBuffer.from_array(ws)
    c = Out(mc, m * n * 4)
    workspace = mc.DeviceBuffer(max(1, mc.matmul_mx4_weights_workspace_bytes(dtype, m, n, k)))
    mc.launch_matmul_mx4_weights(dtype, a.ptr, k + pad, bc.ptr, bs.ptr, ref.F32, c.ptr, m, n, k, None, workspace.ptr)
    mc.synchronize()
    got = c.get(np.float32, (m, n)).astype(np.float64)
    sign = np.where(np.arange(n) % 2 == 0, -1.0, 1.0)
    assert np.array_equal(got[0], np.inf * sign)
    assert np.isnan(got[1]).all()
    if m > 3:
        assert np.isnan(got[2]).all() and np.array_equal(got[m - 1], -np.inf * sign)
        exact, bound = ref.product_bound(ref.from_type(bits, dtype)[3:m - 1], values, 3 * k, ref.F32)
        assert (np.abs(got[3:m - 1] - exact) <= bound).all()
    else:
        assert np.isnan(got[2]).all()
